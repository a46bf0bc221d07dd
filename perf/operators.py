"""Workloads of the categorical operators: what they compute, on which sizes, and how they are called.

  * log probabilities of given categories, with the entropy of each row and its most probable alternatives
    (`demiss_vae_amd.categorical_log_prob`), forward and with its gradient;
  * distillation from a teacher's top logits (`demiss_vae_amd.distill_top_logits`): loss and gradient of one step.

`run` computes them in their plain form, with elementary torch operations in 32 bits, or, where `own` is true, through the
framework's entry points.  Rows are laid out as the framework lays out its samples: logits [S, B, D, V] for S samples of B
datapoints with D categorical entries of up to V categories, the given categories X and their mask M [B, D], the number of
categories of each entry, sizes, [D]."""
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_MOST = 2048 * 65536          # elements of the largest listed case; drawn cases stay below


def _score(name, dtype, S, B, D, V, top=0, entropy=False, given=True, mask=False, ragged=False, train=False):
    return {"name": name, "op": "log_prob", "dtype": dtype, "S": S, "B": B, "D": D, "V": V, "top": top, "entropy": entropy,
            "given": given, "mask": mask, "ragged": ragged, "train": train}


def _distill(name, dtype, S, B, D, V, k, temperature, mask=False, ragged=False):
    return {"name": name, "op": "distill", "dtype": dtype, "S": S, "B": B, "D": D, "V": V, "k": k,
            "temperature": temperature, "mask": mask, "ragged": ragged}


def listed():
    return [
        # one entry answered: its distribution's entropy and five best categories, where latency is all that counts
        _score("one answer", "bfloat16", 1, 1, 1, 50000, top=5, entropy=True, given=False),
        # a batch of mixture posteriors: log weight of the chosen component and entropy, 25 components at batch size 512
        _score("mixture weights", "float32", 1, 512, 1, 25, entropy=True),
        # imputing a table: five samples, 4096 datapoints, 8 columns with 2 to 32 categories each, missing entries masked,
        # three candidates for every entry
        _score("table columns", "float32", 5, 4096, 8, 32, top=3, mask=True, ragged=True),
        # 8-bit pixels of 28 x 28 images as categories, with entropy and four candidates
        _score("pixels", "bfloat16", 1, 128, 784, 256, top=4, entropy=True),
        # normalised importance weights of 50 test points at 50 000 importance samples: entropy, and the 64 that carry the sum
        _score("importance weights", "float32", 1, 50, 1, 50000, top=64, entropy=True, given=False),
        # large vocabulary: scoring given categories with entropy and eight alternatives
        _score("vocabulary", "bfloat16", 1, 2048, 1, 65536, top=8, entropy=True),
        # a training pass of the masked categorical likelihood of pixels: log-probabilities and the gradient of the logits
        _score("pixels training", "bfloat16", 1, 128, 784, 256, mask=True, train=True),
        # likelihood and entropy with their gradient over long rows of odd length
        _score("vocabulary training", "float16", 1, 1024, 1, 50001, entropy=True, train=True),
        # a small batch of soft targets: the latency of a loss with its gradient
        _distill("few rows distilled", "float32", 1, 64, 1, 1000, 10, 2.0),
        # missing pixels trained against a teacher's eight best categories, observed ones left out
        _distill("pixels distilled", "bfloat16", 1, 128, 784, 256, 8, 1.0, mask=True),
        # a large vocabulary distilled from the 32 best categories
        _distill("vocabulary distilled", "bfloat16", 1, 2048, 1, 65536, 32, 2.0),
        # few rows of great odd length, in 32 bits
        _distill("long rows distilled", "float32", 1, 96, 1, 262147, 64, 1.0),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    V = _log_uniform(rng, 2, 262147)
    rows = _log_uniform(rng, 1, max(1, min(262144, _MOST // (2 * V))))
    dtype = rng.choice(("float32", "bfloat16", "float16"))
    D = rng.choice((1, 1, 8, 21, 43)) if V <= 1024 else 1
    S = rng.choice((1, 1, 5))
    B = max(1, rows // (D * S))
    mask, ragged = rng.random() < 0.4, V >= 4 and rng.random() < 0.4
    if rng.random() < 0.55:
        train = rng.random() < 0.4
        c = _score("", dtype, S, B, D, V, top=0 if train else min(V, rng.choice((0, 1, 3, 5, 8, 20, 64))),
                   entropy=rng.random() < 0.5, given=True, mask=mask, ragged=ragged, train=train)
    else:
        c = _distill("", dtype, S, B, D, V, min(V, _log_uniform(rng, 1, 128)), rng.choice((1.0, 2.0, 0.7)), mask=mask, ragged=ragged)
    del c["name"]
    return c


def _shape(c):
    return c["S"], c["B"], c["D"], c["V"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = {"device": "cuda", "generator": g}
    S, B, D, V = _shape(case)
    dtype = DTYPES[case["dtype"]]
    # the few large logits of a trained network's output over a broad background
    logits = torch.randn(S, B, D, V, **dev)
    logits = logits.mul_(2.0).add_(logits.pow(3), alpha=0.05)
    st = {"case": case, "sizes": None, "M": None, "X": None}
    if case["ragged"]:
        st["sizes"] = torch.randint(max(1, V // 2), V + 1, (D,), dtype=torch.int32, **dev)
    if case["mask"]:
        st["M"] = torch.rand(B, D, **dev) < 0.5
    if case["op"] == "log_prob":
        st["logits"] = logits.to(dtype)
        if case["given"]:
            most = st["sizes"] if case["ragged"] else V
            st["X"] = (torch.rand(B, D, **dev) * most).long().clamp_(max=V - 1)
            if case["ragged"]:
                st["X"] = torch.minimum(st["X"], st["sizes"].long() - 1)
        if case["train"]:
            st["g_log_prob"] = -(0.5 + torch.rand(S, B, D, **dev))
            st["g_entropy"] = 0.1 * torch.rand(S, B, D, **dev) if case["entropy"] else None
    else:
        st["logits"] = logits.to(dtype)
        # a teacher that has learned more than the student: the two agree on part of the background
        teacher = torch.randn(S, B, D, V, **dev).mul_(1.5).add_(logits, alpha=0.7)
        if case["ragged"]:
            teacher = teacher.masked_fill_(torch.arange(V, device="cuda") >= st["sizes"][:, None], float("-inf"))
        k = min(case["k"], int(st["sizes"].min())) if case["ragged"] else case["k"]
        top = torch.topk(teacher, k, dim=-1)
        st["top_logits"], st["top_index"] = top.values.to(dtype), top.indices
        w = 0.5 + torch.rand(S, B, D, **dev)
        st["weight"] = w * ~st["M"] if case["mask"] else w
    return st


# ------------------------------------------------------------------------------------------ plain forms
def _allowed(st, dtype):
    x = st["logits"].to(dtype)
    if st["sizes"] is not None:
        x = x.masked_fill(torch.arange(x.shape[-1], device=x.device) >= st["sizes"][:, None], float("-inf"))
    return x


def _log_softmax(x):
    """(log q, q) of the rows of x.  The sum of a row that is nearly certain of one category is 1 plus what the others
    add, which 32 bits would lose: it is formed in 64."""
    d = x - x.amax(-1, keepdim=True)
    e = d.exp()
    s = e.sum(-1, keepdim=True, dtype=torch.float64)
    return d - s.log().float(), e / s.float()


def _plain_log_prob(st):
    c = st["case"]
    x = _allowed(st, torch.float32)
    V = x.shape[-1]
    log_q, q = _log_softmax(x)
    out = {}
    if st["X"] is not None:
        X = st["X"].expand(x.shape[:-1])[..., None]
        log_q_X = log_q.gather(-1, X)
        out["log_prob"] = log_q_X[..., 0]
        if st["M"] is not None:
            out["log_prob"] = out["log_prob"] * st["M"]
    if c["entropy"]:
        out["entropy"] = -(torch.where(q > 0, q * log_q, 0.0)).sum(-1)
    if c["top"]:
        # larger logits first, the lower index first among equal ones: one 64-bit key holds both
        bits = (x + 0.0).view(torch.int32)
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * 2 ** 32 + torch.arange(V - 1, -1, -1, device=x.device)
        index = key.topk(c["top"], dim=-1).indices
        out["top_log_prob"] = log_q.gather(-1, index)
        out["top_index"] = torch.where(out["top_log_prob"] > float("-inf"), index, -1)
    if c["train"]:
        g = (st["g_log_prob"] if st["M"] is None else st["g_log_prob"] * st["M"])[..., None]
        slope = -g * q
        slope.scatter_(-1, X, -g * torch.expm1(log_q_X))       # 1 - q without its cancellation
        if c["entropy"]:
            slope -= st["g_entropy"][..., None] * torch.where(q > 0, q * (log_q + out["entropy"][..., None]), 0.0)
        out["d_logits"] = slope.to(st["logits"].dtype)
    return out


def _plain_distill(st):
    T = st["case"]["temperature"]
    log_q, q = _log_softmax(_allowed(st, torch.float32) / T)
    log_p, p = _log_softmax(st["top_logits"].float() / T)
    i = st["top_index"]
    w = st["weight"]
    off = log_q.gather(-1, i) - log_p
    kl = torch.where(w != 0, -(p * off).sum(-1), 0.0)
    slope = q.scatter_(-1, i, p * torch.expm1(off))            # q - p without its cancellation
    d_logits = (slope * (w / T)[..., None]).to(st["logits"].dtype)
    return {"loss": (w.double() * kl.double()).sum().float(), "per_row": kl, "d_logits": d_logits}


# ------------------------------------------------------------------------------------------ the framework's calls
def _own_log_prob(st):
    import demiss_vae_amd as dmv
    c = st["case"]
    z = st["logits"].detach()
    if c["train"]:
        z.requires_grad_()
    r = dmv.categorical_log_prob(z, st["X"], st["M"], sizes=st["sizes"], entropy=c["entropy"], top=c["top"])
    out = {}
    if st["X"] is not None:
        out["log_prob"] = r.log_prob.detach()
    if c["entropy"]:
        out["entropy"] = r.entropy.detach()
    if c["top"]:
        out["top_log_prob"], out["top_index"] = r.top_log_prob, r.top_index
    if c["train"]:
        if c["entropy"]:
            (out["d_logits"],) = torch.autograd.grad((r.log_prob, r.entropy), z, (st["g_log_prob"], st["g_entropy"]))
        else:
            (out["d_logits"],) = torch.autograd.grad(r.log_prob, z, st["g_log_prob"])
    return out


def _own_distill(st):
    import demiss_vae_amd as dmv
    z = st["logits"].detach().requires_grad_()
    loss, per_row = dmv.distill_top_logits(z, st["top_logits"], st["top_index"], sizes=st["sizes"], weight=st["weight"],
                                           temperature=st["case"]["temperature"])
    (d_logits,) = torch.autograd.grad(loss, z)
    return {"loss": loss.detach(), "per_row": per_row, "d_logits": d_logits}


def run(state):
    if state["case"]["op"] == "log_prob":
        return _own_log_prob(state) if own else _plain_log_prob(state)
    return _own_distill(state) if own else _plain_distill(state)


# ------------------------------------------------------------------------------------------ work and 64-bit values
def work(case):
    S, B, D, V = _shape(case)
    rows, esize = S * B * D, DTYPES[case["dtype"]].itemsize
    # (ragged rows hold three quarters of V on average; their gradient is written whole)
    read = rows * V * esize * (0.75 if case["ragged"] else 1.0)
    written = 0.0
    flops = 4.0 * rows * V
    if case["op"] == "log_prob":
        if case["train"] and case["mask"] and not case["entropy"]:
            read *= 0.5                      # rows whose only output is masked need not be read
        read += 8 * B * D if case["given"] else 0
        read += B * D if case["mask"] else 0
        written += 4 * rows * (case["given"] + case["entropy"]) + 12 * rows * case["top"]
        flops += 3.0 * rows * V * case["entropy"]
        if case["train"]:
            read += 4 * rows * (1 + case["entropy"])
            written += rows * V * esize
            flops += 3.0 * rows * V
    else:
        if case["mask"]:
            read *= 0.5                      # rows of weight zero need not be read
        read += rows * (case["k"] * (8 + esize) + 4)
        written += rows * (V * esize + 4)
        flops += 4.0 * rows * V
    return {"bytes": read + written, "flops": flops}


def exact(case, seed):
    st = prepare(case, seed)
    x = _allowed(st, torch.float64)
    if case["op"] == "log_prob":
        log_z = torch.logsumexp(x, -1)
        out = {}
        if case["given"]:
            X = st["X"].expand(x.shape[:-1])
            seen = 1.0 if st["M"] is None else st["M"].double()
            out["log_prob"] = (x.gather(-1, X[..., None])[..., 0] - log_z) * seen
        if case["entropy"] or case["train"]:
            q = torch.exp(x - log_z[..., None])
            H = log_z - (q * x.clamp(min=-1e30)).sum(-1)     # H = log Z - E_q[x]
        if case["entropy"]:
            out["entropy"] = H
        if case["top"]:
            out["top_log_prob"] = x.topk(case["top"], dim=-1).values - log_z[..., None]
            out["top_index"] = None
        if case["train"]:
            g = st["g_log_prob"].double() * seen
            slope = -g[..., None] * q
            if case["entropy"]:
                slope += st["g_entropy"].double()[..., None] * q * ((log_z - H)[..., None] - x.clamp(min=-1e30))
            at = X[..., None]
            out["d_logits"] = slope.scatter(-1, at, slope.gather(-1, at) + g[..., None])
        return out
    T = case["temperature"]
    log_q = torch.log_softmax(x / T, -1)
    p = torch.softmax(st["top_logits"].double() / T, -1)
    w = st["weight"].double()
    kl = -torch.special.entr(p).sum(-1) - (p * log_q.gather(-1, st["top_index"])).sum(-1)
    kl = kl * (w != 0)
    slope = log_q.exp_()
    slope.scatter_(-1, st["top_index"], slope.gather(-1, st["top_index"]) - p)
    return {"loss": (w * kl).sum(), "per_row": kl, "d_logits": slope * (w / T)[..., None]}
