"""The categorical operators against plain implementations in 64 bits.

Tolerances (e = 2^-24, half a step of float32; h = finfo(dtype).eps / 2, half a step of the logits' type).  With d = (x - m)
/ T and Z the row's sum: the exponent's argument has three roundings (difference, factor, and the factor's own), so a term
2^(c d) is off by at most 3 |d| e + 2 e (the exp2 unit) relatively; a thread adds up to V / 256 + 16 terms and the joins
add 24 more levels.  Hence, with C = V / 256 + 64 and D = E_q|d| the row's mean distance:
  log q_v:    e (2 |d_v| + 3 D + C);          entropy: e (4 E_q[d^2] + 4 D + C (1 + H))
  q_v:        q_v e (3 |d_v| + 3 D + C)
and a result in the logits' type is off by another h of itself (or half the smallest subnormal step).  The exp2 unit gives 0
for results below the smallest normal number: 2^c d < 2^-126 becomes 0, an absolute 2^-126 in 2^(c d) and so at most 2^-126
in q_v = 2^(c d) / s (s >= 1)."""
import math

import pytest
import torch

import demiss_vae_amd as dmv

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
FLUSH = 2.0 ** -126
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# lengths around the tiles of the kernels: single elements, 16-byte slots, lane groups, whole wavefronts, workgroups,
# several workgroups a row
LENGTHS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 25, 31, 33, 64, 65, 127, 128, 200, 257, 511, 512, 513, 1000, 1023, 1024, 1025, 1031, 2049, 4100,
           8191, 16385, 50001, 65537, 131075, 262147]


def rows_for(V):
    return 300 if V <= 300 else 37 if V <= 5000 else 5


def make(shape, dtype, seed=0, scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, device="cuda", generator=g) * scale
    return (x + 0.05 * x ** 3).to(dtype)


def ints(high, shape, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, high, shape, device="cuda", generator=g)


def rand(shape, seed=2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.rand(shape, device="cuda", generator=g)


class Ref:
    """q = softmax(x / T) over the allowed categories of x [rows, V], in 64 bits, and the error units of its outputs."""

    def __init__(self, x, sizes=None, T=1.0):
        self.x = x.double() / T
        self.V, self.T = x.shape[-1], T
        if sizes is not None:
            self.x = self.x.masked_fill(torch.arange(self.V, device=x.device) >= sizes[..., None], -math.inf)
        m = self.x.amax(-1, keepdim=True)
        self.empty = (m == -math.inf)
        self.d = torch.where(self.empty, -math.inf, self.x - m)
        # log of the sum over all but the largest: relative accuracy next to 0
        rest = self.d.exp().scatter(-1, self.x.argmax(-1, keepdim=True), 0.0).sum(-1, keepdim=True)
        self.log_q = self.d - torch.log1p(rest)
        self.q = self.log_q.exp()
        dist = torch.where(self.q > 0, self.d, 0.0).abs()
        self.dist = dist
        self.D = (self.q * dist).sum(-1, keepdim=True)
        self.D2 = (self.q * dist * dist).sum(-1, keepdim=True)
        self.C = self.V / 256 + 64
        self.H = -(torch.where(self.q > 0, self.q * self.log_q, 0.0)).sum(-1, keepdim=True)

    def tol_log_q(self):
        return E * (2 * torch.where(self.d == -math.inf, 0.0, self.d.abs()) + 3 * self.D + self.C)

    def tol_H(self):
        return E * (4 * self.D2 + 4 * self.D + self.C * (1 + self.H))

    def tol_q(self):
        return E * (3 * self.dist + 3 * self.D + self.C)          # times q

    def top(self, k):
        """stable descending order: the lower index first among equal values"""
        v, i = torch.sort(self.x, dim=-1, descending=True, stable=True)
        v, i = v[..., :k], i[..., :k]
        if k > self.V:
            pad = (*v.shape[:-1], k - self.V)
            v = torch.cat([v, v.new_full(pad, -math.inf)], -1)
            i = torch.cat([i, i.new_full(pad, -1)], -1)
        none = v == -math.inf
        i = torch.where(none, -1, i)
        lp = torch.where(none, -math.inf, self.log_q.gather(-1, i.clamp(min=0)))
        return lp, i


def close(got, want, tol, what):
    got, tol = got.double(), torch.as_tensor(tol, dtype=torch.float64, device=got.device).expand(want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got - want).abs() / tol)[bad].nan_to_num(1e30).max()),
                                 got[bad][:3].tolist(), want[bad][:3].tolist())


def narrow(t, dtype):
    """half a step of a value of this type, and of its subnormal numbers"""
    f = torch.finfo(dtype)
    return t.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


def grad_ref(r, g_lp, X, g_ent, top_idx, g_top):
    """formula's gradient and its tolerance (float32 part); g_lp 0 where not seen"""
    a = torch.zeros_like(r.q)
    if g_lp is not None:
        a.scatter_add_(-1, X[..., None], g_lp.double()[..., None])
    if g_top is not None:
        a.scatter_add_(-1, top_idx.clamp(min=0), torch.where(top_idx >= 0, g_top.double(), 0.0))
    S = a.sum(-1, keepdim=True)
    S_abs = a.abs().sum(-1, keepdim=True)
    gh = torch.zeros_like(S) if g_ent is None else g_ent.double()[..., None]
    lq = r.log_q.clamp(min=-1e30)
    want = -a * torch.expm1(r.log_q) - (S - a) * r.q - torch.where(r.q > 0, gh * r.q * (lq + r.H), 0.0)
    want = torch.where(r.empty, 0.0, want)
    # S itself is a sum of up to 65 terms; H enters with its own error
    slope = S_abs + gh.abs() * (torch.where(r.q > 0, lq.abs(), 0.0) + r.H)
    tol = slope * (r.q * (r.tol_q() + 70 * E) + FLUSH) + gh.abs() * r.q * (r.tol_log_q() + r.tol_H()) + a.abs() * (
        torch.expm1(r.log_q).abs() * 4 * E + torch.exp(r.log_q) * r.tol_log_q())
    return want, tol


def check_log_prob(x, X=None, M=None, sizes=None, entropy=False, top=0, grads=False, seed=5):
    """forward and gradient of one call against 64 bits"""
    lead, V = x.shape[:-1], x.shape[-1]
    z = x.detach()
    if grads:
        z = z.requires_grad_()
    got = dmv.categorical_log_prob(z, X, M, sizes=sizes, entropy=entropy, top=top)
    r = Ref(x.detach(), None if sizes is None else sizes.expand(lead))
    seen = torch.ones(lead, dtype=torch.bool, device=x.device) if M is None else M.expand(lead)
    if X is not None:
        Xe = torch.where(seen, X.expand(lead), 0)
        want = torch.where(r.empty[..., 0], -math.inf, r.log_q.gather(-1, Xe[..., None])[..., 0])
        close(got.log_prob, torch.where(seen, want, 0.0), torch.where(seen, r.tol_log_q().gather(-1, Xe[..., None])[..., 0], 0.0), "log_prob")
        assert got.log_prob.dtype == torch.float32 and got.log_prob.shape == lead
    else:
        assert got.log_prob is None
    if entropy:
        close(got.entropy, r.H[..., 0], r.tol_H()[..., 0], "entropy")
    else:
        assert got.entropy is None
    if top:
        lp, idx = r.top(top)
        assert torch.equal(got.top_index, idx), (got.top_index[got.top_index != idx][:5], idx[got.top_index != idx][:5])
        close(got.top_log_prob, lp, r.tol_log_q().gather(-1, idx.clamp(min=0)), "top_log_prob")
    else:
        assert got.top_index is None and got.top_log_prob is None
    if not grads:
        return got
    outs, ups = [], []
    g_lp = g_ent = g_top = None
    if X is not None:
        g_lp = rand(lead, seed) - 0.3
        outs.append(got.log_prob), ups.append(g_lp)
    if entropy:
        g_ent = rand(lead, seed + 1) - 0.5
        outs.append(got.entropy), ups.append(g_ent)
    if top:
        g_top = rand((*lead, top), seed + 2) - 0.5
        outs.append(got.top_log_prob), ups.append(g_top)
    (dx,) = torch.autograd.grad(outs, z, ups)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    want, tol = grad_ref(r, None if g_lp is None else torch.where(seen, g_lp, 0.0), None if X is None else Xe, g_ent,
                         got.top_index, g_top)
    close(dx, want, tol + narrow(want, x.dtype), "gradient")
    if sizes is not None:
        past = torch.arange(V, device=x.device) >= sizes.expand(lead)[..., None]
        assert not bool(dx[past].any())
    return got


# ------------------------------------------------------------------------------------------ log-probabilities
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", LENGTHS)
def test_log_prob_lengths(V, dtype):
    n = rows_for(V)
    x = make((n, V), dtype, seed=V)
    X = ints(V, (n,), seed=V + 1)
    check_log_prob(x, X=X, entropy=True, top=min(64, V + 2), grads=True)
    check_log_prob(x, X=X)
    check_log_prob(x, top=1)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V, rows", [(64, 4000), (1025, 700), (3000, 2050), (9000, 1100), (20000, 129)])
def test_log_prob_many_rows(V, rows, dtype):
    x = make((rows, V), dtype, seed=V)
    check_log_prob(x, X=ints(V, (rows,)), M=rand((rows,)) < 0.5, entropy=True, top=8, grads=True)
    check_log_prob(x, X=ints(V, (rows,)), M=rand((rows,)) < 0.5, grads=True)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [2, 6, 32, 300, 1500, 40000])
def test_samples_data_mask_and_sizes(V, dtype):
    """logits [S, B, D, V] with X, M [B, D] and sizes [D]; masked places hold no category, what lies past a row's size is
    NaN"""
    S, B, D = 3, 4, 5
    x = make((S, B, D, V), dtype, seed=V)
    sizes = torch.tensor([V, 1, max(1, V // 2), V - 1, max(1, V - V // 3)], dtype=torch.int32, device="cuda")
    X = (rand((B, D)) * sizes).long()
    M = rand((B, D), 3) < 0.6
    X = torch.where(M, X, -7)
    past = torch.arange(V, device="cuda") >= sizes[:, None]
    x = x.masked_fill(past, float("nan"))
    clean = x.masked_fill(past, 0.0)
    got = check_log_prob_nan_past(x, clean, X, M, sizes)
    assert bool((got.log_prob[:, ~M] == 0).all())


def check_log_prob_nan_past(x, clean, X, M, sizes):
    want = check_log_prob(clean, X=X, M=M, sizes=sizes, entropy=True, top=3, grads=True)
    z = x.detach().requires_grad_()
    got = dmv.categorical_log_prob(z, X, M, sizes=sizes, entropy=True, top=3)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    (dx,) = torch.autograd.grad(got.log_prob.sum(), z)
    assert bool(torch.isfinite(dx).all())
    return got


@pytest.mark.parametrize("V", [10, 700, 3000, 60000])
def test_broadcast_shapes(V):
    x = make((2, 3, 4, V), torch.float32, seed=1)
    for shape in [(2, 3, 4), (3, 4), (4,), (1, 3, 4), (2, 1, 4), (2, 3, 1), (1, 1, 1), ()]:
        X, M = ints(V, shape), rand(shape) < 0.7
        sizes = torch.full(shape, V, dtype=torch.int64, device="cuda")
        check_log_prob(x, X=X, M=M, sizes=sizes, entropy=True)
        check_log_prob(x, X=X.to(torch.int32))
    check_log_prob(x, X=ints(V, (4,)), sizes=torch.tensor(2 ** 40, device="cuda").expand(4), entropy=True)
    check_log_prob(make((V,), torch.float32), X=ints(V, ()), entropy=True, top=2, grads=True)      # one row without leading dimensions


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [1, 5, 24, 100, 1000, 1500, 33333])
def test_strides_and_alignment(V, dtype):
    n = 9
    big = make((n, V + 7), dtype, seed=3)
    X = ints(V, (n,))
    for off in (0, 1, 3):
        check_log_prob(big[:, off:off + V], X=X, entropy=True, top=min(V, 4), grads=True)      # a pitch, and any element alignment
    check_log_prob(make((V, n), dtype).t(), X=X, entropy=True, top=1, grads=True)              # categories not contiguous
    check_log_prob(make((2 * n, V), dtype)[::2], X=X, entropy=True, grads=True)
    check_log_prob(make((1, V), dtype).expand(n, V), X=X, entropy=True, grads=True)            # one row for all: pitch 0
    check_log_prob(make((3, n, V), dtype).transpose(0, 1), X=ints(V, (n, 3)), grads=True)


def test_gradient_of_broadcast_logits_adds_up():
    x = make((1, 40), torch.float32).requires_grad_()
    X = ints(40, (6,))
    dmv.categorical_log_prob(x.expand(6, 40), X).log_prob.sum().backward()
    r = Ref(x.detach().expand(6, 40))
    want, tol = grad_ref(r, torch.ones(6, device="cuda"), X, None, None, None)
    close(x.grad, want.sum(0, keepdim=True), tol.sum(0, keepdim=True) + 6 * E * want.abs().sum(0, keepdim=True), "sum")


def test_no_rows():
    x = torch.empty(0, 9, device="cuda", requires_grad=True)
    got = dmv.categorical_log_prob(x, torch.empty(0, dtype=torch.long, device="cuda"), entropy=True, top=2)
    assert got.log_prob.shape == (0,) and got.top_index.shape == (0, 2)
    got.log_prob.sum().backward()
    assert x.grad.shape == (0, 9)
    loss, per_row = dmv.distill_top_logits(x, torch.empty(0, 3, device="cuda"), torch.empty(0, 3, dtype=torch.long, device="cuda"))
    assert float(loss) == 0.0 and per_row.shape == (0,)


# ------------------------------------------------------------------------------------------ special values
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [4, 40, 1000, 2000, 70000])
def test_masked_logits_and_empty_rows(V, dtype):
    """-inf, the type's lowest value, rows that are nothing but those, NaN and +inf"""
    n = 12
    x = make((n, V), dtype, seed=4)
    low = torch.finfo(dtype).min
    x[0] = -math.inf                                   # nothing of non-zero probability
    x[1, 1:] = -math.inf                               # certain
    x[2, ::2] = -math.inf
    x[3] = low                                         # all equal, however low
    x[4, :-1] = low                                    # certain of the last
    x[5] = torch.finfo(dtype).max
    x[6] = 0.0
    x[7, 0] = torch.finfo(dtype).max
    sizes = torch.full((n,), V, dtype=torch.int32, device="cuda")
    sizes[8] = 0                                       # no categories at all
    sizes[9] = -3
    X = torch.zeros(n, dtype=torch.long, device="cuda")
    X[2], X[4] = 1, V - 1
    M = torch.ones(n, dtype=torch.bool, device="cuda")
    M[8] = M[9] = False
    top = min(V, 20)
    check_log_prob(x, X=X, M=M, sizes=sizes.clamp(min=0), entropy=True, top=top, grads=True)
    got = dmv.categorical_log_prob(x, X, M, sizes=sizes, entropy=True, top=top)
    for row in (0, 8, 9):
        assert float(got.entropy[row]) == 0.0 and bool((got.top_index[row] == -1).all()) and bool((got.top_log_prob[row] == -math.inf).all())
    assert float(got.log_prob[0]) == -math.inf
    # a category that cannot be: -inf, and the formula's finite gradient
    z = x[1:2].detach().requires_grad_()
    lp = dmv.categorical_log_prob(z, torch.tensor([1], device="cuda")).log_prob
    assert float(lp) == -math.inf
    (dx,) = torch.autograd.grad(lp.sum(), z)
    assert float(dx[0, 1]) == 1.0 and float(dx[0, 0]) == -1.0


@pytest.mark.parametrize("V", [4, 40, 1000, 2000, 70000])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_nan_and_inf_show(V, value):
    x = make((3, V), torch.float32, seed=6)
    x[1, V // 2] = value
    z = x.clone().requires_grad_()
    X = torch.zeros(3, dtype=torch.long, device="cuda")
    got = dmv.categorical_log_prob(z, X, entropy=True, top=3)
    for t in (got.log_prob, got.entropy, got.top_log_prob):
        assert bool(t[1].isnan().all()) and bool(torch.isfinite(t[0]).all()) and bool(torch.isfinite(t[2]).all())
    assert bool((got.top_index[1] == -1).all()) and bool((got.top_index[0] >= 0).all())
    (dx,) = torch.autograd.grad(got.log_prob.sum(), z)
    assert bool(dx[1].isnan().all()) and bool(torch.isfinite(dx[::2]).all())
    # where the row is not seen its NaN stays out
    M = torch.tensor([True, False, True], device="cuda")
    z2 = x.clone().requires_grad_()
    lp = dmv.categorical_log_prob(z2, X, M).log_prob
    assert float(lp[1].detach()) == 0.0
    (dx,) = torch.autograd.grad(lp.sum(), z2)
    assert bool((dx[1] == 0).all()) and bool(torch.isfinite(dx).all())


@pytest.mark.parametrize("V", [5, 300, 3000, 70000])
def test_given_category_out_of_range_shows(V):
    x = make((4, V), torch.float32).requires_grad_()
    X = torch.tensor([0, V, -1, 2], device="cuda")
    got = dmv.categorical_log_prob(x, X, entropy=True)
    assert got.log_prob.isnan().tolist() == [False, True, True, False] and bool(torch.isfinite(got.entropy).all())
    (dx,) = torch.autograd.grad(got.log_prob.sum(), x)
    assert dx.isnan().all(-1).tolist() == [False, True, True, False] and bool(torch.isfinite(dx[0]).all())


@pytest.mark.parametrize("V", [2, 12, 500, 2500, 50000, 200000])
def test_nearly_certain_rows_keep_relative_accuracy(V):
    """log q next to 0: the largest category's own rounding must not show (relative accuracy of the small numbers)"""
    x = make((6, V), torch.float32, seed=8, scale=1.0)
    at = ints(V, (6,))
    x.scatter_(-1, at[:, None], torch.tensor([18.0, 20.0, 25.0, 30.0, 22.0, 60.0], device="cuda")[:, None])
    z = x.requires_grad_()
    got = dmv.categorical_log_prob(z, at, entropy=True, top=1)
    r = Ref(x.detach())
    want = r.log_q.gather(-1, at[:, None])[:, 0]
    rel = E * (4 * 80 + r.C + 40)      # exponents of up to 80, times 3 roundings and the sum's
    close(got.log_prob, want, rel * want.abs(), "log_prob")
    close(got.top_log_prob[:, 0], want, rel * want.abs(), "top")
    close(got.entropy, r.H[:, 0], 2 * rel * r.H[:, 0], "entropy")
    (dx,) = torch.autograd.grad(got.log_prob.sum(), z)
    close(dx.gather(-1, at[:, None])[:, 0], -torch.expm1(want), 2 * rel * want.abs(), "gradient")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [6, 64, 1000, 1025, 5000, 66000, 140000])
@pytest.mark.parametrize("top", [1, 5, 64])
def test_equal_logits_rank_by_index(V, top, dtype):
    x = make((8, V), dtype, seed=V)
    x[0] = 1.5                                                  # all equal
    x[1] = -0.0
    x[1, 1::2] = 0.0                                            # equal too
    x[2] = (x[2].float() * 2).round().clamp(-3, 3)              # a few values, many times each
    x[3] = x[3].float().round()
    x[4, :] = -2.0
    x[4, -1] = 3.0
    x[5, V // 3:] = -math.inf
    x[6] = torch.arange(V, device="cuda").float().mul(8.0 / V).to(dtype)      # rising
    x[7] = -torch.arange(V, device="cuda").float().mul(8.0 / V).to(dtype)     # falling
    check_log_prob(x, top=top)
    check_log_prob(x.repeat(40, 1), top=top)                    # one workgroup per row


@pytest.mark.parametrize("dtype, slot", [(torch.float32, 4), (torch.bfloat16, 8), (torch.float16, 8)], ids=str)
@pytest.mark.parametrize("rows", [1, 300])
def test_selection_when_few_threads_hold_all_large_values(rows, dtype, slot):
    """large values in the slots of 63 of 256 threads only, more of them than the candidate list holds, distinct or equal"""
    V = 65536
    s = torch.arange(V, device="cuda") // slot % 256
    for large in (4.0 + rand((rows, V), 9), torch.full((rows, V), 4.0, device="cuda")):
        x = torch.where(s < 63, large, -large - rand((rows, V), 10)).to(dtype)
        check_log_prob(x, top=64)
        check_log_prob(x, top=7, entropy=True)


@pytest.mark.parametrize("dtype, slot", [(torch.float32, 4), (torch.bfloat16, 8), (torch.float16, 8)], ids=str)
@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("threads", [1, 3, 20])
def test_selection_when_few_threads_have_any_value(rows, threads, dtype, slot):
    """fewer threads with a finite value than alternatives asked for, and more such values than the candidate list holds"""
    V = 65536
    s = torch.arange(V, device="cuda") // slot % 256
    for v in (make((rows, V), torch.float32, seed=3), torch.full((rows, V), -1.0, device="cuda"), make((rows, V), torch.float32).round()):
        x = torch.where(s < threads, v, -math.inf).to(dtype)
        check_log_prob(x, top=64)
        check_log_prob(x, top=5, entropy=True)


# ------------------------------------------------------------------------------------------ differences
@pytest.mark.parametrize("V", [3, 50, 1500, 40000])
def test_gradient_against_differences(V):
    """directional derivative of the weighted outputs.  With |direction| <= 1 an element, the third derivative of log-sum-exp
    and of the entropy along it is below 8 (1 + max|log q|), so the central difference of step s is off by s^2 / 6 of that
    per row; its rounding is the outputs' tolerance over s."""
    n, s = 4, 2.0 ** -6
    x = make((n, V), torch.float32, seed=11)
    X = ints(V, (n,))
    w, v, d = rand((n,), 12), rand((n,), 13), 2 * rand((n, V), 14) - 1
    z = x.clone().requires_grad_()
    o = dmv.categorical_log_prob(z, X, entropy=True)
    (dx,) = torch.autograd.grad((o.log_prob, o.entropy), z, (w, v))
    along = (dx.double() * d.double()).sum(-1)
    f = lambda t: dmv.categorical_log_prob(t, X, entropy=True)  # noqa: E731
    up, dn = f(x + s * d), f(x - s * d)
    diff = (w.double() * (up.log_prob.double() - dn.log_prob.double()) + v.double() * (up.entropy.double() - dn.entropy.double())) / (2 * s)
    r = Ref(x)
    noise = (r.tol_log_q().gather(-1, X[:, None])[:, 0] + r.tol_H()[:, 0] + 2 * E * (x.abs().amax(-1) + s)) / s * 1.5
    close(diff, along, s * s / 6 * 8 * (1 + r.dist.amax(-1)) * 2 + noise, "difference")


# ------------------------------------------------------------------------------------------ distillation
def teacher_of(x, k, seed=20, dtype=None):
    t = 0.6 * x.float() + 1.5 * make(x.shape, torch.float32, seed=seed, scale=1.0)
    v, i = torch.sort(t, dim=-1, descending=True)
    return v[..., :k].contiguous().to(dtype or x.dtype), i[..., :k].contiguous()


def distill_ref(x, t, idx, w, T, sizes=None):
    r = Ref(x, sizes, T)
    counts = (idx >= 0) & (t != -math.inf)
    tt = torch.where(counts, t.double() / T, -math.inf)
    some = counts.any(-1, keepdim=True)
    log_p = torch.where(some, torch.log_softmax(torch.where(some, tt, 0.0), -1), -math.inf)
    p = log_p.exp()
    at = idx.clamp(min=0)
    lq = r.log_q.gather(-1, at)
    kl = torch.where(p > 0, p * (log_p - lq), 0.0).sum(-1)
    # errors of log p and log q, and of p itself
    dt = (tt - tt.amax(-1, keepdim=True)).abs().nan_to_num(0.0, 0.0, 0.0)
    e_lp = E * (5 * dt + 3 * (p * dt).sum(-1, keepdim=True) + 64)
    e_lq = r.tol_log_q().gather(-1, at) * 1.5
    tol_kl = torch.where(p > 0, p * (e_lp + e_lq + (log_p - lq).abs() * (e_lp + 16 * E)), 0.0).sum(-1)
    sp = torch.zeros_like(r.q).scatter_add_(-1, at, torch.where(counts, p, 0.0))
    P = p.sum(-1, keepdim=True)
    g = P * r.q - sp
    e_p = torch.zeros_like(r.q).scatter_add_(-1, at, torch.where(counts, p * (e_lp + 8 * E), 0.0))
    tol_g = r.q * (r.tol_q() + r.tol_log_q() + 8 * E) + e_p + FLUSH
    scale = (w.double() / T)[..., None]
    return kl, tol_kl, g * scale, tol_g * scale.abs() + 3 * E * (g * scale).abs()


def check_distill(x, t, idx, weight=None, T=1.0, sizes=None, upstream=None):
    lead = x.shape[:-1]
    z = x.detach().requires_grad_()
    loss, per_row = dmv.distill_top_logits(z, t, idx, sizes=sizes, weight=weight, temperature=T)
    (dx,) = torch.autograd.grad(loss if upstream is None else loss * upstream, z)
    w = torch.ones(lead, device="cuda") if weight is None else weight.expand(lead)
    te, ie = t.expand(*lead, t.shape[-1]), idx.expand(*lead, t.shape[-1])
    kl, tol, g, tol_g = distill_ref(x.detach(), te, ie, w, T, None if sizes is None else sizes.expand(lead))
    live = w != 0
    close(per_row, torch.where(live, kl, 0.0), torch.where(live, tol, 0.0), "per_row")
    assert not per_row.requires_grad and loss.dtype == per_row.dtype == torch.float32
    total = torch.where(live, w.double() * kl, 0.0).sum()
    close(loss.detach(), total, (w.abs().double() * tol).sum() + 2 * E * total.abs(), "loss")
    u = 1.0 if upstream is None else upstream
    close(dx, torch.where(live[..., None], u * g, 0.0), abs(u) * (tol_g + 2 * E * g.abs()) + narrow(u * g, x.dtype), "gradient")
    # the loss alone, without its gradient, is the same
    loss2, per_row2 = dmv.distill_top_logits(x.detach(), t, idx, sizes=sizes, weight=weight, temperature=T)
    assert torch.equal(loss2, loss.detach()) and torch.equal(per_row2, per_row) and not loss2.requires_grad
    return loss, per_row, dx


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", LENGTHS)
def test_distill_lengths(V, dtype):
    n = rows_for(V)
    x = make((n, V), dtype, seed=V)
    for k, T in ((1, 1.0), (min(V, 10), 2.0), (min(V, 256), 0.7)):
        t, idx = teacher_of(x, k)
        check_distill(x, t, idx, T=T)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V, rows", [(20, 5000), (256, 3000), (1025, 300), (2600, 150), (9001, 150), (20000, 140), (33000, 130),
                                     (65600, 130), (131000, 130)])
def test_distill_many_rows(V, rows, dtype):
    """every register tile of the kernels that hold a whole row"""
    x = make((rows, V), dtype, seed=V)
    t, idx = teacher_of(x, 8)
    w = rand((rows,)) * (rand((rows,), 7) < 0.6)
    check_distill(x, t, idx, weight=w, T=2.0)


@pytest.mark.parametrize("V", [30, 1000, 3000, 90000])
@pytest.mark.parametrize("rows", [3, 200])
def test_distill_upstream_gradient(V, rows):
    """any upstream gradient, powers of two that only half precision would lose among them, with one rounding"""
    x = make((rows, V), torch.float16, seed=V)
    t, idx = teacher_of(x, 5)
    w = torch.full((rows,), 2.0 ** -20, device="cuda")
    for u in (2.0 ** 16, -0.3, 1.0, 0.0):
        check_distill(x, t, idx, weight=w, upstream=u)


@pytest.mark.parametrize("V", [30, 3000, 90000])
@pytest.mark.parametrize("rows", [3, 200])
def test_distill_backward_twice_and_accumulation(V, rows):
    x = make((rows, V), torch.float32, seed=V).requires_grad_()
    t, idx = teacher_of(x.detach(), 5)
    loss, _ = dmv.distill_top_logits(x, t, idx)
    loss.backward(retain_graph=True)
    once = x.grad.clone()
    loss.backward(retain_graph=True)
    assert torch.equal(x.grad, 2 * once)
    x.grad = None
    (3.0 * loss).backward()
    _, _, g, tol = distill_ref(x.detach(), t, idx, torch.ones(rows, device="cuda"), 1.0)
    close(x.grad, 3 * g, 3 * tol + 6 * E * g.abs(), "scaled")
    # two losses of the same logits add up
    x.grad = None
    (dmv.distill_top_logits(x, t, idx)[0] + dmv.distill_top_logits(x, t, idx)[0]).backward()
    assert torch.equal(x.grad, 2 * once)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [6, 40, 1000, 2000, 66000])
@pytest.mark.parametrize("rows", [11, 150])
def test_distill_entries(V, rows, dtype):
    """empty entries, categories given more than once, rows without any entry, ragged sizes"""
    k = 6
    x = make((rows, V), dtype, seed=V)
    t, idx = teacher_of(x, k)
    idx[0, 2:] = -1
    t[1, 1:] = -math.inf
    idx[2] = -1                                       # nothing given
    idx[3, 1] = idx[3, 0]                             # the same category twice
    idx[4] = idx[4, 0]                                # ... and all the time
    idx[5, 3], idx[5, 5] = idx[5, 0], idx[5, 1]
    t[6, 0] = 80.0                                    # certain: the others underflow
    x[7, idx[7, 0]] = 50.0                            # the student is certain
    t[8] = -math.inf
    idx[9, 0] = -5
    w = rand((rows,), 4) + 0.1
    loss, per_row, dx = check_distill(x, t, idx, weight=w, T=2.0)
    for row in (2, 8):
        assert float(per_row[row]) == 0.0 and not bool(dx[row].any())
    # the same with sizes, where nothing past them is given
    sizes = torch.full((rows,), V, dtype=torch.int32, device="cuda")
    sizes[::2] = V - 1
    idx = idx.clamp(max=V - 2)
    y = x.clone()
    y[::2, V - 1] = float("nan")
    z = x.clone()
    z[::2, V - 1] = 0.0
    a = check_distill(z, t, idx, weight=w, T=0.5, sizes=sizes)
    zz = y.requires_grad_()
    loss, per_row = dmv.distill_top_logits(zz, t, idx, sizes=sizes, weight=w, temperature=0.5)
    (dy,) = torch.autograd.grad(loss, zz)
    assert torch.equal(per_row, a[1]) and torch.equal(dy, a[2])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [2, 7, 30, 100, 128, 200, 256, 700, 3000, 70000])
@pytest.mark.parametrize("k", [65, 129, 256])
@pytest.mark.parametrize("rows", [3, 700])
def test_distill_many_entries(V, k, rows, dtype):
    """as many entries as may be given, more than there are categories: most of them given several times, some empty"""
    rows = min(rows, 20_000_000 // V)
    x = make((rows, V), dtype, seed=V)
    idx = ints(V, (rows, k), seed=k)
    idx[rand((rows, k), 6) < 0.1] = -1
    check_distill(x, make((rows, k), torch.float32, seed=k), idx, weight=rand((rows,)) + 0.1, T=1.5)


def test_temperatures():
    x = make((5, 900), torch.float32, seed=2)
    t, idx = teacher_of(x, 9)
    for T in (0.05, 0.7, 30.0, 1e4):
        check_distill(x, t, idx, T=T)
    for T in (1e-30, 1e30):
        loss, per_row = dmv.distill_top_logits(x, t, idx, temperature=T)
        assert not bool(per_row.isnan().any())


@pytest.mark.parametrize("V", [40, 5000])
def test_saved_logits_and_second_derivatives(V):
    x = make((4, V), torch.float32)
    X = ints(V, (4,))
    t, idx = teacher_of(x, 3)
    for f in (lambda z: dmv.categorical_log_prob(z, X).log_prob.sum(), lambda z: dmv.distill_top_logits(z, t, idx)[0]):
        z = x.clone().requires_grad_()
        y = 1.0 * z
        loss = f(y)
        with torch.no_grad():
            y.add_(1.0)                                # written over after the forward pass
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        (g,) = torch.autograd.grad(f(z), z, create_graph=True)
        (want,) = torch.autograd.grad(f(z), z)
        assert torch.equal(g.detach(), want)
        with pytest.raises(RuntimeError, match="no second derivative"):
            g.sum().backward()


@pytest.mark.parametrize("V", [6, 1000, 2000, 66000])
@pytest.mark.parametrize("rows", [5, 140])
def test_distill_special_rows(V, rows):
    x = make((rows, V), torch.float32, seed=V)
    t, idx = teacher_of(x, 3)
    idx[0, 1] = V                                     # no such category
    x[1] = -math.inf                                  # the student allows nothing
    x[2, idx[2, 1]] = -math.inf                       # ... or not what the teacher gives
    t[3, 2] = math.nan
    x[4, 0] = math.nan
    z = x.clone().requires_grad_()
    loss, per_row = dmv.distill_top_logits(z, t, idx)
    (dx,) = torch.autograd.grad(loss, z)
    assert per_row[0].isnan() and dx[0].isnan().all()
    assert float(per_row[1]) == math.inf and not bool(dx[1].any())
    assert float(per_row[2]) == math.inf and bool(torch.isfinite(dx[2]).all()) and float(dx[2, idx[2, 1]]) < 0
    assert per_row[3].isnan() and dx[3].isnan().all() and per_row[4].isnan() and loss.isnan()
    assert bool(torch.isfinite(per_row[5:]).all()) and bool(torch.isfinite(dx[5:]).all())
    # weight 0 leaves all of them out
    w = torch.ones(rows, device="cuda")
    w[:5] = 0
    z2 = x.clone().requires_grad_()
    loss, per_row = dmv.distill_top_logits(z2, t, idx, weight=w)
    (dx,) = torch.autograd.grad(loss, z2)
    assert bool(torch.isfinite(loss)) and not bool(per_row[:5].any()) and not bool(dx[:5].any()) and bool(torch.isfinite(dx).all())


@pytest.mark.parametrize("V", [9, 700, 3000, 70000])
def test_distill_broadcast_strides_and_types(V):
    S, B, D, k = 2, 3, 4, 5
    x = make((S, B, D, V), torch.bfloat16, seed=V)
    t, idx = teacher_of(x[0], k, dtype=torch.float32)            # one teacher for all samples
    w = rand((B, D)) * (rand((B, D), 8) < 0.7)
    check_distill(x, t, idx, weight=w)
    check_distill(x, t[:1, :1], idx[:1, :1], weight=w[:1])
    check_distill(x, t.to(torch.float16), idx, weight=rand((D,)))
    wide = make((7, V + 5), torch.float32, seed=1)
    t, idx = teacher_of(wide[:, 3:3 + V], k)
    check_distill(wide[:, 3:3 + V], t, idx)
    check_distill(make((V, 7), torch.float32).t(), t, idx.to(torch.int32))
    check_distill(make((1, V), torch.float32).expand(7, V), t, idx)
    check_distill(make((V,), torch.float32), t[0], idx[0])


@pytest.mark.parametrize("V", [40, 2000, 40000])
def test_distill_gradient_against_differences(V):
    """as above: KL differs from -sum p log q by a constant, its third derivative along a direction of at most 1 is below 8"""
    n, s = 4, 2.0 ** -6
    x = make((n, V), torch.float32, seed=15)
    t, idx = teacher_of(x, 6)
    d, w = 2 * rand((n, V), 16) - 1, rand((n,), 17) + 0.5
    z = x.clone().requires_grad_()
    loss, _ = dmv.distill_top_logits(z, t, idx, weight=w)
    (dx,) = torch.autograd.grad(loss, z)
    along = (dx.double() * d.double()).sum(-1)
    f = lambda y: dmv.distill_top_logits(y, t, idx, weight=w)[1].double()  # noqa: E731
    diff = w.double() * (f(x + s * d) - f(x - s * d)) / (2 * s)
    _, tol, _, _ = distill_ref(x, t, idx, w, 1.0)
    close(diff, along, w.double() * (s * s / 6 * 8 + (1.5 * tol + 2 * E * (x.abs().amax(-1) + s)) / s), "difference")


# ------------------------------------------------------------------------------------------ as they are used
def test_results_repeat_and_inputs_stay():
    for V, rows in ((200, 500), (5000, 300), (100000, 3)):
        x = make((rows, V), torch.bfloat16, seed=V)
        keep = x.clone()
        X = ints(V, (rows,))
        t, idx = teacher_of(x, 16)
        once = [check_distill(x, t, idx), check_log_prob(x, X=X, entropy=True, top=16, grads=True)]
        for _ in range(3):
            a, b = check_distill(x, t, idx), dmv.categorical_log_prob(x, X, entropy=True, top=16)
            assert all(torch.equal(p, q) for p, q in zip(a, once[0])) and all(torch.equal(p, q) for p, q in zip(b, once[1]))
        assert torch.equal(x, keep)


def test_side_stream():
    x, X = make((64, 3000), torch.float32), ints(3000, (64,))
    want = dmv.categorical_log_prob(x, X, entropy=True, top=4)
    t, idx = teacher_of(x, 4)
    wloss, _ = dmv.distill_top_logits(x, t, idx)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = dmv.categorical_log_prob(x, X, entropy=True, top=4)
        z = x.detach().requires_grad_()
        loss, _ = dmv.distill_top_logits(z, t, idx)
        loss.backward()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(loss.detach(), wloss)


@pytest.mark.parametrize("V", [25, 3000, 70000])
def test_a_step_of_both_records_into_graphs(V):
    """Imputation by distillation: the teacher's alternatives of every entry, the observed entries' log-likelihood, the
    missing ones' distillation, gradients of both - eager, and recorded twice into graphs that are replayed in turn, with
    eager work in between."""
    B, D, k = 6, 3, 4
    teacher, x = make((B, D, V), torch.float32, seed=1), make((B, D, V), torch.float32, seed=2)
    X, M = ints(V, (B, D)), rand((B, D)) < 0.5
    sizes = torch.tensor([V, V - 1, max(k, V // 2)], dtype=torch.int32, device="cuda")
    X = torch.minimum(X, sizes.long() - 1)
    miss = (~M).float()

    def step(student, teach):
        z = student.detach().requires_grad_()
        a = dmv.categorical_log_prob(teach, sizes=sizes, entropy=True, top=k)
        loss, kl = dmv.distill_top_logits(z, a.top_log_prob, a.top_index, sizes=sizes, weight=miss)
        lp = dmv.categorical_log_prob(z, X, M, sizes=sizes, entropy=True)
        total = loss - lp.log_prob.sum() - 0.1 * lp.entropy.sum()
        (g,) = torch.autograd.grad(total, z)
        return a.entropy, a.top_index, kl, lp.log_prob.detach(), total.detach(), g

    # against 64 bits
    got = step(x, teacher)
    r, rt = Ref(x, sizes), Ref(teacher, sizes)
    lp, idx = rt.top(k)
    assert torch.equal(got[1], idx)
    kl, tol, g, tol_g = distill_ref(x, lp.float(), idx, miss, 1.0, sizes)
    close(got[2], torch.where(M, 0.0, kl), torch.where(M, 0.0, tol + 16 * E), "kl")
    ones = -torch.ones(B, D, device="cuda")
    g2, tol2 = grad_ref(r, torch.where(M, ones, 0.0), X, 0.1 * ones, None, None)
    close(got[5], torch.where(M[..., None], 0.0, g) + g2, tol_g + tol2 + 32 * E * (g.abs() + g2.abs() + r.q), "gradient")

    bufs = [(x.clone(), teacher.clone()) for _ in range(2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for b in bufs:
            step(*b)
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for b in bufs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*b))
        graphs.append(graph)
    for it in range(3):
        for i in (0, 1):
            bufs[i][0].copy_(make((B, D, V), torch.float32, seed=100 + 2 * it + i))
            bufs[i][1].copy_(make((B, D, V), torch.float32, seed=200 + 2 * it + i))
        for graph in graphs:
            graph.replay()
        eager = [step(*b) for b in bufs]
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert all(torch.equal(p, q) for p, q in zip(o, e)), it


def test_offsets_past_32_bits():
    """rows whose byte offset passes 2^32, and whose element offset passes 2^31"""
    V, rows = 65536 + 1, 34000
    x = torch.empty(rows, V, dtype=torch.bfloat16, device="cuda")
    x.copy_(make((1, V), torch.bfloat16).expand(rows, V))
    last = make((3, V), torch.bfloat16, seed=31)
    x[-3:] = last
    X = ints(V, (rows,), seed=32)
    got = dmv.categorical_log_prob(x, X, entropy=True, top=3)
    want = check_log_prob(last, X=X[-3:], entropy=True, top=3)
    tail = [t[-3:] for t in got]
    assert torch.equal(tail[3], want.top_index)
    close(tail[0], want.log_prob.double(), 2 * E * (100 + V / 128), "log_prob")       # another split of the same row
    close(tail[1], want.entropy.double(), 2 * E * (500 + V / 64), "entropy")
    del got
    z = x.requires_grad_()
    lp = dmv.categorical_log_prob(z, X).log_prob
    (dx,) = torch.autograd.grad(lp.sum(), z)
    r = Ref(last)
    w, tol = grad_ref(r, torch.ones(3, device="cuda"), X[-3:], None, None, None)
    close(dx[-3:], w, tol + narrow(w, torch.bfloat16), "gradient")
    del dx, lp
    t, idx = teacher_of(last, 4)
    weight = torch.zeros(rows, device="cuda")
    weight[-3:] = 1
    T, I = torch.zeros(rows, 4, dtype=torch.bfloat16, device="cuda"), torch.zeros(rows, 4, dtype=torch.long, device="cuda")
    T[-3:], I[-3:] = t, idx
    loss, per_row = dmv.distill_top_logits(z, T, I, weight=weight)
    (dx,) = torch.autograd.grad(loss, z)
    kl, tol, g, tol_g = distill_ref(last, t, idx, torch.ones(3, device="cuda"), 1.0)
    close(per_row[-3:], kl, tol, "kl")
    close(dx[-3:], g, tol_g + narrow(g, torch.bfloat16), "gradient")
    assert not bool(dx[:-3].any())


# ------------------------------------------------------------------------------------------ what a backward pass holds
def _losses(V, n=4):
    x = make((n, V), torch.float32)
    X = ints(V, (n,))
    t, idx = teacher_of(x, 3)
    return x, [lambda z: dmv.categorical_log_prob(z, X, entropy=True).log_prob.sum(), lambda z: dmv.distill_top_logits(z, t, idx)[0] * 2.0]


@pytest.mark.parametrize("V", [40, 5000, 90000])
def test_saved_logits_come_back_from_elsewhere(V):
    """saved tensors kept on the host, or computed again: the first copy's memory is somebody else's by then"""
    from torch.utils.checkpoint import checkpoint
    x, losses = _losses(V)
    for f in losses:
        z = x.clone().requires_grad_()
        (want,) = torch.autograd.grad(f(1.0 * z), z)
        for rows in (lambda y: y, lambda y: torch.cat([y, y], -1)[:, :V], lambda y: (1.0 * y.t()).t()):     # a pitch; a copy
            with torch.autograd.graph.save_on_cpu():
                loss = f(rows(1.0 * z))
            others = [torch.full((4, V), 7.0, device="cuda") for _ in range(8)]
            (got,) = torch.autograd.grad(loss, z)
            assert torch.equal(got, want)
            loss = checkpoint(lambda z: f(rows(1.0 * z)), z, use_reentrant=False)
            others += [torch.full((4, V), 7.0, device="cuda") for _ in range(8)]
            (got,) = torch.autograd.grad(loss, z)
            assert torch.equal(got, want)


@pytest.mark.parametrize("V", [40, 5000])
def test_arguments_modified_before_the_backward_pass(V):
    n = 4
    x = make((n, V), torch.float32)

    def refused(loss, z, t):
        t.add_(1) if t.dtype != torch.bool else t.logical_not_()
        with pytest.raises(RuntimeError, match="modified in place"):
            torch.autograd.grad(loss, z)

    for name in ("X", "M", "sizes"):
        a = dict(X=ints(V - 1, (n,)), M=rand((n,)) < 0.5, sizes=torch.full((n,), V - 1, dtype=torch.int32, device="cuda"))
        z = x.clone().requires_grad_()
        refused(dmv.categorical_log_prob(z, **a).log_prob.sum(), z, a[name])
    for name in ("top_logits", "top_index", "weight", "sizes"):
        t, idx = teacher_of(x[:, :V - 1], 3)
        a = dict(top_logits=t, top_index=idx, weight=rand((n,)), sizes=torch.full((n,), V - 1, dtype=torch.int32, device="cuda"))
        z = x.clone().requires_grad_()
        refused(dmv.distill_top_logits(z, **a)[0], z, a[name])


@pytest.mark.parametrize("V", [40, 5000])
def test_a_teacher_in_inference_mode(V):
    x = make((4, V), torch.float32, seed=2)
    with torch.inference_mode():
        a = dmv.categorical_log_prob(make((4, V), torch.float32, seed=1), top=5)
    check_distill(x, a.top_log_prob.clone(), a.top_index.clone())
    z = x.clone().requires_grad_()
    (got,) = torch.autograd.grad(dmv.distill_top_logits(z, a.top_log_prob, a.top_index)[0], z)
    (want,) = torch.autograd.grad(dmv.distill_top_logits(z, a.top_log_prob.clone(), a.top_index.clone())[0], z)
    assert torch.equal(got, want)


@pytest.mark.parametrize("V", [40, 5000, 90000])
def test_forward_and_backward_in_graphs_of_their_own(V):
    """the backward pass replayed twice for one forward pass, with another upstream gradient each time"""
    x = make((4, V), torch.float32)
    t, idx = teacher_of(x, 3)
    z, u = x.clone().requires_grad_(), torch.ones((), device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        loss, _ = dmv.distill_top_logits(z, t, idx)
        want = torch.autograd.grad(loss, z)[0].clone()
    del loss
    torch.cuda.synchronize()
    fwd, bwd = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(fwd, stream=s):
        loss, _ = dmv.distill_top_logits(z, t, idx)
    with torch.cuda.graph(bwd, stream=s):
        (g,) = torch.autograd.grad(loss, z, u)
    for _ in range(2):
        fwd.replay()
        for up in (2.0, 1.0, -4.0, 1.0):
            u.fill_(up)
            bwd.replay()
            torch.cuda.synchronize()
            assert torch.equal(g, want if up == 1.0 else up * want), up      # (powers of two)


# ------------------------------------------------------------------------------------------ arguments
@pytest.mark.parametrize("V", [300, 3000])
def test_sizes_of_every_integer_type(V):
    x = make((3, V), torch.float32)
    for dtype in (torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64):
        sizes = torch.tensor([3, 100, 127], dtype=dtype, device="cuda")
        check_log_prob(x, sizes=sizes, entropy=True)


@pytest.mark.parametrize("V", [40, 3000])
def test_weight_as_a_number(V):
    x = make((4, V), torch.float32)
    t, idx = teacher_of(x, 3)
    z = x.clone().requires_grad_()
    a = dmv.distill_top_logits(z, t, idx, weight=0.25)
    b = dmv.distill_top_logits(z, t, idx, weight=torch.full((4,), 0.25, device="cuda"))
    assert torch.equal(a[0], b[0]) and torch.equal(*(torch.autograd.grad(o[0], z)[0] for o in (a, b)))


@pytest.mark.parametrize("V", [40, 5000])
def test_large_upstream_gradient_of_the_entropy_leaves_masked_places(V):
    x = make((3, V), torch.float32)
    x[:, ::2] = -math.inf
    z = x.requires_grad_()
    (dx,) = torch.autograd.grad(dmv.categorical_log_prob(z, entropy=True).entropy.sum() * 2.0 ** 80, z)
    assert bool((dx[:, ::2] == 0).all()) and bool(torch.isfinite(dx).all())


@pytest.mark.parametrize("V", [40, 5000, 90000])
def test_distillation_looks_at_weights_and_not_at_the_rows_mask(V):
    """rows of weight 0 hold NaN; the C entry given the rows' X and M as well"""
    import ctypes as C
    from demiss_vae_amd import _lib as L
    x = make((5, V), torch.float32)
    t, idx = teacher_of(x, 3)
    w = torch.tensor([1.0, 0.0, 2.0, 0.0, 1.0], device="cuda")
    loss, per_row = dmv.distill_top_logits(x, t, idx, weight=w)
    x[w == 0] = math.nan
    again = dmv.distill_top_logits(x, t, idx, weight=w)
    assert torch.equal(again[0], loss) and torch.equal(again[1], per_row)
    X, M = ints(V, (5,)), torch.zeros(5, dtype=torch.bool, device="cuda")
    r = L.DmvCatRows(logits=x.data_ptr(), ld=V, rows=5, V=V, dtype=0, X=X.data_ptr(), x_period=5, M=M.data_ptr(), m_period=5)
    tc = L.DmvCatTeacher(logits=t.data_ptr(), index=idx.data_ptr(), period=5, k=3, dtype=0, weight=w.data_ptr(), w_period=5, temperature=1.0)
    n = L.lib().dmv_cat_distill_ws_bytes(C.byref(r), 3)
    ws = torch.empty(n // 4 + 4, device="cuda")
    out, rows = torch.empty((), device="cuda"), torch.empty(5, device="cuda")
    L.check(L.lib().dmv_cat_distill(C.byref(r), C.byref(tc), rows.data_ptr(), out.data_ptr(), None, None, 0, ws.data_ptr(), n,
                                    torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out, loss) and torch.equal(rows, per_row)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V, top", [(132, 16), (132, 32), (264, 32), (264, 64), (300, 17), (520, 33), (520, 64), (1030, 20), (1092, 64), (1500, 64)])
def test_alternatives_of_rows_that_fill_little_of_their_tile(V, top, dtype):
    """a lane group's width doubles at these lengths; sizes down to none, next to full rows in the same wavefront"""
    x = make((200, V), dtype, seed=V)
    check_log_prob(x, top=top)
    sizes = torch.randint(0, V + 1, (200,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(top), dtype=torch.int32)
    sizes[:8] = torch.tensor([0, 1, top - 1, top, top + 1, 2 * top, V // 4, V], device="cuda")
    check_log_prob(x, sizes=sizes, entropy=True, top=top, grads=True)
    check_log_prob(-x.abs() - 1, sizes=sizes, top=top)                      # nothing but negative values
    check_log_prob(torch.where(rand((200, V), 41) < 0.9, -math.inf, x.float()).to(dtype), sizes=sizes, top=top)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V, rows", [(2049, 5000), (4100, 300), (66000, 8), (140001, 3), (262147, 1), (262147, 9), (600000, 3)])
def test_alternatives_of_long_rows_with_few_elements(V, rows, dtype):
    """sizes down to none: threads and parts of a row without elements, and a last part with a few"""
    x = make((rows, V), dtype, seed=V)
    sizes = (rand((rows,), rows) ** 2 * V).int() + 1
    few = torch.tensor([V, 500, 70, 520, 1, 0, 64, 65], dtype=torch.int32, device="cuda")[:rows]
    sizes[:len(few)] = few
    for top in (64, 17, 3):
        check_log_prob(x, top=top)
        check_log_prob(x, sizes=sizes, entropy=True, top=top)
    low = torch.where(torch.arange(V, device="cuda") < V - 40, -math.inf, x.float()).to(dtype)      # the last part's elements only
    check_log_prob(low, top=64)
    check_log_prob(low, sizes=sizes, top=64)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V, rows", [(2049, 70), (2049, 4100), (50001, 9), (66001, 300), (262147, 8), (600000, 2)])
def test_alternatives_of_equal_values_in_long_rows(V, rows, dtype):
    """rows of one value (an untrained network's), of two, and of one value behind a few larger ones in every part"""
    x = torch.zeros(rows, V, dtype=dtype, device="cuda")
    check_log_prob(x, top=64)
    check_log_prob(x, top=1)
    x[:, ::3] = -1.5
    check_log_prob(x, top=64)
    x[:, V // 100::V // 37 + 1] = 2.0
    check_log_prob(x, top=50, sizes=torch.full((rows,), V - 3, dtype=torch.int32, device="cuda"))


# ------------------------------------------------------------------------------------------ more entries than categories
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [1, 2, 3, 7, 8, 10, 12, 16, 17, 31, 33])
@pytest.mark.parametrize("k", [17, 20, 33, 64, 65, 200])
@pytest.mark.parametrize("rows", [60, 700])
def test_distill_more_entries_than_categories(V, k, rows, dtype):
    """The alternatives of short rows, with nothing behind them, and entries given several times; rows of small and of
    large |log p|, many row groups in a workgroup.  The first entry of a row is its most probable one, and in every other
    row its least probable one, whose log p is the largest."""
    x = make((rows, V), dtype, seed=V)
    w = rand((rows,)) + 0.1
    a = dmv.categorical_log_prob(make((rows, V), torch.float32, seed=k, scale=3.0), top=min(k, 64))
    t, idx = a.top_log_prob, a.top_index
    t, idx = torch.nn.functional.pad(t, (0, k - t.shape[1]), value=-math.inf), torch.nn.functional.pad(idx, (0, k - idx.shape[1]), value=-1)
    have = min(V, k)
    order = torch.arange(k, device="cuda").repeat(rows, 1)
    order[1::2, :have] = torch.arange(have - 1, -1, -1, device="cuda")
    t, idx = t.gather(-1, order), idx.gather(-1, order)
    assert bool((idx[:, :have] >= 0).all()) and not bool((idx[:, have:] >= 0).any())
    once = check_distill(x, t, idx, weight=w, T=1.5)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(check_distill(x, t, idx, weight=w, T=1.5), once))
    check_distill(x, t, idx, weight=w, upstream=0.5)
    again = ints(V, (rows, k), seed=k)
    again[rand((rows, k), 6) < 0.1] = -1
    logits = make((rows, k), torch.float32, seed=k + 1, scale=4.0)
    once = check_distill(x, logits, again, weight=w)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(check_distill(x, logits, again, weight=w), once))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V, rows", [(3000, 700), (9000, 300), (9000, 40), (50001, 50), (262147, 5)])
def test_alternatives_from_many_candidates(V, rows, dtype):
    """Long rows of which 70 to 512 elements come into question, which are thinned out before they are ranked: few categories,
    and as many among the others, by workgroups of four and of sixteen wavefronts and in parts of rows.  Every call of
    the same rows gives the same."""
    x = make((rows, V), dtype, seed=V)
    few = torch.full((rows, V), -math.inf, dtype=dtype, device="cuda")
    at = torch.argsort(rand((rows, V), 51), dim=-1)[:, :400]
    few.scatter_(-1, at, x.gather(-1, at))
    for z, sizes in ((x, 500), (x, 300), (few, V)):
        sizes = torch.full((rows,), sizes, dtype=torch.int32, device="cuda")
        for top in (64, 20, 1):
            once = check_log_prob(z, sizes=sizes, entropy=True, top=top)
            for _ in range(5):
                again = dmv.categorical_log_prob(z, sizes=sizes, entropy=True, top=top)
                assert torch.equal(again.top_index, once.top_index) and torch.equal(again.top_log_prob, once.top_log_prob)


@pytest.mark.parametrize("V", [40, 5000, 90000])
def test_saved_logits_come_back_to_the_same_address(V):
    """... in rows of another pitch: what a hook kept elsewhere may get the memory of the first logits again"""
    x, losses = _losses(V)
    for f in losses:
        z = x.clone().requires_grad_()
        (want,) = torch.autograd.grad(f(1.0 * z), z)
        memory = torch.empty(4 * (V + 9), device="cuda")
        for ours, back in ((V + 9, V), (V, V + 9)):
            def pack(t):
                return t.clone()

            def unpack(t):
                if t.shape != (4, V):
                    return t
                again = memory.as_strided((4, V), (back, 1))
                return again.copy_(t)

            y = memory.as_strided((4, V), (ours, 1))
            y.copy_(x)
            y.requires_grad_()
            with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
                loss = f(y)
            memory.fill_(7.0)
            (got,) = torch.autograd.grad(loss, y)
            assert torch.equal(got, want)
            memory = torch.empty(4 * (V + 9), device="cuda")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [3, 40, 1000, 2000, 5000, 70000, 262147])
@pytest.mark.parametrize("rows", [8, 300])
def test_observed_entries_without_categories(V, rows, dtype):
    """Rows of size 0 and rows of nothing but -inf that are observed: -inf and a zero gradient, whatever category is given; a
    category that is none of the row's shows in every other row."""
    rows = min(rows, 20_000_000 // V)
    x = make((rows, V), dtype, seed=V)
    sizes = torch.full((rows,), V, dtype=torch.int32, device="cuda")
    X = ints(V, (rows,))
    sizes[:3] = torch.tensor([0, 0, -5], device="cuda")
    X[:3] = torch.tensor([0, V, -1], device="cuda")
    x[3:6] = -math.inf
    sizes[4] = V - 1
    X[3:6] = torch.tensor([0, V - 1, -1], device="cuda")
    sizes[6] = V - 1
    X[6] = V - 1
    for top in (0, min(V, 5)):
        for entropy in (False, True):
            z = x.clone().requires_grad_()
            got = dmv.categorical_log_prob(z, X, sizes=sizes, entropy=entropy, top=top)
            assert bool((got.log_prob[:6] == -math.inf).all()) and bool(got.log_prob[6].isnan())
            assert bool(torch.isfinite(got.log_prob[7:]).all())
            (dx,) = torch.autograd.grad(got.log_prob.sum(), z)
            assert not bool(dx[:6].any()) and bool(dx[6, :V - 1].isnan().all()) and float(dx[6, V - 1]) == 0.0
            assert bool(torch.isfinite(dx[7:]).all())
            if entropy:
                assert not bool(got.entropy[:6].any())
            if top:
                assert bool((got.top_index[:6] == -1).all()) and bool((got.top_log_prob[:6] == -math.inf).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V", [2, 3, 9, 40, 300, 1000, 2000, 2600, 9001, 70000, 200001])
@pytest.mark.parametrize("rows", [12, 300])
def test_distill_invalid_rows_with_sizes(V, rows, dtype):
    """What makes a row NaN makes its gradient NaN at each of its categories, and leaves 0 past its size, by every kernel and
    for every upstream gradient; a row without categories has a loss to tell and nothing to write."""
    rows = min(rows, 20_000_000 // V)
    x = make((rows, V), dtype, seed=V)
    k = 2 if V < 40 else 20
    sizes = torch.full((rows,), V - 1, dtype=torch.int32, device="cuda")
    t, idx = teacher_of(x[:, :V - 1], min(k, V - 1), dtype=torch.float32)
    t, idx = torch.nn.functional.pad(t, (0, k - t.shape[1]), value=-math.inf), torch.nn.functional.pad(idx, (0, k - idx.shape[1]), value=-1)
    w = rand((rows,)) + 0.1
    x[:, V - 1] = math.inf                              # past the size: not looked at
    idx[0, 0] = V - 1                                   # an index past the row's size
    t[1, 0] = math.nan
    t[2, 0] = math.inf
    x[3, 0] = math.nan
    x[4, V - 2] = math.inf
    x[5, :V - 1] = -math.inf                            # no probability anywhere ...
    x[6, :V - 1] = -math.inf
    idx[6, 0] = V - 1                                   # ... and an index past the row's size
    sizes[7] = 0                                        # no categories, and so every index past the row's size
    sizes[8] = 0
    idx[8] = -1                                         # ... and no entries either
    w[9] = math.nan
    for up in (None, 0.5, math.inf):
        z = x.clone().requires_grad_()
        loss, per_row = dmv.distill_top_logits(z, t, idx, sizes=sizes, weight=w)
        (dx,) = torch.autograd.grad(loss if up is None else loss * up, z)
        assert per_row[[0, 1, 2, 3, 4, 6, 7]].isnan().all() and float(per_row[5]) == math.inf and float(per_row[8]) == 0.0
        assert bool(torch.isfinite(per_row[9:]).all()) and bool(loss.isnan())
        past = torch.arange(V, device="cuda") >= sizes[:, None]
        assert not bool(dx[past].any())
        nan = dx[:, :V - 1].isnan()
        assert nan[[0, 1, 2, 3, 4, 6, 9]].all(), nan.float().mean(-1)[:10]
        assert not bool(dx[[7, 8]].any())
        if up != math.inf:
            assert not bool(dx[5].any()) and bool(torch.isfinite(dx[10:]).all())
