"""Categorical entries: log-probabilities of given categories, entropy and the most probable alternatives of rows of
logits, and distillation from a teacher's top logits (dmv_cat_* in include/dmv.h).

Rows follow the layout of the samples everywhere else: logits [..., B, D, V] for D categorical entries of a datapoint, the
data X and its mask M [B, D] (1 = observed) without the sample dimensions, the number of categories of each column,
sizes, [D].  An unobserved entry contributes no log-probability (the masked log p(x|z) of vgiwae/shared/iwae.py:9-100);
its entropy and alternatives say what could stand there, and `distill_top_logits` trains it against the alternatives
another model gave:

    teacher = categorical_log_prob(teacher_logits, entropy=True, top=8)
    loss, kl = distill_top_logits(logits, teacher.top_log_prob, teacher.top_index, sizes=sizes, weight=(~M).float())
    log_px = (categorical_log_prob(logits, X, M, sizes=sizes).log_prob).sum(-1)

Both are differentiable with respect to the logits (float32, bfloat16 or float16), in reverse mode and once, run on the
current stream, allocate through torch only and record into HIP graphs.  There is no CPU path."""
import ctypes as C
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _lib as L


class CategoricalLogProb(NamedTuple):
    log_prob: Optional[torch.Tensor]        # [...]       None without X
    entropy: Optional[torch.Tensor]         # [...]       None unless asked for
    top_log_prob: Optional[torch.Tensor]    # [..., top]  None for top = 0
    top_index: Optional[torch.Tensor]       # [..., top]  int64, -1 past the categories of non-zero probability


_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _rows(logits):
    """The logits as rows of one pitch: (tensor, rows, V, pitch).  Copies only what has no such form."""
    V = logits.shape[-1]
    if logits.is_contiguous():
        return logits, logits.numel() // V, V, V
    flat = logits.reshape(-1, V)
    if V > 1 and flat.stride(1) != 1:
        flat = flat.contiguous()
    return flat, flat.shape[0], V, flat.stride(0)


def _per_row(t, lead, dtype, what, device, tail=()):
    """A per-row argument as a contiguous array that repeats over the leading dimensions: (tensor, period)."""
    if t.dtype == dtype and t.device == device and (t.shape[:-1] if tail else t.shape) == lead and t.is_contiguous():
        return t, t.numel() // tail[0] if tail else t.numel()
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, the logits on {device}")
    if t.dtype != dtype:
        t = t.to(dtype)
    shape = tuple(t.shape[:t.dim() - len(tail)])
    if len(shape) > len(lead):
        raise ValueError(f"{what} of shape {tuple(t.shape)} does not fit rows of shape {tuple(lead)}")
    while shape and shape[0] == 1:
        shape = shape[1:]
    if shape != tuple(lead[len(lead) - len(shape):]):
        try:
            t = t.expand(*lead, *tail)
        except RuntimeError:
            raise ValueError(f"{what} of shape {tuple(t.shape)} does not fit rows of shape {tuple(lead)}") from None
        shape = tuple(lead)
    period = 1
    for n in shape:
        period *= n
    return t.contiguous(), period


def _check_logits(logits):
    if not isinstance(logits, torch.Tensor) or logits.dim() < 1:
        raise ValueError("logits: a tensor [..., V]")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits of type {logits.dtype}: float32, bfloat16 or float16")
    if not 1 <= logits.shape[-1] < 2 ** 31:
        raise ValueError(f"logits of {logits.shape[-1]} categories: 1 .. 2^31 - 1")


def _need_gpu(logits):
    if not logits.is_cuda:
        raise RuntimeError(f"the categorical operators have no CPU path: the logits are on {logits.device}")


def _no_tangent(*tensors):
    """Forward-mode gradients are not formed; inside a forward-mode level a tensor that carries one is refused."""
    if forward_ad._current_level < 0:
        return
    for t in tensors:
        if isinstance(t, torch.Tensor) and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("the categorical operators have no forward-mode gradient")


def _integers(t, what):
    if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
        raise TypeError(f"{what} of type {t.dtype}: integers")


def _row_args(logits, X, M, sizes):
    """DmvCatRows without its logits, and the tensors its pointers need alive."""
    lead, dev = logits.shape[:-1], logits.device
    r = L.DmvCatRows()
    r.V, r.dtype = logits.shape[-1], _DTYPES[logits.dtype]
    keep = []
    if X is not None:
        _integers(X, "X")
        X, r.x_period = _per_row(X, lead, torch.int64, "X", dev)
        r.X = X.data_ptr()
        keep.append(X)
    if M is not None:
        if M.dtype.is_floating_point or M.dtype.is_complex:
            raise TypeError(f"M of type {M.dtype}: a mask")
        M, r.m_period = _per_row(M, lead, torch.bool, "M", dev)
        r.M = M.data_ptr()
        keep.append(M)
    if sizes is not None:
        _integers(sizes, "sizes")
        if sizes.dtype != torch.int32:
            sizes = sizes.to(torch.int64).clamp(0, r.V)
        sizes, r.size_period = _per_row(sizes, lead, torch.int32, "sizes", dev)
        r.sizes = sizes.data_ptr()
        keep.append(sizes)
    return r, keep


def _set_logits(r, logits, keep):
    """The logits of a call: its rows in `r`; what they had to be copied to is kept alive with the call's other arrays."""
    flat, r.rows, _, r.ld = _rows(logits)
    r.logits = flat.data_ptr()
    if r.logits != logits.data_ptr():
        keep.append(flat)


def _keep(ctx, logits, r, keep):
    """What a backward pass needs of a call's arguments.  Its arrays are held here, and their versions, because pointers to
    them are: saved tensors may come back from elsewhere, and may not have been made for saving (a teacher's, say)."""
    ctx.kept = r, keep, _versions(keep), logits.stride() if r.logits == logits.data_ptr() else None


def _versions(keep):
    try:
        return [t._version for t in keep]
    except RuntimeError:                    # one made in inference mode, which counts no versions
        return [0 if t.is_inference() else t._version for t in keep]


def _kept(ctx, logits):
    """The call's rows for its backward pass, with the saved logits where they are now; and what has to stay alive."""
    r, keep, versions, strides = ctx.kept
    if _versions(keep) != versions:
        raise RuntimeError("a tensor that the gradient of a categorical operator needs (X, M, sizes, weight or the teacher's) "
                           "was modified in place after the forward call")
    if strides is None or (r.logits == logits.data_ptr() and strides == logits.stride()):
        return r, None
    r, moved = L.DmvCatRows.from_buffer_copy(r), []
    _set_logits(r, logits, moved)
    return r, moved


def _like(logits):
    return torch.empty_like(logits, memory_format=torch.contiguous_format, requires_grad=False)


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def _capture(stream):
    """The graph capture that the current stream is in, 0 outside any."""
    return L.lib().dmv_capture_id(stream) if torch._C._cuda_isCurrentStreamCapturing() else 0


def _on_device(f):
    """Runs f(device, ...) with the tensors' device as the current one: launches go to its current stream."""
    def call(device, *args):
        if device.index == torch._C._cuda_getDevice():
            return f(device, *args)
        with torch.cuda.device(device):
            return f(device, *args)
    return call


class _Once(torch.autograd.Function):
    """A gradient that autograd records (create_graph=True): it may be used, not differentiated."""
    @staticmethod
    def forward(ctx, d, logits):
        return d.view_as(d)

    @staticmethod
    def backward(ctx, g):
        raise RuntimeError("the categorical operators have no second derivative")


@_on_device
def _log_prob(dev, logits, r, keep, want_lp, entropy, top, want_stats):
    lib, lead = L.lib(), logits.shape[:-1]
    _set_logits(r, logits, keep)
    f32 = torch.float32
    lp = torch.empty(lead, dtype=f32, device=dev) if want_lp else None
    ent = torch.empty(lead, dtype=f32, device=dev) if entropy else None
    top_lp = torch.empty((*lead, top), dtype=f32, device=dev) if top else None
    top_idx = torch.empty((*lead, top), dtype=torch.int64, device=dev) if top else None
    n_stats = 4 * r.rows if want_stats else 0
    n_ws = lib.dmv_cat_log_prob_ws_bytes(C.byref(r), top) if r.V > L.CAT_SHORT_ROW else 0
    # the row statistics that the gradient reads, and behind them the workspace
    stats = torch.empty(n_stats + n_ws // 4, dtype=f32, device=dev) if n_stats or n_ws else None
    at = L.addr(stats)
    L.check(lib.dmv_cat_log_prob(C.byref(r), L.addr(lp), L.addr(ent), top, L.addr(top_lp), L.addr(top_idx), at if n_stats else None,
                                 at + 4 * n_stats if n_ws else None, n_ws, _stream(dev)))
    return lp, ent, top_lp, top_idx, stats


@_on_device
def _log_prob_backward(dev, logits, r, stats, g_lp, g_ent, top, top_idx, g_top):
    d = _like(logits)
    L.check(L.lib().dmv_cat_log_prob_backward(C.byref(r), L.addr(stats), L.addr(g_lp), L.addr(g_ent), top, L.addr(top_idx),
                                              L.addr(g_top), L.addr(d), r.V, _stream(dev)))
    return d


class _LogProb(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, r, keep, want_lp, entropy, top):
        lp, ent, top_lp, top_idx, stats = _log_prob(logits.device, logits, r, keep, want_lp, entropy, top, True)
        _keep(ctx, logits, r, keep)
        ctx.top = top
        ctx.save_for_backward(logits, stats, top_idx)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(top_idx)
        return lp, ent, top_lp, top_idx

    @staticmethod
    def backward(ctx, g_lp, g_ent, g_top, _):
        d = None
        if g_lp is not None or g_ent is not None or g_top is not None:
            logits, stats, top_idx = ctx.saved_tensors
            g_lp, g_ent, g_top = (None if g is None else g.contiguous() for g in (g_lp, g_ent, g_top))
            r, moved = _kept(ctx, logits)
            d = _log_prob_backward(logits.device, logits, r, stats, g_lp, g_ent, ctx.top, top_idx, g_top)
            if torch.is_grad_enabled():
                d = _Once.apply(d, logits)
        return d, None, None, None, None, None


def categorical_log_prob(logits, X=None, M=None, *, sizes=None, entropy=False, top=0) -> CategoricalLogProb:
    """log q(X), entropy and the `top` most probable categories of q = softmax(logits), each row in one pass.

    logits [..., V]; X (integers) and M (a mask, 1 = observed) broadcast over the leading dimensions: an unobserved entry
    has log-probability 0 whatever its X holds; sizes (integers): the number of categories of a row, the logits past it
    are not looked at.  top: 0 .. 64; equal logits rank by their index, and places past the categories of non-zero
    probability hold -1 and -inf.  An observed entry whose X is none of its categories is NaN; one that has no category of
    non-zero probability at all is -inf, with entropy 0 and a zero gradient.  Results are float32.  log_prob, entropy and
    top_log_prob are differentiable."""
    _check_logits(logits)
    _no_tangent(logits)
    top = int(top)
    if not 0 <= top <= L.CAT_MAX_TOP:
        raise ValueError(f"top = {top}: 0 .. {L.CAT_MAX_TOP}")
    if X is None and not entropy and not top:
        raise ValueError("nothing asked for: give X, entropy=True or top")
    if X is None and M is not None:
        raise ValueError("M masks the log-probability of X: give X")
    r, keep = _row_args(logits, X, M, sizes)
    _need_gpu(logits)
    if logits.requires_grad and torch.is_grad_enabled():
        return CategoricalLogProb(*_LogProb.apply(logits, r, keep, X is not None, bool(entropy), top))
    return CategoricalLogProb(*_log_prob(logits.device, logits, r, keep, X is not None, bool(entropy), top, False)[:4])


@_on_device
def _distill(dev, logits, r, t, keep, training):
    lib = L.lib()
    _set_logits(r, logits, keep)
    per_row = torch.empty(logits.shape[:-1], dtype=torch.float32, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    d = _like(logits) if training else None
    n_stats = 4 * r.rows if training and r.V > L.CAT_SHORT_ROW else 0
    n_ws = lib.dmv_cat_distill_ws_bytes(C.byref(r), t.k)
    stats = torch.empty(n_stats + n_ws // 4, dtype=torch.float32, device=dev) if n_stats or n_ws else None      # as in _log_prob
    at, stream = L.addr(stats), _stream(dev)
    L.check(lib.dmv_cat_distill(C.byref(r), C.byref(t), per_row.data_ptr(), loss.data_ptr(), at if n_stats else None, L.addr(d), r.V,
                                at + 4 * n_stats if n_ws else None, n_ws, stream))
    return loss, per_row, stats, (d, _capture(stream)) if training else None


@_on_device
def _distill_backward(dev, logits, r, t, g, stats, formed):
    # the forward pass has written the gradient for g = 1 (a loss that is not scaled further): any other g forms it again
    # from the logits, on the device; a second backward pass has a gradient of its own, and so has one that is recorded
    # without its forward pass, which may be replayed more often
    stream = _stream(dev)
    unless_one = formed is not None and formed[1] == _capture(stream)
    d = formed[0] if unless_one else _like(logits)
    L.check(L.lib().dmv_cat_distill_backward(C.byref(r), C.byref(t), L.addr(g), unless_one, L.addr(stats), L.addr(d), r.V, stream))
    return d


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, r, t, keep):
        loss, per_row, stats, ctx.formed = _distill(logits.device, logits, r, t, keep, True)
        _keep(ctx, logits, r, keep)
        ctx.t = t
        ctx.save_for_backward(logits, stats)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(per_row)
        return loss, per_row

    @staticmethod
    def backward(ctx, g, _):
        if g is None:
            return None, None, None, None
        logits, stats = ctx.saved_tensors
        r, moved = _kept(ctx, logits)
        formed, ctx.formed = ctx.formed, None
        d = _distill_backward(logits.device, logits, r, ctx.t, g, stats, formed)
        return _Once.apply(d, logits) if torch.is_grad_enabled() else d, None, None, None


def distill_top_logits(logits, top_logits, top_index, *, sizes=None, weight=None, temperature=1.0):
    """Distillation from a teacher that gives its k (1 .. 256) largest logits, or log-probabilities, and their categories:

        KL_row = sum_j p_j (log p_j - log q_{i_j}),   p = softmax(top_logits / T),   q = softmax(logits / T)

    Returns (loss, per_row): loss = sum over rows of weight * KL_row (a tensor or a number, 1 unless given; 1 / rows for a mean,
    T^2 for the customary scale, 0 for the rows to leave out: those are not read), differentiable with respect to the
    logits, and KL_row itself, float32, without gradient.  The gradient is formed in the pass that forms the loss; an
    upstream gradient other than 1 costs a second pass.

    top_logits (float32, bfloat16 or float16) and top_index [..., k], weight and sizes broadcast over the leading
    dimensions of logits [..., V].  Entries with a negative index or a logit of -inf are empty (what categorical_log_prob
    leaves past a row's categories); a category given twice counts twice."""
    _check_logits(logits)
    temperature = float(temperature)
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"temperature = {temperature}: 1e-30 .. 1e30")
    if top_logits.shape != top_index.shape or top_logits.dim() < 1:
        raise ValueError(f"top_logits {tuple(top_logits.shape)} and top_index {tuple(top_index.shape)}: one shape [..., k]")
    if top_logits.dtype not in _DTYPES:
        raise TypeError(f"top_logits of type {top_logits.dtype}: float32, bfloat16 or float16")
    _integers(top_index, "top_index")
    if isinstance(weight, (int, float)):
        weight = torch.full((), float(weight), device=logits.device)
    if torch.is_grad_enabled() and (top_logits.requires_grad or (weight is not None and weight.requires_grad)):
        raise ValueError("the teacher's logits and the weights have no gradient: detach them")
    _no_tangent(logits, top_logits, weight)
    k = top_logits.shape[-1]
    if not 1 <= k <= L.CAT_MAX_TEACHER:
        raise ValueError(f"{k} entries per row: 1 .. {L.CAT_MAX_TEACHER}")
    r, keep = _row_args(logits, None, None, sizes)
    lead, dev = logits.shape[:-1], logits.device
    t = L.DmvCatTeacher()
    top_logits, t.period = _per_row(top_logits, lead, top_logits.dtype, "top_logits", dev, (k,))
    top_index, _ = _per_row(top_index, lead, torch.int64, "top_index", dev, (k,))
    t.logits, t.index, t.k, t.dtype, t.temperature = top_logits.data_ptr(), top_index.data_ptr(), k, _DTYPES[top_logits.dtype], temperature
    keep += [top_logits, top_index]
    if weight is not None:
        weight, t.w_period = _per_row(weight, lead, torch.float32, "weight", dev)
        t.weight = weight.data_ptr()
        keep.append(weight)
    _need_gpu(logits)
    if logits.requires_grad and torch.is_grad_enabled():
        return _Distill.apply(logits, r, t, keep)
    return _distill(logits.device, logits, r, t, keep, False)[:2]
