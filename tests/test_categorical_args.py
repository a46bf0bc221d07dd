"""What the categorical operators refuse, on the CPU: the Python entry points' checks of their arguments, and the C entry
points' error codes (argument checks come before any launch, so none of these calls reaches a GPU)."""
import ctypes as C

import pytest
import torch

import demiss_vae_amd as dmv
from demiss_vae_amd import _lib as L


def _logits(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("kw, error, what", [
    (dict(), ValueError, "nothing asked"),
    (dict(M=torch.ones(4, dtype=torch.bool), entropy=True), ValueError, "give X"),
    (dict(top=-1), ValueError, "top"),
    (dict(top=65), ValueError, "top"),
    (dict(X=torch.zeros(4)), TypeError, "X of type"),
    (dict(X=torch.zeros(4, dtype=torch.bool)), TypeError, "X of type"),
    (dict(X=torch.zeros(3, dtype=torch.long)), ValueError, "does not fit"),
    (dict(X=torch.zeros(2, 4, dtype=torch.long)), ValueError, "does not fit"),
    (dict(X=torch.zeros(4, dtype=torch.long), M=torch.ones(4)), TypeError, "a mask"),
    (dict(X=torch.zeros(4, dtype=torch.long), M=torch.ones(5, dtype=torch.bool)), ValueError, "does not fit"),
    (dict(entropy=True, sizes=torch.ones(4)), TypeError, "sizes"),
    (dict(entropy=True, sizes=torch.ones(2, dtype=torch.int32)), ValueError, "does not fit"),
    (dict(entropy=True), RuntimeError, "no CPU path"),
])
def test_log_prob_refuses(kw, error, what):
    with pytest.raises(error, match=what):
        dmv.categorical_log_prob(_logits(4, 7), **kw)


@pytest.mark.parametrize("logits, error", [
    (_logits(4, 0), ValueError), (torch.zeros(4, 3, dtype=torch.int32), TypeError), (_logits(4, 3, dtype=torch.float64), TypeError),
    (torch.tensor(1.0), ValueError), ([1.0, 2.0], ValueError)])
def test_both_refuse_logits(logits, error):
    with pytest.raises(error):
        dmv.categorical_log_prob(logits, entropy=True)
    with pytest.raises(error):
        dmv.distill_top_logits(logits, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.long))


@pytest.mark.parametrize("top, index, kw, error, what", [
    (torch.zeros(4, 2), torch.zeros(4, 3, dtype=torch.long), {}, ValueError, "one shape"),
    (torch.zeros(4, 2), torch.zeros(4, 2), {}, TypeError, "top_index"),
    (torch.zeros(4, 2, dtype=torch.float64), torch.zeros(4, 2, dtype=torch.long), {}, TypeError, "top_logits"),
    (torch.zeros(4, 0), torch.zeros(4, 0, dtype=torch.long), {}, ValueError, "entries per row"),
    (torch.zeros(4, 257), torch.zeros(4, 257, dtype=torch.long), {}, ValueError, "entries per row"),
    (torch.zeros(5, 2), torch.zeros(5, 2, dtype=torch.long), {}, ValueError, "does not fit"),
    (torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.long), dict(temperature=0.0), ValueError, "temperature"),
    (torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.long), dict(temperature=float("nan")), ValueError, "temperature"),
    (torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.long), dict(temperature=float("inf")), ValueError, "temperature"),
    (torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.long), dict(weight=torch.ones(3)), ValueError, "does not fit"),
    (torch.zeros(4, 2, requires_grad=True), torch.zeros(4, 2, dtype=torch.long), {}, ValueError, "detach"),
    (torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.long), dict(weight=torch.ones(4, requires_grad=True)), ValueError, "detach"),
    (torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.long), {}, RuntimeError, "no CPU path"),
])
def test_distill_refuses(top, index, kw, error, what):
    with pytest.raises(error, match=what):
        dmv.distill_top_logits(_logits(4, 7), top, index, **kw)


# ------------------------------------------------------------------------------------------ the C entry points
FAKE = 4096          # an address that is only looked at: every call below is refused before it would be read


def _rows(**kw):
    r = L.DmvCatRows(logits=FAKE, ld=8, rows=4, V=8, dtype=0, X=FAKE, x_period=4)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def _teacher(**kw):
    t = L.DmvCatTeacher(logits=FAKE, index=FAKE, period=4, k=2, dtype=0, temperature=1.0)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


BAD, UNSUPPORTED, WORKSPACE = L.E_BADARG, L.E_UNSUPPORTED, L.E_WORKSPACE
ROWS_REFUSED = [(dict(rows=-1), BAD), (dict(V=0), BAD), (dict(ld=-1), BAD), (dict(logits=None), BAD), (dict(logits=FAKE + 2), BAD),
                (dict(dtype=1, logits=FAKE + 1), BAD), (dict(x_period=0), BAD), (dict(M=FAKE, m_period=0), BAD),
                (dict(sizes=FAKE, size_period=0), BAD), (dict(dtype=3), UNSUPPORTED), (dict(dtype=-1), UNSUPPORTED),
                (dict(rows=1 << 26), UNSUPPORTED), (dict(V=0x7fffffff), UNSUPPORTED)]


@pytest.mark.parametrize("kw, code", ROWS_REFUSED)
def test_entry_points_refuse_rows(kw, code):
    lib = L.lib()
    r, t = C.byref(_rows(**kw)), C.byref(_teacher())
    assert lib.dmv_cat_log_prob(r, FAKE, None, 0, None, None, None, None, 0, None) == code
    assert lib.dmv_cat_log_prob_backward(r, FAKE, FAKE, None, 0, None, None, FAKE, 1 << 40, None) == code
    assert lib.dmv_cat_distill(r, t, FAKE, FAKE, None, None, 0, FAKE, 1 << 40, None) == code
    assert lib.dmv_cat_distill_backward(r, t, FAKE, 0, FAKE, FAKE, 1 << 40, None) == code
    assert lib.dmv_cat_log_prob_ws_bytes(r, 1) == 0 and lib.dmv_cat_distill_ws_bytes(r, 2) == 0


@pytest.mark.parametrize("args, code", [
    ((None, None, 0, None, None, None, None, 0), BAD),                   # nothing asked for
    ((FAKE, None, -1, None, None, None, None, 0), BAD),
    ((FAKE, None, 65, FAKE, FAKE, None, None, 0), UNSUPPORTED),
    ((FAKE, None, 2, None, FAKE, None, None, 0), BAD),
    ((FAKE, None, 2, FAKE, None, None, None, 0), BAD),
    ((FAKE, None, 0, None, None, FAKE + 4, None, 0), BAD),               # misaligned stats
    ((FAKE, None, 0, None, None, None, FAKE + 8, 0), BAD)])              # misaligned workspace
def test_log_prob_entry_refuses(args, code):
    assert L.lib().dmv_cat_log_prob(C.byref(_rows()), *args, None) == code


def test_log_prob_entry_needs_x_and_workspace():
    lib = L.lib()
    assert lib.dmv_cat_log_prob(C.byref(_rows(X=None)), FAKE, None, 0, None, None, None, None, 0, None) == BAD
    r = _rows(V=1 << 20, ld=1 << 20)
    need = lib.dmv_cat_log_prob_ws_bytes(C.byref(r), 5)
    assert need > 0 and need % 8 == 0
    for ws, n in ((None, 0), (FAKE, need - 1)):
        assert lib.dmv_cat_log_prob(C.byref(r), FAKE, None, 5, FAKE, FAKE, None, ws, n, None) == WORKSPACE


@pytest.mark.parametrize("args, code", [
    ((FAKE, FAKE, None, 0, None, None, FAKE, 7), BAD),                   # pitch below V
    ((FAKE, FAKE, None, 0, None, FAKE, FAKE, 8), BAD),                   # gradient of alternatives that were not asked for
    ((FAKE, FAKE, None, 65, FAKE, FAKE, FAKE, 8), UNSUPPORTED),
    ((None, FAKE, None, 0, None, None, FAKE, 8), BAD),
    ((FAKE, FAKE, None, 0, None, None, None, 8), BAD),
    ((FAKE, FAKE, None, 0, None, None, FAKE + 1, 8), BAD)])
def test_backward_entry_refuses(args, code):
    assert L.lib().dmv_cat_log_prob_backward(C.byref(_rows()), *args, None) == code


@pytest.mark.parametrize("kw, code", [
    (dict(logits=None), BAD), (dict(index=None), BAD), (dict(period=0), BAD), (dict(k=0), BAD), (dict(k=257), UNSUPPORTED),
    (dict(dtype=5), UNSUPPORTED), (dict(temperature=0.0), BAD), (dict(temperature=-1.0), BAD), (dict(temperature=1e-40), BAD), (dict(temperature=1e38), BAD), (dict(temperature=float("nan")), BAD),
    (dict(weight=FAKE, w_period=0), BAD), (dict(logits=FAKE + 1), BAD)])
def test_distill_entry_refuses_teacher(kw, code):
    lib = L.lib()
    t = C.byref(_teacher(**kw))
    assert lib.dmv_cat_distill(C.byref(_rows()), t, FAKE, FAKE, None, None, 0, FAKE, 1 << 30, None) == code
    assert lib.dmv_cat_distill_backward(C.byref(_rows()), t, FAKE, 0, FAKE, FAKE, 8, None) == code


def test_entries_refuse_launches_beyond_the_grid():
    """2^32 threads and more in one launch"""
    lib = L.lib()
    r = C.byref(_rows(rows=(1 << 24) + 5, V=70000, ld=70000))
    assert lib.dmv_cat_log_prob(r, FAKE, None, 0, None, None, None, None, 0, None) == UNSUPPORTED
    assert lib.dmv_cat_log_prob_backward(r, FAKE, FAKE, None, 0, None, None, FAKE, 70000, None) == UNSUPPORTED
    need = lib.dmv_cat_distill_ws_bytes(r, 2)
    assert lib.dmv_cat_distill(r, C.byref(_teacher()), None, FAKE, None, None, 0, FAKE, need, None) == UNSUPPORTED


def test_distill_entry_refuses_outputs_and_workspace():
    lib = L.lib()
    r, t = C.byref(_rows(rows=100000)), C.byref(_teacher())
    need = lib.dmv_cat_distill_ws_bytes(r, 2)
    assert need >= 8 and need % 16 == 0
    assert lib.dmv_cat_distill_ws_bytes(C.byref(_rows()), 2) == 0           # a small launch forms the loss itself
    call = lambda loss=FAKE, stats=None, d=None, ld=8, ws=FAKE, n=need: lib.dmv_cat_distill(r, t, None, loss, stats, d, ld, ws, n, None)  # noqa: E731
    assert call(loss=None) == BAD and call(d=FAKE, ld=7) == BAD and call(d=FAKE + 1) == BAD and call(stats=FAKE + 4) == BAD
    assert call(ws=None) == WORKSPACE and call(n=need - 1) == WORKSPACE and call(ws=FAKE + 8) == WORKSPACE
    big = C.byref(_rows(V=5000, ld=5000))
    assert lib.dmv_cat_distill_backward(big, t, FAKE, 0, None, FAKE, 5000, None) == BAD      # long rows need their statistics
    assert lib.dmv_cat_distill_backward(r, t, None, 0, FAKE, FAKE, 8, None) == BAD


def test_more_categories_than_an_index_holds():
    x = torch.empty(1, 2 ** 31, dtype=torch.float16, device="meta")
    with pytest.raises(ValueError, match="categories"):
        dmv.categorical_log_prob(x, entropy=True)
    with pytest.raises(ValueError, match="categories"):
        dmv.distill_top_logits(x, torch.zeros(1, 2), torch.zeros(1, 2, dtype=torch.long))


def test_entries_refuse_rows_beyond_the_grid_of_the_widest_tile():
    """64 lanes a row: 2^26 - 4 rows would take 2^32 threads"""
    r = C.byref(_rows(rows=(1 << 26) - 4, V=2048, ld=2048))
    assert L.lib().dmv_cat_log_prob(r, FAKE, None, 0, None, None, None, None, 0, None) == UNSUPPORTED
    assert L.lib().dmv_cat_distill(r, C.byref(_teacher()), None, FAKE, None, None, 0, FAKE, 1 << 40, None) == UNSUPPORTED


def test_a_number_as_weight_is_an_argument():
    with pytest.raises(RuntimeError, match="no CPU path"):
        dmv.distill_top_logits(_logits(4, 7), torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.long), weight=0.25)


def test_a_view_of_the_logits_is_not_held():
    """Rows with a pitch are read where they are.  What autograd saves of them is autograd's: they may be written over
    where its hooks have put them elsewhere, and are not kept alive; a copy that a call has made is."""
    from types import SimpleNamespace
    from demiss_vae_amd import categorical as cat
    memory = torch.arange(48.0).view(4, 12)
    for logits, copies in ((memory[:, :7], 0), (memory[:, :, None].transpose(1, 2)[:, :, 2:9], 0), (memory, 0), (memory.t(), 1),
                           (memory.view(2, 2, 12).transpose(0, 1), 1)):
        r, keep = cat._row_args(logits, None, None, None)
        cat._set_logits(r, logits, keep)
        assert len(keep) == copies
        ctx = SimpleNamespace()
        cat._keep(ctx, logits, r, keep)
        saved = logits.clone()
        memory.add_(1.0)
        assert cat._kept(ctx, saved)[0].V == logits.shape[-1]


# ------------------------------------------------------------------------------------------ what a backward pass holds
def _held(logits):
    from types import SimpleNamespace
    from demiss_vae_amd import categorical as cat
    r, keep = cat._row_args(logits, None, None, None)
    cat._set_logits(r, logits, keep)
    ctx = SimpleNamespace()
    cat._keep(ctx, logits, r, keep)
    return lambda saved: cat._kept(ctx, saved)[0]


@pytest.mark.parametrize("ours, back", [((12, 1), (7, 1)), ((7, 1), (12, 1)), ((12, 1), (1, 4)), ((0, 1), (7, 1))])
def test_saved_logits_of_another_pitch_at_the_same_address(ours, back):
    """Logits that autograd's hooks hand back may lie where the first ones lay (that memory is free again) in rows of
    another pitch."""
    memory = torch.arange(48.0)
    first, again = memory.as_strided((4, 7), ours), memory.as_strided((4, 7), back)
    kept = _held(first)
    same = kept(first)
    assert (same.logits, same.ld, same.rows, same.V) == (first.data_ptr(), ours[0], 4, 7)
    r = kept(again)
    assert (r.rows, r.V) == (4, 7)
    if back[1] == 1:
        assert (r.logits, r.ld) == (again.data_ptr(), back[0])
    else:
        assert r.logits != again.data_ptr() and r.ld == 7       # copied to rows


# ------------------------------------------------------------------------------------------ forward-mode gradients
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_gradients_are_refused(grad):
    """A tangent of the logits, of the teacher's or of the weights would be dropped."""
    import torch.autograd.forward_ad as fw
    idx = torch.zeros(4, 2, dtype=torch.long)
    with fw.dual_level():
        x = fw.make_dual(_logits(4, 7).requires_grad_(grad), torch.ones(4, 7))
        t, w = fw.make_dual(torch.zeros(4, 2), torch.ones(4, 2)), fw.make_dual(torch.ones(4), torch.ones(4))
        for no_grad in (False, True):
            with torch.set_grad_enabled(not no_grad):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    dmv.categorical_log_prob(x, entropy=True)
                with pytest.raises(RuntimeError, match="forward-mode"):
                    dmv.distill_top_logits(x, torch.zeros(4, 2), idx)
                with pytest.raises(RuntimeError, match="forward-mode"):
                    dmv.distill_top_logits(_logits(4, 7), t, idx)
                with pytest.raises(RuntimeError, match="forward-mode"):
                    dmv.distill_top_logits(_logits(4, 7), torch.zeros(4, 2), idx, weight=w)
        # without a tangent they are ordinary arguments
        with pytest.raises(RuntimeError, match="no CPU path"):
            dmv.categorical_log_prob(_logits(4, 7), entropy=True)
        with pytest.raises(RuntimeError, match="no CPU path"):
            dmv.distill_top_logits(_logits(4, 7), torch.zeros(4, 2), idx, weight=0.5)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda z: dmv.categorical_log_prob(z, entropy=True).entropy, (_logits(4, 7),), (torch.ones(4, 7),))
