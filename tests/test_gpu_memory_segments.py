"""Walks cut into segments (a first pass over the segments without outputs, a scan, a second pass) at the types, widths,
alignments and orders that short walks are tested at, against the float64 restatement under the same bounds."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a HIP device", allow_module_level=True)

import ctypes  # noqa: E402

from ilrl_amd import _native as N  # noqa: E402
from ilrl_amd import memory as M  # noqa: E402
from test_gpu_memory import Case, TYPES  # noqa: E402


def cut(c, backward):
    """The walk is cut: it needs scratch beyond what shared heads' partial gradients take."""
    b, s, h, dk = c.q.shape
    g, dv = c.k.shape[2], c.v.shape[3]
    e, need = M._e(), ctypes.c_uint64(0)
    a = M._attn(e, c.q, c.k, c.v, c.log_decay, c.state, None, c.reset, c.lengths, c.scale, (b, s, h, g, dk, dv))
    N.check(e.workspace(a, backward, ctypes.byref(need)), "hum_decay_attn_workspace")
    partial = 4 * b * s * h * (dk + dv) + 16 if backward and h != g else 0
    return need.value > partial


def check(c):
    assert cut(c, 0) and cut(c, 1)
    c.check_forward()
    c.check_backward()


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("order", ["lane", "time"])
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("h,g,dk,dv", [(2, 1, 40, 72), (2, 2, 117, 22), (2, 1, 5, 128), (4, 2, 32, 32), (2, 2, 64, 64), (1, 1, 128, 128),
                                       (2, 2, 24, 120), (3, 1, 3, 6)])
def test_cut_walks(h, g, dk, dv, odd, order, kind):
    s = 431
    check(Case(3, s, h, g, dk, dv, kind=kind, order=order, resets=0.006, lengths=[s, 0, s // 2 + 7], odd=odd, seed=3))


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("s,dk,dv", [(907, 117, 22), (900, 40, 72), (640, 64, 64)])
def test_longer_cut_walks(s, dk, dv, kind):
    check(Case(2, s, 2, 1, dk, dv, kind=kind, order="time", resets=0.003, lengths=[s, s - 65], seed=4))


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("d", [64, 13])
def test_cut_walks_of_steps_far_apart(d, kind):
    """Rows of a wide time-major batch, and more than 32 MB from a step to the next."""
    check(Case(2, 400, 4, 4, d, d, kind=kind, order="time", resets=0.01, far=32768 + 64))
    check(Case(1, 400, 1, 1, d, d, kind=kind, order="time", resets=0.01, far=(2 ** 25 + 64) // TYPES[kind].itemsize))


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("dk,dv,odd", [(32, 32, False), (40, 72, True)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_non_finite_rows_and_the_reset_behind_them_in_other_segments(dk, dv, odd, bad, kind):
    """An episode diverges in one segment and ends some segments later: what comes before it and the next episode are as
    without it, in both directions; a lane whose first state is not finite starts afresh."""
    s, at, start = 500, 70, 330
    c = Case(3, s, 2, 2, dk, dv, kind=kind, lengths=[s, s, 450], odd=odd)
    c.reset = torch.zeros(3, s, dtype=torch.uint8, device="cuda")
    c.reset[:2, start] = 1
    assert cut(c, 0) and cut(c, 1)
    clean, clean_state = c.check_forward()
    grads = c.check_backward()
    for x in (c.q, c.k, c.v, c.d_out):
        x[0, at] = bad
        x[2, 450:] = bad
    c.state[1] = bad
    out, state = c.forward()
    dq, dk_, dv_, ds = c.backward()
    for lane in range(3):
        assert torch.equal(state[lane], clean_state[lane])
    assert torch.equal(out[0, :at], clean[0, :at]) and torch.equal(out[0, start:], clean[0, start:])
    assert not out[0, at:start].isfinite().any() and not out[1, :start].isfinite().any()
    assert torch.equal(out[1, start:], clean[1, start:]) and torch.equal(out[2], clean[2])
    assert torch.equal(dq[0, :at], grads[0][0, :at]) and torch.equal(dq[0, start:], grads[0][0, start:])
    for x, y in ((dk_, grads[1]), (dv_, grads[2])):   # backwards: the steps from the bad one to the episode's first see it
        assert torch.equal(x[0, at + 1:], y[0, at + 1:]) and not x[0, :at + 1].isfinite().any()
        assert torch.equal(x[1], y[1]) and torch.equal(x[2], y[2])
    assert torch.equal(dq[1, start:], grads[0][1, start:]) and torch.equal(dq[2], grads[0][2])
    assert not ds[0].isfinite().any() and torch.equal(ds[1:], grads[3][1:])
    assert (out[2, 450:] == 0).all() and (dq[2, 450:] == 0).all()


def test_cut_walks_in_place():
    """The state after the walk over the one before it, also where segments are scanned in between."""
    c = Case(2, 600, 2, 1, 40, 72, kind="bf16", resets=0.004)
    out, state = c.check_forward()
    e = M._e()
    b, s, h, dk = c.q.shape
    here, into = c.state.clone(), torch.empty_like(out)
    a = M._attn(e, c.q, c.k, c.v, c.log_decay, here, here, c.reset, c.lengths, c.scale, (b, s, h, 1, dk, 72))
    ws = M._scratch(e, a, 0, c.q.device)
    N.check(e.attn(a, M._rows(into), ws.data_ptr(), ws.numel(), e.stream(0)), "hum_decay_attn")
    assert torch.equal(into, out) and torch.equal(here, state)
