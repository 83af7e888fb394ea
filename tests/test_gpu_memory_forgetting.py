"""Heads without memory (log_decay -inf): what is not finite ends with its step, in every form of the operator."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a HIP device", allow_module_level=True)

from ilrl_amd import memory as M  # noqa: E402
from test_gpu_memory import Case  # noqa: E402

INF = float("inf")


@pytest.mark.parametrize("bad", [float("nan"), INF, -INF])
@pytest.mark.parametrize("dk,dv", [(32, 32), (3, 9), (128, 70)])
def test_step_without_memory_forgets_a_state_that_is_not_finite(dk, dv, bad):
    c = Case(3, 1, 2, 2, dk, dv, kind="fp32")
    c.log_decay = torch.tensor([-INF, -0.1], device="cuda")
    c.state[1] = bad
    state = c.state.clone()
    out = M.decay_attention_step(c.q[:, 0], c.k[:, 0], c.v[:, 0], c.log_decay, state, scale=c.scale)
    got, last = M.decay_attention(c.q, c.k, c.v, c.log_decay, state=c.state, scale=c.scale)
    for o, s in ((out, state), (got[:, 0], last)):
        assert o[:, 0].isfinite().all() and s[:, 0].isfinite().all()
        assert not o[1, 1].isfinite().any() and not s[1, 1].isfinite().any()
    clean = c.state.clone()
    clean[1] = 0
    want = M.decay_attention_step(c.q[:, 0], c.k[:, 0], c.v[:, 0], c.log_decay, clean, scale=c.scale)
    assert torch.equal(out[:, 0], want[:, 0]) and torch.equal(state[:, 0], clean[:, 0])


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("bad", [float("nan"), INF])
@pytest.mark.parametrize("dk,dv", [(32, 32), (64, 64), (128, 128), (13, 7)])
def test_fragment_without_memory_sees_the_step_itself(dk, dv, bad, kind):
    """Rows of every operand that are not finite, at steps inside a chunk, at its ends and in the next one."""
    b, s, h = 4, 70, 2
    c = Case(b, s, h, h, dk, dv, kind=kind)
    c.log_decay = torch.tensor([-INF, -0.1], device="cuda")
    clean, clean_state = c.check_forward()
    grads = c.check_backward()
    at = [5, 31, 32, 68]
    for lane, t in enumerate(at):
        for x in (c.q, c.k, c.v, c.d_out):
            x[lane, t, :, 1] = bad
    out, state = c.forward()
    dq, dk_, dv_, ds = c.backward()
    assert torch.equal(state[:, 0], clean_state[:, 0]) and torch.equal(ds[:, 0], grads[3][:, 0])
    for lane, t in enumerate(at):
        others = torch.arange(s) != t
        for x, y in zip((out, dq, dk_, dv_), (clean,) + grads[:3]):
            assert torch.equal(x[lane, others, 0], y[lane, others, 0]), (lane, t)
            assert not x[lane, t, 0].isfinite().all()
        # a head that remembers: nothing before the step, everything behind it
        assert out[lane, :t, 1].isfinite().all() and not out[lane, t:, 1].isfinite().all(-1).any()


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_what_is_not_finite_in_the_last_step_reaches_the_state(kind):
    c = Case(2, 40, 2, 2, 32, 32, kind=kind, state=False)
    c.log_decay = torch.tensor([-INF, -0.1], device="cuda")
    c.v[0, 39, :, 1] = INF
    out, state = c.forward()
    assert not state[0, :, 1].isfinite().any() and state[0, :, 2:].isfinite().all() and state[1].isfinite().all()
    assert not out[0, 39, :, 1].isfinite().any() and out[0, :39].isfinite().all()


@pytest.mark.parametrize("order,far,d", [("time", 32768 + 64, 64), ("time", 0, 64), ("lane", 0, 32), ("lane", 0, 33)])
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_heads_that_forget_beside_heads_that_remember(order, far, d, kind):
    """Heads of one lane (one workgroup's, with steps far apart) whose decays mask different steps of a chunk."""
    c = Case(3, 100, 4, 4, d, d, kind=kind, order=order, far=far, resets=0.02)
    c.reset[1] = 0
    c.log_decay = torch.tensor([-INF, -0.1, -8.0, 0.0], device="cuda")   # -8: float32 holds 2^-149, 12 steps of it
    clean, clean_state = c.check_forward()
    grads = c.check_backward()
    for x in (c.q, c.k, c.v, c.d_out):
        x[1, 40, :, 1] = INF
    out, state = c.forward()
    dq, dk_, dv_, ds = c.backward()
    for x, y in zip((out, dq, dk_, dv_, state, ds), (clean,) + grads[:3] + (clean_state, grads[3])):
        assert torch.equal(x[::2], y[::2])   # the other lanes
    for x, y in zip((out, dq, dk_, dv_), (clean,) + grads[:3]):
        others = torch.arange(100) != 40
        assert torch.equal(x[1, others, 0], y[1, others, 0])
        assert torch.equal(x[1, 80:, 2], y[1, 80:, 2]) and torch.equal(x[1, :20, 2], y[1, :20, 2])
        assert not x[1, 40].isfinite().all(-1).any()
    for h in (1, 3):
        assert out[1, :40, h].isfinite().all() and not out[1, 40:, h].isfinite().all(-1).any() and not state[1, h].isfinite().all()
    assert torch.equal(state[1, ::2], clean_state[1, ::2]) and torch.equal(ds[1, ::2], grads[3][1, ::2])
