"""What a policy memory's tensors mean to the calls around them: states that move between a forward pass and its gradient."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a HIP device", allow_module_level=True)

from ilrl_amd import memory as M  # noqa: E402
from ilrl_amd.policy import DevicePolicy  # noqa: E402
from ilrl_amd.vec_env import HumanoidVecEnv  # noqa: E402


def rows(*shape, seed=0, **kw):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).cuda().requires_grad_(kw.get("grad", False))


@pytest.mark.parametrize("how", ["state", "state_out", "out", "rollout"])
def test_gradient_notices_that_a_saved_tensor_was_overwritten(how):
    """A step writes into a tensor that a fragment's pass has saved: backward() raises, as it does behind torch's own
    in-place operators."""
    n, h, d = 8, 2, 16
    ld = M.decay_schedule(h)
    q, k, v = (rows(n, 5, h, d, seed=i, grad=True) for i in range(3))
    state = rows(n, h, d, d, seed=4)
    one = [rows(n, h, d, seed=5 + i) for i in range(3)]
    if how == "out":
        held = rows(n, 1, h, d, seed=9)   # the values of the fragment
        out, _ = M.decay_attention(q[:, :1], k[:, :1], held, ld, state=state)
        M.decay_attention_step(*one, ld, state.clone(), out=held[:, 0])
    elif how == "rollout":
        pol, mem, env = DevicePolicy.random_init(seed=1), M.PolicyMemory(heads=h, channels=d), HumanoidVecEnv(n, seed=2)
        env.reset()
        with torch.no_grad():
            mem.w_out += 0.1
        state = mem.begin(n)
        out, _ = mem.forward(rows(3, n, 70), state=state)
        pol.rollout(env, 1, memory=mem, state=state)
        env.close()
        pol.close()
    else:
        out, _ = M.decay_attention(q, k, v, ld, state=state)
        if how == "state":
            M.decay_attention_step(*one, ld, state)
        else:
            M.decay_attention_step(*one, ld, state.clone(), state_out=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_gradient_notices_that_a_norms_input_was_overwritten():
    x, w = rows(6, 40), rows(40, grad=True)
    y = M.layer_norm(x, w)
    M.layer_norm_forward(rows(6, 40, seed=1), out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_step_elsewhere_leaves_the_gradient():
    """A step of a copy, and one into other tensors, raise nothing; tensors made under inference_mode can be stepped."""
    n, h, d = 4, 2, 16
    ld = M.decay_schedule(h)
    q, k, v = (rows(n, 5, h, d, seed=i, grad=True) for i in range(3))
    state = rows(n, h, d, d, seed=4)
    one = [rows(n, h, d, seed=5 + i) for i in range(3)]
    out, _ = M.decay_attention(q, k, v, ld, state=state)
    M.decay_attention_step(*one, ld, state.clone())
    M.decay_attention_step(*one, ld, state, state_out=torch.empty_like(state))
    out.sum().backward()
    assert q.grad.isfinite().all()
    with torch.inference_mode():
        s = torch.zeros(n, h, d, d, device="cuda")
        M.decay_attention_step(*one, ld, s)
        assert s.any()
        y = torch.zeros(3, 8, device="cuda")
        M.layer_norm_forward(y, out=y)
