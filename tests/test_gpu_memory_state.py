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


@pytest.mark.parametrize("between", ["masked", "all", "masked, stepped", "twice"])
def test_reset_between_rollouts_starts_an_episode(between):
    """Lanes that venv.reset() takes to a new episode forget the old one, and the trajectory says so to the learner."""
    n = 12
    pol, mem, env = DevicePolicy.random_init(seed=1), M.PolicyMemory(heads=2, channels=16, seed=3), HumanoidVecEnv(n, seed=2)
    with torch.no_grad():
        mem.w_out += 0.1 * rows(32, 70, seed=8)
    mask = torch.arange(n).remainder(3).eq(0).to(torch.uint8).cuda()
    env.reset()
    assert not env.episode_start().any()   # no episode came before
    state = mem.begin(n)
    first = pol.rollout(env, 3, memory=mem, state=state)
    assert not first["resets"][0].any() and state.flatten(1).any(1).all()
    starts = env.done.bool()
    env.reset(None if between == "all" else mask)
    starts = torch.ones_like(starts) if between == "all" else starts | mask.bool()
    if between == "twice":
        env.reset(1 - mask)
        starts.fill_(True)
    assert torch.equal(env.episode_start().bool(), starts)
    if between == "masked, stepped":   # the marked step is not the rollout's
        env.step(torch.zeros(n, 17), autoreset=True)
        starts = env.done.bool()
    before, want = state.clone(), state.clone()
    obs = torch.where(env.done.bool()[:, None], env.obs_reset, env.obs)
    tr = pol.rollout(env, 2, memory=mem, state=state)
    assert torch.equal(tr["resets"][0].bool(), starts) and torch.equal(tr["resets"][1], tr["dones"][0])
    assert torch.equal(tr["obs"][0], obs)
    mem.step(obs, want, reset=starts)
    mem.step(tr["obs"][1], want, reset=tr["resets"][1])
    assert torch.equal(state, want)
    if starts.any():
        blank = mem.begin(n)
        mem.step(obs, blank)
        mem.step(tr["obs"][1], blank, reset=tr["resets"][1])
        assert torch.equal(state[starts], blank[starts])   # nothing of the old episode is left
    # the learner's pass over the fragment does not see it either
    _, last = mem.forward(tr["obs"], state=before, reset=tr["resets"])
    torch.testing.assert_close(last.detach(), state, rtol=1e-4, atol=1e-5)
    assert not (env.episode_start().bool() & ~env.done.bool()).any()
    env.close()
    pol.close()


def test_other_rollouts_end_the_start_of_an_episode():
    """Every call that steps the lanes ends what reset() marked."""
    n, pol, env = 8, DevicePolicy.random_init(seed=1), HumanoidVecEnv(8, seed=2)
    env.reset()
    env.step(torch.zeros(n, 17))
    for advance in (lambda: pol.rollout(env, 1), lambda: env.step_k(torch.zeros(2, n, 17), autoreset=True),
                    lambda: env.step(torch.zeros(n, 17))):
        env.reset()
        assert env.episode_start().all()
        advance()
        assert not env.begun.any()
    env.close()
    pol.close()


def test_a_replayed_step_ends_the_start_of_an_episode():
    """A step captured into a graph clears the marks on every replay, also of resets that came after the capture."""
    n, env = 8, HumanoidVecEnv(8, seed=2)
    act = torch.zeros(n, 17, device="cuda")
    env.reset()
    env.step(act)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        env.step(act, autoreset=True)
    for _ in range(3):
        env.reset()
        assert env.episode_start().all()
        graph.replay()
        torch.cuda.synchronize()
        assert not env.begun.any()
    env.close()


@pytest.mark.parametrize("how", ["plain", "memory", "fused"])
@pytest.mark.parametrize("field", ["obs", "actions"])
def test_gradient_notices_that_a_trajectory_was_recorded_over(how, field):
    """rollout(out=) writes into the trajectory a learner's pass has saved: backward() raises."""
    n = 256
    pol, mem, env = DevicePolicy.random_init(seed=1), M.PolicyMemory(heads=2, channels=16), HumanoidVecEnv(n, seed=2)
    env.reset()
    kw = dict(memory=mem, state=mem.begin(n)) if how == "memory" else dict(fused=how == "fused")
    tr = pol.rollout(env, 2, **kw)
    w = torch.ones(tr[field].shape[-1], device="cuda", requires_grad=True)
    loss = (M.layer_norm(tr[field], w) if field == "obs" else tr[field] * w).sum()
    pol.rollout(env, 2, out=tr, **kw)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    env.close()
    pol.close()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_padding_that_is_not_finite_stays_out_of_the_gradients(bad):
    """Observations behind a lane's length are whatever the batch holds there: the held steps' features and every parameter's
    gradient are what they are with zeros in their place."""
    k, n = 40, 6
    mem = M.PolicyMemory(heads=2, channels=16, seed=3)
    with torch.no_grad():
        mem.w_out += 0.1 * rows(32, 70, seed=8)
    obs, weight = rows(k, n, 70), rows(k, n, 70, seed=1)
    lengths = torch.tensor([40, 0, 1, 33, 17, 39], dtype=torch.int32, device="cuda")
    held = (torch.arange(k, device="cuda")[:, None] < lengths)[..., None]
    runs = []
    for pad in (0.0, bad):
        x = torch.where(held, obs, torch.full_like(obs, pad)).requires_grad_(True)
        f, state = mem.forward(x, state=rows(n, 2, 16, 16, seed=2), lengths=lengths)
        loss = torch.where(held, f * weight, torch.zeros_like(f)).sum() + state.sum()
        runs.append((torch.where(held, f, torch.zeros_like(f)), state) + torch.autograd.grad(loss, mem.parameters() + [x]))
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    assert all(g.isfinite().all() for g in runs[1])


def test_lengths_of_the_core_are_checked():
    mem, obs = M.PolicyMemory(heads=2, channels=16), rows(4, 3, 70)
    ok = torch.tensor([4, 2, 0], dtype=torch.int32, device="cuda")
    assert mem.forward(obs, lengths=ok)[0].shape == (4, 3, 70)
    for bad in (ok.long(), ok[:2], ok.cpu(), ok[:, None]):
        with pytest.raises(ValueError, match="lengths"):
            mem.forward(obs, lengths=bad)
