"""The policy memory as it is used: DevicePolicy.rollout(memory=) acts through PolicyMemory.step, the learner's columns and
gradients come from PolicyMemory.forward over the recorded fragment."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a HIP device", allow_module_level=True)

import memory_reference as R  # noqa: E402
from ilrl_amd import memory as M  # noqa: E402
from ilrl_amd.policy import DevicePolicy  # noqa: E402
from ilrl_amd.vec_env import HumanoidVecEnv  # noqa: E402

U = 2.0 ** -24


def trained(seed=0, **kw):
    """A memory that does something: every parameter moved off its initial value."""
    mem = M.PolicyMemory(seed=seed, **kw)
    g = torch.Generator().manual_seed(seed + 1)
    with torch.no_grad():
        for p in mem.parameters():
            p += 0.1 * torch.randn(p.shape, generator=g).to(p.device)
    return mem


def test_fresh_memory_is_the_plain_rollout():
    n, k = 64, 20
    pol = DevicePolicy.random_init(seed=2)
    runs = []
    for mem in (None, M.PolicyMemory()):
        env = HumanoidVecEnv(n, seed=5)
        env.reset()
        runs.append(pol.rollout(env, k) if mem is None else pol.rollout(env, k, memory=mem, state=mem.begin(n)))
        env.close()
    for f in ("obs", "actions", "rewards", "dones"):
        assert torch.equal(runs[0][f], runs[1][f]), f
    pol.close()


def core(mem, obs, state, resets):
    """The core in float64 on the CPU: (features, the bound of a float32 evaluation's error).  First order: e is the error a
    float32 value carries, taken through each operator on magnitudes; 1.1 covers the products of errors."""
    p = {f: getattr(mem, f).detach().double().cpu() for f in mem.NAMES}
    x = obs.double().cpu()
    k, n, _ = x.shape
    h, c = mem.heads, mem.channels

    def norm(v, e, w, b):
        rstd = 1 / torch.sqrt(v.var(-1, unbiased=False, keepdim=True) + 1e-5)
        hat = (v - v.mean(-1, keepdim=True)) * rstd
        d = e + e.mean(-1, keepdim=True)
        eh = rstd * d + hat.abs() * rstd * (d * d).mean(-1, keepdim=True).sqrt()
        eh = eh + 64 * U * (rstd * (v.abs().mean(-1, keepdim=True) + v.abs()) + hat.abs())
        return hat * w + b, w.abs() * eh + 4 * U * ((hat * w).abs() + b.abs())

    y, e = norm(x, torch.zeros_like(x), p["norm_weight"], p["norm_bias"])
    qkv = (y @ p["w_qkv"]).view(k, n, 3, h, c)
    eq = (e @ p["w_qkv"].abs() + (mem.n_in + 2) * U * (y.abs() @ p["w_qkv"].abs())).view(k, n, 3, h, c)
    t = lambda z: z.transpose(0, 1)
    ops = [t(qkv[:, :, i]) for i in range(3)]
    err = [t(eq[:, :, i]) for i in range(3)]
    args = (mem.log_decay, state, resets.t(), None, c ** -0.5)
    o, _ = R.attention(*ops, *args)
    mags = [a.abs() for a in ops]
    ma = (mem.log_decay, state.abs(), resets.t(), None, c ** -0.5)
    size, _ = R.attention(*mags, *ma)
    eo = (c + k + 64) * U * size
    z = (mem.log_decay, None, resets.t(), None, c ** -0.5)
    eo = eo + R.attention(err[0], mags[1], mags[2], *ma)[0] + R.attention(mags[0], err[1], mags[2], *z)[0] + R.attention(mags[0], mags[1], err[2], *z)[0]
    y, e = norm(t(o), t(eo), p["head_weight"], p["head_bias"])
    y, e = y.reshape(k, n, h * c), e.reshape(k, n, h * c)
    f = x + y @ p["w_out"]
    return f, 1.1 * (e @ p["w_out"].abs() + (h * c + 4) * U * (y.abs() @ p["w_out"].abs() + x.abs()))


def test_rollout_acts_on_what_the_learner_sees():
    n, k = 96, 60
    pol, val, mem = DevicePolicy.random_init(seed=2), DevicePolicy.random_init_value(seed=3), trained()
    env = HumanoidVecEnv(n, seed=5)
    env.reset()
    state = mem.begin(n)
    first = pol.rollout(env, 3, memory=mem, state=state)   # the fragment below starts from a state that holds something
    before = state.clone()
    assert before.any() and not first["resets"][0].any()
    tr = pol.rollout(env, k, explore=False, step0=3, memory=mem, state=state)
    assert tr["resets"].any() and not tr["resets"].all()
    assert torch.equal(tr["resets"][1:], tr["dones"][:-1])
    # the sampler's steps and the learner's fragment are both the core, each within its rounding
    want, tol = core(mem, tr["obs"], before, tr["resets"])
    with torch.no_grad():
        feat, last = mem.forward(tr["obs"], state=before, reset=tr["resets"])
    assert ((feat.double().cpu() - want).abs() <= tol).all()
    s, steps = before.clone(), []
    for i in range(k):
        steps.append(mem.step(tr["obs"][i], s, reset=tr["resets"][i]))
    assert ((torch.stack(steps).double().cpu() - want).abs() <= tol).all()
    assert torch.equal(s, state)
    # without exploration the recorded actions are the network's means on the core's features: the columns' first half.
    # 2e-5 as between the network's own two evaluations; the features' difference shrinks in the 0.01-normed last layer
    cols = pol.sample_batch_columns(tr["obs"], tr["actions"], value=val, memory=mem, state=before, resets=tr["resets"])
    assert (cols["action_dist_inputs"][..., :17] - tr["actions"]).abs().max().item() < 2e-5
    plain = pol.sample_batch_columns(feat, tr["actions"], value=val)
    for f in plain:
        assert torch.equal(plain[f], cols[f])
    # without the marks the learner would see other features
    with torch.no_grad():
        other, _ = mem.forward(tr["obs"], state=before, reset=torch.zeros_like(tr["resets"]))
    assert ((other.double().cpu() - want).abs() > tol).any()
    env.close()
    pol.close()
    val.close()


def test_learner_gradient():
    """Gradients of every parameter through the whole core against float64 autograd of the plain formulas.  Yardstick: the
    same plain formulas under float32 autograd; the core may be 8 times as far off, and 64 float32 roundings."""
    k, n = 45, 24
    mem = trained(seed=4, heads=3, channels=16)
    g = torch.Generator().manual_seed(8)
    obs = torch.randn(k, n, 70, generator=g).cuda()
    resets = (torch.rand(k, n, generator=g) < 0.05).to(torch.uint8).cuda()
    state = torch.randn(n, 3, 16, 16, generator=g).cuda()
    weight = torch.randn(k, n, 70, generator=g).cuda()
    lengths = torch.randint(0, k + 1, (n,), generator=g, dtype=torch.int32).cuda()
    f, _ = mem.forward(obs, state=state, reset=resets, lengths=lengths)
    (f * weight).sum().backward()

    def plain(dt):
        p = [x.detach().to(dt).requires_grad_(True) for x in mem.parameters()]
        nw, nb, wqkv, hw, hb, wo = p
        ln = lambda v, w, b: (v - v.mean(-1, keepdim=True)) / torch.sqrt(v.var(-1, unbiased=False, keepdim=True) + 1e-5) * w + b
        x = obs.to(dt)
        q, kk, v = (ln(x, nw, nb) @ wqkv).view(k, n, 3, 3, 16).permute(2, 1, 3, 0, 4)   # [n, heads, k, c]
        at = torch.arange(k, device="cuda")
        held = at[None] < lengths[:, None]
        ep = torch.cumsum(resets.t().long(), 1)
        seen = (at[None, :] <= at[:, None]) & (ep[:, :, None] == ep[:, None, :]) & held[:, :, None] & held[:, None, :]
        decay = torch.exp(mem.log_decay.to(dt)[:, None, None] * (at[:, None] - at[None, :]).clamp(min=0))
        o = ((q * 0.25) @ kk.transpose(2, 3).contiguous() * decay * seen[:, None]) @ v
        w_in = torch.exp(mem.log_decay.to(dt)[:, None] * (at + 1)) * (held & (ep == 0))[:, None]
        o = o + 0.25 * w_in[..., None] * (q @ state.to(dt).transpose(2, 3).contiguous())
        y = ln(o.permute(2, 0, 1, 3), hw, hb).reshape(k, n, 48)
        ((x + y @ wo) * weight.to(dt)).sum().backward()
        return [x.grad for x in p]
    want, yard = plain(torch.float64), plain(torch.float32)
    for name, p, w, y in zip(mem.NAMES, mem.parameters(), want, yard):
        scale = w.abs().max()
        err, ref = (p.grad - w).abs().max() / scale, (y - w).abs().max() / scale
        assert err <= 8 * ref + 64 * U, (name, err.item(), ref.item())


def test_refusals():
    pol, mem = DevicePolicy.random_init(seed=2), M.PolicyMemory()
    env = HumanoidVecEnv(8, seed=5)
    env.reset()
    s = mem.begin(8)
    for kw, text in [(dict(memory=mem), "needs its lanes' state"), (dict(state=s), "needs memory"),
                     (dict(memory=mem, state=s, fused=True), "neither fused"),
                     (dict(memory=M.PolicyMemory(n_in=44), state=s), "input width"),
                     (dict(memory=mem, state=mem.begin(7)), "state must be"),
                     (dict(memory=mem, state=s, out={"obs": torch.zeros(1)}), "out")]:
        with pytest.raises(ValueError, match=text):
            pol.rollout(env, 2, **kw)
    tr = pol.rollout(env, 2, memory=mem, state=s)
    for kw, text in [(dict(memory=mem), "resets"), (dict(state=s), "need memory"), (dict(resets=tr["resets"]), "need memory"),
                     (dict(memory=mem, resets=tr["resets"], mean=tr["actions"]), "neither mean")]:
        with pytest.raises(ValueError, match=text):
            pol.sample_batch_columns(tr["obs"], tr["actions"], **kw)
    with pytest.raises(ValueError, match="obs must be"):
        mem.forward(tr["obs"][..., :44])
    assert pol.rollout(env, 2, memory=mem, state=s, trajectories=False) == {}
    env.close()
    pol.close()
