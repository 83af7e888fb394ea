"""The policy memory's operators (csrc/decay_attn.hip, csrc/layer_norm.hip through ilrl_amd.memory) against float64
restatements (tests/memory_reference.py), at the sizes, strides and masks where they can go wrong.

Bounds.  u = 2^-24.  A result is a sum of products; `size` is the same sum over the magnitudes of its terms (the
reference run on absolute values).  Every float32 rounding on the way to it - the products over at most 128 channels, the
sums over the steps, the decays' powers (one exp2 of a product, at most 32 steps at a time) - changes it by at most u of
`size`; at most C = 128 + steps + 64 of them lie on one path.  bf16 operands formed from float32 values are split in two
parts, whose remainder is 2^-18 of the value; three such operands meet on a path at most.  The result's own rounding is
half a step, eps / 2 of its value (fp16: at least half its smallest number, 2^-25)."""
import copy

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a HIP device", allow_module_level=True)

import memory_reference as R  # noqa: E402
from ilrl_amd import memory as M  # noqa: E402

U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF = {"fp32": U, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
DEV = "cuda"


def close(got, want, size, kind, steps, state=False):
    got, want, size = got.detach().double().cpu(), want.double().cpu(), size.double().cpu()
    rel = (128 + steps + 64) * U + (3 * 2.0 ** -18 if kind == "bf16" and not state else 0.0)
    half = U if state else HALF[kind]
    tol = half * want.abs() + rel * (1 + half) * size + (2.0 ** -25 if kind == "fp16" and not state else 1e-37)
    err = (got - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), "worst %.3g of its bound at %s" % ((err / tol).max().item(), bad.nonzero()[:3].tolist())


class Case:
    def __init__(self, b, s, h, g, dk, dv, kind="bf16", order="lane", resets=0.0, lengths=None, state=True, seed=0, odd=False,
                 far=0):
        r = torch.Generator().manual_seed(seed * 7919 + b * 31 + s)
        self.kind, self.scale, self.steps = kind, dk ** -0.5, s
        dt = TYPES[kind]

        def rows(heads, d):
            extra = 3 if odd else 0   # rows cut out of a wider, unaligned buffer
            shape = (s, b, heads, d + extra) if order == "time" else (b, s, heads, d + extra)
            x = torch.randn(shape, generator=r).to(dt).to(DEV)
            if far:   # time-major steps `far` elements apart
                wide = torch.empty(s, far, dtype=dt, device=DEV)
                x = wide[:, :b * heads * d].copy_(x.reshape(s, -1)).view(s, b, heads, d)
            x = x[..., 1:1 + d] if odd else x
            return x.transpose(0, 1) if order == "time" else x
        self.q, self.k, self.v, self.d_out = rows(h, dk), rows(g, dk), rows(g, dv), rows(h, dv)
        self.log_decay = (-torch.rand(h, generator=r) * 0.3).to(DEV)
        self.state = torch.randn(b, h, dv, dk, generator=r).to(DEV) if state else None
        self.d_state = torch.randn(b, h, dv, dk, generator=r).to(DEV) if state else None
        self.reset = (torch.rand(b, s, generator=r) < resets).to(torch.uint8).to(DEV) if resets else None
        if order == "time" and self.reset is not None:
            self.reset = self.reset.t().contiguous().t()
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=DEV) if lengths is not None else None

    def masks(self):
        return dict(state=self.state, reset=self.reset, lengths=self.lengths, scale=self.scale)

    def forward(self):
        return M.decay_attention(self.q, self.k, self.v, self.log_decay, **self.masks())

    def backward(self, **kw):
        return M.decay_attention_backward(self.d_out, self.d_state, self.q, self.k, self.v, self.log_decay, **self.masks(), **kw)

    def _ref(self, fn, magnitude, *first):
        ops = list(first) + [self.q, self.k, self.v, self.log_decay, self.state]
        if magnitude:
            ops = [x if x is None or x is self.log_decay else x.abs() for x in ops]
        return fn(*ops, self.reset, self.lengths, self.scale)

    def check_forward(self, got=None):
        out, state = got or self.forward()
        for x, w, m, st in zip((out, state), self._ref(R.attention, False), self._ref(R.attention, True), (False, True)):
            close(x, w, m, self.kind, self.steps, st)
        return out, state

    def check_backward(self, got=None):
        grads = got or self.backward()
        want = self._ref(R.attention_grad, False, self.d_out, self.d_state)
        size = self._ref(R.attention_grad, True, self.d_out, self.d_state)
        for i, (x, w, m) in enumerate(zip(grads, want, size)):
            close(x, w, m, self.kind, self.steps + 8, i == 3)
        return grads


SHAPES = [
    # lanes, steps, heads, kv_heads, dk, dv
    (1, 1, 1, 1, 1, 1), (2, 2, 1, 1, 7, 3), (3, 31, 2, 2, 32, 32), (2, 32, 4, 4, 64, 64), (2, 33, 2, 1, 33, 65),
    (1, 65, 3, 3, 64, 32), (2, 95, 2, 2, 128, 128), (1, 64, 6, 2, 40, 72), (5, 20, 4, 4, 96, 16), (1, 40, 1, 1, 5, 128),
    (9, 3, 5, 5, 16, 48), (1, 130, 2, 2, 100, 36),
]


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_and_gradient(shape, kind):
    c = Case(*shape, kind=kind, resets=0.1, order="time" if sum(shape) % 2 else "lane")
    out, _ = c.check_forward()
    assert out.dtype == c.q.dtype
    c.check_backward()


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("dk,dv", [(32, 32), (8, 64), (24, 128), (64, 32), (64, 64), (56, 128), (128, 16), (128, 40), (120, 128)])
def test_widths_of_keys_and_values(dk, dv, kind):
    """Every pair of width classes, aligned."""
    c = Case(2, 75, 2, 1, dk, dv, kind=kind, resets=0.03, lengths=[75, 34])
    c.check_forward()
    c.check_backward()


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("dk", [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 17, 23, 31, 33, 34, 61, 66, 99, 127])
def test_rows_that_end_inside_a_load(dk, kind):
    """Rows of any width at any alignment, cut out of a buffer of NaN: nothing beside a row is read into it, and a result's
    row is written beside others that keep theirs."""
    dv = dk * 37 % 128 + 1
    c = Case(2, 37, 2, 1, dk, dv, kind=kind, order="time" if dk % 2 else "lane", resets=0.05, lengths=[37, 20], odd=True)
    for name in ("q", "k", "v", "d_out"):
        x = getattr(c, name)
        wide = torch.full((*x.shape[:3], x.shape[3] + 3), float("nan"), dtype=x.dtype, device=DEV)
        wide[..., 1:1 + x.shape[3]] = x
        setattr(c, name, wide[..., 1:1 + x.shape[3]])
    c.check_forward()
    c.check_backward()


@pytest.mark.parametrize("kind,d", [("bf16", 64), ("bf16", 63), ("fp32", 5), ("fp16", 6)])
def test_steps_very_far_apart(kind, d):
    """32 MB and more from one step to the next."""
    c = Case(2, 36, 2, 1, d, d, kind=kind, order="time", resets=0.04, lengths=[36, 33], far=(2 ** 25 + 64) // TYPES[kind].itemsize)
    c.check_forward()
    c.check_backward()


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("h,g,d", [(4, 4, 64), (4, 1, 64), (4, 2, 32), (8, 8, 32), (3, 3, 64), (6, 3, 32), (2, 2, 128)])
def test_steps_far_apart(h, g, d, kind):
    """Time-major steps of a wide batch (64 KB and more from one to the next), where a workgroup takes several heads."""
    c = Case(3, 70, h, g, d, d, kind=kind, order="time", resets=0.04, lengths=[70, 41, 0], far=32768 + 64)
    c.check_forward()
    c.check_backward()


def check_many(c, n):
    """The case's lanes n times over: every copy is the first, and the first is right."""
    def many(x):
        if x is None:
            return None
        if x.dim() == 4 and x.stride(0) < x.stride(1):   # time-major
            return x.transpose(0, 1).repeat(1, n, 1, 1).transpose(0, 1)
        return x.repeat(n, *[1] * (x.dim() - 1))
    big = copy.copy(c)
    for name in ("q", "k", "v", "d_out", "state", "d_state", "reset", "lengths"):
        setattr(big, name, many(getattr(c, name)))
    b = c.q.shape[0]
    got, grads = big.forward(), big.backward()
    for x in got + grads:
        copies = x.reshape(n, b, *x.shape[1:])
        assert torch.equal(copies, copies[:1].expand_as(copies))
    c.check_forward(tuple(x[:b] for x in got))
    c.check_backward(tuple(x[:b] for x in grads))


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("dk,dv", [(32, 32), (32, 64), (16, 128), (64, 24), (64, 64), (48, 128), (128, 32), (128, 64), (120, 128), (99, 127), (31, 63)])
def test_more_walks_than_the_card_has_waves(dk, dv, kind):
    """Batches of thousands of walks (each wave has wider slices there, for some types and widths)."""
    check_many(Case(3, 43, 2, 1, dk, dv, kind=kind, resets=0.05, lengths=[43, 0, 34]), 240)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("h,g,d", [(4, 4, 64), (4, 1, 64), (4, 2, 32), (8, 8, 32), (3, 3, 64), (2, 2, 128)])
def test_many_walks_of_steps_far_apart(h, g, d, kind):
    """The same time-major, 64 KB and more from a step to the next (a workgroup takes several heads)."""
    check_many(Case(4, 37, h, g, d, d, kind=kind, order="time", resets=0.04, lengths=[37, 20, 0, 33]), 130)


@pytest.mark.parametrize("kind,dk,dv", [("bf16", 64, 64), ("bf16", 128, 128), ("fp16", 128, 128), ("bf16", 127, 99)])
def test_many_walks_meet_values_that_are_not_finite(kind, dk, dv):
    c = Case(2, 50, 2, 2, dk, dv, kind=kind, state=False)
    c.reset = torch.zeros(2, 50, dtype=torch.uint8, device=DEV)
    c.reset[:, 40] = 1
    c.v[1, 36, :, 3] = float("inf")
    q, k, v = (x.repeat(300, 1, 1, 1) for x in (c.q, c.k, c.v))
    got, state = M.decay_attention(q, k, v, c.log_decay, reset=c.reset.repeat(300, 1), scale=c.scale)
    few, few_state = M.decay_attention(c.q, c.k, c.v, c.log_decay, reset=c.reset, scale=c.scale)
    for x, y in ((got, few), (state, few_state)):
        bad = ~x.reshape(300, *y.shape).isfinite()
        assert torch.equal(bad, (~y.isfinite()).expand_as(bad))
    bad = ~got.isfinite()
    want = torch.zeros_like(bad)
    want[1::2, 36:40, :, 3] = True
    assert torch.equal(bad, want) and state.isfinite().all()


@pytest.mark.parametrize("steps", [700, 1500])
@pytest.mark.parametrize("kind,dk", [("bf16", 64), ("fp32", 32), ("bf16", 128)])
def test_long_walks_of_few_lanes(steps, kind, dk):
    """Few lanes and many steps (the walk is split over time there), with episodes ending and lanes of many lengths."""
    c = Case(3, steps, 2, 1, dk, dk, kind=kind, resets=0.004, lengths=[steps, 0, steps // 2 + 7], seed=1)
    c.check_forward()
    c.check_backward()
    c = Case(1, steps, 2, 2, dk, dk, kind=kind, state=False, seed=2)
    c.check_forward()
    c.check_backward()


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("odd", [False, True])
def test_lengths_and_strides(kind, odd):
    c = Case(6, 70, 4, 2, 24, 56, kind=kind, order="time", resets=0.05, lengths=[70, 0, 1, 33, -5, 900], odd=odd)
    out, state = c.check_forward()
    assert torch.equal(state[1], c.state[1]) and torch.equal(state[4], c.state[4])   # nothing held: as it came
    grads = c.check_backward()
    assert torch.equal(grads[3][1], c.d_state[1])
    for x in (out,) + grads[:3]:   # steps behind a lane's length
        for lane, n in enumerate([70, 0, 1, 33, 0, 70]):
            assert not x[lane, n:].any()


def test_no_steps_and_no_lanes():
    c = Case(3, 0, 2, 2, 8, 8)
    out, state = c.forward()
    assert out.shape == (3, 0, 2, 8) and torch.equal(state, c.state)
    grads = c.backward()
    assert torch.equal(grads[3], c.d_state) and grads[0].shape == c.q.shape
    c = Case(0, 5, 2, 2, 8, 8)
    out, state = c.forward()
    assert out.shape == (0, 5, 2, 8) and state.shape == (0, 2, 8, 8)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_every_step_starts_an_episode(kind):
    c = Case(2, 50, 2, 2, 32, 32, kind=kind, resets=2.0)
    assert c.reset.all()
    c.check_forward()
    c.check_backward()


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_no_memory_and_full_memory(kind):
    """log_decay -inf sees the step itself only; 0 forgets nothing."""
    c = Case(2, 70, 2, 2, 32, 32, kind=kind)
    c.log_decay = torch.tensor([-float("inf"), 0.0], device=DEV)
    c.check_forward()
    c.check_backward()


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_rows_that_are_not_seen(kind, bad):
    """Steps behind a lane's length, an episode that diverged before the next one starts, and later steps: outputs that
    must not see them are what they are without them."""
    b, s, h, d = 4, 90, 2, 32
    lengths = [90, 61, 90, 90]
    c = Case(b, s, h, h, d, d, kind=kind, lengths=lengths)
    c.reset = torch.zeros(b, s, dtype=torch.uint8, device=DEV)
    c.reset[2, 40] = 1
    c.reset[0, 17] = 1
    clean_out, clean_state = c.check_forward()
    clean = c.check_backward()
    for x in (c.q, c.k, c.v, c.d_out):
        x[1, 61:] = bad       # behind the length
        x[2, 35] = bad        # lane 2: the first episode diverged at step 35
        x[3, 80, 0, 5] = bad  # lane 3, head 0: from step 80 on
    c.state[0] = bad          # lane 0: the state it came with; step 17 starts afresh
    out, state = c.forward()
    dq, dk, dv, ds = c.backward()
    rel = dict(atol=0.0, rtol=0.0)
    assert torch.equal(out[1], clean_out[1]) and torch.equal(state[1], clean_state[1])
    for x, y in zip((dq, dk, dv, ds), clean):
        assert torch.equal(x[1], y[1])
    torch.testing.assert_close(out[2, :35], clean_out[2, :35], **rel)      # before it
    torch.testing.assert_close(out[2, 40:], clean_out[2, 40:], **rel)      # the next episode
    torch.testing.assert_close(state[2], clean_state[2], **rel)
    assert not out[2, 35:40].isfinite().any()
    torch.testing.assert_close(dq[2, :35], clean[0][2, :35], **rel)
    torch.testing.assert_close(dq[2, 40:], clean[0][2, 40:], **rel)
    for x, y in ((dk, clean[1]), (dv, clean[2])):                           # backwards: earlier steps of its episode see it
        torch.testing.assert_close(x[2, 36:], y[2, 36:], **rel)
    torch.testing.assert_close(out[3, :80], clean_out[3, :80], **rel)
    torch.testing.assert_close(out[3, :, 1], clean_out[3, :, 1], **rel)    # the other head
    torch.testing.assert_close(out[0, 17:], clean_out[0, 17:], **rel)
    torch.testing.assert_close(state[0], clean_state[0], **rel)
    torch.testing.assert_close(dk[0], clean[1][0], **rel)


def test_heads_that_share_keys_by_expansion():
    """An expanded key head (stride 0) is the same as a shared one."""
    c = Case(2, 45, 4, 1, 32, 48)
    out, state = c.check_forward()
    c.k, c.v = c.k.expand(-1, -1, 4, -1), c.v.expand(-1, -1, 4, -1)
    out2, state2 = c.forward()
    assert torch.equal(out, out2) and torch.equal(state, state2)


def test_autograd_is_the_functional_gradient():
    c = Case(3, 40, 4, 2, 32, 32, kind="fp32", resets=0.1, order="time")
    ops = [x.detach().clone().requires_grad_(True) for x in (c.q, c.k, c.v, c.state)]
    out, state = M.decay_attention(*ops[:3], c.log_decay, state=ops[3], reset=c.reset, scale=c.scale)
    ((out * c.d_out).sum() + (state * c.d_state).sum()).backward()
    for x, g in zip(ops, c.backward()):
        assert torch.equal(x.grad, g)
    # one output alone, an expanded gradient, a leaf that needs none
    q = c.q.detach().clone().requires_grad_(True)
    M.decay_attention(q, c.k, c.v, c.log_decay, state=c.state, reset=c.reset, scale=c.scale)[0].sum().backward()
    c.d_out, c.d_state = torch.ones_like(c.d_out), None
    c.check_backward((q.grad,) + c.backward()[1:])
    k = c.k.detach().clone().requires_grad_(True)
    M.decay_attention(c.q, k, c.v, c.log_decay, reset=c.reset)[1].sum().backward()
    assert k.grad.isfinite().all() and k.grad.any()


def test_gradient_against_differences():
    """Along one operand the output is linear, so a difference quotient of float32 forward passes is the derivative up
    to their rounding: (C u) of the magnitude sum, on each of the two passes."""
    c = Case(2, 60, 2, 2, 32, 32, kind="fp32", resets=0.05)
    grads = c.backward()
    for name, g in zip(("q", "k", "v", "state"), grads):
        x = getattr(c, name)
        step = torch.randn(x.shape, generator=torch.Generator().manual_seed(5)).to(DEV)
        vals, size = [], 0.0
        for sign in (1, -1):
            setattr(c, name, (x + sign * step).contiguous())
            out, st = c.forward()
            vals.append((out.double() * c.d_out.double()).sum() + (st.double() * c.d_state.double()).sum())
            mag = c._ref(R.attention, True)
            size += (mag[0] * c.d_out.abs().double().cpu()).sum() + (mag[1] * c.d_state.abs().double().cpu()).sum()
            size += (x.abs().double() * g.abs().double()).sum().cpu()   # x + step rounds too
        setattr(c, name, x)
        quotient = (vals[0] - vals[1]).item() / 2
        assert abs(quotient - (g.double() * step.double()).sum().item()) <= 2 * (128 + 60 + 64) * U * size.item()


# ---------------------------------------------------------------------------------------------- the single step
@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("n,h,g,dk,dv", [(1, 4, 4, 64, 64), (1, 1, 1, 1, 1), (7, 6, 2, 40, 72), (33, 4, 4, 128, 128), (5, 3, 1, 13, 127),
                                         (300, 2, 2, 32, 17), (3, 2, 2, 4, 9), (2, 2, 2, 8, 70), (4, 2, 1, 16, 33)])
def test_step_is_one_step_of_the_walk(n, h, g, dk, dv, kind):
    c = Case(n, 1, h, g, dk, dv, kind=kind, resets=0.3)
    idle = torch.rand(n, generator=torch.Generator().manual_seed(n)) < 0.25
    active = (~idle).to(DEV)
    old = c.state.clone()
    c.lengths = active.int()
    into = torch.full_like(c.state, 7.0)
    out = M.decay_attention_step(c.q[:, 0], c.k[:, 0], c.v[:, 0], c.log_decay, c.state, reset=c.reset[:, 0], active=active,
                                 scale=c.scale, state_out=into)
    assert torch.equal(c.state, old)
    c.check_forward((out[:, None], into))
    assert torch.equal(into[~active], old[~active]) and not out[~active].any()
    here = old.clone()
    out2 = M.decay_attention_step(c.q[:, 0], c.k[:, 0], c.v[:, 0], c.log_decay, here, reset=c.reset[:, 0], active=active, scale=c.scale)
    assert torch.equal(out, out2) and torch.equal(here, into)


@pytest.mark.parametrize("dk", [2, 3, 5, 6, 7, 9, 11, 15, 18, 29, 31, 33, 62, 63, 65, 95, 126, 127])
def test_step_of_rows_that_end_inside_a_load(dk):
    """Also of states that begin 4 bytes behind a multiple of 16, and what lies beside a state stays as it was."""
    n, h, dv = 3, 2, 21
    c = Case(n, 1, h, h, dk, dv, kind="fp32", resets=0.3)
    size = n * h * dv * dk
    flat = torch.full((size + 2,), 7.0, device=DEV)
    state = flat[1:-1].view(n, h, dv, dk).copy_(c.state)
    out = M.decay_attention_step(c.q[:, 0], c.k[:, 0], c.v[:, 0], c.log_decay, state, reset=c.reset[:, 0], scale=c.scale)
    c.check_forward((out[:, None], state))
    assert flat[0] == 7 and flat[-1] == 7


def test_step_forgets_a_state_that_is_not_finite():
    c = Case(4, 1, 2, 2, 32, 32)
    c.state[1] = float("nan")
    c.state[2] = float("inf")
    c.reset = torch.tensor([[0], [1], [1], [0]], dtype=torch.uint8, device=DEV)
    out = M.decay_attention_step(c.q[:, 0], c.k[:, 0], c.v[:, 0], c.log_decay, c.state, reset=c.reset[:, 0], scale=c.scale)
    assert out.isfinite().all() and c.state.isfinite().all()


def test_steps_walk_like_the_fragment():
    c = Case(5, 40, 4, 4, 32, 32, kind="fp32", resets=0.1, order="time")
    state, outs = c.state.clone(), []
    for t in range(40):
        outs.append(M.decay_attention_step(c.q[:, t], c.k[:, t], c.v[:, t], c.log_decay, state, reset=c.reset[:, t], scale=c.scale))
    c.check_forward((torch.stack(outs, 1), state))


# ---------------------------------------------------------------------------------------------- where they run
def test_offsets_past_32_bits():
    """Lanes further apart than 2^31 elements (a slice of a long buffer)."""
    far, s, h, d = 2 ** 31 + 64, 40, 2, 64
    c = Case(2, s, h, h, d, d)
    buf = torch.empty(far + s * h * d, dtype=torch.bfloat16, device=DEV)
    for name in ("q", "k", "v", "d_out"):
        x = getattr(c, name)
        view = buf.as_strided((2, s, h, d), (far, h * d, d, 1))
        view.copy_(x)
        setattr(c, name, view)
        c.check_forward()
        c.check_backward()
        setattr(c, name, x)
    rows = buf.as_strided((2, d), (far, 1))
    rows.copy_(torch.randn(2, d, generator=torch.Generator().manual_seed(1)))
    y = M.layer_norm(rows)
    assert torch.equal(y, M.layer_norm(rows.contiguous()))


def test_streams_and_captured_graphs():
    """The calls follow the current stream, and captured once give on every replay what an eager call gives."""
    c = Case(3, 400, 2, 1, 64, 64, resets=0.02, order="time")
    x = torch.randn(300, 70, device=DEV)
    w, b = torch.randn(70, device=DEV), torch.randn(70, device=DEV)

    def calls():
        out, state = c.forward()
        grads = c.backward()
        y, mean, rstd = M.layer_norm_forward(x, w, b)
        dn = M.layer_norm_backward(y, x, mean, rstd, w)
        step = M.decay_attention_step(c.q[:, 0], c.k[:, 0], c.v[:, 0], c.log_decay, state.clone(), scale=c.scale)
        return (out, state, y, step) + tuple(grads) + tuple(dn)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    eager = calls()
    with torch.cuda.stream(side):
        for a, e in zip(calls(), eager):
            assert torch.equal(a, e)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):   # two graphs that hold the same operators
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            got = calls()
        graphs.append((gr, got))
    for turn in range(4):
        for t in (c.q, c.k, c.v, c.d_out, x):
            t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(turn)).to(t.dtype))
        c.state.normal_()
        for gr, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        eager = calls()
        for _, got in graphs:
            for a, e in zip(got, eager):
                assert torch.equal(a, e)


# ---------------------------------------------------------------------------------------------- layer norm
def norm_bounds(x, w, b, y, kind):
    """|y - exact| from float32 sums: at most 64 roundings on the path to a mean or a variance."""
    xd = x.double().cpu()
    rstd = 1 / torch.sqrt(xd.var(-1, unbiased=False, keepdim=True) + 1e-5)
    h = (xd - xd.mean(-1, keepdim=True)) * rstd
    dh = 64 * U * (rstd * (xd.abs().mean(-1, keepdim=True) + xd.abs()) + h.abs())
    wa = 1.0 if w is None else w.double().cpu().abs()
    ba = 0.0 if b is None else b.double().cpu().abs()
    return HALF[kind] * y.abs() * 1.01 + wa * dh + 4 * U * (wa * h.abs() + ba) + (2.0 ** -25 if kind == "fp16" else 0)


def test_captured_gradients_follow_their_inputs():
    """Forward and gradient through autograd, captured together: every replay is the eager result for the inputs of then."""
    c = Case(4, 70, 4, 2, 32, 64, kind="bf16", resets=0.05, order="time")
    x, w = torch.randn(90, 64, device=DEV), torch.randn(64, device=DEV)
    leaves = [t.detach().clone().requires_grad_(True) for t in (c.q, c.k, c.v, c.state, x, w)]

    def step():
        q, k, v, s, x, w = leaves
        out, state = M.decay_attention(q, k, v, c.log_decay, state=s, reset=c.reset, scale=c.scale)
        y = M.layer_norm(x, w)
        return torch.autograd.grad((out, state, y), leaves, (c.d_out, c.d_state, y.detach()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()   # (its graph is gone with its results)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step()
    for turn in range(3):
        with torch.no_grad():
            for i, t in enumerate(leaves):
                t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(10 * turn + i)).to(t.dtype))
        graph.replay()
        torch.cuda.synchronize()
        got = [g.clone() for g in grads]
        for a, e in zip(got, step()):
            assert torch.equal(a, e)


NORMS = [(1, 70), (3, 1), (5, 7), (1000, 64), (17, 44), (33, 128), (257, 256), (9, 257), (40, 512), (6, 1000), (5, 2048), (3, 4096), (2, 5000),
         (3, 8192), (2, 16384), (4, 9001), (2500, 32)]


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("rows,c", NORMS)
def test_norm_and_gradient(rows, c, kind):
    r = torch.Generator().manual_seed(rows + c)
    dt = TYPES[kind]
    pitch = c + (0 if rows % 2 else 5)
    x = (torch.randn(rows, pitch, generator=r) * 2 + 0.7).to(dt).to(DEV)[:, :c]
    dy = torch.randn(rows, pitch, generator=r).to(dt).to(DEV)[:, :c]
    for pd in (torch.float32, dt):
        w, b = torch.randn(c, generator=r).to(pd).to(DEV), torch.randn(c, generator=r).to(pd).to(DEV)
        y, mean, rstd = M.layer_norm_forward(x, w, b)
        want = R.norm(x, w, b, 1e-5)
        assert ((y.double().cpu() - want).abs() <= norm_bounds(x, w, b, want, kind)).all()
        dx, dw, db = M.layer_norm_backward(dy, x, mean, rstd, w)
        wx, ww, wb = R.norm_grad(dy, x, mean, rstd, w)
        # the statistics are inputs here: 64 roundings on the way to each of dx's sums and to dw, db
        h = ((x.double().cpu() - mean.double().cpu()[:, None]) * rstd.double().cpu()[:, None]).abs()
        g = (dy.double().cpu() * w.double().cpu()).abs()
        size = rstd.double().cpu()[:, None] * (g + g.mean(-1, keepdim=True) + h * (g * h).mean(-1, keepdim=True))
        assert ((dx.double().cpu() - wx).abs() <= HALF[kind] * wx.abs() * 1.01 + 64 * U * size + (2.0 ** -25 if kind == "fp16" else 0)).all()
        half = U if pd == torch.float32 else HALF[kind]
        tiny = 2.0 ** -25 if pd == torch.float16 else 0
        assert ((dw.double().cpu() - ww).abs() <= half * ww.abs() * 1.01 + 64 * U * (dy.double().cpu().abs() * h).sum(0) + tiny).all()
        assert ((db.double().cpu() - wb).abs() <= half * wb.abs() * 1.01 + 64 * U * dy.double().cpu().abs().sum(0) + tiny).all()
        again = M.layer_norm_backward(dy, x, mean, rstd, w)
        assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("rows,c", [(5, 1), (7, 3), (70, 4), (9, 6), (13, 9), (40, 15), (21, 63), (300, 65), (11, 250), (37, 511), (6, 1030),
                                    (5, 1537), (3, 3001), (3, 6003), (2, 12001)])
def test_norm_rows_that_end_inside_a_load(rows, c, kind):
    """Rows of any width at any alignment, cut out of a buffer of NaN, and parameters that begin anywhere: the results are
    those of the same rows by themselves, to the rounding of another order of the sums; nothing beside a row is read or
    written."""
    r = torch.Generator().manual_seed(rows * 31 + c)
    dt = TYPES[kind]

    def cut(*shape, type=dt):
        x = torch.randn(shape, generator=r).to(type).to(DEV)
        wide = torch.full((*shape[:-1], c + 3), float("nan"), dtype=type, device=DEV)
        wide[..., 1:1 + c] = x
        return wide[..., 1:1 + c]
    x, dy = cut(rows, c), cut(rows, c)
    for pd in (torch.float32, dt):
        w, b = cut(c, type=pd), cut(c, type=pd)
        y, mean, rstd = M.layer_norm_forward(x, w, b)
        want = R.norm(x, w, b, 1e-5)
        assert ((y.double().cpu() - want).abs() <= norm_bounds(x, w, b, want, kind)).all()
        dx, dw, db = M.layer_norm_backward(dy, x, mean, rstd, w)
        for got in (dx, dw, db):
            assert got.isfinite().all()
        one = M.layer_norm_backward(dy[:1].clone(), x[:1].clone(), mean[:1].clone(), rstd[:1].clone(), w.clone())[0]
        torch.testing.assert_close(dx[:1], one, atol=0.0, rtol=0.0)


def test_norm_without_parameters_empty_and_in_place():
    x = torch.randn(4, 3, 48, device=DEV)
    y = M.layer_norm(x)
    assert ((y.double().cpu() - R.norm(x, None, None, 1e-5)).abs() <= norm_bounds(x, None, None, R.norm(x, None, None, 1e-5), "fp32")).all()
    assert torch.equal(y, M.layer_norm(x, torch.ones(48, device=DEV)))
    z = x.clone()
    out, _, _ = M.layer_norm_forward(z, out=z)
    assert out is z and torch.equal(z, y)
    e = torch.empty(0, 48, device=DEV)
    assert M.layer_norm(e).shape == (0, 48)
    dx, dw, db = M.layer_norm_backward(e, e, torch.empty(0, device=DEV), torch.empty(0, device=DEV), torch.ones(48, device=DEV))
    assert dx.shape == (0, 48) and not dw.any() and not db.any()


def test_norm_of_a_large_mean():
    """The variance is summed from differences: a mean far above the spread costs no more than the inputs' own rounding."""
    x = (torch.randn(64, 256, generator=torch.Generator().manual_seed(2)) + 1000).to(DEV)
    want = R.norm(x, None, None, 1e-5)
    assert ((M.layer_norm(x).double().cpu() - want).abs() <= norm_bounds(x, None, None, want, "fp32")).all()


def test_norm_autograd_and_differences():
    r = torch.Generator().manual_seed(9)
    x, w, b = (torch.randn(s, generator=r).to(DEV).requires_grad_(True) for s in ((12, 3, 70), (70,), (70,)))
    dy = torch.randn(12, 3, 70, generator=r).to(DEV)
    M.layer_norm(x, w, b).backward(dy)
    xd, wd = x.detach().reshape(-1, 70), w.detach()
    _, mean, rstd = M.layer_norm_forward(xd, wd, b.detach())
    dx, dw, db = M.layer_norm_backward(dy.reshape(-1, 70), xd, mean, rstd, wd)
    assert torch.equal(x.grad.reshape(-1, 70), dx) and torch.equal(w.grad, dw) and torch.equal(b.grad, db)
    # a central difference of the float64 definition along one direction (its error is the cubic term, 1e-4 squared)
    step = torch.randn(12, 3, 70, generator=r)
    f = lambda e: (R.norm(x.detach().cpu().double() + e * step.double(), w.detach(), b.detach(), 1e-5) * dy.double().cpu()).sum()
    quotient = ((f(1e-4) - f(-1e-4)) / 2e-4).item()
    assert abs(quotient - (x.grad.double().cpu() * step.double()).sum().item()) <= 1e-4 * (x.grad.double().cpu() * step.double()).abs().sum().item()
    b2 = torch.zeros(70, device=DEV, requires_grad=True)
    M.layer_norm(x.detach(), None, b2).sum().backward()
    assert torch.equal(b2.grad, torch.full((70,), 36.0, device=DEV))


# ---------------------------------------------------------------------------------------------- refusals of the front
def test_front_refusals():
    c = Case(2, 5, 4, 2, 16, 24)
    ok = lambda **kw: M.decay_attention(kw.pop("q", c.q), kw.pop("k", c.k), kw.pop("v", c.v), kw.pop("ld", c.log_decay), **kw)
    f32 = torch.float32
    for kw, text in [(dict(q=c.q[0]), "lanes, steps"), (dict(k=c.k[:, :3]), "k must be"), (dict(k=c.k.float()), "of type"),
                     (dict(v=c.v[:, :, :1]), "v must be"), (dict(k=c.k.cpu()), "is on"), (dict(ld=c.log_decay[:2]), "log_decay"),
                     (dict(ld=c.log_decay.double()), "log_decay"), (dict(state=c.state.half()), "state"),
                     (dict(state=c.state[:1]), "state"), (dict(state=c.state.transpose(2, 3).contiguous().transpose(2, 3)), "contiguous"),
                     (dict(reset=torch.zeros(2, 5, device=DEV)), "reset"), (dict(reset=torch.zeros(5, 2, dtype=torch.uint8, device=DEV)), "reset"),
                     (dict(lengths=torch.zeros(2, dtype=torch.int64, device=DEV)), "lengths"),
                     (dict(q=c.q.double(), k=c.k.double(), v=c.v.double()), "float32, bfloat16"),
                     (dict(q=torch.zeros(2, 5, 3, 16, device=DEV, dtype=c.q.dtype), ld=c.log_decay[:3]), "shared evenly"),
                     (dict(q=torch.zeros(2, 5, 4, 129, device=DEV), k=torch.zeros(2, 5, 2, 129, device=DEV), v=c.v.to(f32)), "1 to 128")]:
        with pytest.raises(ValueError, match=text):
            ok(**kw)
    step = lambda **kw: M.decay_attention_step(c.q[:, 0], c.k[:, 0], c.v[:, 0], c.log_decay, kw.pop("state", c.state), **kw)
    for kw, text in [(dict(state=None), "state is required"), (dict(active=torch.ones(3, dtype=torch.uint8, device=DEV)), "active"),
                     (dict(state_out=c.state[:1]), "state_out"), (dict(out=c.q[:, 0].float()), "out"),
                     (dict(reset=torch.zeros(2, 1, dtype=torch.uint8, device=DEV)), "reset"),
                     (dict(state=c.state.clone().requires_grad_(True)), "not differentiable")]:
        with pytest.raises(ValueError, match=text):
            step(**kw)
    with pytest.raises(ValueError, match="d_out"):
        M.decay_attention_backward(c.d_out[:, :3], None, c.q, c.k, c.v, c.log_decay)
    with pytest.raises(ValueError, match="d_state"):
        M.decay_attention_backward(c.d_out, c.d_state[:1], c.q, c.k, c.v, c.log_decay)
    x = torch.randn(3, 8, device=DEV)
    for call, text in [(lambda: M.layer_norm(x.double()), "float32, bfloat16"), (lambda: M.layer_norm(x, x[0, :4]), "weight"),
                       (lambda: M.layer_norm(x, x[0], x[0].half()), "one type"), (lambda: M.layer_norm(x, x[0].cpu()), "is on"),
                       (lambda: M.layer_norm(x[:, :0]), "channels"), (lambda: M.layer_norm(torch.zeros(1, 16385, device=DEV)), "channels"),
                       (lambda: M.layer_norm_backward(x, x, x[:2, 0], x[:, 0], x[0]), "mean"),
                       (lambda: M.layer_norm_backward(x[:2], x, x[:, 0], x[:, 0], x[0]), "dy")]:
        with pytest.raises(ValueError, match=text):
            call()
