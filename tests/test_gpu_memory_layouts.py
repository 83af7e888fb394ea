"""The policy memory's operators on slices of packed buffers, as one projection gives q, k and v, and the same buffers' free
slices as outputs."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a HIP device", allow_module_level=True)

from ilrl_amd import _native as N  # noqa: E402
from ilrl_amd import memory as M  # noqa: E402
from test_gpu_memory import Case  # noqa: E402


def pack(c, order):
    """The case's q, k, v, d_out side by side in one buffer, with room for an output, steps or lanes outside."""
    parts = (c.q, c.k, c.v, c.d_out, torch.full_like(c.d_out, 7.0))
    flat = [x.transpose(0, 1) if order == "time" else x for x in parts]
    wide = torch.cat([x.reshape(*x.shape[:2], -1) for x in flat], -1)
    got, at = [], 0
    for x in flat:
        size = x.shape[2] * x.shape[3]
        y = wide[..., at:at + size].view(x.shape)
        got.append(y.transpose(0, 1) if order == "time" else y)
        at += size
    c.q, c.k, c.v, c.d_out, free = got
    return wide, free


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("order", ["time", "lane"])
@pytest.mark.parametrize("b,s,h,g,dk,dv", [(3, 45, 4, 4, 32, 32), (2, 70, 4, 2, 64, 64), (5, 33, 3, 1, 13, 7), (300, 40, 4, 4, 32, 32),
                                           (2, 500, 2, 2, 32, 32)])
def test_slices_of_one_projection(b, s, h, g, dk, dv, order, kind):
    c = Case(b, s, h, g, dk, dv, kind=kind, order=order, resets=0.05, lengths=[s - i % 3 * (s // 3) for i in range(b)])
    pack(c, order)
    c.check_forward()
    c.check_backward()


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("h,g,dk,dv", [(4, 4, 32, 32), (4, 2, 128, 128), (3, 1, 13, 7)])
def test_step_into_a_slice_of_the_buffer(h, g, dk, dv, kind):
    """The free slice beside the inputs takes the output; nothing beside it changes.  A slice that is an input's, or reaches
    into one, is refused."""
    c = Case(6, 1, h, g, dk, dv, kind=kind)
    wide, free = pack(c, "lane")
    before, state = wide.clone(), c.state.clone()
    one = (c.q[:, 0], c.k[:, 0], c.v[:, 0], c.log_decay)
    plain = M.decay_attention_step(*one, state.clone(), scale=c.scale)
    out = M.decay_attention_step(*one, state, scale=c.scale, out=free[:, 0])
    assert torch.equal(out, plain)
    size = h * dv
    assert torch.equal(wide[..., :-size], before[..., :-size]) and torch.equal(wide[..., -size:].reshape(6, h, dv), plain)
    c.check_forward((out[:, None], state))
    into = wide.view(6, -1)
    for at in (0, h * dk - 1, h * dk + 1, into.shape[1] - 2 * size - g * dv):
        with pytest.raises(N.NativeError, match="overlap"):
            M.decay_attention_step(*one, state, out=into[:, at:at + size].view(6, h, dv))
    with pytest.raises(N.NativeError, match="overlap"):
        M.decay_attention_step(*one, state, out=torch.empty(h, dv, dtype=wide.dtype, device="cuda").expand(6, h, dv))
    with pytest.raises(N.NativeError, match="overlap"):
        M.decay_attention_step(*one, state, state_out=shifted(state))


def shifted(state):
    """A contiguous state that shares all but its last element with `state`'s storage."""
    flat = torch.cat([state.flatten(), state.new_zeros(1)])
    state.set_(flat.untyped_storage(), 0, state.shape, state.stride())
    return flat[1:].view(state.shape)


def test_norm_into_its_input_or_beside_it():
    """Row for row over the input, or apart from it: another place inside the input's rows is refused."""
    rows, c = 300, 64
    flat = torch.randn(rows * c + 2 * c, generator=torch.Generator().manual_seed(1)).cuda()
    x = flat[:rows * c].view(rows, c)
    want = M.layer_norm(x)
    for shift in (1, 4, c, 2 * c):
        with pytest.raises(N.NativeError, match="overlap"):
            M.layer_norm_forward(x, out=flat[shift:shift + rows * c].view(rows, c))
    with pytest.raises(N.NativeError, match="overlap"):
        M.layer_norm_forward(x, x[7], out=x)   # a weight among the rows it replaces
    assert torch.equal(M.layer_norm(x), want)
    half = flat[:rows * c].view(2, rows // 2, c)
    y, _, _ = M.layer_norm_forward(half[0], out=half[1])   # the buffer's other half
    assert torch.equal(y, want[:rows // 2])
    M.layer_norm_forward(half[0], out=half[0])
    assert torch.equal(half[0], half[1])


def test_calls_of_two_threads_on_their_own_streams():
    """Nothing is shared between calls: every thread gets what it gets alone, refusals of one do not reach the other."""
    import threading
    cases = [Case(3, 431, 2, 1, 40, 72, kind="bf16", resets=0.01), Case(40, 45, 4, 2, 32, 32, kind="fp32", order="time", resets=0.05)]
    alone = [c.forward() + c.backward() for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(c, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = c.forward() + c.backward()
                    x = torch.ones(5, 64, device="cuda")
                    with pytest.raises(N.NativeError, match="hum_layer_norm: .*overlap"):
                        M.layer_norm_forward(x, x[2], out=x)
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want))
        except BaseException as e:   # (else the thread would end without the test knowing)
            wrong.append(e)
    threads = [threading.Thread(target=work, args=a) for a in zip(cases, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
