"""A policy that remembers: linear attention with a decay for each head and layer norm over the C-ABI
(include/humanoid_env.h: hum_decay_attn / _backward / _step, hum_layer_norm / _backward), and `PolicyMemory`, the
recurrent core made of them that DevicePolicy.rollout and sample_batch_columns (ilrl_amd/policy.py) take as `memory=`.

The reference's policies see one observation (train_config.py:107-111, RLlib's FullyConnectedNetwork); what the
observation leaves out - the heightfield under the feet, what a limb did some steps ago - a policy can only act on by
remembering it.  Per lane and head the memory is a matrix S [dv, dk] in float32:

    S_t = a_t S_{t-1} + v_t k_t^T      a_t = 0 where step t starts an episode, exp(log_decay[head]) elsewhere
    o_t = scale S_t q_t

The sampler advances it a step at a time (`decay_attention_step`: one read and one write of the state); the learner runs
whole fragments (`decay_attention`, differentiable, on the matrix cores) and gets the same numbers up to rounding.

Rows are [lanes, steps, heads, channels]; a rollout's time-major [steps, lanes, ...] tensors are passed as
x.transpose(0, 1), no copy.  float32, bfloat16 and float16; 1 to 128 channels a head; key / value heads may be shared by
equal groups of query heads.  There is no CPU path.
"""
import ctypes
import struct

from . import _native as N

MAX_HEAD_CHANNELS, MAX_NORM_CHANNELS = 128, 16384

# The argument structures as packed bytes (hum_decay_attn_args, hum_rows, hum_norm_args): building them field by field with
# ctypes took longer than a single step's kernel
_ATTN = struct.Struct("=8if4xQ" + "Qqqq" * 3 + "QQQqqQ")
_ROWS = struct.Struct("=Qqqq")
_NORM = struct.Struct("=4i2q2Q")

_entry = None


class _Entry:
    """torch and the entry points, found once (torch is only imported when an operator is called)."""

    def __init__(self):
        import torch
        self.t = torch
        self.types = {torch.float32: N.HUM_F32, torch.bfloat16: N.HUM_BF16, torch.float16: N.HUM_F16}
        self.marks = (torch.uint8, torch.bool)
        L, c = N.lib(), ctypes
        b, vp, i32, i64, u64, f32 = c.c_char_p, c.c_void_p, c.c_int32, c.c_int64, c.c_uint64, c.c_float
        need = c.POINTER(u64)

        def bind(name, *args):
            return c.CFUNCTYPE(c.c_int, *args)((name, L))
        self.workspace = bind("hum_decay_attn_workspace", b, i32, need)
        self.attn = bind("hum_decay_attn", b, b, vp, u64, vp)
        self.attn_backward = bind("hum_decay_attn_backward", b, b, vp, b, b, b, vp, vp, u64, vp)
        self.step = bind("hum_decay_attn_step", b, vp, b, vp)
        self.norm = bind("hum_layer_norm", b, vp, f32, vp, i64, vp, vp, vp)
        self.norm_workspace = bind("hum_layer_norm_workspace", b, need)
        self.norm_backward = bind("hum_layer_norm_backward", b, vp, i64, vp, vp, vp, i64, vp, vp, vp, u64, vp)
        self.raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        self.forward_ad = torch.autograd.forward_ad
        self.written = torch.autograd.graph.increment_version   # for tensors of the caller's that a kernel wrote into

    def stream(self, index):
        if self.raw_stream is not None:
            return self.raw_stream(index)
        return self.t.cuda.current_stream(index).cuda_stream


def _e():
    global _entry
    if _entry is None:
        _entry = _Entry()
    return _entry


def _no_tangents(e, *xs):
    """Forward-mode derivatives are refused: past the autograd functions they would be dropped without a word."""
    if getattr(e.forward_ad, "_current_level", 0) < 0:   # outside dual_level no tensor has one
        return
    if any(x is not None and e.forward_ad.unpack_dual(x).tangent is not None for x in xs):
        raise NotImplementedError("the policy memory's operators have no forward-mode derivative")


def _type(e, x, what):
    code = e.types.get(x.dtype)
    if code is None:
        raise ValueError("%s: float32, bfloat16 or float16, got %s" % (what, x.dtype))
    return code


def _p(x):
    return x.data_ptr() if x is not None else None


def _unit(x):
    """x with adjacent channels."""
    return x if x.stride(-1) == 1 or x.shape[-1] <= 1 else x.contiguous()


def _rows(x):
    s = x.stride()
    return _ROWS.pack(x.data_ptr(), s[0], s[1], s[2])


def _same_order(like, shape):
    """An empty [lanes, steps, heads, channels] tensor in `like`'s memory order (time-major where its steps are the outer
    axis)."""
    t = _e().t
    st, sh = like.stride(), like.shape
    if shape == sh and st[3] == 1 and st[2] == sh[3]:
        row = sh[2] * sh[3]
        if (st[1] == row and st[0] == sh[1] * row) or (st[0] == row and st[1] == sh[0] * row):
            return t.empty_like(like)   # (packed: half the host time of what follows)
    if st[0] < st[1]:
        return t.empty((shape[1], shape[0]) + shape[2:], dtype=like.dtype, device=like.device).transpose(0, 1)
    return t.empty(shape, dtype=like.dtype, device=like.device)


def _on(x, device, what, shape=None, dtypes=None):
    if x.device != device:
        raise ValueError("%s is on %s, expected %s" % (what, x.device, device))
    if shape is not None and x.shape != shape:
        raise ValueError("%s must be %s, got %s" % (what, list(shape), list(x.shape)))
    if dtypes is not None and x.dtype not in dtypes:
        raise ValueError("%s must be of type %s, got %s" % (what, " or ".join(str(d) for d in dtypes), x.dtype))
    return x


def _check(e, q, k, v, log_decay, state, reset, lengths, axes):
    """The checks fragments (axes 4: [lanes, steps, heads, channels]) and single steps (axes 3) share; returns (q, k, v with
    adjacent channels, log_decay, lengths, the sizes (lanes, steps, heads, kv_heads, dk, dv))."""
    t, f32 = e.t, e.t.float32
    qs, ks, vs = q.shape, k.shape, v.shape
    if len(qs) != axes or len(ks) != axes or len(vs) != axes:
        raise ValueError("q, k, v must be [lanes, %sheads, channels], got %s, %s, %s"
                         % ("steps, " if axes == 4 else "", list(qs), list(ks), list(vs)))
    if not q.is_cuda:
        raise ValueError("q must be on a GPU (there is no CPU path)")
    dev, dt, index = q.device, q.dtype, q.get_device()
    lead, h, dk = qs[:-2], qs[-2], qs[-1]
    g, dv = ks[-2], vs[-1]
    # (one expression for what is nearly always so: the single step's host time is its time)
    if not (k.dtype == dt == v.dtype and ks == lead + (g, dk) and vs == lead + (g, dv) and k.get_device() == index
            and v.get_device() == index):
        _on(k, dev, "k", lead + (g, dk), (dt,))
        _on(v, dev, "v", lead + (g, dv), (dt,))
    if g < 1 or h % g:
        raise ValueError("%d key / value heads cannot be shared evenly by %d query heads" % (g, h))
    if not (1 <= dk <= MAX_HEAD_CHANNELS and 1 <= dv <= MAX_HEAD_CHANNELS):
        raise ValueError("1 to %d channels a head, got %d (keys) and %d (values)" % (MAX_HEAD_CHANNELS, dk, dv))
    if not (log_decay.dtype == f32 and log_decay.shape == (h,) and log_decay.get_device() == index):
        _on(log_decay, dev, "log_decay", (h,), (f32,))
    if log_decay.requires_grad:
        raise ValueError("log_decay is a constant schedule and has no gradient: pass log_decay.detach()")
    if not log_decay.is_contiguous():
        log_decay = log_decay.contiguous()
    if state is not None:
        if not (state.dtype == f32 and state.shape == (lead[0], h, dv, dk) and state.get_device() == index):
            _on(state, dev, "state", (lead[0], h, dv, dk), (f32,))
        if not state.is_contiguous():
            raise ValueError("state must be contiguous")
    if reset is not None:
        _on(reset, dev, "reset", lead, e.marks)
    if lengths is not None:
        _on(lengths, dev, "lengths", lead[:1], (t.int32,))
        lengths = lengths.contiguous()
    return _unit(q), _unit(k), _unit(v), log_decay, lengths, (lead[0], lead[1] if axes == 4 else 1, h, g, dk, dv)


def _attn(e, q, k, v, log_decay, state, state_out, reset, lengths, scale, sizes):
    """hum_decay_attn_args of a fragment."""
    sq, sk, sv = q.stride(), k.stride(), v.stride()
    sr = reset.stride() if reset is not None else (0, 0)
    return _ATTN.pack(q.get_device(), _type(e, q, "q"), *sizes, sizes[4] ** -0.5 if scale is None else float(scale),
                      log_decay.data_ptr(), q.data_ptr(), sq[0], sq[1], sq[2], k.data_ptr(), sk[0], sk[1], sk[2],
                      v.data_ptr(), sv[0], sv[1], sv[2], _p(state) or 0, _p(state_out) or 0, _p(reset) or 0, sr[0], sr[1],
                      _p(lengths) or 0)


def _scratch(e, a, backward, device):
    need = ctypes.c_uint64(0)
    N.check(e.workspace(a, backward, ctypes.byref(need)), "hum_decay_attn_workspace")
    return e.t.empty(need.value, dtype=e.t.uint8, device=device) if need.value else None


def _forward(q, k, v, log_decay, state, reset, lengths, scale):
    e = _e()
    q, k, v, log_decay, lengths, sizes = _check(e, q, k, v, log_decay, state, reset, lengths, 4)
    n, s, h, _, dk, dv = sizes
    out = _same_order(q, (n, s, h, dv))
    state_out = e.t.empty(n, h, dv, dk, dtype=e.t.float32, device=q.device)
    a = _attn(e, q, k, v, log_decay, state, state_out, reset, lengths, scale, sizes)
    ws = _scratch(e, a, 0, q.device)
    N.check(e.attn(a, _rows(out), _p(ws), ws.numel() if ws is not None else 0, e.stream(q.get_device())), "hum_decay_attn")
    return out, state_out


def decay_attention_backward(d_out, d_state, q, k, v, log_decay, state=None, reset=None, lengths=None, scale=None,
                             needs=(True, True, True, True)):
    """(dq, dk, dv, d_state_in) of decay_attention for the gradients d_out [lanes, steps, heads, dv] of its output and
    d_state [lanes, heads, dv, dk] of its final state (None = zeros), from the same inputs.  needs: which of the four to
    compute (the others are None)."""
    e = _e()
    q, k, v, log_decay, lengths, sizes = _check(e, q, k, v, log_decay, state, reset, lengths, 4)
    n, s, h, _, dk, dv = sizes
    a = _attn(e, q, k, v, log_decay, state, None, reset, lengths, scale, sizes)
    d_out = _unit(_on(d_out, q.device, "d_out", (n, s, h, dv), (q.dtype,)))
    if d_state is not None:
        d_state = _on(d_state, q.device, "d_state", (n, h, dv, dk), (e.t.float32,)).contiguous()
    grads = [_same_order(x, x.shape) if need else None for x, need in zip((q, k, v), needs)]
    d_in = e.t.empty(n, h, dv, dk, dtype=e.t.float32, device=q.device) if needs[3] else None
    ws = _scratch(e, a, 1, q.device)
    rows = [_rows(x) if x is not None else None for x in grads]
    N.check(e.attn_backward(a, _rows(d_out), _p(d_state), *rows, _p(d_in), _p(ws), ws.numel() if ws is not None else 0,
                            e.stream(q.get_device())), "hum_decay_attn_backward")
    return grads[0], grads[1], grads[2], d_in


_functions = None


def _autograd():
    """The autograd functions (torch is only imported when an operator is called)."""
    global _functions
    if _functions is not None:
        return _functions
    t = _e().t
    once = t.autograd.function.once_differentiable

    class DecayAttention(t.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v, log_decay, state, reset, lengths, scale):
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(q, k, v, log_decay, state, reset, lengths)
            ctx.scale = scale
            return _forward(q, k, v, log_decay, state, reset, lengths, scale)

        @staticmethod
        @once
        def backward(ctx, d_out, d_state):
            if d_out is None and d_state is None:
                return (None,) * 8
            q, k, v, log_decay, state, reset, lengths = ctx.saved_tensors
            if d_out is None:
                d_out = t.zeros(tuple(q.shape[:3]) + (v.shape[3],), dtype=q.dtype, device=q.device)
            n = ctx.needs_input_grad
            dq, dk, dv, ds = decay_attention_backward(d_out, d_state, q, k, v, log_decay, state, reset, lengths,
                                                      ctx.scale, (n[0], n[1], n[2], n[4]))
            return dq, dk, dv, None, ds, None, None, None

    class LayerNorm(t.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, bias, eps):
            y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
            ctx.save_for_backward(x, weight, mean, rstd)
            ctx.bias_dtype = bias.dtype if bias is not None else None
            return y

        @staticmethod
        @once
        def backward(ctx, dy):
            x, weight, mean, rstd = ctx.saved_tensors
            n = ctx.needs_input_grad
            dx, dw, db = layer_norm_backward(dy, x, mean, rstd, weight, (n[0], n[1], n[2]),
                                             weight.dtype if weight is not None else ctx.bias_dtype)
            return dx, dw, db, None

    _functions = DecayAttention, LayerNorm
    return _functions


def decay_attention(q, k, v, log_decay, state=None, reset=None, lengths=None, scale=None):
    """Whole fragments: q [lanes, steps, heads, dk], k [lanes, steps, kv_heads, dk], v [lanes, steps, kv_heads, dv] of one
    type -> (out [lanes, steps, heads, dv] of that type, final state [lanes, heads, dv, dk] float32).

    log_decay [heads] float32, <= 0: a constant schedule (decay_schedule), it has no gradient.  state: the state before
    the first step (None = zeros), contiguous float32.  reset [lanes, steps] uint8 or bool: nonzero where an episode starts,
    whatever came before is not seen from there on, also where it is not finite.  lengths [lanes] int32: steps behind a
    lane's length are not read and give zeros; the final state is the one after the last step held.  scale: default
    dk ** -0.5.  Differentiable in q, k, v and state, once and backwards."""
    e = _e()
    t = e.t
    _no_tangents(e, q, k, v, log_decay, state)
    if t.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                or (state is not None and state.requires_grad)):
        if log_decay.requires_grad:
            raise ValueError("log_decay is a constant schedule and has no gradient: pass log_decay.detach()")
        return _autograd()[0].apply(q, k, v, log_decay, state, reset, lengths, scale)
    return _forward(q, k, v, log_decay, state, reset, lengths, scale)


def decay_attention_step(q, k, v, log_decay, state, reset=None, active=None, scale=None, state_out=None, out=None):
    """One step of every lane: q [lanes, heads, dk], k [lanes, kv_heads, dk], v [lanes, kv_heads, dv], state
    [lanes, heads, dv, dk] float32 -> out [lanes, heads, dv].  The new state goes to state_out, by default into `state`
    itself.  reset [lanes] uint8 or bool: this step starts an episode; active [lanes] uint8 or bool: lanes that step
    (None = all), the others keep their state and give zeros.  out and state_out may be slices of a buffer that holds the
    inputs too, but must not overlap them (state_out may be state).  Not differentiable (the learner's pass over the
    recorded fragment is): inputs that require a gradient are refused while gradients are recorded."""
    e = _e()
    t = e.t
    if t.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (state is not None and state.requires_grad)):
        raise ValueError("decay_attention_step is not differentiable: use decay_attention, or torch.no_grad()")
    _no_tangents(e, q, k, v, log_decay, state)
    if state is None:
        raise ValueError("state is required (PolicyMemory.begin, or zeros)")
    q, k, v, log_decay, _, sizes = _check(e, q, k, v, log_decay, state, reset, None, 3)
    dev, n = q.device, sizes[0]
    if active is not None:
        active = _on(active, dev, "active", (n,), e.marks).contiguous()
    if state_out is None:
        state_out = state
    elif state_out is not state:
        _on(state_out, dev, "state_out", state.shape, (t.float32,))
        if not state_out.is_contiguous():
            raise ValueError("state_out must be contiguous")
    shape, made = (n, sizes[2], sizes[5]), out is None
    if made:
        out = t.empty_like(v) if v.shape == shape and v.is_contiguous() else t.empty(shape, dtype=q.dtype, device=dev)
    elif _unit(_on(out, dev, "out", shape, (q.dtype,))) is not out:
        raise ValueError("out must have adjacent channels")
    sq, sk, sv, so, index = q.stride(), k.stride(), v.stride(), out.stride(), q.get_device()
    a = _ATTN.pack(index, _type(e, q, "q"), *sizes, sizes[4] ** -0.5 if scale is None else float(scale), log_decay.data_ptr(),
                   q.data_ptr(), sq[0], 0, sq[1], k.data_ptr(), sk[0], 0, sk[1], v.data_ptr(), sv[0], 0, sv[1],
                   state.data_ptr(), state_out.data_ptr(), reset.data_ptr() if reset is not None else 0,
                   reset.stride(0) if reset is not None else 0, 0, 0)
    N.check(e.step(a, active.data_ptr() if active is not None else None, _ROWS.pack(out.data_ptr(), so[0], 0, so[1]),
                   e.stream(index)), "hum_decay_attn_step")
    e.written(state_out)   # (a gradient that has saved them raises)
    if not made:
        e.written(out)
    return out


# ---------------------------------------------------------------------------------------------- layer norm
def _norm_args(e, x, weight, bias, param_dtype):
    """(x as rows with adjacent channels, weight, bias, hum_norm_args)."""
    if not x.is_cuda:
        raise ValueError("x must be on a GPU (there is no CPU path)")
    c = x.shape[-1] if x.dim() else 0
    if not 1 <= c <= MAX_NORM_CHANNELS:
        raise ValueError("layer norm takes 1 to %d channels, got %s" % (MAX_NORM_CHANNELS, list(x.shape)))
    code = _type(e, x, "x")
    x2 = _unit(x if x.dim() == 2 else x.reshape(-1, c))
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("weight and bias must have one type, got %s and %s" % (weight.dtype, bias.dtype))
    index, f32 = x.get_device(), e.t.float32
    if weight is not None:
        if not (weight.dtype == f32 and weight.shape == (c,) and weight.get_device() == index):
            _on(weight, x.device, "weight", (c,), (f32, x.dtype))
        weight = weight.contiguous()
    if bias is not None:
        if not (bias.dtype == f32 and bias.shape == (c,) and bias.get_device() == index):
            _on(bias, x.device, "bias", (c,), (f32, x.dtype))
        bias = bias.contiguous()
    a = _NORM.pack(index, code, N.HUM_F32 if param_dtype == f32 else code, c, x2.shape[0], x2.stride(0),
                   x2.data_ptr(), weight.data_ptr() if weight is not None else 0)
    return x2, weight, bias, a


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, out=None, stats=True):
    """(y, mean, rstd): layer_norm without autograd and what its backward pass needs (mean, rstd [rows] float32, None
    without stats).  out: a contiguous tensor for y, x itself or one that does not overlap an input."""
    e = _e()
    t, dev = e.t, x.device
    p = weight if weight is not None else bias
    x2, weight, bias, a = _norm_args(e, x, weight, bias, p.dtype if p is not None else t.float32)
    made = out is None
    if made:
        out = t.empty_like(x) if x2 is x and x.is_contiguous() else t.empty(x.shape, dtype=x.dtype, device=dev)
    else:
        _on(out, dev, "out", x.shape, (x.dtype,))
        if not out.is_contiguous():
            raise ValueError("out must be contiguous")
    rows, c = x2.shape
    mean = t.empty(rows, dtype=t.float32, device=dev) if stats else None
    rstd = t.empty(rows, dtype=t.float32, device=dev) if stats else None
    N.check(e.norm(a, _p(bias), eps, out.data_ptr(), c, _p(mean), _p(rstd), e.stream(x.get_device())), "hum_layer_norm")
    if not made:
        e.written(out)
    return out, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight=None, needs=(True, True, True), param_dtype=None):
    """(dx, d_weight, d_bias) for the gradient dy of layer_norm's output, from its input x and the statistics
    layer_norm_forward returned.  needs: which of the three to compute (the others are None).  The parameter gradients are
    of the weight's type; without a weight they are computed only if param_dtype names their type, float32 or x's."""
    e = _e()
    t, dev = e.t, x.device
    if param_dtype is None:
        param_dtype = weight.dtype if weight is not None else None
    elif param_dtype not in (t.float32, x.dtype) or (weight is not None and param_dtype != weight.dtype):
        # (the kernel has one type for the weight and both gradients)
        raise ValueError("param_dtype must be the weight's type, without one float32 or x's, got %s" % param_dtype)
    x2, weight, _, a = _norm_args(e, x, weight, None, param_dtype if param_dtype is not None else t.float32)
    rows, c = x2.shape
    if not (dy.dtype == x.dtype and dy.shape == x.shape and dy.get_device() == x.get_device()):
        _on(dy, dev, "dy", x.shape, (x.dtype,))
    dy2 = _unit(dy if dy.dim() == 2 else dy.reshape(-1, c))
    mean = _on(mean, dev, "mean", (rows,), (t.float32,)).contiguous()
    rstd = _on(rstd, dev, "rstd", (rows,), (t.float32,)).contiguous()
    dx = dw = db = None
    if needs[0]:
        dx = t.empty_like(x) if x2 is x and x.is_contiguous() else t.empty(x.shape, dtype=x.dtype, device=dev)
    if param_dtype is not None and (needs[1] or needs[2]):
        dw, db = t.empty((2, c), dtype=param_dtype, device=dev).unbind(0)
        dw, db = dw if needs[1] else None, db if needs[2] else None
    ws, size = None, 0
    if dw is not None or db is not None:
        need = ctypes.c_uint64(0)
        N.check(e.norm_workspace(a, ctypes.byref(need)), "hum_layer_norm_workspace")
        size = need.value
        ws = t.empty(size, dtype=t.uint8, device=dev)
    N.check(e.norm_backward(a, dy2.data_ptr(), dy2.stride(0), mean.data_ptr(), rstd.data_ptr(), _p(dx), c, _p(dw), _p(db),
                            _p(ws), size, e.stream(x.get_device())), "hum_layer_norm_backward")
    return dx, dw, db


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last dimension of x (any leading shape, 1 to 16384 channels): (x - mean) / sqrt(var + eps) *
    weight + bias, sums in float32.  weight, bias: float32 or x's type, None = ones / zeros.  Differentiable in x, weight
    and bias, once and backwards; the parameter gradients have the same bits every time."""
    e = _e()
    _no_tangents(e, x, weight, bias)
    if e.t.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                  or (bias is not None and bias.requires_grad)):
        return _autograd()[1].apply(x, weight, bias, eps)
    return layer_norm_forward(x, weight, bias, eps, stats=False)[0]


# ---------------------------------------------------------------------------------------------- the core
def decay_schedule(heads, shortest=2.5, longest=8.0, device="cuda"):
    """log_decay [heads]: the heads' decays 1 - 2^-e with e evenly spread from `shortest` to `longest` - half-lives from 4
    to some 180 steps, a step's reflex to a gait's cycle."""
    t = _e().t
    return t.log1p(-t.exp2(-t.linspace(shortest, longest, heads, dtype=t.float64))).float().to(device)


class PolicyMemory:
    """The recurrent core before a policy: x + W_out norm(attend(W_qkv norm(x))) over observations x [..., n_in], so the
    policy network behind it keeps its shape.  W_out starts at zero: a fresh memory changes nothing.

    begin(n) gives n lanes' empty state, step(obs, state, reset) advances it in place (the sampler), forward(obs, state,
    reset) runs fragments [steps, lanes, n_in] and is differentiable in `parameters()` (the learner)."""

    NAMES = ("norm_weight", "norm_bias", "w_qkv", "head_weight", "head_bias", "w_out")

    def __init__(self, n_in=N.HUM_NOBS, heads=4, channels=32, device=0, seed=0, log_decay=None):
        t = _e().t
        self.device = t.device("cuda", device)
        self.n_in, self.heads, self.channels = n_in, heads, channels
        g = t.Generator().manual_seed(seed)
        w = t.randn(n_in, 3 * heads * channels, generator=g) * n_in ** -0.5
        self.norm_weight, self.norm_bias = t.ones(n_in, device=self.device), t.zeros(n_in, device=self.device)
        self.w_qkv = w.to(self.device)
        self.head_weight, self.head_bias = t.ones(channels, device=self.device), t.zeros(channels, device=self.device)
        self.w_out = t.zeros(heads * channels, n_in, device=self.device)
        self.log_decay = decay_schedule(heads, device=self.device) if log_decay is None else log_decay
        for p in self.parameters():
            p.requires_grad_(True)

    def parameters(self):
        return [getattr(self, n) for n in self.NAMES]

    def begin(self, n):
        """The empty state of n lanes [n, heads, channels, channels]."""
        t = _e().t
        return t.zeros(n, self.heads, self.channels, self.channels, dtype=t.float32, device=self.device)

    def _project(self, obs):
        if obs.shape[-1] != self.n_in:
            raise ValueError("obs must be [..., %d], got %s" % (self.n_in, list(obs.shape)))
        qkv = layer_norm(obs, self.norm_weight, self.norm_bias) @ self.w_qkv
        return qkv.view(obs.shape[:-1] + (3, self.heads, self.channels)).unbind(-3)

    def _join(self, obs, out):
        y = layer_norm(out, self.head_weight, self.head_bias)
        return obs + y.reshape(obs.shape[:-1] + (self.heads * self.channels,)) @ self.w_out

    def step(self, obs, state, reset=None, active=None):
        """Features [n, n_in] for the lanes' observations obs [n, n_in]; `state` moves on in place.  reset [n]: this step
        starts an episode (HumanoidVecEnv.episode_start(); behind a step with auto-reset its done flags); active [n]:
        lanes that step."""
        with _e().t.no_grad():
            q, k, v = self._project(obs)
            return self._join(obs, decay_attention_step(q, k, v, self.log_decay, state, reset=reset, active=active))

    def forward(self, obs, state=None, reset=None, lengths=None):
        """(features [steps, lanes, n_in], final state) for a fragment's observations obs [steps, lanes, n_in] from the
        state before its first step; reset [steps, lanes] as in step; lengths [lanes]: steps held (RLlib's seq_lens), the
        observations behind them may be anything."""
        t, seen = _e().t, obs
        if lengths is not None:   # what pads a lane passes the norm and the product, whose gradients would meet it with zeros
            _on(lengths, obs.device, "lengths", tuple(obs.shape[1:2]), (t.int32,))
            held = t.arange(obs.shape[0], device=obs.device)[:, None] < lengths
            seen = t.where(held[..., None], obs, t.zeros((), dtype=obs.dtype, device=obs.device))
        q, k, v = (x.transpose(0, 1) for x in self._project(seen))
        out, state = decay_attention(q, k, v, self.log_decay, state=state,
                                     reset=reset.transpose(0, 1) if reset is not None else None, lengths=lengths)
        return self._join(obs, out.transpose(0, 1)), state
