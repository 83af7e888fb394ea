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

from . import _native as N

MAX_HEAD_CHANNELS, MAX_NORM_CHANNELS = 128, 16384


def _torch():
    import torch
    return torch


_TYPES = None


def _type(x, what):
    global _TYPES
    if _TYPES is None:
        t = _torch()
        _TYPES = {t.float32: N.HUM_F32, t.bfloat16: N.HUM_BF16, t.float16: N.HUM_F16}
    code = _TYPES.get(x.dtype)
    if code is None:
        raise ValueError("%s: float32, bfloat16 or float16, got %s" % (what, x.dtype))
    return code


def _p(x):
    return x.data_ptr() if x is not None else None


def _stream(device):
    return _torch().cuda.current_stream(device).cuda_stream


def _unit(x):
    """x with adjacent channels."""
    return x if x.stride(-1) == 1 or x.shape[-1] <= 1 else x.contiguous()


def _rows(x):
    return N.HumRows(x.data_ptr(), x.stride(0), x.stride(1), x.stride(2))


def _same_order(like, shape):
    """An empty [lanes, steps, ...] tensor in `like`'s memory order (time-major where its steps are the outer axis)."""
    t = _torch()
    if like.stride(0) < like.stride(1):
        return t.empty((shape[1], shape[0]) + shape[2:], dtype=like.dtype, device=like.device).transpose(0, 1)
    return t.empty(shape, dtype=like.dtype, device=like.device)


def _on(x, device, what, shape=None, dtypes=None):
    if x.device != device:
        raise ValueError("%s is on %s, expected %s" % (what, x.device, device))
    if shape is not None and tuple(x.shape) != shape:
        raise ValueError("%s must be %s, got %s" % (what, list(shape), list(x.shape)))
    if dtypes is not None and x.dtype not in dtypes:
        raise ValueError("%s must be of type %s, got %s" % (what, " or ".join(str(d) for d in dtypes), x.dtype))
    return x


def _check(q, k, v, log_decay, state, reset, lengths):
    """The operands of a fragment as (q, k, v with adjacent channels, HumDecayAttnArgs); [lanes, steps, ...]."""
    t = _torch()
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k, v must be [lanes, steps, heads, channels], got %s, %s, %s"
                         % (list(q.shape), list(k.shape), list(v.shape)))
    if not q.is_cuda:
        raise ValueError("q must be on a GPU (there is no CPU path)")
    b, s, h, dk = q.shape
    g, dv = k.shape[2], v.shape[3]
    _on(k, q.device, "k", (b, s, g, dk), (q.dtype,))
    _on(v, q.device, "v", (b, s, g, dv), (q.dtype,))
    if g < 1 or h % g:
        raise ValueError("%d key / value heads cannot be shared evenly by %d query heads" % (g, h))
    if not (1 <= dk <= MAX_HEAD_CHANNELS and 1 <= dv <= MAX_HEAD_CHANNELS):
        raise ValueError("1 to %d channels a head, got %d (keys) and %d (values)" % (MAX_HEAD_CHANNELS, dk, dv))
    _on(log_decay, q.device, "log_decay", (h,), (t.float32,))
    if log_decay.requires_grad:
        raise ValueError("log_decay is a constant schedule and has no gradient: pass log_decay.detach()")
    if not log_decay.is_contiguous():
        log_decay = log_decay.contiguous()
    if state is not None:
        _on(state, q.device, "state", (b, h, dv, dk), (t.float32,))
        if not state.is_contiguous():
            raise ValueError("state must be contiguous")
    if reset is not None:
        _on(reset, q.device, "reset", (b, s), (t.uint8, t.bool))
    if lengths is not None:
        _on(lengths, q.device, "lengths", (b,), (t.int32,))
        lengths = lengths.contiguous()
    q, k, v = _unit(q), _unit(k), _unit(v)
    a = N.HumDecayAttnArgs(q.device.index, _type(q, "q"), b, s, h, g, dk, dv, 0.0, log_decay.data_ptr(), _rows(q),
                           _rows(k), _rows(v), _p(state), None, _p(reset), 0, 0, _p(lengths))
    if reset is not None:
        a.reset_lane, a.reset_step = reset.stride(0), reset.stride(1)
    return q, k, v, log_decay, lengths, a


def _scratch(a, backward, device):
    need = ctypes.c_uint64(0)
    N.check(N.lib().hum_decay_attn_workspace(ctypes.byref(a), backward, ctypes.byref(need)), "hum_decay_attn_workspace")
    if not need.value:
        return None
    t = _torch()
    return t.empty(need.value, dtype=t.uint8, device=device)


def _forward(q, k, v, log_decay, state, reset, lengths, scale):
    t = _torch()
    q, k, v, log_decay, lengths, a = _check(q, k, v, log_decay, state, reset, lengths)
    a.scale = q.shape[3] ** -0.5 if scale is None else float(scale)
    out = _same_order(q, tuple(q.shape[:3]) + (v.shape[3],))
    state_out = t.empty(q.shape[0], q.shape[2], v.shape[3], q.shape[3], dtype=t.float32, device=q.device)
    a.state_out = state_out.data_ptr()
    ws = _scratch(a, 0, q.device)
    N.check(N.lib().hum_decay_attn(ctypes.byref(a), ctypes.byref(_rows(out)), _p(ws), ws.numel() if ws is not None else 0,
                                   _stream(q.device)), "hum_decay_attn")
    return out, state_out


def decay_attention_backward(d_out, d_state, q, k, v, log_decay, state=None, reset=None, lengths=None, scale=None,
                             needs=(True, True, True, True)):
    """(dq, dk, dv, d_state_in) of decay_attention for the gradients d_out [lanes, steps, heads, dv] of its output and
    d_state [lanes, heads, dv, dk] of its final state (None = zeros), from the same inputs.  needs: which of the four to
    compute (the others are None)."""
    t = _torch()
    q, k, v, log_decay, lengths, a = _check(q, k, v, log_decay, state, reset, lengths)
    a.scale = q.shape[3] ** -0.5 if scale is None else float(scale)
    d_out = _unit(_on(d_out, q.device, "d_out", tuple(q.shape[:3]) + (v.shape[3],), (q.dtype,)))
    sshape = (q.shape[0], q.shape[2], v.shape[3], q.shape[3])
    if d_state is not None:
        d_state = _on(d_state, q.device, "d_state", sshape, (t.float32,)).contiguous()
    grads = [_same_order(x, tuple(x.shape)) if need else None for x, need in zip((q, k, v), needs)]
    d_in = t.empty(sshape, dtype=t.float32, device=q.device) if needs[3] else None
    ws = _scratch(a, 1, q.device)
    rows = [ctypes.byref(_rows(x)) if x is not None else None for x in grads]
    N.check(N.lib().hum_decay_attn_backward(ctypes.byref(a), ctypes.byref(_rows(d_out)), _p(d_state), *rows, _p(d_in),
                                            _p(ws), ws.numel() if ws is not None else 0, _stream(q.device)),
            "hum_decay_attn_backward")
    return grads[0], grads[1], grads[2], d_in


_functions = None


def _autograd():
    """The autograd functions (torch is only imported when an operator is called)."""
    global _functions
    if _functions is not None:
        return _functions
    t = _torch()
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
    dk ** -0.5.  Differentiable in q, k, v and state."""
    t = _torch()
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
    (None = all), the others keep their state and give zeros.  Not differentiable (the learner's pass over the recorded
    fragment is): inputs that require a gradient are refused while gradients are recorded."""
    t = _torch()
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k, v must be [lanes, heads, channels], got %s, %s, %s" % (list(q.shape), list(k.shape), list(v.shape)))
    if t.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, state)):
        raise ValueError("decay_attention_step is not differentiable: use decay_attention, or torch.no_grad()")
    n = q.shape[0]
    if reset is not None and reset.dim() != 1:
        raise ValueError("reset must be [%d], got %s" % (n, list(reset.shape)))
    if state is None:
        raise ValueError("state is required (PolicyMemory.begin, or zeros)")
    q4, k4, v4, log_decay, _, a = _check(q[:, None], k[:, None], v[:, None], log_decay, state,
                                         reset[:, None] if reset is not None else None, None)
    a.scale = q.shape[2] ** -0.5 if scale is None else float(scale)
    if active is not None:
        active = _on(active, q.device, "active", (n,), (t.uint8, t.bool)).contiguous()
    if state_out is None:
        state_out = state
    elif state_out is not state:
        _on(state_out, q.device, "state_out", tuple(state.shape), (t.float32,))
        if not state_out.is_contiguous():
            raise ValueError("state_out must be contiguous")
    a.state_out = state_out.data_ptr()
    shape = (n, q.shape[1], v.shape[2])
    if out is None:
        out = t.empty(shape, dtype=q.dtype, device=q.device)
    elif _unit(_on(out, q.device, "out", shape, (q.dtype,))) is not out:
        raise ValueError("out must have adjacent channels")
    N.check(N.lib().hum_decay_attn_step(ctypes.byref(a), _p(active),
                                        ctypes.byref(N.HumRows(out.data_ptr(), out.stride(0), 0, out.stride(1))),
                                        _stream(q.device)), "hum_decay_attn_step")
    return out


# ---------------------------------------------------------------------------------------------- layer norm
def _norm_args(x, weight, param_dtype):
    t = _torch()
    if not x.is_cuda:
        raise ValueError("x must be on a GPU (there is no CPU path)")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_NORM_CHANNELS:
        raise ValueError("layer norm takes 1 to %d channels, got %s" % (MAX_NORM_CHANNELS, list(x.shape)))
    c = x.shape[-1]
    x2 = _unit(x.reshape(-1, c))
    if weight is not None:
        _on(weight, x.device, "weight", (c,), (t.float32, x.dtype))
        weight = weight.contiguous()
    a = N.HumNormArgs(x.device.index, _type(x, "x"), N.HUM_F32 if param_dtype == t.float32 else _type(x, "x"), c, x2.shape[0],
                      x2.stride(0), x2.data_ptr(), _p(weight))
    return x2, weight, a


def layer_norm_forward(x, weight=None, bias=None, eps=1e-5, out=None, stats=True):
    """(y, mean, rstd): layer_norm without autograd and what its backward pass needs (mean, rstd [rows] float32, None
    without stats)."""
    t = _torch()
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError("weight and bias must have one type, got %s and %s" % (weight.dtype, bias.dtype))
    p = weight if weight is not None else bias
    x2, weight, a = _norm_args(x, weight, p.dtype if p is not None else t.float32)
    if bias is not None:
        bias = _on(bias, x.device, "bias", (x.shape[-1],), (t.float32, x.dtype)).contiguous()
    if out is None:
        out = t.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        _on(out, x.device, "out", tuple(x.shape), (x.dtype,))
        if not out.is_contiguous():
            raise ValueError("out must be contiguous")
    rows, c = x2.shape
    mean = t.empty(rows, dtype=t.float32, device=x.device) if stats else None
    rstd = t.empty(rows, dtype=t.float32, device=x.device) if stats else None
    N.check(N.lib().hum_layer_norm(ctypes.byref(a), _p(bias), eps, out.data_ptr(), c, _p(mean), _p(rstd), _stream(x.device)),
            "hum_layer_norm")
    return out, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, weight=None, needs=(True, True, True), param_dtype=None):
    """(dx, d_weight, d_bias) for the gradient dy of layer_norm's output, from its input x and the statistics
    layer_norm_forward returned.  needs: which of the three to compute (the others are None).  Without a weight the
    parameter gradients are computed only if param_dtype names their type."""
    t = _torch()
    if param_dtype is None:
        param_dtype = weight.dtype if weight is not None else None
    x2, weight, a = _norm_args(x, weight, param_dtype if param_dtype is not None else t.float32)
    rows, c = x2.shape
    dy2 = _unit(_on(dy, x.device, "dy", tuple(x.shape), (x.dtype,)).reshape(-1, c))
    _on(mean, x.device, "mean", (rows,), (t.float32,))
    _on(rstd, x.device, "rstd", (rows,), (t.float32,))
    mean, rstd = mean.contiguous(), rstd.contiguous()
    dx = t.empty(x.shape, dtype=x.dtype, device=x.device) if needs[0] else None
    dw = t.empty(c, dtype=param_dtype, device=x.device) if needs[1] and param_dtype is not None else None
    db = t.empty(c, dtype=param_dtype, device=x.device) if needs[2] and param_dtype is not None else None
    ws, size = None, 0
    if dw is not None or db is not None:
        need = ctypes.c_uint64(0)
        N.check(N.lib().hum_layer_norm_workspace(ctypes.byref(a), ctypes.byref(need)), "hum_layer_norm_workspace")
        size = need.value
        ws = t.empty(size, dtype=t.uint8, device=x.device)
    N.check(N.lib().hum_layer_norm_backward(ctypes.byref(a), dy2.data_ptr(), dy2.stride(0), mean.data_ptr(), rstd.data_ptr(),
                                            _p(dx), c, _p(dw), _p(db), _p(ws), size, _stream(x.device)),
            "hum_layer_norm_backward")
    return dx, dw, db


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last dimension of x (any leading shape, 1 to 16384 channels): (x - mean) / sqrt(var + eps) *
    weight + bias, sums in float32.  weight, bias: float32 or x's type, None = ones / zeros.  Differentiable in x, weight
    and bias; the parameter gradients have the same bits every time."""
    t = _torch()
    if t.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                or (bias is not None and bias.requires_grad)):
        return _autograd()[1].apply(x, weight, bias, eps)
    return layer_norm_forward(x, weight, bias, eps, stats=False)[0]


# ---------------------------------------------------------------------------------------------- the core
def decay_schedule(heads, shortest=2.5, longest=8.0, device="cuda"):
    """log_decay [heads]: the heads' decays 1 - 2^-e with e evenly spread from `shortest` to `longest` - half-lives from 4
    to some 180 steps, a step's reflex to a gait's cycle."""
    t = _torch()
    return t.log1p(-t.exp2(-t.linspace(shortest, longest, heads, dtype=t.float64))).float().to(device)


class PolicyMemory:
    """The recurrent core before a policy: x + W_out norm(attend(W_qkv norm(x))) over observations x [..., n_in], so the
    policy network behind it keeps its shape.  W_out starts at zero: a fresh memory changes nothing.

    begin(n) gives n lanes' empty state, step(obs, state, reset) advances it in place (the sampler), forward(obs, state,
    reset) runs fragments [steps, lanes, n_in] and is differentiable in `parameters()` (the learner)."""

    NAMES = ("norm_weight", "norm_bias", "w_qkv", "head_weight", "head_bias", "w_out")

    def __init__(self, n_in=N.HUM_NOBS, heads=4, channels=32, device=0, seed=0, log_decay=None):
        t = _torch()
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
        t = _torch()
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
        starts an episode (the previous step's done flags); active [n]: lanes that step."""
        with _torch().no_grad():
            q, k, v = self._project(obs)
            return self._join(obs, decay_attention_step(q, k, v, self.log_decay, state, reset=reset, active=active))

    def forward(self, obs, state=None, reset=None, lengths=None):
        """(features [steps, lanes, n_in], final state) for a fragment's observations obs [steps, lanes, n_in] from the
        state before its first step; reset [steps, lanes] as in step; lengths [lanes]: steps held (RLlib's seq_lens)."""
        q, k, v = (x.transpose(0, 1) for x in self._project(obs))
        out, state = decay_attention(q, k, v, self.log_decay, state=state,
                                     reset=reset.transpose(0, 1) if reset is not None else None, lengths=lengths)
        return self._join(obs, out.transpose(0, 1)), state
