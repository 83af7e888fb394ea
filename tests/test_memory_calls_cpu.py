"""Calls of the policy memory's operators that are refused before anything reaches a GPU."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from ilrl_amd import _native as N  # noqa: E402
from ilrl_amd import memory as M  # noqa: E402

r = ctypes.byref


@pytest.mark.parametrize("x,weight,param", [
    (torch.bfloat16, torch.bfloat16, torch.float32), (torch.float16, torch.float16, torch.float32),
    (torch.bfloat16, torch.float32, torch.bfloat16), (torch.float16, torch.float32, torch.float16),
    (torch.bfloat16, None, torch.float16), (torch.float32, None, torch.bfloat16), (torch.float32, None, torch.float64),
    (torch.bfloat16, None, torch.int32), (torch.float32, torch.float32, torch.float64)])
def test_norm_gradient_refuses_a_parameter_type_that_is_not_the_weights(x, weight, param):
    """One type describes the weight and both of its gradients to the kernel: another one's rows would be read past their
    end or as other numbers."""
    a = torch.zeros(3, 8, dtype=x)
    w = torch.zeros(8, dtype=weight) if weight is not None else None
    with pytest.raises(ValueError, match="param_dtype"):
        M.layer_norm_backward(a, a, torch.zeros(3), torch.ones(3), w, param_dtype=param)


# ---------------------------------------------------------------------------------------------- outputs over inputs
# (addresses that nothing is at: every call here is refused)
LANES, STEPS, HEADS, D = 2, 3, 4, 8
Q, K, V, OUT, STATE, NEXT, RESET, DECAY, GRAD, SPACE = (0x1000000 * i for i in range(1, 11))


def rows(at, step=HEADS * D, head=D, lane=None):
    return N.HumRows(at, STEPS * step if lane is None else lane, step, head)


def attn(**kw):
    d = dict(device=0, type=N.HUM_F32, lanes=LANES, steps=STEPS, heads=HEADS, kv_heads=HEADS, dk=D, dv=D, scale=1.0,
             log_decay=DECAY, q=rows(Q), k=rows(K), v=rows(V), state_in=STATE, state_out=NEXT, reset=RESET, reset_lane=STEPS,
             reset_step=1)
    d.update(kw)
    return N.HumDecayAttnArgs(**d)


def refused(rc):
    assert rc == N.HUM_ERR_ARG and b"overlap" in N.lib().hum_last_error(), (rc, N.lib().hum_last_error())


SIZE, ALL = 4 * STEPS * HEADS * D * LANES, 4 * LANES * HEADS * D * D


@pytest.mark.parametrize("at", [Q, K, V, Q + SIZE - 4, V - SIZE + 4, STATE + ALL - 4, NEXT, DECAY, RESET + 4])
def test_out_that_overlaps_is_refused(at):
    """Waves that store out beside others that still read: the whole of q and k by every wave of a head."""
    L = N.lib()
    refused(L.hum_decay_attn(r(attn()), r(rows(at)), None, 0, None))
    one = dict(steps=1, q=rows(Q, lane=HEADS * D), k=rows(K, lane=HEADS * D), v=rows(V, lane=HEADS * D), reset_lane=STEPS)
    small = SIZE // STEPS
    at = {Q + SIZE - 4: Q + small - 4, V - SIZE + 4: V - small + 4, RESET + 4: RESET}.get(at, at)
    refused(L.hum_decay_attn_step(r(attn(**one)), None, r(rows(at, lane=HEADS * D)), None))
    refused(L.hum_decay_attn_step(r(attn(**one)), GRAD, r(rows(GRAD, lane=HEADS * D)), None))   # active


@pytest.mark.parametrize("at", [Q, K, V, DECAY, STATE + 4, STATE - ALL + 4])
def test_state_out_that_overlaps_is_refused(at):
    L = N.lib()
    refused(L.hum_decay_attn(r(attn(state_out=at)), r(rows(OUT)), None, 0, None))
    refused(L.hum_decay_attn_step(r(attn(steps=1, state_out=at)), None, r(rows(OUT)), None))


def test_rows_of_out_that_lie_on_each_other_are_refused():
    L = N.lib()
    for bad in (rows(OUT, head=0), rows(OUT, head=D - 1), rows(OUT, lane=0), rows(OUT, step=(HEADS - 1) * D)):
        refused(L.hum_decay_attn(r(attn()), r(bad), None, 0, None))
        refused(L.hum_decay_attn_backward(r(attn()), r(rows(GRAD)), None, r(bad), None, None, None, None, 0, None))
    refused(L.hum_decay_attn_step(r(attn(steps=1)), None, r(rows(OUT, lane=0)), None))


@pytest.mark.parametrize("at", [Q, K, V, GRAD, DECAY, STATE, NEXT])
def test_gradients_that_overlap_are_refused(at):
    L = N.lib()
    own = [rows(OUT), rows(OUT + 0x10000), rows(OUT + 0x20000)]
    for i in range(3):
        g = [rows(at) if j == i else own[j] for j in range(3)]
        refused(L.hum_decay_attn_backward(r(attn()), r(rows(GRAD)), NEXT, *map(r, g), None, None, 0, None))
        g[i] = own[i - 1]
        refused(L.hum_decay_attn_backward(r(attn()), r(rows(GRAD)), NEXT, *map(r, g), None, None, 0, None))
    refused(L.hum_decay_attn_backward(r(attn()), r(rows(GRAD)), NEXT, *map(r, own), at, None, 0, None))


def test_workspaces_that_overlap_are_refused():
    L, need = N.lib(), ctypes.c_uint64(0)
    shared = attn(kv_heads=2)
    assert L.hum_decay_attn_workspace(r(shared), 1, r(need)) == 0 and need.value
    for at in (Q, K + 16, V, GRAD, OUT, STATE, NEXT):
        refused(L.hum_decay_attn_backward(r(shared), r(rows(GRAD)), NEXT, r(rows(OUT)), None, None, None, at, need.value, None))
    long = dict(steps=1000, lanes=1)
    assert L.hum_decay_attn_workspace(r(attn(**long)), 0, r(need)) == 0 and need.value
    for at in (Q, V, STATE, NEXT, OUT):
        refused(L.hum_decay_attn(r(attn(**long)), r(rows(OUT)), at, need.value, None))


C, ROWS = 64, 5


def norm(**kw):
    d = dict(device=0, type=N.HUM_F32, param_type=N.HUM_F32, channels=C, rows=ROWS, x_row=80, x=Q, weight=K)
    d.update(kw)
    return N.HumNormArgs(**d)


# (rows of x are 64 of 80 elements wide: 4 x 16 elements lie between one row and the next)
@pytest.mark.parametrize("at,row", [(Q + 4, 80), (Q - 4, 80), (Q + 320, 80), (Q + 3 * 320, 80), (Q + 4 * 65, 96), (Q, 96), (Q, 64),
                                    (Q + 4 * 320 + 252, 64), (K, 80), (K + 252, 80), (V, 80)])
def test_norm_rows_that_overlap_are_refused(at, row):
    """Rows at another place inside x's: a workgroup would store over rows that others have yet to read."""
    L = N.lib()
    refused(L.hum_layer_norm(r(norm()), V, 1e-5, at, row, None, None, None))
    refused(L.hum_layer_norm_backward(r(norm()), V, 64, DECAY, GRAD, at, row if at != V else 80, None, None, None, 0, None))
    refused(L.hum_layer_norm_backward(r(norm(x=V, x_row=64)), Q, 80, DECAY, GRAD, at, row if at != V else 80, None, None, None, 0, None))


def test_norm_statistics_and_sums_that_overlap_are_refused():
    L, need = N.lib(), ctypes.c_uint64(0)
    for mean, rstd in ((Q, STATE), (STATE, K), (V + 4, STATE), (STATE, STATE + 16), (OUT, STATE), (STATE, OUT + 4 * 320)):
        refused(L.hum_layer_norm(r(norm()), V, 1e-5, OUT, 80, mean, rstd, None))
    assert L.hum_layer_norm_workspace(r(norm()), r(need)) == 0 and need.value
    back = lambda dw, db, space, dx=OUT: L.hum_layer_norm_backward(r(norm()), V, 64, DECAY, GRAD, dx, 80, dw, db, space, need.value, None)
    for dw, db, space in ((STATE, STATE + 252, SPACE), (OUT, STATE, SPACE), (STATE, SPACE + 64, SPACE), (STATE, NEXT, OUT), (STATE, NEXT, Q),
                          (STATE, NEXT, V + 16), (STATE, NEXT, K), (STATE, NEXT, DECAY), (STATE, NEXT, GRAD)):
        refused(back(dw, db, space))
    for dx in (DECAY, GRAD + 16, K):
        refused(back(STATE, NEXT, SPACE, dx))


# ---------------------------------------------------------------------------------------------- forward-mode derivatives
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused_not_dropped(grad):
    """No operator has a forward-mode derivative: a dual tensor raises, also where gradients are not recorded."""
    import torch.autograd.forward_ad as fwd
    x, ld = torch.randn(2, 3, 4, 8), torch.zeros(4)
    s, w = torch.randn(2, 4, 8, 8), torch.ones(8)
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        dual = lambda a: fwd.make_dual(a, torch.ones_like(a))
        for ops in ((dual(x), x, x, None), (x, dual(x), x, None), (x, x, dual(x), None), (x, x, x, dual(s))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                M.decay_attention(*ops[:3], ld, state=ops[3])
            with pytest.raises(NotImplementedError, match="forward-mode"):
                M.decay_attention_step(*(a[:, 0] for a in ops[:3]), ld, s if ops[3] is None else ops[3])
        with pytest.raises(NotImplementedError, match="forward-mode"):
            M.decay_attention(x, x, x, dual(ld))
        for ops in ((dual(x), w, w), (x, dual(w), w), (x, w, dual(w))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                M.layer_norm(*ops)
        with pytest.raises(ValueError, match="no CPU path"):
            M.layer_norm(x, w, w)   # (no tangent: refused for its device)
