"""CPU tests of the policy memory's operators: the ctypes layouts, what the C entry points and the Python front refuse
(nothing of it reaches a GPU), the tests' own float64 reference against autograd and differences."""
import ctypes
import os
import subprocess

import pytest

import memory_reference as R
from ilrl_amd import _native as N

torch = pytest.importorskip("torch")
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("cname,cls", [("hum_rows", "HumRows"), ("hum_decay_attn_args", "HumDecayAttnArgs"),
                                       ("hum_norm_args", "HumNormArgs")])
def test_struct_layouts_match_header(tmp_path, cname, cls):
    S = getattr(N, cls)
    fields = [f[0] for f in S._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "humanoid_env.h"\nint main(void){\n'
                   'printf("%%zu\\n", sizeof(%s));\n' % cname +
                   "".join('printf("%%zu\\n", offsetof(%s, %s));\n' % (cname, f) for f in fields) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)])
    out = [int(x) for x in subprocess.check_output([str(exe)]).split()]
    assert out[0] == ctypes.sizeof(S)
    for f, off in zip(fields, out[1:]):
        assert getattr(S, f).offset == off, f


def test_packed_arguments_are_the_structures():
    """memory.py packs the argument structures itself: the same bytes as the ctypes mirror's."""
    from ilrl_amd import memory as M
    rows = [N.HumRows(0x1000 * i, i, 2 * i, 3 * i) for i in (1, 2, 3)]
    a = N.HumDecayAttnArgs(1, 2, 3, 4, 5, 6, 7, 8, 0.25, 9, *rows, 10, 11, 12, 13, 14, 15)
    flat = [v for r in rows for v in (r.ptr, r.lane, r.step, r.head)]
    assert M._ATTN.pack(1, 2, 3, 4, 5, 6, 7, 8, 0.25, 9, *flat, 10, 11, 12, 13, 14, 15) == bytes(a)
    assert M._ROWS.pack(0x3000, 3, 6, 9) == bytes(rows[2])
    assert M._NORM.pack(1, 2, 3, 4, 5, 6, 7, 8) == bytes(N.HumNormArgs(1, 2, 3, 4, 5, 6, 7, 8))


def _attn(**kw):
    rows = N.HumRows(0x1000, 64, 64, 8)
    d = dict(device=0, type=N.HUM_F32, lanes=2, steps=3, heads=4, kv_heads=2, dk=8, dv=8, scale=1.0, log_decay=0x1000, q=rows,
             k=rows, v=rows)
    d.update({k: N.HumRows(*v) if isinstance(v, tuple) else v for k, v in kw.items()})
    return N.HumDecayAttnArgs(**d)


BAD = [(dict(type=3), b"element type"), (dict(lanes=-1), b">= 0"), (dict(steps=-1), b">= 0"), (dict(heads=0), b"divide"),
       (dict(kv_heads=3), b"divide"), (dict(dk=0), b"\\[1, 128\\]"), (dict(dv=129), b"\\[1, 128\\]"),
       (dict(lanes=1 << 20, heads=4), b"2\\^21"), (dict(scale=float("nan")), b"finite"), (dict(log_decay=None), b"log_decay"),
       (dict(q=(None, 0, 0, 0)), b"required"), (dict(k=(0x1002, 0, 0, 0)), b"aligned"),
       (dict(state_in=0x1002), b"aligned"), (dict(lengths=0x1001), b"aligned")]


@pytest.mark.parametrize("kw,text", BAD)
def test_attention_entry_points_refuse(kw, text):
    """The same checks stand before every attention entry point; none of them gets to a device."""
    L, out = N.lib(), N.HumRows(0x1000, 64, 64, 8)
    a = _attn(**kw)
    need = ctypes.c_uint64(0)
    r = ctypes.byref
    one = _attn(steps=1, state_out=0x1000, **{k: v for k, v in kw.items() if k not in ("steps", "lengths")}) \
        if not {"steps", "lengths"} & set(kw) else None
    calls = [lambda: L.hum_decay_attn_workspace(r(a), 1, r(need)), lambda: L.hum_decay_attn(r(a), r(out), None, 0, None),
             lambda: L.hum_decay_attn_backward(r(a), r(out), None, r(out), None, None, None, None, 0, None)]
    if one is not None:
        calls.append(lambda: L.hum_decay_attn_step(r(one), None, r(out), None))
    import re
    for c in calls:
        assert c() == N.HUM_ERR_ARG
        assert re.search(text, L.hum_last_error())


def test_attention_entry_points_refuse_their_own():
    L, out, r = N.lib(), N.HumRows(0x1000, 64, 64, 8), ctypes.byref
    none, odd = N.HumRows(None, 0, 0, 0), N.HumRows(0x1002, 0, 0, 0)
    need = ctypes.c_uint64(0)

    def refused(rc, text):
        assert rc == N.HUM_ERR_ARG and text in L.hum_last_error(), L.hum_last_error()
    refused(L.hum_decay_attn(None, r(out), None, 0, None), b"null")
    refused(L.hum_decay_attn_workspace(r(_attn()), 0, None), b"null")
    for bad in (none, odd):
        refused(L.hum_decay_attn(r(_attn()), r(bad), None, 0, None), b"out is required")
        refused(L.hum_decay_attn_backward(r(_attn()), r(bad), None, r(out), None, None, None, None, 0, None), b"d_out is required")
    refused(L.hum_decay_attn_backward(r(_attn()), r(out), 0x1002, r(out), None, None, None, None, 0, None), b"aligned")
    # shared heads need scratch
    assert L.hum_decay_attn_workspace(r(_attn()), 1, r(need)) == 0 and need.value >= 4 * 2 * 3 * 4 * 16
    refused(L.hum_decay_attn_backward(r(_attn()), r(out), None, r(out), r(out), r(out), None, None, 0, None), b"workspace")
    refused(L.hum_decay_attn_backward(r(_attn()), r(out), None, r(out), r(out), r(out), None, 0x2008, need.value, None), b"workspace")
    # the state's gradient may overlap neither the state nor its own incoming gradient
    own = _attn(kv_heads=4, state_in=0x100000)
    size = 4 * 2 * 4 * 8 * 8
    for at in (0x100000, 0x100000 + size - 4, 0x100000 - size + 4):
        refused(L.hum_decay_attn_backward(r(own), r(out), None, None, None, None, at, None, 0, None), b"overlap")
        refused(L.hum_decay_attn_backward(r(_attn(kv_heads=4)), r(out), 0x100000, None, None, None, at, None, 0, None), b"overlap")
    refused(L.hum_decay_attn_step(r(_attn()), None, r(out), None), b"steps must be 1")
    refused(L.hum_decay_attn_step(r(_attn(steps=1)), None, r(out), None), b"state_out")
    refused(L.hum_decay_attn_step(r(_attn(steps=1, state_out=0x1000, lengths=0x1000)), None, r(out), None), b"lengths NULL")
    # nothing to do is no error
    assert L.hum_decay_attn(r(_attn(lanes=0)), r(none), None, 0, None) == 0
    assert L.hum_decay_attn_step(r(_attn(lanes=0, steps=1)), None, r(none), None) == 0


def _norm(**kw):
    d = dict(device=0, type=N.HUM_BF16, param_type=N.HUM_F32, channels=64, rows=4, x_row=64, x=0x1000, weight=0x2000)
    d.update(kw)
    return N.HumNormArgs(**d)


def test_norm_entry_points_refuse():
    L, r = N.lib(), ctypes.byref
    need = ctypes.c_uint64(0)

    def refused(rc, text):
        assert rc == N.HUM_ERR_ARG and text in L.hum_last_error(), L.hum_last_error()

    def both(a, text):
        refused(L.hum_layer_norm(r(a) if a else None, None, 1e-5, 0x3000, 64, None, None, None), text)
        refused(L.hum_layer_norm_backward(r(a) if a else None, 0x3000, 64, 0x4000, 0x4000, 0x3000, 64, None, None, None, 0, None), text)
        refused(L.hum_layer_norm_workspace(r(a) if a else None, r(need)), text)
    both(None, b"null")
    both(_norm(type=5), b"element type")
    both(_norm(param_type=N.HUM_F16), b"parameters")
    both(_norm(rows=-1), b"rows must be")
    both(_norm(channels=0), b"channels in")
    both(_norm(channels=16385), b"channels in")
    both(_norm(x=None), b"x is required")
    both(_norm(x=0x1001), b"aligned")
    both(_norm(weight=0x2002), b"aligned")
    a = _norm()
    refused(L.hum_layer_norm(r(a), None, 1e-5, None, 64, None, None, None), b"y is required")
    refused(L.hum_layer_norm(r(a), None, 1e-5, 0x3000, 64, 0x4000, None, None), b"together")
    refused(L.hum_layer_norm(r(a), 0x2002, 1e-5, 0x3000, 64, None, None, None), b"aligned")
    for eps in (-1e-5, float("nan"), float("inf")):
        refused(L.hum_layer_norm(r(a), None, eps, 0x3000, 64, None, None, None), b"eps")
    refused(L.hum_layer_norm_backward(r(a), None, 64, 0x4000, 0x4000, 0x3000, 64, None, None, None, 0, None), b"required")
    refused(L.hum_layer_norm_backward(r(a), 0x3000, 64, 0x4000, None, 0x3000, 64, None, None, None, 0, None), b"required")
    refused(L.hum_layer_norm_backward(r(a), 0x3000, 64, 0x4000, 0x4000, 0x3000, 64, 0x5000, None, None, 0, None), b"workspace")
    assert L.hum_layer_norm_workspace(r(a), r(need)) == 0 and need.value >= 2 * 64 * 4
    refused(L.hum_layer_norm_backward(r(a), 0x3000, 64, 0x4000, 0x4000, 0x3000, 64, 0x5000, None, 0x6000, need.value - 1, None), b"workspace")
    refused(L.hum_layer_norm_backward(r(a), 0x3000, 64, 0x4000, 0x4000, 0x3000, 64, 0x5000, None, 0x6008, need.value, None), b"workspace")
    assert L.hum_layer_norm(r(_norm(rows=0, x=None)), None, 1e-5, None, 64, None, None, None) == 0


def test_outputs_that_overlap_what_is_still_read():
    L, r, out = N.lib(), ctypes.byref, N.HumRows(0x1000, 64, 64, 8)

    def refused(rc, text):
        assert rc == N.HUM_ERR_ARG and text in L.hum_last_error(), L.hum_last_error()
    size = 4 * 2 * 4 * 8 * 8
    for at in (0x100004, 0x100000 + size - 4, 0x100000 - size + 4):
        refused(L.hum_decay_attn(r(_attn(state_in=0x100000, state_out=at)), r(out), None, 0, None), b"overlap")
        refused(L.hum_decay_attn_step(r(_attn(steps=1, state_in=0x100000, state_out=at)), None, r(out), None), b"overlap")
    a = _norm(x_row=80)
    for y, row in ((0x1000, 64), (0x1000, 96), (0x9000, 63), (0x9000, 0), (0x9000, -63)):
        refused(L.hum_layer_norm(r(a), None, 1e-5, y, row, None, None, None), b"overlap")
        refused(L.hum_layer_norm_backward(r(a), 0x5000, 64, 0x4000, 0x4000, y, row, None, None, None, 0, None), b"overlap")
    refused(L.hum_layer_norm_backward(r(a), 0x5000, 64, 0x4000, 0x4000, 0x5000, 80, None, None, None, 0, None), b"overlap")


def test_front_refuses_cpu_tensors():
    from ilrl_amd import memory as M
    x = torch.zeros(2, 3, 4, 8)
    ld = torch.zeros(4)
    with pytest.raises(ValueError, match="no CPU path"):
        M.decay_attention(x, x, x, ld)
    with pytest.raises(ValueError, match="no CPU path"):
        M.decay_attention_step(x[:, 0], x[:, 0], x[:, 0], ld, torch.zeros(2, 4, 8, 8))
    with pytest.raises(ValueError, match="no CPU path"):
        M.layer_norm(x)
    with pytest.raises(ValueError, match="no gradient"):
        M.decay_attention(x.requires_grad_(True), x, x, ld.requires_grad_(True))


def _case(seed, b=2, s=9, h=4, g=2, dk=5, dv=3):
    r = torch.Generator().manual_seed(seed)

    def n(*shape):
        return torch.randn(*shape, generator=r, dtype=torch.float64)
    reset = (torch.rand(b, s, generator=r) < 0.25).to(torch.uint8)
    lengths = torch.tensor([s, s - 4], dtype=torch.int32)
    return n(b, s, h, dk), n(b, s, g, dk), n(b, s, g, dv), -torch.rand(h, generator=r), n(b, h, dv, dk), reset, lengths, n(b, s, h, dv), n(b, h, dv, dk)


def test_reference_gradient_is_the_forward_pass_derivative():
    """The reference's gradient formula against central differences of its forward pass.  The outputs are multilinear in
    (q, k, v, state): along one of them the difference quotient is exact, so only float64 rounding remains."""
    q, k, v, ld, state, reset, lengths, d_out, d_state = _case(0)
    grads = R.attention_grad(d_out, d_state, q, k, v, ld, state, reset, lengths, 0.7)
    for i, (x, g) in enumerate(zip((q, k, v, state), grads)):
        step = torch.randn(x.shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        ops = [q, k, v, state]
        vals = []
        for sign in (1, -1):
            ops[i] = x + sign * step
            out, S = R.attention(ops[0], ops[1], ops[2], ld, ops[3], reset, lengths, 0.7)
            vals.append((out * d_out).sum() + (S * d_state).sum())
        assert abs((vals[0] - vals[1]) / 2 - (g * step).sum()) < 1e-10


def test_reference_norm_gradient_matches_autograd():
    r = torch.Generator().manual_seed(3)
    x = torch.randn(6, 11, generator=r, dtype=torch.float64, requires_grad=True)
    w = torch.randn(11, generator=r, dtype=torch.float64, requires_grad=True)
    b = torch.randn(11, generator=r, dtype=torch.float64, requires_grad=True)
    dy = torch.randn(6, 11, generator=r, dtype=torch.float64)
    torch.nn.functional.layer_norm(x, (11,), w, b, 1e-5).backward(dy)
    xd = x.detach()
    dx, dw, db = R.norm_grad(dy, xd, xd.mean(-1), torch.rsqrt(xd.var(-1, unbiased=False) + 1e-5), w.detach())
    for a, e in ((dx, x.grad), (dw, w.grad), (db, b.grad)):
        assert (a - e).abs().max() < 1e-12
    assert (R.norm(xd, w.detach(), b.detach(), 1e-5) - torch.nn.functional.layer_norm(xd, (11,), w.detach(), b.detach(), 1e-5)).abs().max() < 1e-12
