"""Layer norm and its gradient at every shape of its kernels (threads a row, channels a thread) with rows of 16-byte units
and without, and over enough rows that workgroups take several and their partial sums are joined.  Bounds as in
tests/test_gpu_memory.py: 64 float32 roundings on the way to each sum (24 channels a thread or 16, 6 exchanges in a wave, 16
waves, some rows a workgroup)."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a HIP device", allow_module_level=True)

import memory_reference as R  # noqa: E402
from ilrl_amd import memory as M  # noqa: E402
from test_gpu_memory import HALF, TYPES, U, norm_bounds  # noqa: E402


def check(x, dy, w, b, kind):
    y, mean, rstd = M.layer_norm_forward(x, w, b)
    want = R.norm(x, w, b, 1e-5)
    assert ((y.double().cpu() - want).abs() <= norm_bounds(x, w, b, want, kind)).all()
    dx, dw, db = M.layer_norm_backward(dy, x, mean, rstd, w)
    wx, ww, wb = R.norm_grad(dy, x, mean, rstd, w)
    r, d = rstd.double().cpu()[:, None], dy.double().cpu().abs()
    h = ((x.double().cpu() - mean.double().cpu()[:, None]) * r).abs()
    g = d * w.double().cpu().abs()
    size = r * (g + g.mean(-1, keepdim=True) + h * (g * h).mean(-1, keepdim=True))
    tiny = lambda t: 2.0 ** -25 if t == torch.float16 else 0
    assert ((dx.double().cpu() - wx).abs() <= HALF[kind] * wx.abs() * 1.01 + 64 * U * size + tiny(x.dtype)).all()
    half = torch.finfo(w.dtype).eps / 2
    assert ((dw.double().cpu() - ww).abs() <= half * ww.abs() * 1.01 + 64 * U * (d * h).sum(0) + tiny(w.dtype)).all()
    assert ((db.double().cpu() - wb).abs() <= half * wb.abs() * 1.01 + 64 * U * d.sum(0) + tiny(w.dtype)).all()
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), M.layer_norm_backward(dy, x, mean, rstd, w)))
    # fewer results, the same bits
    assert torch.equal(M.layer_norm_backward(dy, x, mean, rstd, w, (True, False, False))[0], dx)
    assert torch.equal(M.layer_norm_backward(dy, x, mean, rstd, w, (False, False, True))[2], db)


WIDTHS = [8, 40, 64, 120, 128, 200, 256, 264, 512, 520, 1000, 1024, 1032, 1280, 1536, 1544, 2048, 2056, 4096, 4104, 8192, 8200, 12000, 16384]
ODD = [7, 63, 65, 129, 257, 511, 513, 1023, 1025, 1111, 1535, 1537, 2047, 2049, 4095, 4097, 8191, 8193, 12001, 16383]


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("wide", ["rows", "params"])
@pytest.mark.parametrize("c,pitch", [(c, c) for c in WIDTHS] + [(c, c + 8) for c in (64, 512, 1280, 16384)] +
                         [(c, c + 5) for c in (64, 512, 1024, 1280, 2048, 4096, 8192, 16384)] + [(c, c) for c in ODD] + [(1111, 1148)])
def test_every_shape(c, pitch, wide, kind):
    rows = 45 if c <= 2048 else 7
    r = torch.Generator().manual_seed(c + pitch)
    dt = TYPES[kind]
    x = (torch.randn(rows, pitch, generator=r) * 2 + 0.7).to(dt).cuda()[:, :c]
    dy = torch.randn(rows, pitch, generator=r).to(dt).cuda()[:, :c]
    pd = dt if wide == "rows" else torch.float32
    w, b = torch.randn(c, generator=r).to(pd).cuda(), torch.randn(c, generator=r).to(pd).cuda()
    check(x, dy, w, b, kind)


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("rows,c,pitch", [(5000, 64, 64), (3001, 70, 70), (3000, 264, 264), (3000, 512, 517), (2500, 1024, 1024), (2500, 1111, 1148),
                                          (2500, 1280, 1280), (700, 2048, 2048), (700, 2500, 2500), (600, 8192, 8192), (600, 9000, 9000)])
def test_rows_that_workgroups_share(rows, c, pitch, kind):
    """More rows than the gradient has groups of threads for: several turns a workgroup, hundreds of partial rows."""
    r = torch.Generator().manual_seed(rows + c)
    dt = TYPES[kind]
    x = (torch.randn(rows, pitch, generator=r) * 2 + 0.7).to(dt).cuda()[:, :c]
    dy = torch.randn(rows, pitch, generator=r).to(dt).cuda()[:, :c]
    check(x, dy, torch.randn(c, generator=r).cuda(), torch.randn(c, generator=r).cuda(), kind)


@pytest.mark.parametrize("kind", ["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("c", [70, 512, 1024, 1111, 1280, 16384])
def test_rows_and_parameters_that_begin_anywhere(c, kind):
    """Cut out of buffers of NaN at an element's alignment."""
    r = torch.Generator().manual_seed(c)
    dt = TYPES[kind]

    def cut(*lead, type=dt):
        wide = torch.full((*lead, c + 3), float("nan"), dtype=type, device="cuda")
        wide[..., 1:1 + c] = torch.randn((*lead, c), generator=r).to(type)
        return wide[..., 1:1 + c]
    for pd in (torch.float32, dt):
        check(cut(45), cut(45), cut(type=pd), cut(type=pd), kind)
