"""Weight gradients from rows in 8 bits against float64. Every product is exact. A chain of the tensor core's additions (16 rows
each, at most 1024 rows, three instructions per 16 rows for fp32) cuts off at most 2^-22 of what it has added so far, and every
later fp32 addition rounds by 2^-24: with S the sum of the products' absolute values at most (3 * 64 * 2^-22 + (m / 512 + 160) *
2^-24) * S, below 2^-14 * S for the sizes here. For a dy of few columns every addition rounds by 2^-24, and an element goes through
at most 8 * 1.7 in its lane, 40 in its block and 600 between blocks: less than 2^-14 too."""
import pytest
import torch

from helpers import randn
from rows8_ref import held_values

pytestmark = pytest.mark.gpu

BOUND = 2.0 ** -14


def _close(got, want, mag):
    return bool(((got.double().cpu() - want).abs() <= BOUND * mag + 1e-300).all())


def _inputs(m, k, n, dtype, seed=0):
    x = randn((m, k), seed + 1).clamp(min=0).to(dtype)
    dy = (randn((m, n), seed + 2) * torch.exp2(randn((m, 1), seed + 3) * 4)).to(dtype)
    return x, dy


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (5, 32, 8), (63, 47, 47), (64, 64, 64), (65, 100, 65), (200, 128, 128), (1000, 33, 200),
                                   (3000, 257, 130), (20000, 100, 47), (40000, 16, 300), (500, 40, 50), (500, 40, 100),
                                   (300, 64, 180), (1000, 20, 16), (255, 7, 11), (3000, 33, 7), (257, 64, 8), (700, 90, 3),
                                   (20000, 128, 4), (100000, 32, 1), (70000, 50, 2), (60000, 10, 13)])
def test_weight_grad(cuda, m, k, n, dtype):
    import cxgnncomp_backend as be
    x, dy = _inputs(m, k, n, dtype, m)
    rows = be.quantize_rows(x.cuda())
    dw, db = be.rows8_weight_grad(rows, dy.cuda(), bias=True)
    assert dw.shape == (n, k) and dw.dtype == torch.float32 and db.shape == (n,)
    v, g = be.dequantize_rows(rows).double().cpu(), dy.double()  # the values themselves are tested elsewhere
    assert _close(dw, g.t() @ v, g.t().abs() @ v.abs())
    assert _close(db, g.sum(0), g.abs().sum(0))
    assert torch.equal(dw, be.rows8_weight_grad(rows, dy.cuda()))
    be.check_device_status("linear")


def test_all_bits_of_fp32_gradients_count(cuda):
    """One row: the gradient is a single product per element, exact in fp32 but for its own rounding."""
    import cxgnncomp_backend as be
    x = torch.full((1, 32), 127.0)
    x[0, 5] = 1.0
    dy = randn((1, 64), 3)
    dw = be.rows8_weight_grad(be.quantize_rows(x.cuda()), dy.cuda())
    want = dy.double().t() @ held_values(x)
    # three exact products of 15 bits, added with at most 2^-22 of the sum cut off
    assert bool(((dw.double().cpu() - want).abs() <= 2.0 ** -22 * want.abs()).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k,n", [(40, 70), (30, 8), (100, 4), (60, 7)])
def test_gradients_that_are_not_finite_and_large(cuda, k, n, dtype):
    import cxgnncomp_backend as be
    x, dy = _inputs(300, k, n, dtype)
    x[:, 3] = 1.0
    dy[7, 3] = float("inf")
    dy[9, 1] = float("nan")
    dy[11, 2] = torch.finfo(dtype).max / 256
    rows = be.quantize_rows(x.cuda())
    dw, db = be.rows8_weight_grad(rows, dy.cuda(), bias=True)
    v, g = be.dequantize_rows(rows).double().cpu(), dy.double()
    want = g.t() @ v
    assert torch.equal(torch.isnan(dw.cpu()), torch.isnan(want)) and torch.equal(torch.isinf(dw.cpu()), torch.isinf(want))
    keep = torch.isfinite(want)
    mag = torch.nan_to_num(g.abs(), 0.0, 0.0).t() @ v.abs()
    assert bool(((dw.double().cpu() - want).abs() <= BOUND * mag)[keep].all())
    assert bool(torch.isinf(db[3])) and bool(torch.isnan(db[1]))


def test_rows_that_are_not_finite(cuda):
    import cxgnncomp_backend as be
    x, dy = _inputs(100, 96, 20, torch.float32)
    x[50, 40] = float("nan")
    dw = be.rows8_weight_grad(be.quantize_rows(x.cuda()), dy.cuda())
    assert bool(torch.isnan(dw[:, 32:64]).all()) and not bool(torch.isnan(dw[:, :32]).any()) and not bool(torch.isnan(dw[:, 64:]).any())


@pytest.mark.parametrize("k,n", [(40, 70), (30, 8), (100, 3)])
@pytest.mark.parametrize("size", [1e35, 1e-34])
def test_rows_of_any_magnitude(cuda, k, n, size):
    import cxgnncomp_backend as be
    x, dy = _inputs(300, k, n, torch.float32)
    x *= size
    dy /= dy.abs().max()
    rows = be.quantize_rows(x.cuda())
    v, g = be.dequantize_rows(rows).double().cpu(), dy.double()
    got = be.rows8_weight_grad(rows, dy.cuda())
    # (small operands of the tensor cores lose bits below 2^-133)
    assert _close(got, g.t() @ v, g.t().abs() @ v.abs() + 300 * 2.0 ** -133 / BOUND)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_few_columns_anywhere(cuda, dtype):
    """In a wider matrix, and behind an odd start."""
    import cxgnncomp_backend as be
    x, wide = _inputs(500, 48, 24, dtype)
    rows = be.quantize_rows(x.cuda())
    v = be.dequantize_rows(rows).double().cpu()
    flat = torch.zeros(1 + 500 * 5, dtype=dtype)
    flat[1:] = wide[:, :5].reshape(-1)
    for g, on_gpu in ((wide[:, 3:10], wide.cuda()[:, 3:10]), (wide[:, :5], flat.cuda()[1:].view(500, 5)),
                      (wide[:77, :1], wide.cuda()[:77, :1])):
        dw, db = be.rows8_weight_grad(rows, on_gpu, bias=True)
        assert _close(dw, g.double().t() @ v[:g.shape[0]], g.double().t().abs() @ v[:g.shape[0]].abs())
        assert _close(db, g.double().sum(0), g.double().abs().sum(0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_gradients_and_more_rows_than_gradients(cuda, dtype):
    import cxgnncomp_backend as be
    x, wide = _inputs(500, 48, 90, dtype)
    rows = be.quantize_rows(x.cuda())
    g = wide[:300, 11:58]
    got = be.rows8_weight_grad(rows, wide.cuda()[:300, 11:58])
    v = be.dequantize_rows(rows).double().cpu()[:300]
    assert _close(got, g.double().t() @ v, g.double().t().abs() @ v.abs())
    got = be.rows8_weight_grad(rows, wide.cuda()[:0])
    assert got.shape == (90, 48) and not bool(got.any())


def _linear_grads(be, x, w, b, add, dy, **kw):
    leaves = [t.detach().cuda().requires_grad_(True) for t in (x, w, b, add) if t is not None]
    it = iter(leaves)
    args = [None if t is None else next(it) for t in (x, w, b, add)]
    y = be.linear_kept8(*args, **kw)
    return y, torch.autograd.grad(y, leaves, dy.cuda())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", [(1, 3, 5), (70, 47, 33), (500, 128, 96)])
@pytest.mark.parametrize("bias,add", [(True, True), (False, False), (False, True), (True, False)])
def test_linear(cuda, m, k, n, dtype, bias, add):
    import cxgnncomp_backend as be
    x, dy = _inputs(m, k, n, dtype)
    w, b = randn((n, k), 5, dtype), randn((n,), 6, dtype) if bias else None
    a = randn((m, n), 7, dtype) if add else None
    y, grads = _linear_grads(be, x, w, b, a, dy)
    half = torch.finfo(dtype).eps / 2
    d = lambda t: t.double()
    want = d(x) @ d(w).t() + (0 if b is None else d(b)) + (0 if a is None else d(a))
    mag = d(x).abs() @ d(w).abs().t() + (0 if b is None else d(b).abs()) + (0 if a is None else d(a).abs())
    # products in fp32; bf16 results round the product, and again with `add`
    assert bool(((y.double().cpu() - want).abs() <= (3 * half + (k + 4) * 2.0 ** -23) * mag).all())
    assert bool(((grads[0].double().cpu() - d(dy) @ d(w)).abs() <= (2 * half + (n + 4) * 2.0 ** -23) * (d(dy).abs() @ d(w).abs())).all())
    kept = held_values(x)
    assert bool(((grads[1].double().cpu() - d(dy).t() @ kept).abs() <= (half + BOUND) * (d(dy).t().abs() @ kept.abs())).all())
    rest = list(grads[2:])
    if bias:
        assert bool(((rest.pop(0).double().cpu() - d(dy).sum(0)).abs() <= (half + BOUND) * d(dy).abs().sum(0)).all())
    if add:
        assert torch.equal(rest.pop(0).cpu(), dy)
    assert all(g.dtype == dtype for g in grads)


def test_linear_with_rows_that_are_there(cuda):
    import cxgnncomp_backend as be
    x, dy = _inputs(300, 64, 48, torch.float32)
    w, b = randn((48, 64), 5), randn((48,), 6)
    y, grads = _linear_grads(be, x, w, b, None, dy)
    rows = be.quantize_rows(x.cuda())
    y2, grads2 = _linear_grads(be, x, w, b, None, dy, kept=rows)
    assert torch.equal(y, y2) and all(torch.equal(a, c) for a, c in zip(grads, grads2))
    # rows that are written in between are noticed
    wg = w.cuda().requires_grad_(True)
    out = be.linear_kept8(x.cuda(), wg, kept=rows)
    be.quantize_rows(x.cuda()[:1], out=rows)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_linear_keeps_a_quarter(cuda):
    """What lives between the two directions: the rows in 8 bits and the weight, not x."""
    import cxgnncomp_backend as be
    w = randn((16, 256), 1).cuda().requires_grad_(True)
    base = torch.cuda.memory_allocated()
    x = torch.randn(40000, 256, device="cuda")
    y = be.linear_kept8(x, w)
    del x
    held = torch.cuda.memory_allocated() - base - y.numel() * 4
    assert held < 1.1 * 40001 * (256 + 8)
    y.sum().backward()
    assert w.grad.shape == w.shape


def test_only_the_gradients_that_are_asked_for(cuda):
    import cxgnncomp_backend as be
    x, dy = _inputs(200, 32, 24, torch.float32)
    w, b = randn((24, 32), 5), randn((24,), 6)
    for need in [(True, False, False), (False, True, False), (False, False, True), (False, True, True)]:
        args = [t.cuda().requires_grad_(r) for t, r in zip((x, w, b), need)]
        be.linear_kept8(*args).backward(dy.cuda())
        assert [a.grad is not None for a in args] == list(need)
    with torch.no_grad():
        y = be.linear_kept8(x.cuda(), w.cuda().requires_grad_(True))
    assert not y.requires_grad
    y = be.linear_kept8(x.cuda(), w.cuda().requires_grad_(True))
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), [y.grad_fn.next_functions[1][0].variable], create_graph=True)


def test_under_autocast(cuda):
    import cxgnncomp_backend as be
    x, dy = _inputs(100, 32, 24, torch.float32)
    w = randn((24, 32), 5)
    xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = be.linear_kept8(xg, wg)
    assert y.dtype == torch.bfloat16
    y.backward(dy.cuda().bfloat16())
    y2, grads = _linear_grads(be, x.bfloat16(), w.bfloat16(), None, None, dy.bfloat16())
    assert torch.equal(y, y2) and torch.equal(xg.grad, grads[0].float()) and torch.equal(wg.grad, grads[1].float())


def test_waits_that_run_out_are_reported(cuda):
    """The producers never hand over their first stage: every role leaves, the status says so, the next call is right."""
    import ctypes
    import cxgnncomp_backend as be
    x, dy = _inputs(500, 64, 64, torch.float32)
    rows, g = be.quantize_rows(x.cuda()), dy.cuda()
    want = be.rows8_weight_grad(rows, g)
    be.check_device_status("linear")
    vp, i64, ci, sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t
    fn = be._sig("cxg_rows8_wgrad", [vp, vp, i64, ci, vp, ci, i64, ci, ctypes.c_uint32, vp, vp, ci, vp, sz, vp])
    ws, dw = torch.empty(1 << 22, dtype=torch.uint8, device="cuda"), torch.zeros(64, 64, device="cuda")
    be.set_wait_limit_cycles(2_000_000)
    try:
        assert fn(rows.codes.data_ptr(), rows.scales.data_ptr(), 500, 64, g.data_ptr(), 0, 64, 64, 1, dw.data_ptr(), None, 0,
                  ws.data_ptr(), ws.numel(), None) == 0
        torch.cuda.synchronize()
    finally:
        be.set_wait_limit_cycles(0)
    with pytest.raises(RuntimeError, match="wait ran out"):
        be.check_device_status("linear")
    be.check_device_status("linear")
    assert torch.equal(be.rows8_weight_grad(rows, g), want)
