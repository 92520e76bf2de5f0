"""Rows in 8 bits: writing and reading against the definition in float64. Every value that is held is exact in both types, so
there is no tolerance."""
import pytest
import torch

from helpers import randn
from rows8_ref import held_values

pytestmark = pytest.mark.gpu

NAN = float("nan")


def _same(got, want):
    """Equal bit for bit, NaN for NaN."""
    got = got.double().cpu()
    return torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got, 0.0, 0.0, 0.0),
                                                                            torch.nan_to_num(want, 0.0, 0.0, 0.0))


def _spread(n, width, seed, dtype):
    """Rows whose sizes lie far apart, values with a ReLU's zeros among them."""
    x = randn((n, width), seed) * torch.exp2(torch.randint(-30, 30, (n, 1), generator=torch.Generator().manual_seed(seed)).float())
    return torch.where(randn((n, width), seed + 1) > 0.7, torch.zeros(()), x).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,width", [(1, 1), (3, 4), (5, 31), (1, 32), (17, 33), (40, 47), (33, 64), (21, 100), (9, 257), (300, 128),
                                     (2, 2000), (1000, 5), (700, 50), (333, 99), (100, 130)])
def test_write_and_read(cuda, n, width, dtype):
    import cxgnncomp_backend as be
    x = _spread(n, width, n + width, dtype)
    rows = be.quantize_rows(x.cuda())
    assert rows.shape == (n, width) and len(rows) == n and rows.device == torch.device("cuda:0")
    want = held_values(x)
    for out in (torch.float32, torch.bfloat16):
        got = be.dequantize_rows(rows, dtype=out)
        assert got.dtype == out and _same(got, want)
    # the row behind the last, and what lies behind the width, are zeros
    assert bool((rows.codes[n] == 128).all()) and bool((rows.codes[:, width:] == 128).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_borders_of_the_format(cuda, dtype):
    import cxgnncomp_backend as be
    top = torch.finfo(dtype).max
    tiny = 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -149
    rows = [
        [0.0] * 32,
        [-0.0] * 32,
        [127.0, 126.5, 125.5, 0.5, -0.5, 1.5],       # a step of 1: ties to even
        [127.5, 1.0],                                 # would round to 128: the step is 2
        [-127.5, 3.0, 5.0],
        [127.49999, 1.0],
        [top, -top, top / 3, 1.0],                    # the largest there is
        [tiny, -tiny],                                # below the smallest step
        [2.0 ** -126 * 63, 2.0 ** -126, 2.0 ** -127],
        [float("inf"), 1.0], [NAN, 1.0], [1.0] * 31 + [float("-inf")],
        [1.0] * 32 + [NAN] + [2.0] * 40,              # only its own group
    ]
    x = torch.zeros(len(rows), 80)
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r)
    x = x.to(dtype)
    assert _same(be.dequantize_rows(be.quantize_rows(x.cuda())), held_values(x))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width,offset", [(64, 0), (64, 1), (47, 3), (100, 4), (32, 8)])
def test_rows_of_a_wider_matrix(cuda, width, offset, dtype):
    import cxgnncomp_backend as be
    wide = _spread(37, width + 21, 5, dtype)
    x = wide.cuda()[2:35, offset:offset + width]
    assert _same(be.dequantize_rows(be.quantize_rows(x)), held_values(wide[2:35, offset:offset + width]))
    # columns that do not lie side by side
    t = wide.cuda().t()
    assert _same(be.dequantize_rows(be.quantize_rows(t)), held_values(wide.t()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", [1, 47, 128])
def test_write_at_and_read_at(cuda, width, dtype):
    import cxgnncomp_backend as be
    n = 500
    before, x = _spread(n, width, 1, torch.float32), _spread(800, width, 2, dtype)
    at = torch.randint(-3, n + 3, (800,), generator=torch.Generator().manual_seed(3))
    cache = be.quantize_rows(before.cuda())
    want = held_values(before)
    new = held_values(x)
    for i, r in enumerate(at.tolist()):  # in order: the last of equal ids stays
        if 0 <= r < n:
            want[r] = new[i]
    for _ in range(2):  # the second time the same once more
        assert be.quantize_rows(x.cuda(), out=cache, index=at.cuda()) is cache
        assert _same(be.dequantize_rows(cache), want)
    # a later call's early positions win over an earlier call's late ones
    few = at[:40].flip(0)
    be.quantize_rows(x[:40].cuda(), out=cache, index=few.cuda())
    for i, r in enumerate(few.tolist()):
        if 0 <= r < n:
            want[r] = new[i]
    assert _same(be.dequantize_rows(cache), want)
    ids = torch.randint(-2, n + 2, (900,), generator=torch.Generator().manual_seed(4))
    ids[0], ids[1], ids[2] = 2 ** 40, -2 ** 63, n
    ok = (ids >= 0) & (ids < n)
    picked = torch.where(ok.unsqueeze(1), want[torch.where(ok, ids, torch.zeros_like(ids))], torch.zeros(()).double())
    assert _same(be.dequantize_rows(cache, index=ids.cuda(), dtype=dtype), picked)


@pytest.mark.parametrize("n", [1, 1023, 1025, 4096, 4097, 30000])
def test_equal_ids_of_any_number_of_rows(cuda, n):
    """Every id comes about three times; the last of its rows is told by its values."""
    import cxgnncomp_backend as be
    ids = torch.randint(0, max(1, n // 3), (n,), generator=torch.Generator().manual_seed(n))
    x = (torch.arange(n) % 127 + 1).float().unsqueeze(1).expand(n, 5).contiguous()  # whole numbers up to 127: exact
    cache = be.Rows8(max(1, n // 3), 5)
    be.quantize_rows(x.cuda(), out=cache, index=ids.cuda())
    want = torch.zeros(max(1, n // 3), 5)
    for i, r in enumerate(ids.tolist()):
        want[r] = x[i]
    assert torch.equal(be.dequantize_rows(cache).cpu(), want)


def test_first_rows_and_empty_calls(cuda):
    import cxgnncomp_backend as be
    cache = be.Rows8(10, 40)
    assert not bool(be.dequantize_rows(cache).any())
    x = _spread(4, 40, 9, torch.float32)
    be.quantize_rows(x.cuda(), out=cache)
    want = torch.cat([held_values(x), torch.zeros(6, 40).double()])
    assert _same(be.dequantize_rows(cache), want)
    none = torch.empty(0, 40, device="cuda")
    be.quantize_rows(none, out=cache)
    be.quantize_rows(none, out=cache, index=torch.empty(0, dtype=torch.int64, device="cuda"))
    assert _same(be.dequantize_rows(cache), want)
    assert be.dequantize_rows(cache, index=torch.empty(0, dtype=torch.int64, device="cuda")).shape == (0, 40)
    empty = be.quantize_rows(none)
    assert empty.shape == (0, 40) and be.dequantize_rows(empty).shape == (0, 40)
    assert not bool(be.dequantize_rows(empty, index=torch.tensor([0, 5], device="cuda")).any())


def test_rows_beyond_four_gigabytes(cuda):
    import cxgnncomp_backend as be
    n = 34_000_000  # 4.35 GB of codes
    cache = be.Rows8(n, 128)
    x = _spread(6, 128, 11, torch.bfloat16)
    at = torch.tensor([n - 1, 0, 33_554_432, 33_554_431, n - 2, 16_777_216])
    be.quantize_rows(x.cuda(), out=cache, index=at.cuda())
    assert _same(be.dequantize_rows(cache, index=at.cuda()), held_values(x))
    near = torch.tensor([1, n - 3, 33_554_433, 33_554_430, 16_777_215])
    assert not bool(be.dequantize_rows(cache, index=near.cuda()).any())
    ptr = torch.tensor([0, 3, 3, 6])
    y = be.rows8_aggregate(cache, ptr.cuda(), at.cuda(), 3)
    want = held_values(x)
    want = torch.stack([want[:3].sum(0), torch.zeros(128).double(), want[3:].sum(0)])
    mag = held_values(x).abs().sum(0)
    assert bool(((y.double().cpu() - want).abs() <= 3 * 2.0 ** -24 * mag).all())


def test_another_stream_and_a_captured_write(cuda):
    import cxgnncomp_backend as be
    x = [_spread(64, 47, s, torch.float32) for s in (1, 2, 3)]
    at = [torch.randint(0, 50, (64,), generator=torch.Generator().manual_seed(s)) for s in (4, 5, 6)]

    def expect(steps):
        want = torch.zeros(50, 47).double()
        for s in steps:
            for i, r in enumerate(at[s].tolist()):
                want[r] = held_values(x[s][i:i + 1])[0]
        return want

    cache, xs, ids = be.Rows8(50, 47), x[0].cuda(), at[0].cuda()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        be.quantize_rows(xs, out=cache, index=ids)
        got = be.dequantize_rows(cache)
    stream.synchronize()
    assert _same(got, expect([0]))
    # captured with a cache that has no words yet, replayed twice with an eager write of other rows in between
    fresh = be.Rows8(50, 47)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        be.quantize_rows(xs, out=fresh, index=ids)
        read = be.dequantize_rows(fresh)
    graph.replay()
    assert _same(read, expect([0]))
    be.quantize_rows(x[1].cuda(), out=fresh, index=at[1].cuda())
    xs.copy_(x[2])
    ids.copy_(at[2])
    graph.replay()
    assert _same(read, expect([0, 1, 2]))


def test_a_cache_made_in_inference_mode(cuda):
    """Written and read like any other, in inference mode and outside."""
    import cxgnncomp_backend as be
    x = _spread(30, 40, 3, torch.float32)
    with torch.inference_mode():
        cache = be.Rows8(50, 40)
        be.quantize_rows(x[:9].cuda(), out=cache)
    at = torch.arange(20, 50)
    be.quantize_rows(x.cuda(), out=cache, index=at.cuda())
    assert _same(be.dequantize_rows(cache, index=at.cuda()), held_values(x))
    assert _same(be.dequantize_rows(cache, num_rows=9), held_values(x[:9]))


def test_views_that_stand_for_their_negative(cuda):
    import cxgnncomp_backend as be
    x = randn((40, 33), 7).cuda()
    v = torch._neg_view(x)
    assert _same(be.dequantize_rows(be.quantize_rows(v)), held_values(-x.cpu()))
    rows = be.quantize_rows(x)
    dy = randn((40, 17), 8).cuda()
    assert torch.equal(be.rows8_weight_grad(rows, torch._neg_view(dy)), be.rows8_weight_grad(rows, -dy))
    w = randn((17, 33), 9).cuda()
    assert torch.equal(be.linear_kept8(v, torch._neg_view(w)), be.linear_kept8(-x, -w))
    f = randn((40, 33), 10).cuda()
    scale = randn((33,), 11).cuda()
    a = be.residual_norm(v, torch._neg_view(f), gate=torch._neg_view(f), scale=torch._neg_view(scale))
    b = be.residual_norm(-x, -f, gate=-f, scale=-scale)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ptr, idx = torch.tensor([0, 2, 3]).cuda(), torch.tensor([1, 2, 3]).cuda()
    with pytest.raises(RuntimeError, match="resolve_neg"):
        be.rows8_aggregate(rows, ptr, idx, 2, edge_value=torch._neg_view(torch.ones(3, device="cuda")))
