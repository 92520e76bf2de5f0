"""Aggregation over rows in 8 bits against float64. A row's sum of d exact terms (one more rounding each with edge values) is
added in fp32, in tiles: at most d + 2 roundings of at most 2^-24 of the sum of the terms' absolute values, one for a mean's
division, and that of the output's type."""
import pytest
import torch

from helpers import random_csr, randn
from rows8_ref import aggregate, held_values

pytestmark = pytest.mark.gpu


def _close(got, want, mag, deg):
    half = torch.finfo(got.dtype).eps / 2
    bound = (2 * deg.double().unsqueeze(1) + 4) * 2.0 ** -24 * mag * (1 + half) + half * want.abs()
    return bool(((got.double().cpu() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduce", ["sum", "mean", "value"])
@pytest.mark.parametrize("width", [1, 31, 32, 47, 64, 100, 128, 200, 256, 500, 900, 2048])
def test_aggregate(cuda, width, reduce, dtype):
    import cxgnncomp_backend as be
    index = torch.int32 if width % 2 else torch.int64
    ptr, idx = random_csr(300, 250, 9, seed=width, hub=3000, idx_dtype=index)
    x = randn((250, width), width + 1)
    values = held_values(x)
    ev = torch.rand(idx.shape[0], generator=torch.Generator().manual_seed(2)) - 0.3 if reduce == "value" else None
    rows = be.quantize_rows(x.cuda())
    kind = "mean" if reduce == "mean" else "sum"
    got = be.rows8_aggregate(rows, ptr.cuda(), idx.cuda(), 300, reduce=kind, edge_value=None if ev is None else ev.cuda(), dtype=dtype)
    assert got.dtype == dtype and got.shape == (300, width)
    assert _close(got, *aggregate(values, ptr, idx, kind, ev))
    again = be.rows8_aggregate(rows, ptr.cuda(), idx.cuda(), 300, reduce=kind, edge_value=None if ev is None else ev.cuda(), dtype=dtype)
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduce", ["mean", "value"])
@pytest.mark.parametrize("width", [67, 99, 149, 255, 301, 511])
def test_odd_rows_of_few_edges(cuda, width, reduce, dtype):
    """A graph that is too large for one launch of clusters, with fewer than ten edges per row."""
    import cxgnncomp_backend as be
    ptr, idx = random_csr(30000, 2000, 4, seed=width, hub=5000)
    x = randn((2000, width), width + 1)
    ev = torch.rand(idx.shape[0], generator=torch.Generator().manual_seed(2)) - 0.3 if reduce == "value" else None
    kind = "mean" if reduce == "mean" else "sum"
    got = be.rows8_aggregate(be.quantize_rows(x.cuda()), ptr.cuda(), idx.cuda(), 0, reduce=kind, edge_value=None if ev is None else ev.cuda(),
                             dtype=dtype)
    assert _close(got, *aggregate(held_values(x), ptr, idx, kind, ev))


@pytest.mark.parametrize("edges", [1, 7, 64, 1000])
def test_tiles_that_cut_rows(cuda, edges):
    """Tiles of a few edges: chains of partials, empty rows at every border."""
    import cxgnncomp_backend as be
    ptr, idx = random_csr(200, 100, 3, seed=edges, hub=700, empty_frac=0.4, idx_dtype=torch.int32)
    x = randn((100, 47), 5)
    rows = be.quantize_rows(x.cuda())
    be.SPLIT_EDGES = edges
    try:
        got = be.rows8_aggregate(rows, ptr.int().cuda(), idx.cuda(), 0, reduce="mean")
    finally:
        be.SPLIT_EDGES = 0
    assert _close(got, *aggregate(held_values(x), ptr, idx, "mean"))


def test_rows_without_edges_and_first_rows(cuda):
    import cxgnncomp_backend as be
    x = randn((20, 40), 1)
    rows = be.quantize_rows(x.cuda())
    ptr = torch.zeros(31, dtype=torch.int64)
    y = be.rows8_aggregate(rows, ptr.cuda(), torch.empty(0, dtype=torch.int64).cuda(), 30)
    assert y.shape == (30, 40) and not bool(y.any())
    ptr, idx = random_csr(50, 20, 5, seed=3)
    y = be.rows8_aggregate(rows, ptr.cuda(), idx.cuda(), 17)
    want = aggregate(held_values(x), ptr[:18], idx, "sum")
    assert y.shape == (17, 40) and _close(y, *want)
    assert be.rows8_aggregate(rows, ptr[:1].cuda(), idx.cuda(), 0).shape == (0, 40)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduce", ["sum", "mean", "value"])
@pytest.mark.parametrize("n,edges,width", [(1000, 1, 33), (3000, 200, 4), (3000, 700, 100), (30000, 5000, 47), (30000, 29000, 128),
                                           (31000, 120000, 64),
                                           (9000, 2000, 300), (2000, 400, 900), (100000, 70000, 16)])
def test_graphs_of_mostly_empty_rows(cuda, n, edges, width, reduce, dtype):
    """More rows than edges: whole tiles of one row, rows that tiles cut, empty rows in front, between and behind."""
    import cxgnncomp_backend as be
    gen = torch.Generator().manual_seed(edges)
    dst = torch.randint(n // 10, n - n // 10, (edges,), generator=gen)
    dst[: edges // 4] = n // 2
    ptr = torch.zeros(n + 1, dtype=torch.int64)
    ptr[1:] = torch.bincount(dst, minlength=n).cumsum(0)
    idx = torch.randint(0, 500, (edges,), generator=gen)
    idx[::7], idx[3::11] = -1, 507
    if width % 2:
        ptr, idx = ptr.int(), idx.int()
    x = randn((500, width), width)
    ev = torch.rand(edges, generator=gen) - 0.3 if reduce == "value" else None
    kind = "mean" if reduce == "mean" else "sum"
    rows = be.quantize_rows(x.cuda())
    got = be.rows8_aggregate(rows, ptr.cuda(), idx.cuda(), 0, reduce=kind, edge_value=None if ev is None else ev.cuda(), dtype=dtype)
    assert _close(got, *aggregate(held_values(x), ptr, idx, kind, ev))
    again = be.rows8_aggregate(rows, ptr.cuda(), idx.cuda(), 0, reduce=kind, edge_value=None if ev is None else ev.cuda(), dtype=dtype)
    assert torch.equal(got, again)


def test_ids_outside_and_groups_that_are_not_finite(cuda):
    import cxgnncomp_backend as be
    x = randn((20, 96), 1)
    x[3, 40] = float("inf")
    rows = be.quantize_rows(x.cuda())
    idx = torch.tensor([0, -1, 5, 20, 2 ** 32 + 1, 7, -2 ** 62, 3, 3, 4])
    ptr = torch.tensor([0, 2, 5, 7, 8, 10])
    for reduce in ("sum", "mean"):
        y = be.rows8_aggregate(rows, ptr.cuda(), idx.cuda(), 5, reduce=reduce).double().cpu()
        want, mag, deg = aggregate(held_values(x), ptr, idx, reduce)
        assert torch.equal(torch.isnan(y), torch.isnan(want))
        assert bool(torch.isnan(y[3:, 32:64]).all()) and not bool(torch.isnan(y[:, 64:]).any())
        keep = ~torch.isnan(want)
        assert bool(((y - want).abs() <= 8 * 2.0 ** -24 * mag)[keep].all())


def test_captured(cuda):
    import cxgnncomp_backend as be
    ptr, idx = (t.cuda() for t in random_csr(400, 300, 8, seed=1))
    first, second = randn((300, 64), 1), randn((300, 64), 2)
    rows = be.quantize_rows(first.cuda())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = be.rows8_aggregate(rows, ptr, idx, 400, dtype=torch.bfloat16)
    for x in (first, second):
        be.quantize_rows(x.cuda(), out=rows)
        want = be.rows8_aggregate(rows, ptr, idx, 400, dtype=torch.bfloat16)
        graph.replay()
        assert torch.equal(y, want)
