"""Aggregation over rows in 8 bits where an edge's value takes a group's scale out of the range of fp32: terms are what the held value
times the edge's value is in fp32, infinities where that overflows, and zeros stay zeros."""
import pytest
import torch

from helpers import random_csr, randn
from rows8_ref import held_values

pytestmark = pytest.mark.gpu


def _check(be, x, ptr, idx, ev, dtype):
    n = ptr.shape[0] - 1
    got = be.rows8_aggregate(be.quantize_rows(x.cuda()), ptr.cuda(), idx.cuda(), n, edge_value=ev.cuda(), dtype=dtype).double().cpu()
    terms = (held_values(x).float()[idx] * ev.unsqueeze(1)).double()  # rounded to fp32, infinities among them
    deg = ptr[1:] - ptr[:-1]
    dst = torch.repeat_interleave(torch.arange(n), deg)
    want = torch.zeros((n, x.shape[1]), dtype=torch.float64).index_add_(0, dst, terms)
    mag = torch.zeros_like(want).index_add_(0, dst, torch.nan_to_num(terms.abs(), 0.0, 0.0, 0.0))
    assert bool(torch.isinf(want).any()) and bool(torch.isfinite(want).any())
    # Terms of both signs that overflow: a sum of rounded terms is NaN. A multiply-add does not round its product: where the sum is
    # infinite already, a finite product of the other sign leaves it so. Either is right, a finite sum is not.
    def any_of(which):
        return torch.zeros_like(want).index_add_(0, dst, which.double()) > 0

    both = any_of(terms == float("inf")) & any_of(terms == -float("inf")) & ~any_of(torch.isnan(terms))
    assert not bool(torch.isfinite(got[both]).any())
    got, want = torch.where(both, 0.0, got), torch.where(both, 0.0, want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf])
    keep = torch.isfinite(want)
    # a rounding per term and per addition of 2^-24 each, in fp32; that of the output
    bound = (2 * deg.double().unsqueeze(1) + 4) * 2.0 ** -24 * mag + torch.finfo(dtype).eps / 2 * want.abs()
    assert bool(((got - want).abs() <= bound)[keep].all())


def _rows(n, width, seed):
    """Groups of up to 2^120 and of up to one, half of the values zero."""
    x = randn((n, width), seed).clamp(-4, 4) / 4
    x[randn((n, width), seed + 1) > 0] = 0
    for a in range(0, width, 64):
        x[:, a:a + 32] *= 2.0 ** 120
    return x


# graphs of one launch of clusters, of tiles, and of mostly empty rows; widths of every layout of lanes
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,edges_per_row,width", [(200, 6, 20), (200, 6, 100), (200, 6, 256), (20000, 4, 33), (20000, 4, 60), (20000, 4, 100),
                                                   (20000, 4, 200), (20000, 4, 300), (2000, 5, 900), (2000, 5, 1300), (90000, 0.5, 100)])
def test_values_that_take_scales_out_of_range(cuda, n, edges_per_row, width, dtype):
    import cxgnncomp_backend as be
    ptr, idx = random_csr(n, 64, edges_per_row, seed=width, hub=900)  # a row of many tiles, finite in its small groups
    gen = torch.Generator().manual_seed(n)
    # few large ones: rows of finite sums have to be left. Sums of up to 40 terms of 2^120 are finite.
    ev = torch.tensor([0.5, -0.25, 0.0, 1.0])[torch.randint(0, 4, (idx.shape[0],), generator=gen)]
    large = torch.rand(idx.shape[0], generator=gen) < 0.1
    ev = torch.where(large, torch.tensor([1e6, -1e6, 1e30])[torch.randint(0, 3, (idx.shape[0],), generator=gen)], ev)
    _check(be, _rows(64, width, width), ptr, idx, ev, dtype)


@pytest.mark.parametrize("rows", [12, 80000])
def test_the_largest_scale(cuda, rows):
    import cxgnncomp_backend as be
    top = torch.finfo(torch.float32).max
    x = torch.zeros(3, 96)
    x[0, :4] = torch.tensor([top, -top, top / 4, 2.0 ** 121])
    x[1, 40] = float("inf")
    x[2, 5] = 3.0
    values = torch.tensor([127.99, 128.0, -128.0, top, 0.0, float("inf"), -float("inf"), float("nan"), 2.0 ** -20, -1.0, 1.0, 0.5])
    idx = (torch.arange(rows) // len(values)) % 3
    ptr = torch.arange(rows + 1)
    _check(be, x, ptr, idx, values[torch.arange(rows) % len(values)], torch.float32)
