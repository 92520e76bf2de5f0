"""Graphs of one launch of clusters whose rows have a few edges less than 64 tiles of 64 hold, and so lie in 64 tiles or in 65,
according to where they begin: sums of more than 64 pieces are added in two rounds. Against float64: a sum of d terms is off by at
most 2 d roundings of 2^-24 of the terms' absolute values, and one of the output's type."""
import pytest
import torch

from helpers import randn
from rows8_ref import aggregate, held_values

pytestmark = pytest.mark.gpu


def _graph(n, degree, seed):
    gen = torch.Generator().manual_seed(seed)
    deg = degree + torch.randint(-3, 4, (n,), generator=gen)
    ptr = torch.zeros(n + 1, dtype=torch.int64)
    ptr[1:] = deg.cumsum(0)
    return ptr, torch.randint(0, 50, (int(ptr[-1]),), generator=gen)


def _close(got, want, mag, deg):
    half = torch.finfo(got.dtype).eps / 2
    bound = (2 * deg.double().unsqueeze(1) + 4) * 2.0 ** -24 * mag * (1 + half) + half * want.abs()
    return bool(((got.double().cpu() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,degree", [(1, 4096), (3, 4090), (9, 4093), (9, 4070), (12, 4050), (9, 4110), (5, 8190), (12, 2040)])
@pytest.mark.parametrize("width", [16, 72])
def test_rows_of_64_or_65_tiles(cuda, width, n, degree, dtype):
    import cxgnncomp_backend as be
    for seed in range(3):
        ptr, idx = _graph(n, degree, seed)
        x = randn((50, width), seed).to(dtype)
        got = be.sage_sum_forward(x.cuda(), ptr.cuda(), idx.cuda(), n)
        assert _close(got, *aggregate(x.double(), ptr, idx, "sum"))
        ev = torch.rand(idx.shape[0], generator=torch.Generator().manual_seed(seed)) - 0.3
        got = be.rows8_aggregate(be.quantize_rows(x.cuda()), ptr.cuda(), idx.cuda(), n, edge_value=ev.cuda(), dtype=dtype)
        assert _close(got, *aggregate(held_values(x), ptr, idx, "sum", ev))
