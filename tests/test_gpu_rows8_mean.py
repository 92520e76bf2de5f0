"""A mean over rows in 8 bits is the sum of the same rows, divided by their number and rounded once."""
import pytest
import torch

from helpers import random_csr, randn

pytestmark = pytest.mark.gpu


# one launch of clusters, tiles, and graphs of mostly empty rows; every layout of lanes
@pytest.mark.parametrize("n,edges_per_row,width", [(300, 9, 47), (300, 9, 256), (20000, 5, 20), (20000, 5, 60), (20000, 5, 100), (20000, 5, 128),
                                                   (20000, 5, 200), (20000, 5, 301), (2000, 40, 900), (2000, 40, 2000), (90000, 0.6, 100)])
def test_a_mean_is_the_quotient_of_the_sum(cuda, n, edges_per_row, width):
    import cxgnncomp_backend as be
    ptr, idx = random_csr(n, 500, edges_per_row, seed=width, hub=3000)
    x = randn((500, width), width) * torch.exp2(randn((500, 1), 1) * 8)
    x[7, 0] = 2.0 ** 127
    rows = be.quantize_rows(x.cuda())
    mean, total = (be.rows8_aggregate(rows, ptr.cuda(), idx.cuda(), n, reduce=r).cpu() for r in ("mean", "sum"))
    want = total / (ptr[1:] - ptr[:-1]).clamp(min=1).float().unsqueeze(1)
    assert bool(torch.isinf(want).any()) and torch.equal(torch.isnan(mean), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(mean, 0.0), torch.nan_to_num(want, 0.0))
    # bf16: rounded from the quotient or one of its neighbours in fp32
    low = be.rows8_aggregate(rows, ptr.cuda(), idx.cuda(), n, reduce="mean", dtype=torch.bfloat16).double().cpu()
    keep = torch.isfinite(want)
    assert bool(((low - want.double()).abs() <= (2.0 ** -8 + 2.0 ** -23) * want.double().abs() + 2.0 ** -133)[keep].all())
