"""Layers that keep what they read in 8 bits: what they compute, and what they keep, against the same layers without."""
import copy

import pytest
import torch

from helpers import random_csr, randn

pytestmark = pytest.mark.gpu


def _pair(make):
    torch.manual_seed(1)
    kept = make()
    plain = copy.deepcopy(kept)
    for m in plain.modules():
        if hasattr(m, "kept8"):
            m.kept8 = False
    return kept, plain


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n_in,n_out,root", [(32, 48, True), (48, 48, True), (64, 32, True), (64, 32, False), (100, 47, True), (36, 64, False)])
def test_a_sage_layer_gives_the_same_bits(cuda, n_in, n_out, root, dtype):
    """Another rounding in front of a ReLU would put values within rounding of zero on its other side."""
    import cxgnncomp
    ptr, idx = (t.cuda() for t in random_csr(500, 800, 6, seed=2))
    x = randn((800, n_in), 3, dtype).cuda()
    kept, plain = _pair(lambda: cxgnncomp.MySageConv(n_in, n_out, root_weight=root, kept8=True).cuda().to(dtype))
    a, b = kept(x, ptr, idx, 500), plain(x, ptr, idx, 500)
    assert a.requires_grad and torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(kept(x, ptr, idx, 500), plain(x, ptr, idx, 500))


@pytest.mark.parametrize("gate", [None, "row", "value"])
def test_a_residual_model_gives_the_same_bits(cuda, gate):
    import cxgnncomp
    ptr, idx = (t.cuda() for t in random_csr(600, 600, 7, seed=1, hub=900))
    batch = cxgnncomp.Batch(randn((600, 40), 5).cuda(), ptr, idx, num_node_in_layer=[600] * 4, num_edge_in_layer=[idx.shape[0]] * 3)
    kept, plain = _pair(lambda: cxgnncomp.ResidualGNN("sage", 40, 64, 12, 3, gate=gate, kept8=True).cuda())
    a, b = kept(batch), plain(batch)
    assert a.requires_grad and torch.equal(a, b)


@pytest.mark.parametrize("n_in,n_out", [(40, 64), (64, 24)])
def test_a_layer_over_features_in_8_bits_gives_the_same_bits(cuda, n_in, n_out):
    import cxgnncomp
    import cxgnncomp_backend as be
    ptr, idx = (t.cuda() for t in random_csr(500, 800, 6, seed=2))
    rows = be.quantize_rows(randn((800, n_in), 3).cuda())
    kept, plain = _pair(lambda: cxgnncomp.MySageConv(n_in, n_out, kept8=True).cuda())
    a, b = kept(rows, ptr, idx, 500), plain(rows, ptr, idx, 500)
    assert a.requires_grad and torch.equal(a, b)
