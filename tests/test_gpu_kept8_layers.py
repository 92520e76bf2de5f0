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


@pytest.mark.parametrize("autocast", [False, True])
def test_a_narrowing_layer_keeps_one_copy_of_what_it_reads(cuda, autocast):
    """Both transforms of a layer that narrows read the same rows."""
    import cxgnncomp
    n, n_in, n_out = 20000, 256, 16
    ptr, idx = (t.cuda() for t in random_csr(n, n, 3, seed=2))
    torch.manual_seed(1)
    conv = cxgnncomp.MySageConv(n_in, n_out, kept8=True).cuda()
    x = torch.randn(n, n_in, device="cuda")
    dy = randn((n, n_out), 4).cuda()
    with torch.autocast("cuda", torch.bfloat16, enabled=autocast):
        y = conv(x, ptr, idx, n)  # what is kept once, per graph or library
        del y
        before = torch.cuda.memory_allocated()
        y = conv(x, ptr, idx, n)
    held = torch.cuda.memory_allocated() - before - y.numel() * y.element_size()
    rows = (n + 1) * (n_in + n_in // 32)
    assert rows <= held < 1.5 * rows
    want = torch.autograd.grad(y, list(conv.parameters()), dy.to(y.dtype))
    # the weights' gradients with rows that the caller has are the same
    import cxgnncomp_backend as be
    with torch.autocast("cuda", torch.bfloat16, enabled=autocast):
        z = conv(x, ptr, idx, n, kept=be.quantize_rows(x.bfloat16() if autocast else x))
    got = torch.autograd.grad(z, list(conv.parameters()), dy.to(z.dtype))
    assert torch.equal(y, z) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("inference", [False, True])
def test_a_model_over_features_in_8_bits_keeps_no_matrix_of_them(cuda, inference):
    import cxgnncomp
    import cxgnncomp_backend as be
    n, n_in = 20000, 500
    ptr, idx = (t.cuda() for t in random_csr(n, n, 3, seed=2))
    x = randn((n, n_in), 3).cuda()
    with torch.inference_mode(inference):
        rows = be.quantize_rows(x)
    batch = cxgnncomp.Batch(rows, ptr, idx, num_node_in_layer=[n] * 2, num_edge_in_layer=[idx.shape[0]])
    torch.manual_seed(1)
    model = cxgnncomp.ResidualGNN("sage", n_in, 16, 4, 1, kept8=True).cuda()
    target = torch.randint(0, 4, (n,), generator=torch.Generator().manual_seed(1)).cuda()

    def grads(m, b):
        out = m(b)
        return out.detach(), torch.autograd.grad(torch.nn.functional.nll_loss(out, target), list(m.parameters()))

    out, got = grads(model, batch)
    before = torch.cuda.memory_allocated()
    kept = model(batch)
    held = torch.cuda.memory_allocated() - before
    assert (held < n * n_in) or inference  # the matrix would be four times as much; about 20 vectors of 16 values a row are kept
    del kept
    # the same model over the values that the rows hold
    batch.x = be.dequantize_rows(rows)
    want_out, want = grads(model, batch)
    assert torch.equal(out, want_out)
    for k, a, b in zip(dict(model.named_parameters()), got, want):
        # the first transform's gradients: sums of 20000 terms on either side, each rounded to 2^-24 of terms that cancel to about
        # 1 / sqrt(20000) of their sizes
        first = k in ("lin_in.weight", "lin_in.bias")
        assert torch.equal(a, b) or (first and float((a - b).norm()) <= 2.0 ** -24 * 20000 ** 0.5 * float(b.norm())), k
