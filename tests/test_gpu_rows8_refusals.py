"""What the operators on rows in 8 bits and the step between two blocks refuse with an error."""
import pytest
import torch

from helpers import random_csr, randn

pytestmark = pytest.mark.gpu


def _raises(match, call):
    with pytest.raises(RuntimeError, match=match):
        call()


def test_rows(cuda):
    import cxgnncomp_backend as be
    x = randn((10, 40), 1).cuda()
    rows = be.Rows8(8, 40)
    at = torch.arange(10, device="cuda")
    _raises("there are 8", lambda: be.quantize_rows(x, out=rows))
    _raises("columns", lambda: be.quantize_rows(x[:4, :39], out=rows))
    _raises("for every row", lambda: be.quantize_rows(x, out=rows, index=at[:5]))
    _raises("dtype", lambda: be.quantize_rows(x, out=rows, index=at.int()))
    _raises("dtype", lambda: be.quantize_rows(x.half()))
    _raises("matrix", lambda: be.quantize_rows(x[0]))
    _raises("matrix", lambda: be.quantize_rows(x[:, :0]))
    _raises("CUDA", lambda: be.quantize_rows(x, out=rows, index=at.cpu()))
    _raises("dtype", lambda: be.dequantize_rows(rows, dtype=torch.float16))
    _raises("9 rows of 8", lambda: be.dequantize_rows(rows, num_rows=9))
    _raises("either", lambda: be.dequantize_rows(rows, index=at, num_rows=3))
    _raises("bad sizes", lambda: be.Rows8(-1, 4))
    _raises("bad sizes", lambda: be.Rows8(4, 0))
    _raises("transform", lambda: torch.vmap(lambda t: be.quantize_rows(t).codes)(randn((3, 4, 32), 1).cuda()))


def test_aggregate(cuda):
    import cxgnncomp_backend as be
    rows = be.quantize_rows(randn((20, 40), 1).cuda())
    ptr, idx = (t.cuda() for t in random_csr(10, 20, 3, seed=1))
    ev = torch.ones(idx.shape[0], device="cuda")
    agg = be.rows8_aggregate
    _raises("reduce", lambda: agg(rows, ptr, idx, 10, reduce="max"))
    _raises("exceeds", lambda: agg(rows, ptr, idx, 11))
    _raises("takes no edge values", lambda: agg(rows, ptr, idx, 10, reduce="mean", edge_value=ev))
    _raises("one edge value per edge", lambda: agg(rows, ptr, idx, 10, edge_value=ev[:-1]))
    _raises("no gradient", lambda: agg(rows, ptr, idx, 10, edge_value=ev.clone().requires_grad_(True)))
    _raises("dtype", lambda: agg(rows, ptr, idx.float(), 10))
    _raises("CUDA", lambda: agg(rows, ptr.cpu(), idx, 10))
    _raises("at most 2048", lambda: agg(be.Rows8(20, 2049), ptr, idx, 10))
    # more edges in ptr than idx holds: what is there is read, and the record says so
    agg(rows, ptr, idx[:-2].contiguous(), 10)
    _raises("exceeds the declared", lambda: be.check_device_status("spmm"))


def test_linear_and_weight_grad(cuda):
    import cxgnncomp_backend as be
    x, w = randn((10, 32), 1).cuda(), randn((8, 32), 2).cuda()
    rows = be.quantize_rows(x)
    lin = be.linear_kept8
    _raises("there are 10", lambda: be.rows8_weight_grad(rows, randn((11, 8), 1).cuda()))
    _raises("dtype", lambda: be.rows8_weight_grad(rows, randn((10, 8), 1).cuda().half()))
    _raises("one type", lambda: lin(x, w.bfloat16()))
    _raises("dtype must be", lambda: lin(x.double(), w.double()))
    _raises("weight must be", lambda: lin(x, w[:, :31]))
    _raises("bias must be", lambda: lin(x, w, randn((9,), 1).cuda()))
    _raises("shape of the result", lambda: lin(x, w, add=randn((10, 9), 1).cuda()))
    _raises("rows of x", lambda: lin(x, w, kept=be.quantize_rows(x[:9])))
    _raises("rows of x", lambda: lin(x, w, kept=be.Rows8(10, 40)))
    _raises("CUDA", lambda: lin(x, w.cpu()))
    with torch.autocast("cuda", dtype=torch.float16):
        _raises("dtype must be", lambda: lin(x, w))


def test_residual_norm(cuda):
    import cxgnncomp_backend as be
    x, f, v = randn((10, 32), 1).cuda(), randn((10, 32), 2).cuda(), torch.ones(32, device="cuda")
    res = be.residual_norm
    _raises("shape of x", lambda: res(x, f[:9]))
    _raises("x's type", lambda: res(x, f.bfloat16()))
    _raises("dtype must be", lambda: res(x.half(), f.half()))
    _raises("one value per row", lambda: res(x, f, gate=f[:9]))
    _raises("one value per row", lambda: res(x, f, gate=f[:1]))
    _raises("without f", lambda: res(x, gate=f))
    _raises("without f", lambda: res(x, next=False))
    _raises("not asked for", lambda: res(x, f, next=False, next_weight=v))
    _raises("not asked for", lambda: res(x, f, next=False, keep8=True))
    _raises("not asked for", lambda: res(x, f, post=False, post_bias=v))
    _raises(r"scale must be \[32\]", lambda: res(x, f, scale=v[:31]))
    _raises(r"next_weight must be \[32\]", lambda: res(x, f, next_weight=v[:1]))
    _raises("eps", lambda: res(x, f, eps=-1.0))
    _raises("at most 4096", lambda: res(torch.zeros(2, 4097, device="cuda"), torch.zeros(2, 4097, device="cuda")))
    _raises("matrix", lambda: res(x[0], f[0]))
    _raises("CUDA", lambda: res(x, f, scale=v.cpu()) if False else res(x, f.cpu()))
    _raises("another device", lambda: res(x, f, scale=v.cpu()))
    y, h = res(x.clone().requires_grad_(True), f)
    leaf = x.clone().requires_grad_(True)
    y, h = res(leaf, f)
    _raises("no derivative", lambda: torch.autograd.grad(h.sum(), [leaf], create_graph=True))


def test_captured_while_an_eager_graph_of_the_same_leaves_lives(cuda):
    """torch's engine ends the process in the backward pass of such a capture; the forward call refuses it."""
    import cxgnncomp_backend as be
    x, w = randn((10, 32), 1).cuda(), randn((8, 32), 2).cuda().requires_grad_(True)
    v = torch.ones(32, device="cuda", requires_grad=True)
    calls = [lambda: be.linear_kept8(x, w), lambda: be.residual_norm(x, x, next_weight=v)[1]]
    for call, leaf in zip(calls, (w, v)):
        kept = call()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="still alive"):
            with torch.cuda.graph(graph):
                call()
        del graph
        want = torch.autograd.grad(kept.sum(), [leaf])[0]
        del kept
        graph = torch.cuda.CUDAGraph()  # the same without it
        with torch.cuda.graph(graph):
            got = torch.autograd.grad(call().sum(), [leaf])[0]
        graph.replay()
        assert torch.equal(got, want)


def test_no_rows(cuda):
    import cxgnncomp_backend as be
    x, w = torch.empty(0, 32, device="cuda", requires_grad=True), randn((8, 32), 2).cuda().requires_grad_(True)
    b = randn((8,), 3).cuda().requires_grad_(True)
    y = be.linear_kept8(x, w, b)
    y.sum().backward()
    assert y.shape == (0, 8) and x.grad.shape == (0, 32) and not bool(w.grad.any()) and not bool(b.grad.any())
