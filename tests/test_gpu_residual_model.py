"""The operators on rows in 8 bits and the step between two blocks as a model runs them: a deep residual stack trained with and
without rows in 8 bits, a SAGE layer over features in 8 bits, sampled batches over such features."""
import copy

import pytest
import torch
import torch.nn.functional as F

from helpers import random_csr, randn, rel_err
from rows8_ref import aggregate, held_values, residual

pytestmark = pytest.mark.gpu

N = 600


def _batch(features, layers, seed=1):
    import cxgnncomp
    ptr, idx = (t.cuda() for t in random_csr(N, N, 7, seed=seed, hub=900))
    return cxgnncomp.Batch(features, ptr, idx, num_node_in_layer=[N] * (layers + 1), num_edge_in_layer=[idx.shape[0]] * layers)


def _reference(model, batch, x):
    """The model in float64 from the formulas."""
    p = {k: v.detach().double().cpu().requires_grad_(True) for k, v in model.named_parameters()}
    ptr, idx = batch.ptr.cpu(), batch.idx.cpu()
    deg = ptr[1:] - ptr[:-1]
    dst = torch.repeat_interleave(torch.arange(N), deg)
    layer = model.norm == "layer"

    def step(i, x, f, gate):
        at = lambda name, j: p.get(f"{name}.{j}")
        return residual(x, f, gate, at("scale", i - 1), f is not None, at("post_weight", i - 1), at("post_bias", i - 1), True,
                        at("next_weight", i), at("next_bias", i), layer, 1e-5)

    x, h = step(0, F.linear(x.double(), p["lin_in.weight"], p["lin_in.bias"]), None, None)
    for i in range(model.num_layers):
        mean = torch.zeros_like(h).index_add(0, dst, h[idx]) / deg.clamp(min=1).double().unsqueeze(1)
        f = F.relu(F.linear(mean, p[f"convs.{i}.lin_l.weight"], p[f"convs.{i}.lin_l.bias"]) + F.linear(h, p[f"convs.{i}.lin_r.weight"]))
        gate = F.linear(h, p[f"gates.{i}.weight"], p[f"gates.{i}.bias"]) if model.gate else None
        x, h = step(i + 1, x, f, gate)
    return F.linear(h, p["lin_out.weight"], p["lin_out.bias"]).log_softmax(-1), p


@pytest.mark.parametrize("norm,gate", [("rms", None), ("layer", "row"), ("rms", "value")])
@pytest.mark.parametrize("kept8", [False, True])
def test_training_step(cuda, norm, gate, kept8):
    import cxgnncomp
    torch.manual_seed(3)
    x, y = randn((N, 20), 5), torch.randint(0, 7, (N,), generator=torch.Generator().manual_seed(6))
    model = cxgnncomp.ResidualGNN("sage", 20, 48, 7, 3, norm=norm, gate=gate, kept8=kept8).cuda()
    with torch.no_grad():
        for k, v in model.named_parameters():
            if v.dim() == 1:
                v.add_(0.1 * torch.randn_like(v))
    batch = _batch(x.cuda(), 3)
    out = model(batch)
    F.nll_loss(out, y.cuda()).backward()
    want, p = _reference(model, batch, x)
    F.nll_loss(want, y).backward()
    # Three blocks of a few dozen roundings each, in norms whose factors are near one; a value within 1e-6 of a ReLU's kink may
    # fall on its other side: one value's part of a sum over 600 nodes.
    assert rel_err(out.detach().cpu(), want.detach()) < 1e-4
    through_rows = {f"convs.{i}.{l}.weight" for i in range(3) for l in ("lin_l", "lin_r")} | {f"gates.{i}.weight" for i in range(3)}
    for k, v in model.named_parameters():
        g, w = v.grad.double().cpu(), p[k].grad
        if kept8 and k in through_rows:
            # each kept value is off by at most 2^-7 of its group's largest, with either sign: sums over 600 nodes of errors that
            # average to 2^-7 / sqrt(3) of values up to about 4 times as large as they are on average, and cancel like their
            # terms: 2^-7 * 4 / sqrt(3) of the gradient's norm at most if they cancel no better than these
            assert float((g - w).norm()) <= 2.0 ** -7 * 4 / 3 ** 0.5 * float(w.norm()) + 1e-5, k
        else:
            assert float((g - w).norm()) <= 1e-3 * float(w.norm()) + 1e-6, k


def test_kept_rows_change_nothing_else(cuda):
    """Blocks with and without rows of h from the step before give the same bits: the rows in 8 bits are the same rows."""
    import cxgnncomp
    import cxgnncomp_backend as be
    torch.manual_seed(1)
    conv = cxgnncomp.MySageConv(32, 48, kept8=True).cuda()
    ptr, idx = (t.cuda() for t in random_csr(200, 300, 6, seed=2))
    x = randn((300, 32), 3).cuda().requires_grad_(True)
    dy = randn((200, 48), 4).cuda()
    leaves = [x, *conv.parameters()]
    a = conv(x, ptr, idx, 200)
    ga = torch.autograd.grad(a, leaves, dy)
    b = conv(x, ptr, idx, 200, kept=be.quantize_rows(x.detach()))
    gb = torch.autograd.grad(b, leaves, dy)
    assert torch.equal(a, b) and all(torch.equal(p, q) for p, q in zip(ga, gb))
    plain = copy.deepcopy(conv)
    plain.kept8 = False
    c = plain(x, ptr, idx, 200)
    assert rel_err(a.detach(), c.detach()) < 1e-5
    gc = torch.autograd.grad(c, [x, *plain.parameters()], dy)
    assert rel_err(ga[0], gc[0]) < 1e-5
    # narrowing layers transform first
    conv = cxgnncomp.MySageConv(48, 16, kept8=True).cuda()
    plain = copy.deepcopy(conv)
    plain.kept8 = False
    x = randn((300, 48), 3).cuda()
    assert rel_err(conv(x, ptr, idx, 200).detach(), plain(x, ptr, idx, 200).detach()) < 1e-5


@pytest.mark.parametrize("kept8", [False, True])
def test_sage_layer_over_features_in_8_bits(cuda, kept8):
    import cxgnncomp
    import cxgnncomp_backend as be
    torch.manual_seed(1)
    conv = cxgnncomp.MySageConv(40, 24, kept8=kept8).cuda()
    ptr, idx = (t.cuda() for t in random_csr(200, 300, 6, seed=2))
    x, dy = randn((300, 40), 3), randn((200, 24), 4)
    out = conv(be.quantize_rows(x.cuda()), ptr, idx, 200)
    out.backward(dy.cuda())
    v = held_values(x)
    mean = aggregate(v, ptr.cpu(), idx.cpu(), "mean")[0]
    wl, wr, b = (t.detach().double().cpu() for t in (conv.lin_l.weight, conv.lin_r.weight, conv.lin_l.bias))
    # sums of 40 products and of a few dozen edges in fp32
    assert rel_err(out.detach().cpu(), mean @ wl.t() + b + v[:200] @ wr.t()) < 1e-5
    assert rel_err(conv.lin_r.weight.grad.cpu(), dy.double().t() @ v[:200]) < 1e-5
    want = dy.double().t() @ mean
    assert rel_err(conv.lin_l.weight.grad.cpu(), want) < (2.0 ** -5 if kept8 else 1e-5)


def test_sampled_batches_of_features_in_8_bits(cuda):
    import cxgnncomp
    import cxgnncomp_backend as be
    ptr, idx = (t.cuda() for t in random_csr(3000, 3000, 9, seed=4, empty_frac=0))
    x = randn((3000, 50), 5)
    y = torch.randint(0, 5, (3000,), generator=torch.Generator().manual_seed(6)).cuda()
    rows = be.quantize_rows(x.cuda())
    sampler = cxgnncomp.NeighborSampler(ptr, idx, [5, 4])
    seeds = torch.arange(0, 600, 3).cuda()
    b = sampler.batch(rows, seeds, seed=1, y=y)
    assert torch.equal(b.x.double().cpu(), held_values(x)[b.target.cpu()])
    torch.manual_seed(0)
    model = cxgnncomp.ResidualGNN("sage", 50, 32, 5, 2, gate="row", kept8=True).cuda()
    losses = cxgnncomp.train_epoch(model, torch.optim.SGD(model.parameters(), lr=0.01), sampler, rows, y, torch.arange(3000).cuda(), 500)
    assert losses.shape == (6,) and bool(torch.isfinite(losses).all())
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in model.parameters())


def test_a_captured_step_gives_the_eager_bits(cuda):
    import cxgnncomp
    torch.manual_seed(3)
    x = randn((N, 24), 5).cuda()
    y = torch.randint(0, 7, (N,), generator=torch.Generator().manual_seed(6)).cuda()
    model = cxgnncomp.ResidualGNN("sage", 24, 32, 7, 2, norm="layer", gate="value", kept8=True).cuda()
    batch = _batch(x, 2)

    def step():
        model.zero_grad(set_to_none=True)
        loss = F.nll_loss(model(batch), y)
        loss.backward()
        return loss

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
        eager = [p.grad.clone() for p in model.parameters()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    grads = [p.grad for p in model.parameters()]
    for g in grads:
        g.zero_()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(eager, grads))
    x.mul_(0.5)
    graph.replay()
    assert not all(torch.equal(a, b) for a, b in zip(eager, grads))


@pytest.mark.parametrize("conv", ["gcn", "gin"])
def test_other_blocks(cuda, conv):
    import cxgnncomp
    torch.manual_seed(1)
    model = cxgnncomp.ResidualGNN(conv, 20, 32, 7, 2).cuda()
    out = model(_batch(randn((N, 20), 5).cuda(), 2))
    out.sum().backward()
    assert out.shape == (N, 7) and all(bool(torch.isfinite(p.grad).all()) for p in model.parameters() if p.grad is not None)


@pytest.mark.parametrize("conv,gate,kept8", [("sage", "row", True), ("sage", "value", False), ("gcn", "row", False), ("gcn", None, False),
                                             ("gin", "value", False)])
def test_under_autocast(cuda, conv, gate, kept8):
    import cxgnncomp
    torch.manual_seed(1)
    model = cxgnncomp.ResidualGNN(conv, 20, 32, 7, 2, gate=gate, kept8=kept8).cuda()
    batch = _batch(randn((N, 20), 5).cuda(), 2)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = F.nll_loss(model(batch).float(), torch.zeros(N, dtype=torch.int64, device="cuda"))
    loss.backward()
    grads = [p.grad for p in model.parameters() if p.grad is not None]
    assert len(grads) > 5 and all(g.dtype == torch.float32 and bool(torch.isfinite(g).all()) for g in grads)


def test_features_in_8_bits_on_disk(cuda, tmp_path):
    """The wire format has float32 features: those that the rows hold."""
    import cxgnncomp
    import cxgnncomp_backend as be
    x = randn((N, 20), 5)
    batch = _batch(be.quantize_rows(x.cuda()), 2)
    batch.tofile(str(tmp_path))
    back = cxgnncomp.Batch(None, None, None).fromfile(str(tmp_path), feat_len=20)
    assert back.x.dtype == torch.float32 and torch.equal(back.x.double(), held_values(x)) and torch.equal(back.idx, batch.idx.cpu())
