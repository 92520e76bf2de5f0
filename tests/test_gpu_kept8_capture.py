"""Steps that are captured the way torch's documentation does it: a few eager ones on a side stream, whose loss stays alive, then
the capture."""
import pytest
import torch

from helpers import random_csr, randn

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:The AccumulateGrad node")]


def _captured(step, params):
    """The gradients of an eager step and of the same step captured and replayed."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            for p in params:
                p.grad = None
            loss = step()
            loss.backward()
    torch.cuda.current_stream().wait_stream(side)
    eager = [p.grad.clone() for p in params]
    for p in params:
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
        captured.backward()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(loss, captured)
    return eager, [p.grad for p in params]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_operators(cuda, dtype):
    import cxgnncomp_backend as be
    x, f = randn((300, 64), 1, dtype).cuda(), randn((300, 64), 2, dtype).cuda()
    w, b = randn((32, 64), 3, dtype).cuda().requires_grad_(True), randn((32,), 4, dtype).cuda().requires_grad_(True)
    scale, w1 = torch.ones(64, device="cuda", requires_grad=True), torch.ones(64, device="cuda", requires_grad=True)

    def step():
        y, h, rows = be.residual_norm(x, f, scale=scale, next_weight=w1, keep8=True)
        return be.linear_kept8(h, w, b, kept=rows).float().square().sum() + y.float().sum()

    eager, got = _captured(step, [w, b, scale, w1])
    assert all(torch.equal(a, c) for a, c in zip(eager, got))


def test_a_model(cuda):
    import cxgnncomp
    ptr, idx = (t.cuda() for t in random_csr(500, 500, 6, seed=1))
    torch.manual_seed(1)
    model = cxgnncomp.ResidualGNN("sage", 24, 32, 7, 2, norm="layer", gate="row", kept8=True).cuda()
    batch = cxgnncomp.Batch(randn((500, 24), 5).cuda(), ptr, idx, num_node_in_layer=[500] * 3, num_edge_in_layer=[idx.shape[0]] * 2)
    y = torch.randint(0, 7, (500,), generator=torch.Generator().manual_seed(6)).cuda()
    eager, got = _captured(lambda: torch.nn.functional.nll_loss(model(batch), y), list(model.parameters()))
    assert all(torch.equal(a, c) for a, c in zip(eager, got))
