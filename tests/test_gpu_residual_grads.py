"""Gradients of the step between two blocks, those of its parameters above all, against float64 within bounds from their terms."""
import pytest
import torch

from residual_bounds import CASES, EPS, gradients, inputs

pytestmark = pytest.mark.gpu


def _run(be, t, post, following, layer, **kw):
    return be.residual_norm(t["x"], t["f"], gate=t["gate"], scale=t["scale"], post=post, post_weight=t["w2"], post_bias=t["b2"],
                            next=following, next_weight=t["w1"], next_bias=t["b1"], norm="layer" if layer else "rms", eps=EPS, **kw)


def _check(t, post, following, layer, dy, dh, place=lambda v: v.cuda()):
    import cxgnncomp_backend as be
    dev = {k: None if v is None else place(v).requires_grad_(True) for k, v in t.items()}
    y, h = _run(be, dev, post, following, layer)
    outs = [(o, d.cuda()) for o, d in ((y, dy), (h, dh)) if d is not None]
    leaves = [k for k in t if t[k] is not None]
    got = torch.autograd.grad([o for o, _ in outs], [dev[k] for k in leaves], [d for _, d in outs], allow_unused=True)
    want = gradients(t, post, following, layer, dy, dh)
    for k, g in zip(leaves, got):
        if k not in want:
            assert g is None or not bool(g.any()), k
            continue
        w, bound, _ = want[k]
        assert g.dtype == t[k].dtype and g.shape == w.shape
        off = (g.double().cpu() - w).abs()
        assert bool((off <= bound).all()), (k, float((off / bound).max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c))
def test_gradients(cuda, case, dtype):
    n, w, gate, post, following, layer, scale = case
    t, dy, dh = inputs(n, w, dtype, gate, post, following, layer, scale, seed=n + w)
    _check(t, post, following, layer, dy, dh)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,width", [(5, 2), (33, 47), (40, 64), (21, 256), (5, 257), (3, 512), (9, 1100)])
def test_matrices_that_start_anywhere(cuda, n, width, dtype):
    def place(v):
        flat = torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")
        flat[1:] = v.flatten().cuda()
        return flat[1:].view(v.shape)

    t, dy, dh = inputs(n, width, dtype, "value", True, True, True, "vector", seed=n)
    _check(t, True, True, True, dy, dh, place)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,width", [(70, 40), (30, 300)])
def test_gradients_of_one_output(cuda, n, width, dtype):
    t, dy, dh = inputs(n, width, dtype, "row", True, True, True, "vector", seed=n)
    _check(t, True, True, True, dy, None)
    _check(t, True, True, True, None, dh)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate", ["value", "row"])
@pytest.mark.parametrize("n,width", [(40, 64), (37, 47), (11, 300)])
def test_gates_far_from_zero(cuda, n, width, gate, dtype):
    """The sigmoid's derivative is as exact on its flat sides as between them."""
    t, dy, dh = inputs(n, width, dtype, gate, True, True, False, "vector", seed=n)
    g = torch.linspace(10, 20, t["gate"].numel()).view(t["gate"].shape)
    t["gate"] = torch.where(t["gate"] > 0, g, -g).to(dtype)
    _check(t, True, True, False, dy, dh)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate", ["none", "value", "row"])
@pytest.mark.parametrize("n,width", [(1, 8), (5, 8), (17, 47), (3, 100), (1, 3)])
def test_an_infinity_in_the_last_row(cuda, n, width, gate, dtype):
    """Lanes that have no row of their own add nothing to the sums over rows, whatever the last row holds."""
    import cxgnncomp_backend as be
    t, dy, _ = inputs(n, width, dtype, gate, False, False, False, "vector", seed=n)
    t["f"][-1, 1], t["f"][-1, 2] = float("inf"), -float("inf")
    dev = {k: None if v is None else v.cuda().requires_grad_(True) for k, v in t.items()}
    y, _ = _run(be, dev, False, False, False)
    got = torch.autograd.grad(y, [dev["scale"]], dy.cuda())[0].cpu()
    s = 1.0 if gate == "none" else torch.sigmoid(t["gate"].double())
    terms = dy.double() * s * t["f"].double()
    want = terms.sum(0)
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and not bool(torch.isnan(got).any())
    assert torch.equal(got[1:3].double(), want[1:3])
    keep = torch.isfinite(want)
    assert bool(((got.double() - want).abs() <= 64 * 2.0 ** -24 * terms.abs().sum(0))[keep].all())
