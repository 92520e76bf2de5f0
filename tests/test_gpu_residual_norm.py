"""The step between two blocks against float64, its gradients too. The longest chain behind a value (a mean and a mean square of
a row by trees of at most 8 + 9 additions, the factor, sigmoid, products) has fewer than 64 roundings of 2^-24, each relative
to the largest value of its row; sums over rows add one per row of a lane and one per block."""
import pytest
import torch

from helpers import randn
from rows8_ref import held_values, residual

pytestmark = pytest.mark.gpu

EPS = 1e-5
NAMES = ("x", "f", "gate", "scale", "w2", "b2", "w1", "b1")


def _inputs(n, width, dtype, gate, post, following, layer, scale="vector", seed=0):
    t = dict.fromkeys(NAMES)
    t["x"], t["f"] = randn((n, width), seed + 1, dtype), (randn((n, width), seed + 2) * 3).to(dtype)
    if gate == "value":
        t["gate"] = (randn((n, width), seed + 3) * 3).to(dtype)
    elif gate in ("row", "rows"):
        t["gate"] = (randn((n, 1) if gate == "row" else (n,), seed + 3) * 3).to(dtype)
    if scale == "vector":
        t["scale"] = randn((width,), seed + 4)
    elif scale == "one":
        t["scale"] = randn((1,), seed + 4)
    if post:
        t["w2"], t["b2"] = 1 + 0.2 * randn((width,), seed + 5), randn((width,), seed + 6) if layer else None
    if following:
        t["w1"], t["b1"] = 1 + 0.2 * randn((width,), seed + 7), randn((width,), seed + 8) if layer else None
    return t


def _run(be, t, post, following, layer, **kw):
    return be.residual_norm(t["x"], t["f"], gate=t["gate"], scale=t["scale"], post=post, post_weight=t["w2"], post_bias=t["b2"],
                            next=following, next_weight=t["w1"], next_bias=t["b1"], norm="layer" if layer else "rms", eps=EPS, **kw)


def _rows_close(got, want, mag):
    """mag: per row, what the roundings are relative to."""
    half = torch.finfo(got.dtype).eps / 2
    return bool(((got.double().cpu() - want).abs() <= half * want.abs() + 64 * 2.0 ** -24 * mag).all())


def _check(n, width, dtype, gate, post, following, layer, scale="vector", place=lambda v: v.cuda()):
    import cxgnncomp_backend as be
    t = _inputs(n, width, dtype, gate, post, following, layer, scale, seed=n + width)
    dev = {k: None if v is None else place(v).requires_grad_(True) for k, v in t.items()}
    ref = {k: None if v is None else v.double().requires_grad_(True) for k, v in t.items()}
    outs = [o for o in _run(be, dev, post, following, layer) if o is not None]
    want = [o for o in residual(ref["x"], ref["f"], ref["gate"], ref["scale"], post, ref["w2"], ref["b2"], following, ref["w1"],
                                ref["b1"], layer, EPS) if o is not None]
    with torch.no_grad():
        plain = [o for o in _run(be, dev, post, following, layer) if o is not None]
    ds = [randn((n, width), 20 + i, dtype) for i in range(len(outs))]
    leaves = [k for k in NAMES if t[k] is not None]
    grads = torch.autograd.grad(outs, [dev[k] for k in leaves], [d.cuda() for d in ds])
    wants = torch.autograd.grad(want, [ref[k] for k in leaves], [d.double() for d in ds])
    # sizes that roundings are relative to: values of a row, and a norm's factor that multiplies errors of what goes in
    y = want[0].detach()
    top = lambda v: v.abs().amax(1, keepdim=True)
    r = lambda v: 1 / torch.sqrt(((v - (v.mean(1, keepdim=True) if layer else 0)) ** 2).mean(1, keepdim=True) + EPS)
    f = t["f"].double()
    gain2 = (1 + r(f) * top(f)) if post else 1 + top(f)
    size = top(t["x"].double()) + (3 * gain2 * (1 + (top(f) if not post else 0)))
    gain1 = 1 + r(y) * size if following else torch.ones(n, 1).double()
    for o, p, w in zip(outs, plain, want):
        assert o.dtype == dtype and torch.equal(o, p)
    assert _rows_close(outs[0], y, 4 * size)
    if following:
        assert _rows_close(outs[1], want[1].detach(), 8 * gain1)
    back = 16 * (1 + (r(y) * gain1 if following else 0)) * (1 + r(f) * gain2 if post else gain2) * (1 + gain2)
    for k, g, w in zip(leaves, grads, wants):
        assert g.dtype == dev[k].dtype and g.shape == dev[k].shape
        if k in ("x", "f", "gate"):
            mag = back * (width if t[k].numel() == n and width > 1 else 1)
            assert _rows_close(g.reshape(n, -1), w.reshape(n, -1), mag), k
        else:
            assert _rows_close(g.reshape(1, -1), w.reshape(1, -1), (back * (1 + size) * 4).sum() * (width if k == "scale" and scale == "one" else 1)), k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("gate", ["none", "value", "row", "rows"])
@pytest.mark.parametrize("n,width", [(1, 1), (7, 3), (33, 47), (70, 64), (65, 128)])
def test_kinds(cuda, n, width, gate, layer, dtype):
    _check(n, width, dtype, gate, True, True, layer)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("post,following", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("scale", ["vector", "one", "none"])
def test_parts(cuda, post, following, scale, dtype):
    _check(50, 72, dtype, "value", post, following, True, scale)
    _check(50, 75, dtype, "row", post, following, False, scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,width", [(700, 16), (300, 8), (500, 20), (33, 32), (40, 200), (300, 256), (30, 257), (20, 512), (9, 1000),
                                     (7, 1500), (9, 768), (9, 520), (7, 769), (5, 1536), (4, 2500), (5, 2048), (3, 4096), (3, 4001)])
def test_widths(cuda, n, width, dtype):
    _check(n, width, dtype, "value", True, True, True)


@pytest.mark.parametrize("width", [1, 5, 7, 9, 15, 17, 31, 33, 63, 65, 127, 129, 255])
def test_odd_rows_of_bf16(cuda, width):
    _check(61, width, torch.bfloat16, "value", True, True, width % 4 == 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,width", [(1, 1), (5, 2), (30, 16), (33, 47), (40, 64), (9, 128), (21, 256), (5, 257), (3, 512), (2, 4096)])
def test_matrices_that_start_anywhere(cuda, n, width, dtype):
    def place(v):
        flat = torch.empty(v.numel() + 1, dtype=v.dtype, device="cuda")
        flat[1:] = v.flatten().cuda()
        return flat[1:].view(v.shape)

    _check(n, width, dtype, "value", True, True, False, place=place)


def test_many_rows(cuda):
    """More rows than the grid holds at once; the sums over rows have the same bits on every run."""
    import cxgnncomp_backend as be
    t = _inputs(60000, 64, torch.float32, "row", True, True, True)
    dev = {k: v.cuda().requires_grad_(True) for k, v in t.items()}
    ref = {k: v.double().requires_grad_(True) for k, v in t.items()}
    leaves = list(dev)
    dy = randn((60000, 64), 30)

    def grads():
        y, h = _run(be, dev, True, True, True)
        return torch.autograd.grad([y, h], [dev[k] for k in leaves], [dy.cuda(), dy.cuda()])

    a, b = grads(), grads()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    y, h = residual(*(ref[k] for k in ("x", "f", "gate", "scale")), True, ref["w2"], ref["b2"], True, ref["w1"], ref["b1"], True, EPS)
    want = torch.autograd.grad([y, h], [ref[k] for k in leaves], [dy.double(), dy.double()])
    for k, g, w in zip(leaves, a, want):
        # random signs: sums over 60000 rows, terms of up to about 10
        assert float((g.double().cpu() - w).abs().max()) <= 60000 * 64 * 2.0 ** -24 * (1 if k in ("scale", "w2", "b2", "w1", "b1") else 0.01), k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,width", [(1, 32), (1, 16), (37, 24), (100, 8), (40, 47), (300, 128), (17, 1000), (9, 768), (5, 1400), (5, 264), (0, 64)])
def test_kept_rows_are_those_of_h(cuda, n, width, dtype):
    import cxgnncomp_backend as be
    t = _inputs(n, width, dtype, "value", True, True, False)
    dev = {k: None if v is None else v.cuda() for k, v in t.items()}
    y, h, rows = _run(be, dev, True, True, False, keep8=True)
    want = be.quantize_rows(h)
    assert torch.equal(rows.codes, want.codes) and torch.equal(rows.scales, want.scales)
    y0, h0 = _run(be, dev, True, True, False)
    assert torch.equal(y, y0) and torch.equal(h, h0)


def test_norm_alone(cuda):
    import cxgnncomp_backend as be
    x, w, dh = randn((40, 96), 1), 1 + 0.1 * randn((96,), 2), randn((40, 96), 3)
    xg, wg = x.cuda().requires_grad_(True), w.cuda().requires_grad_(True)
    y, h = be.residual_norm(xg, next_weight=wg, norm="layer", eps=EPS)
    assert y is xg
    gx, gw = torch.autograd.grad(h, [xg, wg], dh.cuda())
    xr, wr = x.double().requires_grad_(True), w.double().requires_grad_(True)
    _, hr = residual(xr, None, None, None, False, None, None, True, wr, None, True, EPS)
    rx, rw = torch.autograd.grad(hr, [xr, wr], dh.double())
    assert _rows_close(h, hr.detach(), 8 * torch.ones(40, 1)) and _rows_close(gx, rx, 64 * torch.ones(40, 1))
    assert _rows_close(gw.view(1, -1), rw.view(1, -1), 40 * 16 * torch.ones(1, 1))


def test_against_differences(cuda):
    """The gradients against central differences of the function itself (float64 of the same formula is tested above): with a
    step of 2^-6 the cubic term is below 1 % of a gradient of this size, the roundings of fp32 below 1 %."""
    import cxgnncomp_backend as be
    t = _inputs(6, 40, torch.float32, "value", True, True, True)
    dev = {k: v.cuda().requires_grad_(True) for k, v in t.items()}
    dy, dh = randn((6, 40), 30).cuda(), randn((6, 40), 31).cuda()

    def value(**change):
        with torch.no_grad():
            y, h = _run(be, {**{k: v.detach() for k, v in dev.items()}, **change}, True, True, True)
            return float((y.double() * dy).sum() + (h.double() * dh).sum())

    y, h = _run(be, dev, True, True, True)
    grads = dict(zip(dev, torch.autograd.grad([y, h], list(dev.values()), [dy, dh])))
    for k, g in grads.items():
        along = randn(tuple(g.shape), 40).cuda()
        along /= along.norm()
        step = 2.0 ** -6
        got = (value(**{k: dev[k].detach() + step * along}) - value(**{k: dev[k].detach() - step * along})) / (2 * step)
        want = float((g.double() * along).sum())
        assert abs(got - want) <= 0.02 * float(g.double().norm()) / g.numel() ** 0.5 + 0.02 * abs(want) + 1e-3, k


def test_gradients_of_one_output_alone(cuda):
    import cxgnncomp_backend as be
    t = _inputs(50, 64, torch.float32, "none", True, True, False)
    dev = {k: None if v is None else v.cuda().requires_grad_(True) for k, v in t.items()}
    y, h = _run(be, dev, True, True, False)
    zero = torch.zeros_like(y)
    for out, both in ((y, [torch.ones_like(y), zero]), (h, [zero, torch.ones_like(y)])):
        leaves = [dev["x"], dev["f"], dev["w2"], dev["scale"]]
        a = torch.autograd.grad(out, leaves, torch.ones_like(y), retain_graph=True)
        b = torch.autograd.grad([y, h], leaves, both, retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_rows_of_zeros_large_values_and_nan(cuda):
    import cxgnncomp_backend as be
    t = _inputs(6, 64, torch.float32, "value", True, True, False)
    t["f"][1] = 0
    t["x"][2], t["f"][2] = 0, 0
    t["gate"][3, :4] = torch.tensor([100.0, -100.0, 1e30, -float("inf")])
    t["f"][4, 7] = float("nan")
    dev = {k: None if v is None else v.cuda().requires_grad_(True) for k, v in t.items()}
    y, h = _run(be, dev, True, True, False)
    g = torch.autograd.grad([y, h], [dev["x"], dev["f"], dev["gate"]], [torch.ones_like(y)] * 2)
    assert bool((y[2] == 0).all()) and bool((h[2] == 0).all())
    rows = torch.tensor([0, 1, 2, 3, 5])
    for v in (y, h, *g):
        assert bool(torch.isfinite(v[rows.cuda()]).all())
    assert bool(torch.isnan(y[4]).all())
    ref = {k: None if v is None else v.double()[rows] if v.dim() == 2 else v.double() for k, v in t.items()}
    yr, _ = residual(ref["x"], ref["f"], ref["gate"], ref["scale"], True, ref["w2"], None, True, ref["w1"], None, False, EPS)
    assert _rows_close(y[rows.cuda()].detach(), yr, 16 * torch.ones(5, 1) * (1 + ref["x"].abs().amax()))


def test_bf16_parameters_no_rows_and_views(cuda):
    import cxgnncomp_backend as be
    t = _inputs(30, 64, torch.bfloat16, "value", True, True, False)
    dev = {k: None if v is None else v.cuda() for k, v in t.items()}
    w = dev["w1"].bfloat16().requires_grad_(True)
    y, h = be.residual_norm(dev["x"], dev["f"], next_weight=w, post=False)
    h.float().sum().backward()
    assert w.grad.dtype == torch.bfloat16 and bool(torch.isfinite(w.grad.float()).all())
    xe = torch.empty(0, 64, device="cuda", requires_grad=True)
    we = torch.ones(64, device="cuda", requires_grad=True)
    y, h = be.residual_norm(xe, xe, next_weight=we)
    (y.sum() + h.sum()).backward()
    assert y.shape == (0, 64) and not bool(we.grad.any())
    wide = randn((30, 130), 9).cuda()
    a = be.residual_norm(wide[:, 1:65], wide[:, 65:129])
    b = be.residual_norm(wide[:, 1:65].contiguous(), wide[:, 65:129].contiguous())
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_under_autocast(cuda):
    """f and gate are taken in x's type; without autocast they have to be of it."""
    import cxgnncomp_backend as be
    x, f, gate = randn((50, 48), 1).cuda().bfloat16(), randn((50, 48), 2).cuda().requires_grad_(True), randn((50,), 3).cuda()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y, h = be.residual_norm(x, f, gate=gate)
    want = be.residual_norm(x, f.detach().bfloat16(), gate=gate.bfloat16())
    assert torch.equal(y, want[0]) and torch.equal(h, want[1])
    h.sum().backward()
    assert f.grad.dtype == torch.float32
    with pytest.raises(RuntimeError, match="f must be of x's type"):
        be.residual_norm(x, f)
