"""Gradients of the step between two blocks in float64, term by term, and how far fp32 arithmetic may be from them.

Every quantity q that is computed carries e(q), in units of K * 2^-24: what its own roundings and the errors of what went into it add
up to, from magnitudes that roundings are relative to (sums of absolute values, not results in which terms cancel). With <.> the
mean over a row, u = r (v - <v>) a normalised row:
    e(u) = r (e(v) + <e(v)>) + |u| <|u| r (e(v) + <e(v)>)>       the second part by r' / r = -<u r v'>
    e(p q) = e(p) |q| + |p| e(q) + |p q|,    e(<q>) = <e(q)> + <|q|>
K: a mean over a row is added in at most 3 (packed values of a lane) + 5 (lanes) + 16 (warps) additions, and 8 further roundings go into
any one step (a sigmoid's: 8 and |gate| of 2^-24 of it for bf16 rows, whose exponential takes a product rounded once). K = 32, for
gates of up to 24. A sum over n rows rounds at most n + 16 times, and at most n / 148 + 616 (rows of a lane where each of 148
processors has a block; lanes, warps and up to 592 blocks), relative to the sum of its terms' absolute values."""
import torch

K = 32
EPS = 1e-5
U = 2.0 ** -24


def _mean(v):
    return v.mean(1, keepdim=True)


def _norm(v, ev, layer):
    """(u, r, e(u))"""
    c = v - _mean(v) if layer else v
    r = 1 / torch.sqrt(_mean(c * c) + EPS)
    u = c * r
    own = r * (ev + v.abs() + (_mean(ev + v.abs()) if layer else 0))
    return u, r, own + u.abs() * _mean(u.abs() * own)


def _back(t, et, u, eu, r, layer):
    """r (t - <t> - u <t u>) and its error; r's own relative error is at most <|u| e(u)> + 1."""
    dot, edot = _mean(t * u), _mean(et * u.abs() + t.abs() * eu + (t * u).abs())
    v = t - u * dot - (_mean(t) if layer else 0)
    ev = et + eu * dot.abs() + u.abs() * edot + t.abs() + (u * dot).abs()
    if layer:
        ev = ev + _mean(et + t.abs())
    return r * v, r * (ev + v.abs() * (1 + _mean(u.abs() * eu)))


def gradients(t, post, following, layer, dy, dh):
    """{leaf: (gradient, bound, terms or None)} in float64 for inputs t (a dict as of residual_norm's arguments); dy, dh may be None.
    terms: per row, what is summed for a parameter."""
    d = {k: None if v is None else v.double() for k, v in t.items()}
    n, w = d["x"].shape
    one = torch.ones(w, dtype=torch.float64)
    zero = torch.zeros(n, w, dtype=torch.float64)
    out = {}

    def per_row(k, terms, errors):
        bound = K * U * errors.sum(0) + (min(n, n // 148 + 600) + 16) * U * terms.abs().sum(0)
        if t[k] is not None and t[k].numel() == 1 and w > 1:  # one value for all columns
            out[k] = (terms.sum().view(1), (bound.sum() + w * U * terms.abs().sum()).view(1), terms)
        else:
            g = terms.sum(0)
            out[k] = (g, bound + U * g.abs(), terms)

    def value(k, g, e):
        half = torch.finfo(t[k].dtype).eps / 2
        out[k] = (g, K * U * e * (1 + half) + half * g.abs(), None)

    y, ey = d["x"], d["x"].abs()
    if d["f"] is not None:
        scale = one if d["scale"] is None else d["scale"].expand(w) if d["scale"].numel() == 1 else d["scale"]
        if post:
            u2, r2, eu2 = _norm(d["f"], zero, layer)
            w2, b2 = one if d["w2"] is None else d["w2"], 0 if d["b2"] is None else d["b2"]
            m = u2 * w2 + b2
            em = eu2 * w2.abs() + (u2 * w2).abs() + m.abs()
        else:
            m, em = d["f"], zero
        if d["gate"] is None:
            s, ds = torch.ones(n, 1, dtype=torch.float64), None
        else:
            g = d["gate"].reshape(n, -1)
            s = torch.sigmoid(g)
            ds = s * torch.sigmoid(-g)
        y = d["x"] + scale * s * m
        ey = d["x"].abs() + scale.abs() * s * (em + 3 * m.abs()) + y.abs()
    G, eG = (zero, zero) if dy is None else (dy.double(), zero)
    if following and dh is not None:
        u1, r1, eu1 = _norm(y, ey, layer)
        w1 = one if d["w1"] is None else d["w1"]
        h = dh.double()
        per_row("w1", h * u1, h.abs() * (eu1 + u1.abs()))
        if d["b1"] is not None:
            per_row("b1", h, zero)
        t1 = h * w1
        b, eb = _back(t1, t1.abs(), u1, eu1, r1, layer)
        G, eG = G + b, eG + eb + G.abs() + (G + b).abs()
    value("x", G, eG)
    if d["f"] is not None:
        if d["scale"] is not None:
            per_row("scale", G * s * m, s * (eG * m.abs() + G.abs() * (em + 3 * m.abs())))
        if ds is not None:
            term, e = G * scale * m * ds, scale.abs() * ds * (eG * m.abs() + G.abs() * (em + 4 * m.abs()))
            if d["gate"].shape == d["x"].shape and w > 1:
                value("gate", term, e)
            else:
                value("gate", term.sum(1).reshape(d["gate"].shape), (e + term.abs()).sum(1).reshape(d["gate"].shape))
        dm, edm = G * scale * s, scale.abs() * s * (eG + 3 * G.abs())
        if post:
            if d["w2"] is not None:
                per_row("w2", dm * u2, edm * u2.abs() + dm.abs() * (eu2 + u2.abs()))
            if d["b2"] is not None:
                per_row("b2", dm, edm)
            a = dm * w2
            df, edf = _back(a, edm * w2.abs() + a.abs(), u2, eu2, r2, layer)
            value("f", df, edf)
        else:
            value("f", dm, edm)
    return out


# (rows, width, gate, post, next, layer, scale): every number of lanes and warps of a row, vectors of every width, sums over more rows
# than there are lanes for
CASES = [(n, w, gate, True, True, layer, "vector")
         for n, w in [(7, 3), (33, 47), (70, 64), (65, 128), (700, 16), (500, 20), (300, 256)]
         for gate in ("none", "value", "row") for layer in (False, True)]
CASES += [(n, w, ("value", "row", "none")[i % 3], True, True, i % 2 == 0, "vector")
          for i, (n, w) in enumerate([(300, 8), (33, 32), (40, 200), (30, 257), (20, 512), (9, 520), (9, 768), (7, 769), (9, 1000), (5, 1536),
                                      (7, 1500), (5, 2048), (4, 2500), (3, 4001), (3, 4096), (61, 1), (61, 5), (61, 9), (61, 15), (61, 33),
                                      (61, 63), (61, 129), (61, 255), (9000, 64), (3000, 272), (2600, 520), (2000, 1025)])]
CASES += [(50, w, gate, post, following, layer, scale)
          for w, gate, layer in [(72, "value", True), (75, "row", False)]
          for post, following in [(True, False), (False, True), (False, False)] for scale in ("vector", "one", "none")]


def inputs(n, width, dtype, gate, post, following, layer, scale, seed=0):
    def randn(shape, k, like=torch.float32):
        return torch.randn(shape, generator=torch.Generator().manual_seed(seed * 100 + k)).to(like)

    t = dict.fromkeys(("x", "f", "gate", "scale", "w2", "b2", "w1", "b1"))
    t["x"], t["f"] = randn((n, width), 1, dtype), (randn((n, width), 2) * 3).to(dtype)
    if gate != "none":
        t["gate"] = (randn((n, width if gate == "value" else 1), 3) * 2).to(dtype)
    if scale != "none":
        t["scale"] = randn((width if scale == "vector" else 1,), 4)
    if post:
        t["w2"], t["b2"] = 1 + 0.2 * randn((width,), 5), randn((width,), 6) if layer else None
    if following:
        t["w1"], t["b1"] = 1 + 0.2 * randn((width,), 7), randn((width,), 8) if layer else None
    return t, randn((n, width), 20, dtype), randn((n, width), 21, dtype) if following else None
