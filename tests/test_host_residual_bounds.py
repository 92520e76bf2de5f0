"""The bounds that gradients of the step between two blocks are tested with: they are those of the right gradients, and gradients
of zero, or without some of the rows, are outside of them. No GPU is needed."""
import pytest
import torch

from residual_bounds import CASES, EPS, gradients, inputs
from rows8_ref import residual


def _case(case, dtype):
    n, w, gate, post, following, layer, scale = case
    t, dy, dh = inputs(*case[:2], dtype, *case[2:], seed=n + w)
    return t, dy, dh, gradients(t, post, following, layer, dy, dh)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_are_those_of_the_formula(dtype):
    for case in CASES:
        n, w, gate, post, following, layer, scale = case
        t, dy, dh, got = _case(case, dtype)
        ref = {k: None if v is None else v.double().requires_grad_(True) for k, v in t.items()}
        outs = [o for o in residual(ref["x"], ref["f"], ref["gate"], ref["scale"], post, ref["w2"], ref["b2"], following, ref["w1"],
                                    ref["b1"], layer, EPS) if o is not None]
        leaves = [k for k in t if t[k] is not None]
        assert set(leaves) == set(got), case
        want = torch.autograd.grad(outs, [ref[k] for k in leaves], [v.double() for v in (dy, dh) if v is not None])
        for k, v in zip(leaves, want):
            assert got[k][0].shape == v.shape and bool(((got[k][0] - v).abs() <= 1e-10 * (1 + v.abs().max())).all()), (case, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_wrong_gradients_are_outside(dtype):
    for case in CASES:
        for k, (g, bound, terms) in _case(case, dtype)[3].items():
            if k == "f" and case[1] == 1:
                continue  # the norm of one value has no slope
            # zeros: for every element but those that cancel
            assert float((g.abs() > 4 * bound).double().mean()) > 0.8, (case, k)
            if terms is not None:  # without any one row, but the half that adds least
                missing = (terms.sum(1, keepdim=True) if g.numel() == 1 else terms).abs()
                seen = (missing > 2 * bound).any(1).double().mean()
                assert float(seen) > 0.5, (case, k, float(seen))
