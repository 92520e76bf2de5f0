"""The residual stack's arguments; no GPU is needed."""
import pytest


def test_arguments():
    import cxgnncomp
    model = cxgnncomp.ResidualGNN("sage", 10, 16, 3, 2, norm="layer", gate="row", kept8=True)
    assert len(model.convs) == 2 and all(c.kept8 for c in model.convs) and len(model.next_bias) == 3
    model.reset_parameters()
    assert float(model.scale[0].detach().min()) == 1.0 and float(model.next_bias[2].detach().abs().max()) == 0.0
    assert not list(cxgnncomp.ResidualGNN("gin", 10, 16, 3, 2).next_bias)
    for kw in (dict(conv="gat"), dict(conv="sage", gate="all"), dict(conv="sage", norm="batch"), dict(conv="gcn", kept8=True)):
        with pytest.raises(ValueError, match="ResidualGNN"):
            cxgnncomp.ResidualGNN(in_channels=4, hidden_channels=4, out_channels=2, num_layers=1, **kw)
