"""Model stacks over the CSR_Layer format: the `forward_cxg` branches of the reference's model zoo
(cxgnncomp/model.py:55-71,166-191,251-273) without its DGL / PyG branches."""
import torch
import torch.nn.functional as F

import cxgnncomp_backend

from .graph_conv import Linear, _plain, MyGATConv, MyGCNConv, MyGINConv, MyRGCNConv, MySageConv


def get_conv_from_str(name, in_channels, out_channels, num_heads=1, num_rel=1, concat=False):
    name = name.upper()
    if name == "SAGE":
        return MySageConv(in_channels, out_channels)
    if name == "GCN":
        return MyGCNConv(in_channels, out_channels)
    if name == "GIN":
        return MyGINConv(in_channels, out_channels)
    if name == "GAT":
        return MyGATConv(in_channels, out_channels, heads=num_heads, concat=concat)
    if name == "RGCN":
        return MyRGCNConv(in_channels, out_channels, num_rel)
    raise ValueError(f"unknown model {name}")


class GNN(torch.nn.Module):
    """conv -> BatchNorm -> ReLU -> dropout per hidden layer, log_softmax at the end (model.py:17-71)."""

    def __init__(self, conv, in_channels, hidden_channels, out_channels, num_layers, dropout=0.5, num_heads=1,
                 num_rel=1):
        super().__init__()
        self.conv_name = conv.upper()
        self.num_layers = num_layers
        self.dropout = dropout
        self.num_rel = num_rel
        dims = [in_channels] + [hidden_channels] * (num_layers - 1) + [out_channels]
        self.convs = torch.nn.ModuleList()
        self.bns = torch.nn.ModuleList()
        for i in range(num_layers):
            concat = self.conv_name == "GAT" and i < num_layers - 1
            width = dims[i + 1] // num_heads if concat else dims[i + 1]
            self.convs.append(get_conv_from_str(conv, dims[i], width, num_heads, num_rel, concat))
            if i < num_layers - 1:
                self.bns.append(torch.nn.BatchNorm1d(dims[i + 1]))

    def reset_parameters(self):
        for c in self.convs:
            c.reset_parameters()
        for b in self.bns:
            b.reset_parameters()

    def forward(self, batch, edge_types=None):
        return self.forward_cxg(batch, edge_types)

    def forward_cxg(self, batch, edge_types=None):
        x = batch.x
        L = self.num_layers
        for i, conv in enumerate(self.convs):
            num_node = int(batch.num_node_in_layer[L - 1 - i])
            num_edge = int(batch.num_edge_in_layer[L - 1 - i]) if batch.num_edge_in_layer is not None else batch.idx.shape[0]
            if self.conv_name == "GAT":
                x = conv(x, batch.ptr, batch.idx, num_node, int(batch.num_node_in_layer[L - i]), num_edge)
            elif self.conv_name == "RGCN":
                x = conv(x, batch.ptr[:num_node + 1], batch.idx[:num_edge], edge_types[:num_edge], num_node)
            else:
                x = conv(x, batch.ptr[:num_node + 1], batch.idx[:num_edge], num_node)
            if i != L - 1:
                x = F.dropout(F.relu(self.bns[i](x)), p=self.dropout, training=self.training)
        return x.log_softmax(dim=-1)


class ResidualGNN(torch.nn.Module):
    """A deep stack of residual SAGE, GCN or GIN blocks, for which the reference has no counterpart:

        x = W_in features;   per block: f = relu(conv(norm(x))),  x = x + scale * sigmoid(gate) * norm(f);   W_out norm(x)

    norm: "rms" or "layer", between two blocks both norms, the gate and the sum in one pass (cxgnncomp_backend.residual_norm).
    gate: None, "row" (one per node) or "value" (one per node and channel), a linear function of the block's input. kept8: what
    the SAGE blocks' and the gates' transforms read is kept in 8 bits for the backward pass; the result has the same bits as
    without. batch.x may be a cxgnncomp_backend.Rows8, which with kept8 is not to be written before the backward pass.
    log_softmax at the end."""

    def __init__(self, conv, in_channels, hidden_channels, out_channels, num_layers, norm="rms", gate=None, kept8=False, dropout=0.0):
        super().__init__()
        self.conv_name = conv.upper()
        if self.conv_name not in ("SAGE", "GCN", "GIN"):
            raise ValueError(f"ResidualGNN: blocks of {conv}")
        if gate not in (None, "row", "value"):
            raise ValueError(f"ResidualGNN: gate must be None, 'row' or 'value', not {gate!r}")
        if norm not in ("rms", "layer"):
            raise ValueError(f"ResidualGNN: norm must be 'rms' or 'layer', not {norm!r}")
        if kept8 and self.conv_name != "SAGE":
            raise ValueError("ResidualGNN: kept8 is there for SAGE blocks")
        self.num_layers, self.norm, self.gate, self.kept8, self.dropout = num_layers, norm, gate, kept8, dropout
        hid = hidden_channels
        self.lin_in = Linear(in_channels, hid)
        self.lin_out = Linear(hid, out_channels)
        make = (lambda: MySageConv(hid, hid, kept8=kept8)) if self.conv_name == "SAGE" else (lambda: get_conv_from_str(conv, hid, hid))
        self.convs = torch.nn.ModuleList(make() for _ in range(num_layers))
        self.gates = torch.nn.ModuleList(Linear(hid, 1 if gate == "row" else hid) for _ in range(num_layers if gate else 0))

        def vectors(n, value):
            return torch.nn.ParameterList(torch.nn.Parameter(torch.full((hid,), float(value))) for _ in range(n))

        layer = norm == "layer"
        self.scale = vectors(num_layers, 1.0)
        self.post_weight, self.post_bias = vectors(num_layers, 1.0), vectors(num_layers if layer else 0, 0.0)
        self.next_weight, self.next_bias = vectors(num_layers + 1, 1.0), vectors(num_layers + 1 if layer else 0, 0.0)

    def reset_parameters(self):
        for m in (self.lin_in, self.lin_out, *self.convs, *self.gates):
            m.reset_parameters()
        with torch.no_grad():
            for ones in (self.scale, self.post_weight, self.next_weight):
                for p in ones:
                    p.fill_(1.0)
            for zeros in (self.post_bias, self.next_bias):
                for p in zeros:
                    p.zero_()

    def forward(self, batch):
        L, layer = self.num_layers, self.norm == "layer"
        x = batch.x
        keep = self.kept8 and torch.is_grad_enabled()
        if isinstance(x, cxgnncomp_backend.Rows8):
            values = cxgnncomp_backend.dequantize_rows(x, dtype=self.lin_in.weight.dtype)
            # the rows hold what is multiplied: the backward pass reads them (rows made in inference mode cannot be kept for one)
            of_rows = keep and _plain(self.lin_in) and not x.codes.is_inference()
            x = (cxgnncomp_backend.linear_kept8(values, self.lin_in.weight, self.lin_in.bias, kept=x, same_bits=True) if of_rows
                 else self.lin_in(values))
            del values
        else:
            x = self.lin_in(x)

        def step(i, x, f, gate):
            """The step in front of block i, or behind the last one."""
            return cxgnncomp_backend.residual_norm(
                x, f, gate=gate, scale=self.scale[i - 1] if i > 0 else None, post_weight=self.post_weight[i - 1] if i > 0 else None,
                post_bias=self.post_bias[i - 1] if i > 0 and layer else None, next_weight=self.next_weight[i],
                next_bias=self.next_bias[i] if layer else None, norm=self.norm, keep8=keep and i < L)

        x, h, *rows = step(0, x, None, None)
        for i, conv in enumerate(self.convs):
            n = int(batch.num_node_in_layer[L - 1 - i])
            e = int(batch.num_edge_in_layer[L - 1 - i]) if batch.num_edge_in_layer is not None else batch.idx.shape[0]
            ptr, idx, kept = batch.ptr[:n + 1], batch.idx[:e], {"kept": rows[0]} if rows else {}
            f = F.dropout(F.relu(conv(h, ptr, idx, n, **kept)), p=self.dropout, training=self.training)
            if n != x.shape[0]:  # (the gradient of a slice is a copy into zeros)
                x, h = x[:n], h[:n]
            gate = None
            if self.gate is not None:
                lin = self.gates[i]
                gate = cxgnncomp_backend.linear_kept8(h, lin.weight, lin.bias, same_bits=True, **kept) if rows else lin(h)
            x, h, *rows = step(i + 1, x, f, gate)
        return self.lin_out(h).log_softmax(dim=-1)


def SAGE(in_c, hid, out_c, num_layers, dropout=0.5):
    return GNN("SAGE", in_c, hid, out_c, num_layers, dropout)


def GCN(in_c, hid, out_c, num_layers, dropout=0.5):
    return GNN("GCN", in_c, hid, out_c, num_layers, dropout)


def GIN(in_c, hid, out_c, num_layers, dropout=0.5):
    return GNN("GIN", in_c, hid, out_c, num_layers, dropout)


def GAT(in_c, hid, out_c, num_layers, heads=4, dropout=0.5):
    return GNN("GAT", in_c, hid, out_c, num_layers, dropout, num_heads=heads)


def RGCN(in_c, hid, out_c, num_layers, num_rel, dropout=0.5):
    return GNN("RGCN", in_c, hid, out_c, num_layers, dropout, num_rel=num_rel)


def get_model_from_str(name, in_c, hid, out_c, num_layers, num_heads=1, num_rel=1, dropout=0.5):
    return GNN(name, in_c, hid, out_c, num_layers, dropout, num_heads=num_heads, num_rel=num_rel)
