"""Rows held in 8 bits and what reads them: caches of features or hidden states, activations kept for a backward pass, and the
step between two blocks of a residual network. None of it is in the reference.

A row is held in groups of 32 values: a power of two s per group and a whole number of -127 .. 127 per value. s is the smallest
with max|x| / s < 127.5 (from 2^-126 to 2^121), so a value is off by at most s / 2, at most 2^-7 of its group's largest; rounding
is to nearest, ties to even. What is held is exact in float32 and bfloat16. A group with a value that is not finite reads as
NaN throughout."""
import torch

from . import _native


class Rows8:
    """`rows` rows of `width` values in 8 bits on a CUDA device, zeros at first: pitch + pitch / 32 bytes a row, pitch being
    `width` in whole groups of 32, and four more from the first write at an index on. quantize_rows writes them, dequantize_rows,
    rows8_aggregate and rows8_weight_grad read them."""
    __slots__ = ("rows", "width", "codes", "scales", "_claims")

    def __init__(self, rows, width, device="cuda"):
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.rows, self.width = int(rows), int(width)
        self.codes, self.scales = _native.rows8_zeros(self.rows, self.width, device)
        self._claims = None

    @classmethod
    def _of(cls, codes, scales, width):
        """codes [rows + 1, pitch] and scales [rows + 1, pitch / 32], the last row of zeros."""
        r = cls.__new__(cls)
        r.rows, r.width, r.codes, r.scales, r._claims = codes.shape[0] - 1, width, codes, scales, None
        return r

    def __getstate__(self):
        return {"rows": self.rows, "width": self.width, "codes": self.codes, "scales": self.scales}

    def __setstate__(self, state):
        state = state[1] if isinstance(state, tuple) else state  # (as it was saved when the words went with it)
        self.rows, self.width, self.codes, self.scales = (state[k] for k in ("rows", "width", "codes", "scales"))
        self._claims = None  # between two calls they hold nothing

    @property
    def shape(self):
        return torch.Size((self.rows, self.width))

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self):
        return self.codes.numel() + self.scales.numel() + (0 if self._claims is None else self._claims.nbytes)

    def __len__(self):
        return self.rows

    def __repr__(self):
        return f"Rows8({self.rows}, {self.width}, device='{self.device}')"

    def _claimed(self):
        """A word per row, by which writes at an index find the last of equal ids."""
        if self._claims is not None:
            return self._claims
        claims = torch.zeros((max(self.rows, 1),), dtype=torch.int32, device=self.device)
        # not what a capture fills when its graph runs; and other streams must not come before the fill
        if not _native.capturing(self.device.index):
            torch.cuda.current_stream(self.device).synchronize()
            self._claims = claims
        return claims


def _rows8(rows, who):
    if not isinstance(rows, Rows8):
        raise TypeError(f"{who}: rows must be a Rows8")
    return rows


def quantize_rows(x, out=None, index=None):
    """The rows of x (float32 or bfloat16 [n, width]) in 8 bits, as a new Rows8; with `out` into its first n rows, with `out`
    and `index` (int64 [n]) row i into row index[i]. Of equal ids the last counts, ids outside out's rows are left out, all
    other rows stay as they are. No gradient goes through."""
    if out is None:
        if index is not None:
            raise RuntimeError("quantize_rows: an index needs the rows it points into (out)")
        codes, scales = _native.rows8_quantize(x)
        return Rows8._of(codes, scales, x.shape[1])
    _rows8(out, "quantize_rows")
    _native.rows8_quantize_into(x, out.codes, out.scales, out.width, index, None if index is None else out._claimed())
    return out


def dequantize_rows(rows, index=None, dtype=torch.float32, num_rows=None):
    """The values of all rows, of the first num_rows, or of rows[index[i]] (int64 [n]; ids outside the rows give zeros), in
    float32 or bfloat16."""
    _rows8(rows, "dequantize_rows")
    if index is not None and num_rows is not None:
        raise RuntimeError("dequantize_rows: either an index or a number of rows")
    return _native.rows8_dequantize(rows.codes, rows.scales, rows.width, index, dtype, rows.rows if num_rows is None else int(num_rows))


def rows8_aggregate(rows, ptr, idx, num_node, reduce="sum", edge_value=None, dtype=torch.float32):
    """out[d] = sum (or mean) over row d of the graph of [edge_value[e] *] rows[idx[e]], [num_node, width] in `dtype`: the
    aggregations of this module over rows in 8 bits, summed in float32 in edge order. ptr ascends from 0; num_node = 0 means all
    rows of ptr, rows without edges give 0, an id outside the rows counts as a row of zeros. Rows and edge values are constants:
    no gradient. Rows of up to 2048 values."""
    from . import SPLIT_EDGES
    _rows8(rows, "rows8_aggregate")
    if reduce not in ("sum", "mean"):
        raise RuntimeError(f"rows8_aggregate: reduce must be 'sum' or 'mean', not {reduce!r}")
    return _native.rows8_aggregate(rows.codes, rows.scales, rows.width, ptr, idx, int(num_node), reduce == "mean", edge_value,
                                   dtype, SPLIT_EDGES)


def rows8_weight_grad(rows, grad, bias=False):
    """grad^T . rows (float32 [out, width]) for grad [n, out] and the first n rows: the gradient of a weight [out, width] from
    the layer's input in 8 bits; with bias=True (that, the sum of grad's rows, float32 [out]). Summed in a fixed order; no gradient
    goes through."""
    _rows8(rows, "rows8_weight_grad")
    dw, db = _native.rows8_weight_grad(rows.codes, rows.scales, rows.width, grad, bool(bias))
    return (dw, db) if bias else dw


def linear_kept8(x, weight, bias=None, add=None, kept=None, same_bits=False):
    """x @ weight^T (+ bias) (+ add) for x [n, in] and weight [out, in], all float32 or all bfloat16, whose backward pass keeps x
    in 8 bits instead of x itself: result and x's gradient are those of `linear` (same_bits as there; the products of bfloat16 are
    torch's), the weight's gradient that of the rows in 8 bits. kept: rows in 8 bits whose first n are x, where the caller has them
    already (not to be written before the backward pass). Once differentiable."""
    if kept is not None:
        _rows8(kept, "linear_kept8")
        if kept.width != x.shape[-1]:
            raise RuntimeError("linear_kept8: kept must hold the rows of x")
    return _native.linear_kept8(x, weight, bias, add, None if kept is None else kept.codes, None if kept is None else kept.scales,
                                bool(same_bits))


def residual_norm(x, f=None, gate=None, scale=None, post=True, post_weight=None, post_bias=None, next=True, next_weight=None,
                  next_bias=None, norm="rms", eps=1e-5, keep8=False):
    """(y, h) of the step between two blocks of a residual network, row by row, in one pass:

        n = norm(f) * post_weight + post_bias        (f itself with post=False)
        y = x + scale * sigmoid(gate) * n
        h = norm(y) * next_weight + next_bias        (None with next=False)

    x, f: float32 or bfloat16 [n, width], width up to 4096. gate: [n, width], or [n] or [n, 1], or None (a factor of 1). scale:
    [width] or one value. norm: "rms" (v / sqrt(mean v^2 + eps)) or "layer" (the mean taken off first). Parameters may be of
    any floating type and count as float32; missing ones are 1 or 0. Under autocast f and gate are taken in x's type. Without
    f: (x, norm of x). With keep8=True the result is (y, h, quantize_rows(h)), in the same pass. Differentiable once in
    everything but the rows in 8 bits."""
    if norm not in ("rms", "layer"):
        raise RuntimeError(f"residual_norm: norm must be 'rms' or 'layer', not {norm!r}")
    y, h, codes, scales = _native.residual_norm(x, f, gate, scale, bool(post), post_weight, post_bias, bool(next), next_weight,
                                                next_bias, norm == "layer", float(eps), bool(keep8))
    return (y, h, Rows8._of(codes, scales, x.shape[1])) if keep8 else (y, h)
