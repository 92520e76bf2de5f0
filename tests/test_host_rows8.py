"""What the entry points of rows in 8 bits and of the step between two blocks refuse before any CUDA call, and the sizes of
scratch they ask for: no GPU is needed."""
import ctypes

import pytest
import torch

vp, i64, ci, sz, fl, u32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t, ctypes.c_float, ctypes.c_uint32
EINVAL, ENULL, EUNSUPPORTED, EWORKSPACE, ELIMIT = -1, -2, -3, -5, -7
P = 4096  # stands for a device address: none of these calls reads it


def _fn(name, types):
    import cxgnncomp_backend as be
    fn = getattr(be._lib, name)
    fn.argtypes, fn.restype = types, ci
    return fn


def test_write_and_read():
    write = _fn("cxg_rows8_write", [vp, ci, i64, i64, ci, vp, vp, ci, vp])
    assert write(P, 0, 40, 10, 40, None, P, 1, None) == ENULL
    assert write(P, 2, 40, 10, 40, P, P, 1, None) == EINVAL  # no such type
    assert write(P, 0, 39, 10, 40, P, P, 1, None) == EINVAL  # rows overlap
    assert write(P, 0, 40, -1, 40, P, P, 1, None) == EINVAL
    assert write(P, 0, 0, 10, 0, P, P, 1, None) == EINVAL
    assert write(P, 0, 40, 10, 40, P + 8, P, 1, None) == EINVAL  # codes off their alignment
    assert write(None, 0, 40, 0, 40, None, None, 0, None) == 0   # nothing to do
    at = _fn("cxg_rows8_write_at", [vp, ci, i64, i64, ci, vp, vp, vp, i64, vp, vp])
    assert at(P, 0, 40, 10, 40, None, P, P, 5, P, None) == ENULL
    assert at(P, 0, 40, 10, 40, P, P, P, 5, None, None) == ENULL
    assert at(P, 0, 40, 10, 40, P, P, P, 5, P + 4, None) == EINVAL
    assert at(P, 0, 40, 2 ** 31, 40, P, P, P, 5, P, None) == ELIMIT
    assert at(P, 0, 40, 0, 40, None, None, None, 5, None, None) == 0
    read = _fn("cxg_rows8_read", [vp, vp, i64, ci, vp, i64, vp, ci, i64, vp])
    assert read(P, P, 5, 40, None, 6, P, 0, 40, None) == EINVAL  # more rows than there are
    assert read(P, P, 5, 40, None, 5, None, 0, 40, None) == ENULL
    assert read(P, P, 5, 40, None, 0, None, 1, 40, None) == 0
    pitch = _fn("cxg_rows8_pitch", [ci])
    assert [pitch(w) for w in (1, 32, 33, 47, 100, 128)] == [32, 32, 64, 64, 128, 128]


def test_aggregate():
    size = _fn("cxg_rows8_aggregate_workspace_size", [i64, ci, ci, ctypes.POINTER(sz)])
    need = sz(0)
    assert size(100000, 128, 0, ctypes.byref(need)) == 0 and need.value > 0
    assert size(100000, 2049, 0, ctypes.byref(need)) == EUNSUPPORTED
    assert size(-1, 128, 0, ctypes.byref(need)) == EINVAL
    call = _fn("cxg_rows8_aggregate", [vp, vp, i64, ci, vp, ci, vp, ci, vp, i64, i64, ci, ci, vp, ci, vp, sz, vp])

    def args(**change):
        a = dict(codes=P, scales=P, n_src=10, width=64, ptr=P, pb=8, idx=P, ib=8, ev=None, n_dst=10, nnz=20, reduce=0, split=0, y=P,
                 dtype=0, ws=P, bytes=1 << 30, st=None)
        a.update(change)
        return list(a.values())

    for change, want in [(dict(codes=None), ENULL), (dict(y=None), ENULL), (dict(idx=None), ENULL), (dict(pb=2), EINVAL),
                         (dict(dtype=2), EINVAL), (dict(reduce=1, ev=P), EINVAL), (dict(reduce=2), EINVAL), (dict(width=3000), EUNSUPPORTED),
                         (dict(nnz=2 ** 31 - 1), ELIMIT), (dict(n_dst=2 ** 31), ELIMIT), (dict(n_src=2 ** 32), ELIMIT),
                         (dict(bytes=16), EWORKSPACE), (dict(ws=None), EWORKSPACE), (dict(n_dst=0, y=None), 0), (dict(codes=P + 4), EINVAL)]:
        assert call(*args(**change)) == want, change


def test_weight_grad():
    size = _fn("cxg_rows8_wgrad_workspace_size", [i64, ci, ci, ctypes.POINTER(sz)])
    need = sz(0)
    assert size(1000, 100, 47, ctypes.byref(need)) == 0 and need.value >= 16 * 128 * 128 * 4
    assert size(1000, 0, 47, ctypes.byref(need)) == EINVAL
    call = _fn("cxg_rows8_wgrad", [vp, vp, i64, ci, vp, ci, i64, ci, u32, vp, vp, ci, vp, sz, vp])
    assert call(P, P, 1000, 100, P, 0, 47, 47, 0, None, None, 0, P, 1 << 30, None) == ENULL
    assert call(P, P, 1000, 100, P, 0, 46, 47, 0, P, None, 0, P, 1 << 30, None) == EINVAL
    assert call(P, P, 1000, 100, P, 3, 47, 47, 0, P, None, 0, P, 1 << 30, None) == EINVAL
    assert call(P, P, 1000, 100, None, 0, 47, 47, 0, P, None, 0, P, 1 << 30, None) == ENULL
    assert call(P, P, 1000, 100, P, 0, 47, 47, 0, P, None, 0, P, 100, None) == EWORKSPACE
    assert call(P, P, 1000, 60000, P, 0, 60000, 60000, 0, P, None, 0, P, 1 << 60, None) == EUNSUPPORTED
    assert call(P, P, 1000, 100, P, 0, 47, 47, 0, P, None, 2, P, 1 << 30, None) == EINVAL


def test_residual_norm():
    import cxgnncomp_backend as be

    class Desc(ctypes.Structure):
        _fields_ = ([(n, vp) for n in ("x", "f", "gate", "scale", "w2", "b2", "w1", "b1", "y", "h", "codes", "scales", "dy", "dh", "dx", "df", "dgate")]
                    + [("n", i64)] + [(n, ctypes.c_int32) for n in ("width", "dtype", "gate_mode", "layer", "post", "next")] + [("eps", fl)])

    fwd = _fn("cxg_residual_norm_forward", [ctypes.POINTER(Desc), vp])
    bwd = _fn("cxg_residual_norm_backward", [ctypes.POINTER(Desc), vp, vp, sz, vp])
    size = _fn("cxg_residual_norm_backward_workspace_size", [i64, ci, ctypes.POINTER(sz)])
    most = _fn("cxg_residual_norm_max_width", [])()

    def desc(**change):
        d = Desc(x=P, f=P, y=P, h=P, n=10, width=64, post=1, next=1, eps=1e-5)
        for k, v in change.items():
            setattr(d, k, v)
        return ctypes.byref(d)

    assert fwd(None, None) == ENULL
    for change, want in [(dict(x=None), ENULL), (dict(h=None), ENULL), (dict(gate_mode=1), ENULL), (dict(gate_mode=3), EINVAL),
                         (dict(width=most + 1), EUNSUPPORTED), (dict(width=0), EINVAL), (dict(eps=-1.0), EINVAL), (dict(dtype=2), EINVAL),
                         (dict(f=None), EINVAL), (dict(f=None, post=0, next=0), EINVAL), (dict(codes=P, scales=P, next=0), EINVAL),
                         (dict(codes=P, scales=P, width=63), EINVAL), (dict(n=0), 0)]:
        assert fwd(desc(**change), None) == want, change
    assert bwd(desc(), None, P, 1 << 30, None) == ENULL
    assert bwd(desc(), P, P, 16, None) == EWORKSPACE
    need = sz(0)
    assert size(1000, most + 1, ctypes.byref(need)) == EUNSUPPORTED
    assert size(10 ** 9, 256, ctypes.byref(need)) == 0 and need.value <= 148 * 16 * 5 * 256 * 4
    assert be._lib.cxg_residual_norm_keeps(desc()) == 1


def test_tensors_on_the_cpu_are_refused():
    import cxgnncomp_backend as be
    x = torch.randn(4, 32)
    for call in (lambda: be.quantize_rows(x), lambda: be.Rows8(4, 32, "cpu"), lambda: be.linear_kept8(x, x), lambda: be.residual_norm(x, x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(TypeError, match="Rows8"):
        be.dequantize_rows(x)
    with pytest.raises(TypeError, match="Rows8"):
        be.quantize_rows(x, out=x)
    with pytest.raises(RuntimeError, match="out"):
        be.quantize_rows(x, index=torch.arange(4))
    with pytest.raises(RuntimeError, match="norm must be"):
        be.residual_norm(x, x, norm="batch")
