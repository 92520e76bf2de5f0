"""Writes by id: of equal ids the last counts, whatever other calls on the cache do to rows of their own."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

vp, i64, ci = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int


def _last_rows(n_rows, ids, x):
    want = torch.zeros(n_rows, x.shape[1])
    for i, r in enumerate(ids.tolist()):
        if 0 <= r < n_rows:
            want[r] = x[i]
    return want


@pytest.mark.parametrize("left", [0, -1, -2 ** 31, -2 ** 31 + 700])
@pytest.mark.parametrize("width", [1, 47, 300])
def test_no_state_that_a_call_leaves_is_above_a_later_call(cuda, width, left):
    """A word is zero before the first call and negative behind one; the next call's positions are above all of these."""
    import cxgnncomp_backend as be
    fn = be._sig("cxg_rows8_write_at", [vp, ci, i64, i64, ci, vp, vp, vp, i64, vp, vp])
    rows, n = 200, 700
    cache = be.Rows8(rows, width)
    words = torch.full((rows,), left, dtype=torch.int32, device="cuda")
    touched = torch.zeros(rows, dtype=torch.bool)
    want = torch.zeros(rows, width)
    for call in range(3):
        m = n if call == 0 else 300  # later calls with smaller positions than those that won before
        gen = torch.Generator().manual_seed(call)
        ids = torch.randint(-2, rows + 2, (m,), generator=gen)
        x = (torch.arange(m) % 127 + 1).float().unsqueeze(1).expand(m, width).contiguous()  # whole numbers: exact
        xg, ig = x.cuda(), ids.cuda()
        assert fn(xg.data_ptr(), 0, width, m, width, ig.data_ptr(), cache.codes.data_ptr(), cache.scales.data_ptr(), rows,
                  words.data_ptr(), None) == 0
        ok = ids[(ids >= 0) & (ids < rows)]
        touched[ok] = True
        new = _last_rows(rows, ids, x)
        want[ok.unique()] = new[ok.unique()]
        assert torch.equal(be.dequantize_rows(cache).cpu(), want)
        got = words.cpu()
        assert bool((got[touched] < 0).all()) and bool((got[~touched] == left).all())


def test_calls_on_two_streams_that_write_different_rows(cuda):
    import cxgnncomp_backend as be
    rows, n, width = 60000, 150000, 8
    cache = be.Rows8(rows, width)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    calls = []
    for s in range(2):
        gen = torch.Generator().manual_seed(s)
        for c in range(4):
            ids = torch.randint(0, rows // 2, (n,), generator=gen) * 2 + s  # even rows, odd rows
            x = torch.randint(-127, 128, (n, 1), generator=gen).float().expand(n, width).contiguous()
            last = torch.full((rows,), -1, dtype=torch.int64).scatter_reduce_(0, ids, torch.arange(n), "amax")
            calls.append((s, x, x.cuda(), ids.cuda(), last))
    cache._claimed()
    want = torch.zeros(rows, width)
    torch.cuda.synchronize()
    for turn in range(12):
        order = [calls[turn % 4], calls[4 + (turn + 1) % 4]]
        for s, x, xg, ig, last in order:
            with torch.cuda.stream(streams[s]):
                for _ in range(2):
                    be.quantize_rows(xg, out=cache, index=ig)
        torch.cuda.synchronize()
        for s, x, xg, ig, last in order:
            at = (last >= 0).nonzero().squeeze(1)
            want[at] = x[last[at]]
        assert torch.equal(be.dequantize_rows(cache).cpu(), want), turn


def test_a_cache_without_rows(cuda):
    import cxgnncomp_backend as be
    cache = be.Rows8(0, 40)
    be.quantize_rows(torch.ones(3, 40, device="cuda"), out=cache, index=torch.tensor([0, -1, 5], device="cuda"))
    assert be.dequantize_rows(cache).shape == (0, 40)


def test_bytes(cuda):
    """All that a cache holds: codes and scales of its rows and of one of zeros, a word per row where rows are written by id."""
    import cxgnncomp_backend as be
    base = torch.cuda.memory_allocated()
    cache = be.Rows8(10000, 47)
    assert cache.nbytes == 10001 * 66
    be.quantize_rows(torch.ones(3, 47, device="cuda"), out=cache, index=torch.arange(3, device="cuda"))
    assert cache.nbytes == 10001 * 66 + 40000
    held = torch.cuda.memory_allocated() - base
    assert cache.nbytes <= held < cache.nbytes + 3 * 512  # (blocks of 512 bytes)


def test_copies_and_saved_caches(cuda):
    """The words stay behind: those of a cache that was saved may be of another form."""
    import copy
    import pickle
    import cxgnncomp_backend as be
    x, at = torch.ones(3, 40, device="cuda"), torch.tensor([4, 1, 4], device="cuda")
    cache = be.Rows8(6, 40)
    be.quantize_rows(x, out=cache, index=at)
    old = be.Rows8.__new__(be.Rows8)
    old.__setstate__((None, {"rows": 6, "width": 40, "codes": cache.codes.clone(), "scales": cache.scales.clone(),
                             "_claims": torch.full((7,), 2 ** 32 + 3, device="cuda")}))
    before = be.dequantize_rows(cache)
    # (the last one shares its rows with the cache itself)
    for other in (copy.deepcopy(cache), pickle.loads(pickle.dumps(cache)), old, copy.copy(cache)):
        assert other.shape == cache.shape and torch.equal(be.dequantize_rows(other), before)
        be.quantize_rows(torch.stack([x[0] * 2, x[0] * 3, x[0] * 5]), out=other, index=at)
        assert float(be.dequantize_rows(other)[4, 0]) == 5 and float(be.dequantize_rows(other)[1, 0]) == 3
