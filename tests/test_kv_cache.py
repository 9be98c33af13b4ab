"""The paged 4-bit KV cache without a GPU: the oracle's format and layout against their definitions,
and the refusals that come before any device work."""
import ctypes

import numpy as np
import pytest
import torch

import long_context_attention as lca
from long_context_attention import _native
from oracle import swa_oracle


@pytest.mark.parametrize("d", [64, 128])
def test_block_bytes_hold_the_values(d):
    rng = np.random.default_rng(d)
    k, v = rng.standard_normal((2, 16, d)).astype(np.float32) * 3
    k[3], v[5], k[7, 2] = 0, 1e-40, np.inf
    v[9] += 100  # a row of one sign
    block = swa_oracle.kv4_block(k, v)
    assert block.size == 16 * (d + 8)
    for x, codes_at, words_at in ((k, 0, 16 * d), (v, 16 * d // 2, 16 * d + 64)):
        words = block[codes_at:codes_at + 16 * d // 2].view("<u4").reshape(16, d // 8)
        rows = block[words_at:words_at + 64].view("<u4")
        codes = np.stack([(words >> (4 * j)) & 15 for j in range(8)], -1).reshape(16, d).astype(np.int64)
        scale = (rows & np.uint32(0xFFFFFFF0)).view(np.float32).astype(np.float64)
        got = scale[:, None] * (codes - (rows & 15)[:, None].astype(np.int64))
        np.testing.assert_array_equal(got, swa_oracle.kv4_values(x))


def test_quantised_rows_are_within_one_step():
    """Inside the range an element is off by half a step, at an end by one (where both z and the code
    round up), plus the 2^-19 by which the scale is cut."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((500, 64)) * rng.uniform(1e-6, 1e4, (500, 1))).astype(np.float32)
    codes, scale, _ = swa_oracle.kv4_quantize(x)
    assert codes.max() == 15 and codes.min() == 0
    step = (np.maximum(x.max(-1), 0) - np.minimum(x.min(-1), 0)).astype(np.float64) / 15
    assert (np.abs(swa_oracle.kv4_values(x) - x) <= step[:, None] * (1 + 2.0 ** -10)).all()
    nan = swa_oracle.kv4_values(np.array([[1.0] * 63 + [np.nan]], np.float32))
    assert np.isnan(nan).all() and (swa_oracle.kv4_values(np.zeros((1, 64))) == 0).all()


def _native_layout(c, **kw):
    a = dict(table=None, batch=1, width=4, seq=None, new=None, free=None, cap=4, count=None, page=16, rows=8, slots=None,
             pos=None, cu=None, kv=None, placed=None, nseq=None, ncount=None)
    a.update(kw)
    return c.lib.lca_kv_layout(*a.values(), None)


def test_layout_and_release_refusals():
    c = _native.cabi()
    for page in (0, 8, 24, -16, 1 << 20):
        assert _native_layout(c, page=page) == c.ERR_INVALID_ARGUMENT
        assert "page_size" in c.last_error()
    assert _native_layout(c, batch=8193) == c.ERR_UNSUPPORTED
    assert _native_layout(c, batch=-1) == c.ERR_INVALID_ARGUMENT
    assert _native_layout(c, width=1 << 40) == c.ERR_UNSUPPORTED
    assert _native_layout(c, rows=-1) == c.ERR_INVALID_ARGUMENT
    assert _native_layout(c, cap=-1) == c.ERR_INVALID_ARGUMENT
    assert _native_layout(c) == c.ERR_INVALID_ARGUMENT and "non-NULL" in c.last_error()
    buf = (ctypes.c_int32 * 64)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    full = dict(table=p, seq=p, new=p, free=p, count=p, slots=p, pos=p, cu=p, kv=p, placed=p, nseq=p + 16, ncount=p + 16)
    assert _native_layout(c, **{**full, "slots": p + 4}) == c.ERR_INVALID_ARGUMENT and "aligned" in c.last_error()
    assert _native_layout(c, **{**full, "nseq": p}) == c.ERR_INVALID_ARGUMENT and "overwrite" in c.last_error()
    assert _native_layout(c, **{**full, "ncount": p}) == c.ERR_INVALID_ARGUMENT

    def release(page=16, batch=1, count=None, nseq=None):
        return c.lib.lca_kv_release(p, batch, 4, p, p, p, 4, count, page, nseq, p + 16, None)

    assert release(page=17) == c.ERR_INVALID_ARGUMENT
    assert release(batch=9000) == c.ERR_UNSUPPORTED
    assert release() == c.ERR_INVALID_ARGUMENT
    assert release(count=p, nseq=p) == c.ERR_INVALID_ARGUMENT


def test_append_and_read_refusals():
    c = _native.cabi()

    def append(pool=None, pages=4, heads=2, page=16, d=64, k=None, dtype=c.DTYPE_F16, tokens=3):
        return c.lib.lca_kv4_append(pool, pages, heads, page, d, k, k, dtype, 128, 64, 128, 64, None, tokens, None)

    def read(pool=None, pages=4, heads=2, page=16, d=64, k=None, dtype=c.DTYPE_F32, tokens=3):
        return c.lib.lca_kv4_read(pool, pages, heads, page, d, None, tokens, k, k, dtype, None)

    for call in (append, read):
        assert call(d=96) == c.ERR_UNSUPPORTED
        assert call(page=40) == c.ERR_INVALID_ARGUMENT
        assert call(heads=0) == c.ERR_INVALID_ARGUMENT
        assert call(pages=-1) == c.ERR_INVALID_ARGUMENT
        assert call(pages=1 << 28) == c.ERR_UNSUPPORTED  # 2^32 tokens
        assert call(dtype=9) == c.ERR_UNSUPPORTED
        assert call() == c.ERR_INVALID_ARGUMENT and "pool" in c.last_error()
        assert call(pool=8) == c.ERR_INVALID_ARGUMENT and "aligned" in c.last_error()
        assert call(pool=16, tokens=-1) == c.ERR_INVALID_ARGUMENT
        assert call(pool=16) == c.ERR_INVALID_ARGUMENT and "non-NULL" in c.last_error()
        assert call(pool=16, tokens=0) == c.OK
    assert append(pool=16, dtype=c.DTYPE_F32) == c.ERR_UNSUPPORTED
    assert read(pool=None, pages=0, tokens=0) == c.OK


def _cached(c, tokens=(), **kw):
    a = dict(q=None, dtype=c.DTYPE_BF16, qrow=256, qhead=64, rows=2, heads=4, pool=16, pages=4, kv_heads=2, page=16, d=64,
             table=None, batch=1, width=4, kv=None, cu=None, window=8)
    tail = dict(out=None, out_dtype=c.DTYPE_F32)
    for name, value in kw.items():
        (tail if name in tail else a)[name] = value
    arr = (ctypes.c_int64 * max(len(tokens), 1))(*tokens)
    return c.lib.lca_swa_forward_cached(*a.values(), arr, len(tokens), ctypes.c_float(0.1), *tail.values(), None, None, 0,
                                        None)


def test_cached_attention_refusals():
    c = _native.cabi()
    assert _cached(c, dtype=c.DTYPE_F32) == c.ERR_UNSUPPORTED
    assert _cached(c, out_dtype=5) == c.ERR_UNSUPPORTED
    assert _cached(c, d=96) == c.ERR_UNSUPPORTED
    assert _cached(c, heads=3) == c.ERR_INVALID_ARGUMENT and "multiple" in c.last_error()
    assert _cached(c, heads=0) == c.ERR_INVALID_ARGUMENT
    assert _cached(c, window=-1) == c.ERR_INVALID_ARGUMENT
    assert _cached(c, page=20) == c.ERR_INVALID_ARGUMENT
    assert _cached(c, batch=9000) == c.ERR_UNSUPPORTED
    assert _cached(c, rows=-2) == c.ERR_INVALID_ARGUMENT
    assert _cached(c, tokens=[-1]) == c.ERR_INDEX  # no end to count from: the requests grow
    assert _cached(c, tokens=[64]) == c.ERR_INDEX and "capacity" in c.last_error()
    assert _cached(c, tokens=list(range(1025)), width=100) == c.ERR_UNSUPPORTED
    assert _cached(c, tokens=[5] * 2000, rows=0) == c.OK
    assert _cached(c, rows=0) == c.OK
    assert _cached(c, batch=0) == c.OK
    assert _cached(c) == c.ERR_INVALID_ARGUMENT and "non-NULL" in c.last_error()
    full = dict(q=16, table=16, kv=16, cu=16, out=16)
    assert _cached(c, **{**full, "q": 24}) == c.ERR_INVALID_ARGUMENT and "aligned" in c.last_error()
    assert _cached(c, **full, qhead=68) == c.ERR_INVALID_ARGUMENT
    assert _cached(c, **{**full, "out": 20}) == c.ERR_INVALID_ARGUMENT
    # long items are cut and need scratch
    assert _cached(c, **full, width=1000, window=10 ** 6) == c.ERR_WORKSPACE and "workspace" in c.last_error()
    assert _cached(c, **full, width=1 << 27) == c.ERR_UNSUPPORTED


def test_cached_workspace_size():
    c = _native.cabi()
    size = ctypes.c_size_t(7)

    def need(rows=64, heads=32, kv_heads=8, d=128, batch=64, capacity=131072, window=256, tokens=0):
        st = c.lib.lca_swa_cached_workspace_size(rows, heads, kv_heads, d, batch, capacity, window, tokens, ctypes.byref(size))
        return st, size.value

    assert need() == (c.OK, 0)  # a band stays whole
    st, one = need(window=131072)
    assert st == c.OK and one > 0
    assert need(window=131072, rows=64 * 500)[1] == 0  # many long items of many rows stay whole too
    assert need(rows=0) == (c.OK, 0) and need(batch=0) == (c.OK, 0)
    assert need(window=-1)[0] == c.ERR_INVALID_ARGUMENT
    assert need(heads=12)[0] == c.ERR_INVALID_ARGUMENT
    assert need(kv_heads=0)[0] == c.ERR_INVALID_ARGUMENT
    assert need(capacity=-5)[0] == c.ERR_INVALID_ARGUMENT
    assert c.lib.lca_swa_cached_workspace_size(1, 1, 1, 64, 1, 64, 1, 0, None) == c.ERR_INVALID_ARGUMENT


def test_python_refusals():
    ints = torch.zeros(1, dtype=torch.int32)
    pool = lca.kv_cache_pool(2, 1, 16, 64, device="cpu")
    assert pool.shape == (2, 1, 16, 72)
    for call in (lambda: lca.kv_cache_layout(ints[None], ints, ints, ints, ints, 16, 1),
                 lambda: lca.kv_cache_release(ints[None], ints, ints.bool(), ints, ints, 16),
                 lambda: lca.kv_cache_append(pool, torch.zeros(1, 1, 64).half(), torch.zeros(1, 1, 64).half(), ints),
                 lambda: lca.kv_cache_read(pool, ints),
                 lambda: lca.sliding_window_attention_cached(torch.zeros(1, 1, 64).half(), pool, ints[None], ints,
                                                             torch.zeros(2, dtype=torch.int32), 4)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="16"):
        lca.kv_cache_pool(2, 1, 24, 64, device="cpu")
    with pytest.raises(ValueError, match="head_dim"):
        lca.kv_cache_pool(2, 1, 16, 80, device="cpu")


def test_layout_oracle_takes_whole_requests_in_order():
    """A request that does not fit leaves no trace, and no later one overtakes it for pages."""
    table = np.full((4, 3), -1)
    table[0, 0] = 9
    got = swa_oracle.kv_layout(table, [10, 0, 0, 0], [3, 40, 5, 0], [0, 1, 2, 3], 3, 16, 60)
    assert got["slots"][:3].tolist() == [154, 155, 156] and got["kv_lens"].tolist() == [13, 40, 0, 0]
    assert got["block_table"][1].tolist() == [2, 1, 0] and got["free_count"][0] == 0
    assert got["slots"][43:48].tolist() == [-1] * 5 and got["placed"].tolist() == [3, 40, 0, 0]
    got = swa_oracle.kv_layout(table, [10, 0, 0, 0], [3, 49, 5, 0], [0, 1, 2, 3], 3, 16, 60)
    assert got["kv_lens"].tolist() == [13, 0, 5, 0]  # 49 tokens pass the table's row, which takes no pages
    got = swa_oracle.kv_layout(table, [10, 0, 0, 0], [3, 40, 5, 0], [0, 1, 2, 3], 3, 16, 42)
    assert got["kv_lens"].tolist() == [13, 0, 0, 0] and got["cu_seqlens"].tolist() == [0, 3, 42, 42, 42]


def test_derivatives_are_refused():
    """A gradient that is asked for, backward or forward, is refused and not dropped."""
    from torch.autograd import forward_ad

    from long_context_attention import kv_cache

    x, leaf = torch.zeros(2), torch.zeros(2, requires_grad=True)
    kv_cache._no_grad(x, x)
    with pytest.raises(NotImplementedError, match="backward"):
        kv_cache._no_grad(x, leaf)
    with torch.no_grad():
        kv_cache._no_grad(leaf)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(2))
        kv_cache._no_grad(x)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            kv_cache._no_grad(x, dual)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: (kv_cache._no_grad(t), t)[1], (x,), (torch.ones(2),))
    kv_cache._no_grad(x)
