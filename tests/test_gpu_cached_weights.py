"""Softmax weights of every size in cached attention: one key far above a long tail of keys whose weights are
small one by one and count together, beside rows of V far larger than the others.

The keys are made so that a score is exact up to a few products: the tail's rows of K are zeros, the sink's
all of one value, the query all ones.  Then, relative to the average of |v|, an output is off by at most

  2 (G 2^-22 + 2^-21)   a weight: its argument of at most G (in units of log 2) after four roundings,
                        and the exponential; twice, for the normalisation
  2^-22                 the two fp16 halves of a weight (2^-11 for an output in bf16, which has one)
  N 2^-33 w             half a step at the bottom of fp16 (2^-25) for each of N keys, where the row's largest
                        weight (of the softmax, times its |v|) is at least 2^8
  C 2^-23               a sum of C steps, each of which may truncate (C 2^-24 for one that rounds).  The keys
                        of a call of one request are shared out over the SMs: a warp (or a row's thread) adds up at
                        most 11 tiles of 64 keys, 16 at a time in O (twice, for the halves) and 2 by 2 in the
                        sum, and the merge at most 444 / 8 + 8 parts.  Of many requests at once a CTA has whole
                        ones: a warp every fourth tile, the kernel for chunks all of them

and half a step of its type.
"""
import math

import numpy as np
import pytest
import torch

import long_context_attention as lca
from lca_testutil import to_np
from oracle import swa_oracle

pytestmark = pytest.mark.gpu

TAIL, D = 100000, 64
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
STEPS = 11 * 32 + 444 // 8 + 8
HEADS = 8


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def cache_of(k, v, heads, batch):
    """(pool, tables) of a request with the rows k, v [tokens, D] in every head, `batch` times over, and the
    values it holds."""
    n, page = len(k), 64
    pages = -(-n // page)
    pool = lca.kv_cache_pool(pages, heads, page, D)
    rows = [torch.tensor(x[:, None], dtype=torch.float32).bfloat16() for x in (k, v)]
    lca.kv_cache_append(pool, *(x.cuda().expand(n, heads, D) for x in rows), torch.arange(n, dtype=torch.int32, device="cuda"))
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].expand(batch, pages).contiguous()
    return pool, table, [swa_oracle.kv4_values(x.float().numpy()) for x in rows]


def check(k, v, gap, new, out_dtype, peak_at=0, batch=1, off=0.0):
    heads = 1 if batch == 1 else HEADS
    pool, table, values = cache_of(k, v, heads, batch)
    n = len(k)
    peak = values[0][peak_at, 0].sum()
    scale = float(np.float32(gap * math.log(2) / peak))
    q = torch.ones(batch * new, heads, D, device="cuda").half()
    got, lse = lca.sliding_window_attention_cached(q, pool, table, ints([n] * batch), ints(np.arange(batch + 1) * new), 2 * n,
                                                   scale=scale, out_dtype=out_dtype, return_lse=True)
    got, lse = to_np(got).reshape(batch, new, heads, D), to_np(lse).reshape(heads, batch, new)
    tiles = -(-n // 64)
    if batch == 1:
        steps = STEPS
    elif new < 64:  # two halves of four blocks a tile, and four warps to merge
        steps = -(-tiles // 4) * 8 + 4
    else:           # the sum takes fewer: 32 pairs a tile and then the tiles, and rounds
        steps = tiles * 8
    for i in sorted({0, new // 2, new - 1}):  # the rows are alike but for a few keys at the end
        length = n - new + 1 + i
        want, want_lse, mean, _ = swa_oracle.cached_attention(np.ones((1, 1, D)), values[0][:length], values[1][:length], 2 * n,
                                                              [], scale)
        share_of = np.exp(scale * values[0][:length, 0].sum(-1) - want_lse[0, 0])
        largest = (share_of * np.abs(values[1][:length, 0]).max(-1)).max()
        share = 2 * (gap * 2.0 ** -22 + 2.0 ** -21 + off) + steps * 2.0 ** -23
        share += 2.0 ** -11 if out_dtype == torch.bfloat16 else 2.0 ** -22
        bound = share * mean[0, 0] + length * 2.0 ** -33 * largest + HALF[out_dtype] * np.abs(want[0, 0])
        err = np.abs(got[:, i] - want[0, 0])  # of every request and head
        assert (err <= bound).all(), f"row {i}: off by {err.max():.3e}, bound {bound.min():.3e}"
        lse_bound = gap * 2.0 ** -22 + 2.0 ** -21 + 3 * off + steps * 2.0 ** -23 + 2.0 ** -22 * abs(want_lse[0, 0])
        assert (np.abs(lse[:, :, i] - want_lse[0, 0]) <= lse_bound).all()
    assert lca.device_error() == 0


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new", [1, 5, 20, 70])  # 8, 16 and 32 rows an item, and the kernel for chunks
@pytest.mark.parametrize("gap,outlier", [(0.0, 1.0), (12.3, 1.0), (17.3, 1.0), (17.3, 3.5), (17.3, 16.0), (16.7, 200.0),
                                         (20.4, 200.0)])
def test_a_sink_above_a_long_even_tail(gap, outlier, new, out_dtype):
    n = TAIL + 1 + new
    k, v = np.zeros((n, D)), np.ones((n, D))  # rows alike: each weight is rounded the same way
    k[0], v[0] = 1.875, -1.0
    v[3] *= outlier  # in the sink's tile
    if gap == 0.0:
        k[:] = 1.875
    check(k, v, gap, new, out_dtype)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("new,batch", [(1, 64), (70, 75)])  # more items than are cut
@pytest.mark.parametrize("gap,outlier", [(16.9, 1.0), (17.3, 3.5), (17.3, 16.0), (16.7, 200.0), (20.61, 1.0), (22.68, 1.0)])
def test_many_requests_with_a_sink_and_a_tail(gap, outlier, new, batch, out_dtype):
    n = TAIL + 1 + new
    k, v = np.zeros((n, D)), np.ones((n, D))  # rows alike: each weight is rounded the same way
    k[0], v[0] = 1.875, -1.0
    v[3] *= outlier
    check(k, v, gap, new, out_dtype, batch=batch)


@pytest.mark.parametrize("new", [1, 70])
def test_a_tail_of_varied_sizes_before_the_sink(new):
    """The tail's keys come first, at several levels below the one that ends up largest."""
    rng = np.random.default_rng(new)
    n = TAIL + new
    k, v = np.zeros((n, D)), np.abs(rng.standard_normal((n, D))) + 0.5
    k[:, :] = rng.choice([0.0, 0.234375, 0.46875, 0.9375], (n, 1), p=[0.9, 0.06, 0.03, 0.01])
    k[TAIL // 2] = 1.875
    v[::1000] *= rng.choice([0.01, 30.0], (len(v[::1000]), 1))
    check(k, v, 18.7, new, torch.float32, peak_at=TAIL // 2)


@pytest.mark.parametrize("new", [1, 70])
@pytest.mark.parametrize("size", [0.0, 2.0 ** -70, 2.0 ** 80])
def test_values_of_every_size(size, new):
    """All of V zero, or far from 1: the sum of the weights stays in range, and its logarithm right."""
    rng = np.random.default_rng(3)
    n = 30000 + new
    k = np.zeros((n, D))
    k[0], k[20000:] = 1.875, 0.46875
    v = size * (np.abs(rng.standard_normal((n, D))) + 0.5)
    check(k, v, 14.2, new, torch.float32)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("new,batch", [(1, 1), (20, 1), (70, 1), (1, 64), (70, 75)])
@pytest.mark.parametrize("sizes", [(0.0, 1e16), (1e16, 0.0), (1e-22, 1e25), (0.0, 1.0, 1e12, 1e-3, 1e28), (1e20, 0.0, 1e20)])
def test_stretches_of_values_far_apart_in_size(sizes, new, batch, out_dtype):
    """Even scores: every key counts in the sum, whatever the sizes of V before and behind it.  The sizes move
    the reference of the weights by more than fp32's exponent holds.  It is then up to 128 away from the
    scores, which are rounded to 2^-18 against it, as are it and the logarithm in the LSE."""
    n = 9000 + new
    k, v = np.full((n, D), 1.875), np.ones((n, D))
    at = np.linspace(0, 9000, len(sizes) + 1).astype(int)
    for size, a, b in zip(sizes, at, [*at[1:-1], n]):
        v[a:b] *= size
    check(k, v, 0.3, new, out_dtype, batch=batch, off=2.0 ** -18)
