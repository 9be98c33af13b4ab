"""A row of cached attention depends, to the bit, on the keys that it sees and on nothing else in the pool: not
on slots behind a request's length, keys in front of every row's window or pages of no request, and
not on tokens behind it that other rows of the same call see."""
import numpy as np
import pytest
import torch

import long_context_attention as lca

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,new,heads,window,tokens", [
    (60, 60, 2, 1000, []),        # one tile, whose last slots were never written
    (60, 60, 2, 10, [3]),
    (200, 70, 4, 20, []),         # the first tile begins in front of the window
    (200, 70, 4, 20, [70, 100]),  # where two of its keys are global
    (333, 150, 2, 30, [2, 250]),  # a global row among the new ones, which sees everything up to itself
    (203, 1, 2, 20, [5]), (203, 9, 2, 20, [60]), (5000, 3, 2, 10000, []), (3990, 70, 2, 10000, []),
])
def test_what_no_row_sees_changes_nothing(n, new, heads, window, tokens, out_dtype):
    rng = np.random.default_rng(n + new)
    d, page, kv_heads = 64, 32, 1
    pages = -(-n // page)
    pool = lca.kv_cache_pool(pages + 2, kv_heads, page, d)
    order = rng.permutation(pages + 2)[:pages].astype(np.int32)
    table = ints(order[None])
    pos = np.arange(n)
    k, v = (torch.tensor(rng.standard_normal((n, kv_heads, d)), dtype=torch.float32).half().cuda() for _ in range(2))
    lca.kv_cache_append(pool, k, v, ints(order[pos // page] * page + pos % page))
    q = torch.tensor(rng.standard_normal((new, heads, d)), dtype=torch.float32).half().cuda()
    rows = n - new + np.arange(new)
    seen = np.zeros(pages * page, dtype=bool)
    for p in rows:
        seen[:p + 1] |= (p - np.arange(p + 1) <= window) | np.isin(np.arange(p + 1), tokens) | (p in tokens)
    unseen = np.flatnonzero(~seen)
    assert len(unseen)
    slots = np.concatenate([order[unseen // page] * page + unseen % page]
                           + [x * page + np.arange(page) for x in set(range(pages + 2)) - set(order.tolist())])
    lens, cu = ints([n]), ints([0, new])

    def call():
        return lca.sliding_window_attention_cached(q, pool, table, lens, cu, window, tokens, out_dtype=out_dtype, return_lse=True)

    want, want_lse = call()
    assert want.isfinite().all()
    for size in (0.0, 1e-3, 300.0, 6e4, float("nan"), float("inf")):
        x = torch.tensor(rng.standard_normal((len(slots), kv_heads, d)), dtype=torch.float32).half().cuda() * size
        lca.kv_cache_append(pool, x, x, ints(slots))
        got, lse = call()
        assert torch.equal(got, want) and torch.equal(lse, want_lse), f"unseen values of size {size}"


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,new,heads,window,tokens", [
    (64, 64, 2, 1000, []), (100, 7, 1, 1000, []), (150, 16, 2, 30, [1]), (300, 30, 1, 40, [100, 285]),
    (500, 130, 2, 50, [3, 400]), (2100, 20, 2, 10000, []), (2100, 300, 1, 10000, []),
])
def test_a_row_does_not_depend_on_later_tokens(n, new, heads, window, tokens, out_dtype):
    rng = np.random.default_rng(n * new)
    d, page = 128, 16
    pages = -(-n // page)
    pool = lca.kv_cache_pool(pages, 1, page, d)

    def rows(count, size):
        return torch.tensor(rng.standard_normal((count, 1, d)) * size, dtype=torch.float32).half().cuda()

    lca.kv_cache_append(pool, rows(n, 1), rows(n, 1), ints(np.arange(n)))
    q = torch.tensor(rng.standard_normal((new, heads, d)), dtype=torch.float32).bfloat16().cuda()

    def call():
        return lca.sliding_window_attention_cached(q, pool, ints(np.arange(pages)[None]), ints([n]), ints([0, new]), window,
                                                   tokens, out_dtype=out_dtype, return_lse=True)

    want, want_lse = call()
    first = n - new // 2  # rows from here on are allowed to change
    keep = new - new // 2
    for k_size, v_size in ((1, 1e-3), (1, 500.0), (30.0, 1), (0.0, 0.0), (float("nan"), 1), (1, float("nan"))):
        lca.kv_cache_append(pool, rows(n - first, k_size), rows(n - first, v_size), ints(np.arange(first, n)))
        got, lse = call()
        assert torch.equal(got[:keep], want[:keep]) and torch.equal(lse[:, :keep], want_lse[:, :keep]), (k_size, v_size)
        assert not torch.equal(got[keep:], want[keep:])
