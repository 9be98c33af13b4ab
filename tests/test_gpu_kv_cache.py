"""The paged 4-bit KV cache on the GPU against the oracle (64 bits, CPU): layout and release, append
and read, and causal sliding-window + global-token attention over the cache; then the
operators together, as a serving loop runs them."""
import math

import numpy as np
import pytest
import torch

import long_context_attention as lca
from lca_testutil import to_np
from oracle import swa_oracle

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ layout and release


def check_layout(table, seq, new, free, count, page, rows):
    want = swa_oracle.kv_layout(table, seq, new, free, count, page, rows)
    t, s, n, f, c = ints(table), ints(seq), ints(new), ints(free), ints([count])
    for _ in range(2):  # the inputs stay as they were, so a second call finds the same
        step = lca.kv_cache_layout(t, s, n, f, c, page, rows)
        for name in ("slots", "positions", "cu_seqlens", "kv_lens", "placed", "seq_lens", "free_count"):
            np.testing.assert_array_equal(getattr(step, name).cpu().numpy(), want[name], err_msg=name)
        np.testing.assert_array_equal(t.cpu().numpy(), want["block_table"])
    assert torch.equal(step.state, torch.cat([step.seq_lens, step.free_count]))
    assert torch.equal(s, ints(seq)) and torch.equal(c, ints([count]))


@pytest.mark.parametrize("batch,page,rows,longest,spare,seed", [
    (1, 16, 1, 500, 1.0, 0), (7, 16, 300, 200, 1.0, 1), (64, 64, 64, 3000, 1.0, 2), (33, 48, 1001, 300, 0.5, 3),
    (513, 32, 5000, 90, 0.8, 4), (1200, 16, 1200, 40, 1.0, 5), (5, 128, 0, 900, 1.0, 6), (3, 16, 9001, 5000, 0.7, 7),
    (8192, 16, 9000, 30, 1.0, 8),
])
def test_layout_matches_the_oracle(batch, page, rows, longest, spare, seed):
    rng = np.random.default_rng(seed)
    seq = rng.integers(0, longest + 1, batch)
    new = rng.integers(0, max(2, 2 * rows // batch + 1), batch) * rng.integers(0, 2, batch)
    width = -(-longest // page) + 1
    held = -(-seq // page)
    order = rng.permutation(int(held.sum()) + 4 * batch)
    table = np.full((batch, width), -1)
    at = 0
    for b in range(batch):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    free = order[at:]
    need = int((-(-(seq + new) // page) - held).sum())
    check_layout(table, seq, new, free, min(len(free), int(need * spare)), page, rows)


def test_layout_edges():
    table = np.full((3, 2), -1)
    free = np.arange(6)
    check_layout(table, [0, 0, 0], [0, 0, 0], free, 6, 16, 5)            # nothing new
    check_layout(table, [0, 0, 0], [32, 33, 1], free, 6, 16, 80)         # the second passes its table row
    check_layout(table, [0, 0, 0], [2 ** 31 - 1, 4, 2 ** 31 - 1], free, 6, 16, 80)  # sums past 32 bits
    check_layout(table, [-5, 0, 3], [-7, 20, 1], free, 6, 16, 30)        # negative lengths; a page of -1
    check_layout(table, [0, 0, 0], [1, 1, 1], free, 100, 16, 3)          # a count above the list's length
    check_layout(table, [0, 0, 0], [1, 1, 1], free, -4, 16, 3)
    check_layout(table, [99, 0, 0], [0, 1, 1], free, 6, 16, 3)           # a length past the table
    check_layout(np.zeros((2, 0)), [0, 0], [1, 0], free, 6, 16, 2)       # a table of no pages
    check_layout(np.zeros((0, 4)), [], [], free, 6, 16, 3)               # no requests
    huge = np.array([[2 ** 30, -1]])
    check_layout(huge, [3], [1], free, 6, 64, 1)                         # a slot past 31 bits


def test_release_returns_pages_in_order():
    rng = np.random.default_rng(5)
    for batch, width in ((1, 3), (40, 9), (700, 5)):
        table = rng.permutation(batch * width).reshape(batch, width)
        seq = rng.integers(0, 16 * width + 1, batch)
        mask = rng.integers(0, 2, batch).astype(bool)
        free = np.full(batch * width + 4, -7)
        back = [table[b, i] for b in range(batch) if mask[b] for i in range(-(-seq[b] // 16))]
        for cap in (len(free), 2 + len(back) // 2):  # the second list overflows
            f = ints(free[:cap])
            s, c, _ = lca.kv_cache_release(ints(table), ints(seq), torch.tensor(mask, device="cuda"), f, ints([2]), 16)
            want = np.concatenate([[-7, -7], back, free[2 + len(back):]])[:cap]
            np.testing.assert_array_equal(f.cpu().numpy(), want)
            assert c.item() == min(2 + len(back), cap)
            np.testing.assert_array_equal(s.cpu().numpy(), np.where(mask, 0, seq))


# ------------------------------------------------------------------ append and read


def random_rows(rng, rows, heads, d, dtype):
    x = rng.standard_normal((rows, heads, d)) * np.exp(rng.uniform(-6, 4, (rows, heads, 1)))
    x += rng.choice([0, 0, 3], (rows, heads, 1))
    return torch.tensor(x, dtype=torch.float32).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,heads,page,tokens", [(64, 1, 16, 1), (64, 5, 48, 130), (128, 8, 64, 77), (128, 3, 32, 400)])
def test_append_stores_the_defined_codes(dtype, d, heads, page, tokens):
    rng = np.random.default_rng(tokens)
    pages = -(-tokens // page) + 2
    pool = torch.randint(0, 256, (pages, heads, page, d + 8), dtype=torch.uint8, device="cuda")
    before = pool.clone()
    slots = rng.permutation(pages * page)[:tokens]
    slots[rng.random(tokens) < 0.1] = -1
    k, v = random_rows(rng, tokens, heads, d, dtype), random_rows(rng, tokens, heads, d, dtype)
    k[0, 0], v[-1, 0] = 0, -2.0
    if tokens > 10:
        k[5, 0, 3], v[6, 0, 1], k[7, 0, 0] = float("inf"), float("nan"), -float("inf")
        k[8, 0], k[8, 0, 1] = 1e-7, 3e-7  # fp16: subnormal values
        v[9, 0, 0], v[9, 0, 1] = torch.finfo(dtype).max, torch.finfo(dtype).min
    lca.kv_cache_append(pool, k.cuda(), v.cuda(), ints(slots))
    kf, vf = k.float().numpy(), v.float().numpy()
    want_bytes = before.cpu().numpy().reshape(pages, heads, page // 16, 16 * (d + 8))
    for t, s in enumerate(slots):
        if s < 0:
            continue
        for h in range(heads):
            block = want_bytes[s // page, h, s % page // 16]
            fresh = swa_oracle.kv4_block(np.repeat(kf[t, h][None], 16, 0), np.repeat(vf[t, h][None], 16, 0))
            row = s % 16
            for at, size in ((0, d // 2), (16 * d // 2, d // 2), (16 * d, 4), (16 * d + 64, 4)):
                block[at + row * size:at + (row + 1) * size] = fresh[at + row * size:at + (row + 1) * size]
    np.testing.assert_array_equal(pool.cpu().numpy().reshape(want_bytes.shape), want_bytes)
    for out_dtype in (None, torch.float16, torch.bfloat16):
        got = lca.kv_cache_read(pool, ints(slots), out_dtype)
        for x, y in zip((kf, vf), got):
            want = torch.tensor(swa_oracle.kv4_values(x)).float() * 1.0
            want[torch.tensor(slots < 0)] = 0
            want = want.to(out_dtype or torch.float32)
            assert y.dtype == want.dtype
            torch.testing.assert_close(y.cpu(), want, rtol=0, atol=0, equal_nan=True)


def test_append_strided_and_unaligned_views():
    rng = np.random.default_rng(3)
    tokens, heads, d, page = 50, 4, 64, 16
    base = random_rows(rng, tokens, 3 * heads, d, torch.bfloat16).cuda()  # a fused projection
    slots = ints(rng.permutation(128)[:tokens])

    def stored(k, v):
        pool = lca.kv_cache_pool(8, heads, page, d)
        lca.kv_cache_append(pool, k, v, slots)
        return pool

    k, v = base[:, heads:2 * heads], base[:, 2 * heads:]
    want = stored(k.contiguous(), v.contiguous())
    assert torch.equal(stored(k, v), want)
    assert torch.equal(stored(k.transpose(0, 1).contiguous().transpose(0, 1), v), want)  # head-major
    odd = torch.zeros(tokens, heads, d + 1, dtype=torch.bfloat16, device="cuda")
    odd[..., 1:] = k
    assert torch.equal(stored(odd[..., 1:], v), want)  # 2-byte aligned rows
    one = base[:1, :heads].expand(tokens, heads, d)      # one row for every token
    assert torch.equal(stored(one, one), stored(one.contiguous(), one.contiguous()))


def test_append_and_read_skip_slots_outside_the_pool():
    pool = torch.randint(0, 256, (3, 2, 32, 136), dtype=torch.uint8, device="cuda")
    before = pool.clone()
    k = torch.randn(4, 2, 128, device="cuda").half()
    slots = ints([-1, 96, 2 ** 31 - 1, -2 ** 31])
    lca.kv_cache_append(pool, k, k, slots)
    assert torch.equal(pool, before)
    a, b = lca.kv_cache_read(pool, slots)
    assert not a.any() and not b.any()
    lca.kv_cache_append(pool, k[:0], k[:0], slots[:0])
    assert lca.kv_cache_read(pool, slots[:0])[0].shape == (0, 2, 128)


# ------------------------------------------------------------------ attention


def filled_cache(rng, lens, kv_heads, d, page, extra_pages=2, std=1.0):
    """(pool, table, per request the K and V values read back): pages in random order, and every byte
    that no token owns random."""
    held = [-(-n // page) for n in lens]
    pages = sum(held) + extra_pages
    pool = torch.randint(0, 256, (pages, kv_heads, page, d + 8), dtype=torch.uint8, device="cuda",
                         generator=torch.Generator("cuda").manual_seed(1))
    order = rng.permutation(pages)
    table = np.full((len(lens), max(held + [1])), -1)
    at, values = 0, []
    for b, n in enumerate(lens):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
        k = torch.tensor(rng.standard_normal((n, kv_heads, d)) * std, dtype=torch.float32).half()
        v = torch.tensor(rng.standard_normal((n, kv_heads, d)) * np.exp(rng.uniform(-3, 2, (n, kv_heads, 1))),
                         dtype=torch.float32).half()
        p = np.arange(n)
        lca.kv_cache_append(pool, k.cuda(), v.cuda(), ints(table[b, p // page] * page + p % page))
        values.append((swa_oracle.kv4_values(k.float().numpy()), swa_oracle.kv4_values(v.float().numpy())))
    return pool, ints(table), values


def check_rows(got, got_lse, want, lse, mean, size, d, what):
    """Bounds.  A score is a sum of d fp32 products of size at most S = `size` in all; every addition
    may lose 2^-23 of it (a tensor-core sum may truncate), so it is off by at most e = (d + 4) 2^-23 S,
    plus 2^-21 for the exponent function and its argument.  A weight is then off by that share, the
    normalised average by twice it, of `mean` = the average of |v|.  A 16-bit output may also round
    the weights to fp16 (2^-11 of mean) and is rounded itself (half a step)."""
    e = np.swapaxes((d + 4) * 2.0 ** -23 * size + 2.0 ** -21 * (1 + size), 0, 1)[..., None]  # [n, heads, 1]
    bound = 2 * e * mean + 2.0 ** -20 * mean + HALF[got.dtype] * np.abs(want)
    if got.dtype != torch.float32:
        bound = bound + 2.0 ** -11 * mean + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    x = to_np(got).astype(np.float64)
    assert np.isfinite(x).all(), what
    worst = np.max(np.abs(x - want) - bound, initial=-1.0)
    assert worst <= 0, f"{what}: {worst:.3e} over the bound (largest error {np.abs(x - want).max():.3e})"
    if got_lse is not None:
        y = to_np(got_lse).astype(np.float64)
        assert np.array_equal(np.isinf(lse), np.isinf(y)) and not np.isnan(y).any(), what
        seen = np.isfinite(lse)
        err = np.abs(y - lse)[seen]
        limit = (e[..., 0].T + 2.0 ** -21 * (1 + np.abs(np.where(seen, lse, 0))))[seen]
        assert np.all(err <= limit), f"{what}: lse off by {err.max():.3e}"


def check_attention(rng, lens, new, heads, kv_heads, d, page, window, tokens, dtype, out_dtype, q_std=1.0, scale=None):
    pool, table, values = filled_cache(rng, lens, kv_heads, d, page)
    cu = np.concatenate([[0], np.cumsum(new)])
    q = torch.tensor(rng.standard_normal((cu[-1] + 3, heads, d)) * q_std, dtype=torch.float32).to(dtype)
    out = torch.full(q.shape, 7.0, dtype=out_dtype, device="cuda")
    scale = 1 / math.sqrt(d) if scale is None else scale
    got, lse = lca.sliding_window_attention_cached(q.cuda(), pool, table, ints(lens), ints(cu), window, tokens, scale,
                                                   return_lse=True, out=out)
    assert got.data_ptr() == out.data_ptr() and (out[cu[-1]:] == 7.0).all()
    for b in range(len(lens)):
        r = slice(cu[b], cu[b + 1])
        want = swa_oracle.cached_attention(q[r].float().numpy(), *values[b], window, tokens, scale)
        check_rows(got[r], lse[:, r], *want, d, f"request {b} of {len(lens)}: {lens[b]} tokens, {new[b]} new")
    assert lca.device_error() == 0


TYPES = [(torch.float16, torch.float16), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
         (torch.float16, torch.float32)]


@pytest.mark.parametrize("dtype,out_dtype", TYPES)
@pytest.mark.parametrize("lens,heads,kv_heads,d,page,window,tokens", [
    ([1], 1, 1, 64, 16, 0, []),
    ([1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 0], 4, 2, 64, 16, 1000, []),
    ([700, 129, 1, 300], 3, 3, 128, 48, 64, [0, 5, 250]),
    ([1000, 513], 16, 2, 128, 32, 200, [0, 1, 2, 999]),
    ([2500], 5, 1, 64, 64, 100, list(range(0, 2400, 37))),
    ([300, 4000, 17], 40, 2, 128, 128, 100000, [3]),
])
def test_single_tokens_match_the_oracle(dtype, out_dtype, lens, heads, kv_heads, d, page, window, tokens):
    rng = np.random.default_rng(len(lens) + d + window)
    check_attention(rng, lens, [min(n, 1) for n in lens], heads, kv_heads, d, page, window, tokens, dtype, out_dtype)


@pytest.mark.parametrize("dtype,out_dtype", TYPES[:3])
@pytest.mark.parametrize("lens,new,heads,kv_heads,d,page,window,tokens", [
    ([40, 5, 300], [3, 5, 1], 4, 4, 64, 16, 7, [0, 2]),
    ([200, 90], [200, 33], 8, 2, 128, 32, 20, [0, 1, 100, 150]),   # a whole prompt, with global rows
    ([1030, 77, 0, 500], [130, 0, 0, 1], 6, 1, 64, 48, 50, [500, 990]),  # a global inside the chunk
    ([600], [600], 2, 2, 128, 64, 10000, []),
    ([350, 350], [64, 65], 16, 1, 64, 16, 33, list(range(200, 350, 3))),
])
def test_chunks_match_the_oracle(dtype, out_dtype, lens, new, heads, kv_heads, d, page, window, tokens):
    rng = np.random.default_rng(sum(lens) + d)
    check_attention(rng, lens, new, heads, kv_heads, d, page, window, tokens, dtype, out_dtype)


def test_many_requests_and_long_lengths():
    rng = np.random.default_rng(9)
    lens = rng.integers(0, 120, 300).tolist()
    check_attention(rng, lens, [min(n, 1) for n in lens], 2, 1, 64, 16, 40, [0], torch.float16, torch.float32)
    check_attention(rng, [20000, 9000], [2, 1], 8, 1, 64, 64, 100000, [], torch.float16, torch.float16)
    check_attention(rng, [20000], [1], 2, 2, 128, 64, 300, list(range(10, 19000, 300)), torch.bfloat16, torch.bfloat16)


@pytest.mark.parametrize("lens,new,heads,kv_heads,d,out_dtype", [
    ([20000, 300], [20, 20], 8, 2, 128, torch.bfloat16),        # few long items of many rows, cut
    ([2500] * 24, [17] * 24, 32, 8, 64, torch.float32),         # more of them than CTAs
    ([1700, 2300, 5] * 5, [40, 2, 5] * 5, 6, 6, 64, torch.float16),
])
def test_long_chunks_that_are_cut(lens, new, heads, kv_heads, d, out_dtype):
    check_attention(np.random.default_rng(len(lens)), lens, new, heads, kv_heads, d, 64, 10 ** 5, [3], torch.bfloat16,
                    out_dtype)


def test_more_items_than_ctas():
    """Hundreds of requests of any length, cut wherever a CTA's share ends."""
    rng = np.random.default_rng(31)
    lens = np.concatenate([rng.integers(0, 60, 250), rng.integers(1000, 2500, 20), [0, 0, 1, 2000]])
    rng.shuffle(lens)
    check_attention(rng, lens.tolist(), [min(int(n), 1) for n in lens], 6, 3, 64, 64, 10 ** 5, [], torch.float16,
                    torch.float16)
    lens = rng.integers(0, 40, 5000)
    check_attention(rng, lens.tolist(), [min(int(n), 1) for n in lens], 1, 1, 64, 16, 20, [0], torch.bfloat16, torch.float32)


def test_a_pool_past_32_bit_offsets():
    """Pages at the end of a 4.7 GB pool, for every operator that addresses it."""
    kv_heads, d, page = 16, 128, 128
    pages = 17000
    pool = torch.empty(pages, kv_heads, page, d + 8, dtype=torch.uint8, device="cuda")
    assert pool.numel() > 2 ** 32
    rng = np.random.default_rng(32)
    n = 300
    table = np.array([[pages - 1, 3, pages - 2]])
    k, v = (torch.tensor(rng.standard_normal((n, kv_heads, d)), dtype=torch.float32).half() for _ in range(2))
    pos = np.arange(n)
    slots = ints(table[0, pos // page] * page + pos % page)
    lca.kv_cache_append(pool, k.cuda(), v.cuda(), slots)
    values = [swa_oracle.kv4_values(x.float().numpy()) for x in (k, v)]
    for got, want in zip(lca.kv_cache_read(pool, slots), values):
        np.testing.assert_array_equal(got.cpu().numpy(), want.astype(np.float32))
    for new, window in ((1, 200), (1, 10 ** 4), (80, 50)):
        q = torch.tensor(rng.standard_normal((new, kv_heads, d)), dtype=torch.float32).bfloat16()
        got, lse = lca.sliding_window_attention_cached(q.cuda(), pool, ints(table), ints([n]), ints([0, new]), window, [2],
                                                       return_lse=True)
        want = swa_oracle.cached_attention(q.float().numpy(), *values, window, [2], d ** -0.5)
        check_rows(got, lse, *want, d, f"{new} new, window {window}")


def test_rising_scores_and_scales_of_every_size():
    """Scores that grow along the keys (the running maximum moves all the time), queries far from 1, and a
    negative and a zero scale."""
    rng = np.random.default_rng(10)
    for q_std, scale in ((8.0, 0.05), (2.0 ** -20, 0.1), (2000.0, 1e-4), (1.0, -0.1), (1.0, 0.0)):
        for new in (2, 70):  # one kernel and the other
            check_attention(rng, [700], [new], 4, 2, 64, 16, 500, [0], torch.bfloat16, torch.float32, q_std, scale)
    lens, d = [500], 64
    pool, table, _ = filled_cache(rng, lens, 1, d, 16)
    ramp = np.linspace(0, 20, 500)[:, None, None] * np.ones((1, 1, d)) + 0.01
    k = torch.tensor(ramp, dtype=torch.float32).half()
    v = torch.tensor(rng.standard_normal((500, 1, d)) * np.linspace(1e-3, 1e3, 500)[::-1, None, None],
                     dtype=torch.float32).half()
    slots = table[0, torch.arange(500) // 16].cpu().numpy() * 16 + np.arange(500) % 16
    lca.kv_cache_append(pool, k.cuda(), v.cuda(), ints(slots))
    values = [swa_oracle.kv4_values(x.float().numpy()) for x in (k, v)]
    for out_dtype, new in ((torch.float32, 1), (torch.float16, 1), (torch.float32, 100), (torch.bfloat16, 100)):
        q = torch.full((new, 2, d), 0.25, dtype=torch.float16)
        got, lse = lca.sliding_window_attention_cached(q.cuda(), pool, table, ints(lens), ints([0, new]), 1000, [], 0.2,
                                                       out_dtype=out_dtype, return_lse=True)
        check_rows(got, lse, *swa_oracle.cached_attention(q.float().numpy(), *values, 1000, [], 0.2), d, "ramp")


def test_masked_infinities_and_nans_do_not_matter_and_visible_ones_do():
    rng = np.random.default_rng(11)
    lens, d, page = [200], 64, 16
    pool, table, values = filled_cache(rng, lens, 2, d, page)
    q = torch.tensor(rng.standard_normal((1, 2, d)), dtype=torch.float32).half()
    args = (table, ints(lens), ints([0, 1]), 50, [0])
    want = lca.sliding_window_attention_cached(q.cuda(), pool, *args)
    bad = torch.full((1, 2, d), float("nan"), device="cuda").half()
    for pos in (1, 100, 148):  # the row at 199 sees 149 on, and 0
        slot = int(table[0, pos // page]) * page + pos % page
        lca.kv_cache_append(pool, bad, bad, ints([slot]))
    assert torch.equal(lca.sliding_window_attention_cached(q.cuda(), pool, *args), want)
    pool2 = pool.clone()
    slot = int(table[0, 160 // page]) * page + 160 % page
    half = bad.clone()
    half[:, 1] = 1.0
    lca.kv_cache_append(pool2, torch.ones_like(bad), half, ints([slot]))  # V of KV head 0 alone
    got = lca.sliding_window_attention_cached(q.cuda(), pool2, *args)
    assert got[0, 0].isnan().all() and got[0, 1].isfinite().all()
    lca.kv_cache_append(pool2, half, torch.ones_like(bad), ints([slot]))  # K of KV head 0 alone
    got = lca.sliding_window_attention_cached(q.cuda(), pool2, *args)
    assert got[0, 0].isnan().all() and got[0, 1].isfinite().all()
    q[0, 1, 7] = float("inf")  # and a query that is not finite
    got = lca.sliding_window_attention_cached(q.cuda(), pool, *args)
    assert got[0, 1].isnan().all() and got[0, 0].isfinite().all()


def test_chunks_with_masked_and_visible_nans():
    """The same of the kernel for many rows: rows that do not see a NaN key are what they were, those that see
    it in K or V, or whose query is not finite, are NaN, and no other."""
    rng = np.random.default_rng(14)
    n, new, d, page = 400, 100, 128, 16
    pool, table, _ = filled_cache(rng, [n], 1, d, page)
    q = torch.tensor(rng.standard_normal((new, 2, d)), dtype=torch.float32).bfloat16()
    args = (table, ints([n]), ints([0, new]), 60, [5])
    want, lse = lca.sliding_window_attention_cached(q.cuda(), pool, *args, return_lse=True)
    bad = torch.full((1, 1, d), float("nan"), device="cuda").half()
    for which in range(2):
        hurt = pool.clone()
        for pos in (100, 350):  # one that no row sees, one that rows 50 to 99 see
            slot = int(table[0, pos // page]) * page + pos % page
            lca.kv_cache_append(hurt, *((bad, torch.ones_like(bad)) if which else (torch.ones_like(bad), bad)), ints([slot]))
        got = lca.sliding_window_attention_cached(q.cuda(), hurt, *args)
        assert torch.equal(got[:50], want[:50]) and got[50:].isnan().all()
    q[7, 1, 3], q[8, 0, 0], q[9, 0, 5] = float("inf"), float("nan"), -float("inf")
    got, got_lse = lca.sliding_window_attention_cached(q.cuda(), pool, *args, return_lse=True)
    hit = torch.zeros(new, 2, dtype=torch.bool)
    hit[7, 1], hit[8, 0], hit[9, 0] = True, True, True
    assert got[hit].isnan().all() and got_lse.t()[hit].isnan().all()
    assert torch.equal(got[~hit], want[~hit]) and torch.equal(got_lse.t()[~hit], lse.t()[~hit])
    # more rows than tokens: the first ones see nothing
    got, got_lse = lca.sliding_window_attention_cached(q[10:].cuda(), pool, table, ints([30]), ints([0, 90]), 60, [5],
                                                       return_lse=True)
    assert not got[:60].any() and (got_lse[:, :60] == -math.inf).all() and got[60:].isfinite().all()


def test_rows_that_see_nothing():
    """More rows than cached tokens, a length of zero, and pages outside the pool."""
    rng = np.random.default_rng(12)
    pool, table, values = filled_cache(rng, [40, 20], 1, 64, 16)
    q = torch.randn(9, 2, 64, device="cuda").half()
    got, lse = lca.sliding_window_attention_cached(q, pool, table, ints([2, 0]), ints([0, 5, 9]), 10, [0], return_lse=True)
    assert not got[:3].any() and not got[5:].any() and (lse[:, :3] == -math.inf).all() and (lse[:, 5:] == -math.inf).all()
    want = swa_oracle.cached_attention(to_np(q[3:5]), values[0][0][:2], values[0][1][:2], 10, [0], 0.125)
    check_rows(got[3:5], lse[:, 3:5], *want, 64, "two tokens, five rows")
    # a page id outside the pool: its keys are left out
    hole = table.clone()
    hole[0, 1] = 10 ** 6
    got, lse = lca.sliding_window_attention_cached(q[:1], pool, hole[:1], ints([40]), ints([0, 1]), 100, [], return_lse=True)
    keep = np.r_[0:16, 32:40]
    want = swa_oracle.cached_attention(to_np(q[:1]), values[0][0][keep], values[0][1][keep], 100, [], 0.125)
    check_rows(got, lse, *want, 64, "a missing page")
    hole[:] = -3
    got, lse = lca.sliding_window_attention_cached(q[:1], pool, hole[:1], ints([40]), ints([0, 1]), 100, [], return_lse=True)
    assert not got.any() and (lse == -math.inf).all()
    # a length past the table's capacity is the capacity
    a = lca.sliding_window_attention_cached(q[:1], pool, table[:1], ints([10 ** 9]), ints([0, 1]), 5)
    b = lca.sliding_window_attention_cached(q[:1], pool, table[:1], ints([48]), ints([0, 1]), 5)
    # tokens 40 to 47 were never written: their random words may be scales of 2^127, whose products
    # with codes overflow to infinities and then NaN, the same in both calls
    torch.testing.assert_close(a, b, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_chunks_that_see_nothing_between_others(out_dtype):
    """Every other chunk has no cached tokens (a request that was not placed): its rows are zeros, and
    the rows of the others are those that they are without it."""
    rng = np.random.default_rng(15)
    lens = [600 + 7 * b for b in range(20)]
    pool, table, values = filled_cache(rng, lens, 8, 64, 32)
    q = torch.randn(20 * 600, 8, 64, device="cuda").bfloat16()
    kept = [n if b % 2 else 0 for b, n in enumerate(lens)]
    cu = ints(range(0, 20 * 600 + 1, 600))
    got, lse = lca.sliding_window_attention_cached(q, pool, table, ints(kept), cu, 100, [3], out_dtype=out_dtype, return_lse=True)
    got, lse = got.view(20, 600, 8, 64), lse.view(8, 20, 600)
    assert not got[::2].any() and (lse[:, ::2] == -math.inf).all()
    want, want_lse = lca.sliding_window_attention_cached(
        q.view(20, 600, 8, 64)[1::2].reshape(-1, 8, 64), pool, table[1::2].contiguous(), ints(kept[1::2]),
        ints(range(0, 10 * 600 + 1, 600)), 100, [3], out_dtype=out_dtype, return_lse=True)
    assert torch.equal(got[1::2], want.view(10, 600, 8, 64)) and torch.equal(lse[:, 1::2], want_lse.view(8, 10, 600))
    for b in (1, 19):
        one = swa_oracle.cached_attention(to_np(q[600 * b:600 * (b + 1)]), *values[b], 100, [3], 0.125)
        check_rows(got[b], lse[:, b], *one, 64, f"request {b}")


def test_strided_queries_streams_and_graphs():
    rng = np.random.default_rng(13)
    lens = [900, 40]
    pool, table, _ = filled_cache(rng, lens, 2, 128, 32)
    base = torch.randn(2, 3 * 8, 128, device="cuda").bfloat16()
    args = (pool, table, ints(lens), ints([0, 1, 2]), 4000, [1])
    want = lca.sliding_window_attention_cached(base[:, 8:16].contiguous(), *args)
    assert torch.equal(lca.sliding_window_attention_cached(base[:, 8:16], *args), want)
    q = base[:, 8:16].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(lca.sliding_window_attention_cached(q, *args), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = lca.sliding_window_attention_cached(q, *args)
    side.synchronize()
    assert torch.equal(other, want)
    # two graphs replayed in turn and at once
    graphs, outs = [], []
    for scale in (0.05, 0.1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(lca.sliding_window_attention_cached(q, *args, scale))
        graphs.append(g)
    want = [lca.sliding_window_attention_cached(q, *args, s) for s in (0.05, 0.1)]
    torch.cuda.synchronize()
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_strides_of_dimensions_of_one_do_not_matter():
    rng = np.random.default_rng(14)
    pool, table, _ = filled_cache(rng, [90], 2, 64, 32)
    row = torch.randn(1, 4 * 64 + 5, device="cuda").half()
    args = (pool, table, ints([90]), ints([0, 1]), 40)
    q = row[:, :4 * 64].view(1, 4, 64)  # one token: the row's stride is odd
    assert torch.equal(lca.sliding_window_attention_cached(q, *args),
                       lca.sliding_window_attention_cached(q.clone(), *args))
    pool, table, _ = filled_cache(rng, [90, 31], 1, 64, 32)
    args = (pool, table, ints([90, 31]), ints([0, 1, 2]), 40)
    q = torch.randn(2, 1, 64, device="cuda").half()
    odd = q.as_strided((2, 1, 64), (64, 5, 1))  # one head
    assert torch.equal(lca.sliding_window_attention_cached(odd, *args), lca.sliding_window_attention_cached(q, *args))


def test_refusals_on_the_device():
    pool = lca.kv_cache_pool(4, 2, 16, 64)
    table, lens, cu = ints([[0, 1]]), ints([5]), ints([0, 1])
    q = torch.zeros(1, 4, 64, device="cuda").half()

    def refuse(match, *a, error=RuntimeError, **kw):
        with pytest.raises(error, match=match):
            lca.sliding_window_attention_cached(*a, **kw)

    refuse("fp16 or bf16", q.float(), pool, table, lens, cu, 4)
    refuse("multiple", q[:, :3].contiguous(), pool, table, lens, cu, 4)
    refuse("head_dim", torch.zeros(1, 4, 128, device="cuda").half(), pool, table, lens, cu, 4)
    refuse("window_size", q, pool, table, lens, cu, -1)
    refuse("window_size", q, pool, table, lens, cu, [4, 4, 4, 4], error=TypeError)
    refuse("capacity", q, pool, table, lens, cu, 4, [32], error=IndexError)
    refuse("int32", q, pool, table, lens, cu.long(), 4)
    refuse("cu_seqlens", q, pool, table, lens, ints([0, 1, 1]), 4)
    refuse("pool", q, pool.float(), table, lens, cu, 4)
    refuse("same device|int32", q, pool, table.cpu(), lens, cu, 4)
    refuse("out must be", q, pool, table, lens, cu, 4, out=torch.empty(2, 4, 64, device="cuda"))
    refuse("float32, float16 or bfloat16", q, pool, table, lens, cu, 4, out_dtype=torch.float64)
    refuse("backward", q.clone().requires_grad_(), pool, table, lens, cu, 4, error=NotImplementedError)
    with pytest.raises(RuntimeError, match="kv_heads"):
        lca.kv_cache_append(pool, q, q, ints([0]))
    with pytest.raises(RuntimeError, match="one type"):
        lca.kv_cache_append(pool, q[:, :2], q[:, :2].bfloat16(), ints([0]))
    with pytest.raises(RuntimeError, match="page_size"):
        lca.kv_cache_layout(table, lens, lens, ints([1]), ints([1]), 20, 4)
    with pytest.raises(RuntimeError, match="one length"):
        lca.kv_cache_layout(table, lens, ints([1, 2]), ints([1]), ints([1]), 16, 4)


# ------------------------------------------------------------------ together


def test_serving_loop_equals_one_causal_pass():
    """Prompts in chunks, then single tokens, requests that end and slots that are used again: every row
    equals the causal definition over the values that the cache holds."""
    rng = np.random.default_rng(20)
    heads, kv_heads, d, page, window, tokens = 4, 2, 64, 16, 20, [0, 1, 30]
    cache = lca.QuantizedKVCache(40, page, kv_heads, d, 3, device="cuda")
    kept = [[], [], []]  # per request the K and V rows so far
    free_before = cache.free_count.item()
    steps = [([30, 7, 0], None), ([25, 1, 50], None), ([1, 1, 1], None), ([1, 1, 1], [0, 1, 0]), ([1, 40, 1], None),
             ([1, 1, 1], [1, 0, 1]), ([16, 1, 0], None), ([1, 1, 0], None)]
    for new, done in steps:
        if done is not None:
            cache.release(torch.tensor(done, dtype=torch.bool, device="cuda"))
            kept = [[] if x else r for x, r in zip(done, kept)]
        total = sum(new)
        step = cache.reserve(ints(new), total + 5)
        assert step.placed.tolist() == new
        q, k, v = (torch.tensor(rng.standard_normal((total + 5, n, d)), dtype=torch.float32).bfloat16()
                   for n in (heads, kv_heads, kv_heads))
        cache.append(k.cuda(), v.cuda(), step)
        out, lse = cache.attention(q.cuda(), step, window, tokens, return_lse=True)
        at = 0
        for b, n in enumerate(new):
            r = slice(at, at + n)
            at += n
            if n == 0:
                continue
            kept[b].append((k[r].float().numpy(), v[r].float().numpy()))
            ks, vs = (swa_oracle.kv4_values(np.concatenate([x[i] for x in kept[b]])) for i in (0, 1))
            assert step.positions[r].tolist() == list(range(len(ks) - n, len(ks)))
            want = swa_oracle.cached_attention(q[r].float().numpy(), ks, vs, window, tokens, 1 / 8)
            check_rows(out[r], lse[:, r], *want, d, f"step {new} request {b}")
            mine, _ = lca.kv_cache_read(cache.pool, step.slots[r])
            np.testing.assert_array_equal(to_np(mine), ks[-n:].astype(np.float32))
    cache.release(torch.ones(3, dtype=torch.bool, device="cuda"))
    assert cache.free_count.item() == free_before and not cache.seq_lens.any()
    assert sorted(cache.free_pages.tolist()) == list(range(40))


def test_captured_step_advances_with_new_lengths():
    """One captured step (reserve, append, attention) replayed with other lengths equals eager calls."""
    heads, d, page = 2, 64, 16
    caches = [lca.QuantizedKVCache(30, page, heads, d, 2) for _ in range(2)]
    new = ints([1, 1])
    q, k, v = (torch.zeros(8, heads, d, device="cuda").half() for _ in range(3))

    def one(cache):
        step = cache.reserve(new, 8)
        cache.append(k, v, step)
        return cache.attention(q, step, 12, [0]), step

    eager = caches[1]
    new.copy_(ints([0, 0]))
    one(caches[0])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, step = one(caches[0])
    rng = np.random.default_rng(21)
    for lens in ([5, 3], [1, 1], [0, 8], [1, 0], [2, 6]):
        new.copy_(ints(lens))
        for t in (q, k, v):
            t.copy_(torch.tensor(rng.standard_normal(t.shape), dtype=torch.float32))
        g.replay()
        want, other = one(eager)
        n = sum(lens)
        assert torch.equal(out[:n], want[:n]) and torch.equal(step.slots, other.slots)
        assert torch.equal(caches[0]._state, eager._state) and torch.equal(caches[0].block_table, eager.block_table)


def test_a_request_that_does_not_fit_attends_to_nothing():
    cache = lca.QuantizedKVCache(2, 16, 1, 64, 2, 2)
    q = torch.randn(40, 1, 64, device="cuda").half()
    step = cache.reserve(ints([20, 20]), 40)
    cache.append(q, q, step)
    out, lse = cache.attention(q, step, 50, return_lse=True)
    assert step.placed.tolist() == [20, 0] and cache.seq_lens.tolist() == [20, 0]
    assert out[:20].any(-1).all() and not out[20:].any() and (lse[:, 20:] == -math.inf).all()
