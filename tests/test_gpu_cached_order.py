"""What follows cached attention in a stream finds its results complete (eager and in a captured graph), also
where the call reckons with items that several CTAs share and none of them is long enough."""
import pytest
import torch

import long_context_attention as lca

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,new", [([1], 1), ([100], 1), ([250], 4), ([60, 3, 128], 1), ([300], 1), ([190, 240], 40), ([190], 70)])
@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16])
def test_what_follows_finds_the_results(lens, new, out_dtype):
    """A window of everything over a table of 8192 tokens, short contexts.  The consumer that matters is
    one that is launched as early as the operators here are: an append of the output as keys."""
    kv_heads, heads, d, page, batch = 8, 8, 128, 16, len(lens)
    gen = torch.Generator("cuda").manual_seed(sum(lens))

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(out_dtype)

    width = 8192 // page
    pool = lca.kv_cache_pool(batch * 20, kv_heads, page, d)
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):
        table[b, :20] = torch.arange(20 * b, 20 * b + 20, device="cuda")
        slots = torch.arange(n, dtype=torch.int32, device="cuda") + 20 * page * b
        lca.kv_cache_append(pool, randn(n, kv_heads, d), randn(n, kv_heads, d), slots)
    kv_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cu = torch.arange(batch + 1, dtype=torch.int32, device="cuda") * new
    rows = batch * new
    q = randn(rows, heads, d)
    out = torch.zeros(rows, heads, d, dtype=out_dtype, device="cuda")
    after = lca.kv_cache_pool(rows // page + 1, heads, page, d)
    at = torch.arange(rows, dtype=torch.int32, device="cuda")
    args = (q, pool, table, kv_lens, cu, 8192)
    lse = None

    def step():
        nonlocal lse
        out.zero_()
        _, lse = lca.sliding_window_attention_cached(*args, out=out, return_lse=True)
        lca.kv_cache_append(after, out, out, at)
        return out.clone(), lse.clone()

    _, want_lse = lca.sliding_window_attention_cached(*args, out=out, return_lse=True)
    torch.cuda.synchronize()
    want, want_lse = out.clone(), want_lse.clone()
    torch.cuda.synchronize()
    lca.kv_cache_append(after, want, want, at)
    torch.cuda.synchronize()
    want_after = after.clone()
    assert want.any()

    bad = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(20):
        after.zero_()
        got, got_lse = step()
        bad += (after != want_after).any() | (got != want).any() | (got_lse != want_lse).any()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, got_lse = step()
    for _ in range(200):
        after.zero_()
        graph.replay()
        bad += (after != want_after).any() | (got != want).any() | (got_lse != want_lse).any()
    assert bad.item() == 0
    assert lca.device_error() == 0
