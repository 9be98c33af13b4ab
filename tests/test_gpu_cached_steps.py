"""Steps as a serving loop makes them, against the oracle: first chunks of prompts, with global tokens among the
new ones, beside later chunks and single tokens; single tokens in a call that was laid out for many rows."""
import math

import numpy as np
import pytest
import torch

import long_context_attention as lca
from oracle import swa_oracle
from test_gpu_kv_cache import check_attention, check_rows, filled_cache, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("lens,new,heads,kv_heads,d,window,tokens", [
    ([500, 1900, 1200, 900, 1, 0], [500, 150, 1, 1, 1, 0], 4, 2, 64, 100, list(range(16))),     # one kernel for all of them
    ([40, 2100, 1300, 7] + [350] * 30, [40, 1, 1, 7] + [1] * 30, 8, 2, 128, 64, [0, 1, 2, 30]),  # and the other
    ([700, 90], [700, 90], 2, 1, 64, 10 ** 5, [0, 650]),                                        # prompts from empty, plain causal
])
def test_mixed_steps(lens, new, heads, kv_heads, d, window, tokens, dtype, out_dtype):
    check_attention(np.random.default_rng(len(lens)), lens, new, heads, kv_heads, d, 32, window, tokens, dtype, out_dtype)


@pytest.mark.parametrize("window", [60, 10 ** 5])
def test_few_tokens_in_a_call_of_many_rows(window):
    rng = np.random.default_rng(window)
    lens, d, heads, rows = [2000, 17, 900], 128, 4, 4096
    pool, table, values = filled_cache(rng, lens, 2, d, 64)
    q = torch.tensor(rng.standard_normal((rows, heads, d)), dtype=torch.float32).bfloat16()
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    got, lse = lca.sliding_window_attention_cached(q.cuda(), pool, table, ints(lens), ints([0, 1, 2, 4]), window, [3], out=out,
                                                   return_lse=True)
    assert (out[4:] == 7.0).all()
    for b, r in enumerate((slice(0, 1), slice(1, 2), slice(2, 4))):
        want = swa_oracle.cached_attention(q[r].float().numpy(), *values[b], window, [3], 1 / math.sqrt(d))
        check_rows(got[r], lse[:, r], *want, d, f"request {b}")
