"""What the operators of the 4-bit cache refuse on the device, beside the refusals of test_gpu_kv_cache.py."""
import pytest
import torch
from torch.autograd import forward_ad

import long_context_attention as lca

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_forward_mode_tangents_are_refused():
    pool = lca.kv_cache_pool(4, 2, 16, 64)
    table, lens, cu = ints([[0, 1]]), ints([5]), ints([0, 1])
    q, k = torch.zeros(1, 4, 64, device="cuda").half(), torch.zeros(1, 2, 64, device="cuda").half()
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            lca.sliding_window_attention_cached(forward_ad.make_dual(q, torch.ones_like(q)), pool, table, lens, cu, 4)
        for pair in ((forward_ad.make_dual(k, torch.ones_like(k)), k), (k, forward_ad.make_dual(k, torch.ones_like(k)))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                lca.kv_cache_append(pool, *pair, ints([0]))
        lca.kv_cache_append(pool, k, k, ints([0]))  # plain tensors pass
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: lca.sliding_window_attention_cached(t, pool, table, lens, cu, 4), (q,), (torch.ones_like(q),))


def test_an_output_that_requires_grad_is_refused():
    """Written in place behind autograd's back, it would leave a graph with values that it never saved."""
    pool = lca.kv_cache_pool(4, 2, 16, 64)
    q = torch.zeros(1, 4, 64, device="cuda").half()
    args = (q, pool, ints([[0, 1]]), ints([5]), ints([0, 1]), 4)
    leaf = torch.full((1, 4, 64), 3.0, device="cuda", requires_grad=True)
    for out in (leaf, leaf * 1.0):
        with pytest.raises(NotImplementedError, match="backward"):
            lca.sliding_window_attention_cached(*args, out=out)
        assert (out == 3.0).all()
        with torch.no_grad():  # there is no graph to mislead
            assert not lca.sliding_window_attention_cached(*args, out=out).any()  # an empty cache's values
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.zeros(1, 4, 64, device="cuda"), torch.ones(1, 4, 64, device="cuda"))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            lca.sliding_window_attention_cached(*args, out=dual)
