"""How window_attention and prefix_attention may be called: threads, transforms and tracers, views, single queries, repeats."""

import pytest
import torch

from cache_attention_ref import check, reference
from test_cache_attention_gpu import PREFIX, WINDOW, cache, no_wait_gave_up, rand  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Hq,Hkv,Sq,P,D", [(13, 14, 2, 3, 5003, 64), (40, 14, 2, 3, 3000, 128), (5, 32, 8, 1, 16000, 128)])
def test_packed_rows_do_not_depend_on_what_ran_before(B, Hq, Hkv, Sq, P, D, dtype):
    """The rows of the packed product that no query fills: the same bits whatever earlier kernels left in shared memory."""
    q, k, v = cache(B, Hq, Hkv, Sq, 40, D, dtype=dtype, seed=B)
    pre = [rand(Hkv, P, D, dtype=dtype, seed=50 + i) for i in range(2)]
    full = cache(64, 8, 2, 4, 40, D, dtype=dtype, seed=3)           # 16 rows per sequence: all 128 rows in use
    long = [rand(2, 20000, D, dtype=dtype, seed=60 + i) for i in range(2)]
    first = None
    for size in (0.0, 1.0, 30.0, 100.0, 0.0, 300.0):
        PREFIX(full[0] * size, *long, *full[1:])
        got = PREFIX(q, *pre, k, v)
        first = got if first is None else first
        assert torch.equal(got, first), size
    check(first, reference(q, k, v, prefix=pre))


@pytest.mark.parametrize("B,Hq,Hkv,Skv,D,window,sinks", [(64, 8, 8, 2000, 128, 16, 1000), (32, 32, 8, 4500, 128, 128, 4096), (150, 8, 8, 700, 64, 1, 333)])
def test_hidden_keys_of_a_single_query_with_many_sinks(B, Hq, Hkv, Skv, D, window, sinks):
    """With one query per sequence hidden keys may hold anything, however many sequences and sinks there are."""
    q, k, v = cache(B, Hq, Hkv, 1, Skv, D)
    want = WINDOW(q, k, v, window, sinks)
    few = slice(0, 3)
    check(want[few], reference(q[few], k[few], v[few], window=window, sinks=sinks))
    k[:, :, sinks:Skv - window], v[:, :, sinks:Skv - window] = float("nan"), float("inf")
    assert torch.equal(WINDOW(q, k, v, window, sinks), want)
