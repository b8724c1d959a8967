"""How window_attention and prefix_attention may be called: threads, transforms and tracers, views, single queries, repeats."""

import pytest
import torch

from cache_attention_ref import check, reference
from test_cache_attention_gpu import WINDOW, cache, no_wait_gave_up  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,Hq,Hkv,Skv,D,window,sinks", [(64, 8, 8, 2000, 128, 16, 1000), (32, 32, 8, 4500, 128, 128, 4096), (150, 8, 8, 700, 64, 1, 333)])
def test_hidden_keys_of_a_single_query_with_many_sinks(B, Hq, Hkv, Skv, D, window, sinks):
    """With one query per sequence hidden keys may hold anything, however many sequences and sinks there are."""
    q, k, v = cache(B, Hq, Hkv, 1, Skv, D)
    want = WINDOW(q, k, v, window, sinks)
    few = slice(0, 3)
    check(want[few], reference(q[few], k[few], v[few], window=window, sinks=sinks))
    k[:, :, sinks:Skv - window], v[:, :, sinks:Skv - window] = float("nan"), float("inf")
    assert torch.equal(WINDOW(q, k, v, window, sinks), want)
