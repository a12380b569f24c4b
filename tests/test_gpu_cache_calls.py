"""Calls of the quantised cache that its documentation allows and that once went wrong: each against what it means."""
import pytest
import torch

import torchpairwise_b200 as tpw
from attention_cases import assert_near
from cache_cases import attended, filled

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def ints(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("queries", [4, 300])
def test_a_window_over_all_keys_is_none(dtype, queries):
    cache = filled(2, 4096, 2, 128, 4, 32, seed=30)
    q = torch.randn(2, queries, 4, 128, generator=torch.Generator().manual_seed(31)).to(dtype).cuda()
    n = ints(4096, 2700)
    want = tpw.cache_attention(q, cache, n, causal=True, return_lse=True)
    assert_near(want[0], attended(q, cache, [4096, 2700], causal=True)[0], dtype, "out")
    for window in (4096, 4097, 2 ** 31, 2 ** 63 - 1 - queries, 2 ** 63 - 1):
        torch.cuda.empty_cache()
        torch.full((16 << 20,), float("nan"), device="cuda")   # scratch is cut from what this leaves: read before it is written, it would show
        got = tpw.cache_attention(q, cache, n, causal=True, window=window, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), window


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("queries", [3, 300])
def test_large_finite_numbers_that_no_query_sees(dtype, queries):
    """Before the first window's block, and from a sequence's length on: numbers near the top, not NaN, change no bit."""
    lengths, window = [900, 640], 100
    cache = filled(2, 1024, 2, 64, 4, 32, seed=32)
    q = torch.randn(2, queries, 4, 64, generator=torch.Generator().manual_seed(33)).to(dtype).cuda()
    n = ints(*lengths)
    want = tpw.cache_attention(q, cache, n, causal=True, window=window, return_lse=True)
    assert_near(want[0], attended(q, cache, lengths, causal=True, window=window)[0], dtype, "out")
    loud = [t.clone() for t in cache[:4]]
    for b, length in enumerate(lengths):
        for part in (slice(0, max(0, length - queries + 1 - window) // 128 * 128), slice(length, None)):
            for scales in loud[2:]:
                scales[b, :, part] = 2.0 ** 60
    got = tpw.cache_attention(q, tpw.QuantizedCache(*loud, 64, 4), n, causal=True, window=window, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
