"""Attention over a quantised cache whose values differ in magnitude within a head: the small ones keep their digits beside the large ones."""
import pytest
import torch

import torchpairwise_b200 as tpw
from attention_cases import assert_near
from cache_cases import attended, values

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
# The bounds are those of any other call, taken over the small values alone: a probability times a step is rounded once (float16's 2^-11, float32 in two
# parts of them), the result once in its type, and neither depends on how large other groups, or tokens with no weight, are.


def scene(ratio, queries, heads=4, key_heads=2, d=128, keys=300, bits=4, group=32):
    g = torch.Generator().manual_seed(ratio + queries)
    k, v = (torch.randn(2, keys, key_heads, d, generator=g).cuda() for _ in range(2))
    q = 2 * torch.randn(2, queries, heads, d, generator=g).cuda()
    n = torch.tensor([keys, keys - 37], dtype=torch.int32, device="cuda")
    cache = tpw.quantized_cache(2, keys, key_heads, d, bits=bits, group=group)
    return q, k, v, n, cache


def stored(cache, k, v):
    tpw.cache_write(cache, k, v, torch.full((k.shape[0],), k.shape[1], dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("queries", [1, 5, 250])
@pytest.mark.parametrize("ratio", [8, 14, 20])
@pytest.mark.parametrize("bits", [4, 8])
def test_a_group_of_large_values_beside_small_ones(dtype, queries, ratio, bits):
    q, k, v, n, cache = scene(ratio, queries, bits=bits)
    v = v * 2.0 ** (-ratio // 2)
    v[..., 32:64] *= 2.0 ** ratio
    stored(cache, k, v)
    q = q.to(dtype)
    out = tpw.cache_attention(q, cache, n, causal=True)
    want = attended(q, cache, n.tolist(), causal=True)[0]
    small = torch.ones(128, dtype=torch.bool, device="cuda")
    small[32:64] = False
    assert_near(out[..., small], want[..., small], dtype, "small groups")
    assert_near(out[..., ~small], want[..., ~small], dtype, "large group")
    assert tpw.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("queries", [1, 5, 250])
@pytest.mark.parametrize("ratio", [8, 14, 20])
@pytest.mark.parametrize("bits,group", [(4, 32), (4, None), (8, None)])
@pytest.mark.parametrize("place", [0, 130, 261])
def test_a_large_token_that_nobody_attends_to(dtype, queries, ratio, bits, group, place):
    """Its score is about 60 below the others', so that it takes e^-60 times the ratio of the result: nothing."""
    q, k, v, n, cache = scene(ratio, queries, bits=bits, group=group)
    q[..., 0] = 4.0
    k[..., 0] = 0.0
    k[:, place, :, 0] = -60 * 128 ** 0.5 / 4
    v = v * 2.0 ** (-ratio // 2)
    v[:, place] *= 2.0 ** ratio
    stored(cache, k, v)
    q = q.to(dtype)
    out = tpw.cache_attention(q, cache, n)
    want = attended(q, cache, n.tolist())[0]
    assert_near(out, want, dtype, "out")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("queries", [1, 3])
@pytest.mark.parametrize("ratio", [8, 20])
@pytest.mark.parametrize("heads", [4, 32])
def test_a_large_token_that_another_head_attends_to(dtype, queries, ratio, heads):
    """Heads that share keys: the first looks at the large token alone, the others at all but that one, each in its own magnitude."""
    q, k, v, n, cache = scene(ratio, queries, heads=heads, key_heads=2 if heads < 8 else 4)
    group = heads // cache.k_codes.shape[1]
    sees = (torch.arange(heads, device="cuda") % group == 0)[None, None, :]
    q[..., 0] = torch.where(sees, 4.0, -4.0)
    k[..., 0] = 0.0
    k[:, 200, :, 0] = 60 * 128 ** 0.5 / 4
    v = v * 2.0 ** (-ratio // 2)
    v[:, 200] *= 2.0 ** ratio
    stored(cache, k, v)
    q = q.to(dtype)
    out = tpw.cache_attention(q, cache, n)
    want = attended(q, cache, n.tolist())[0]
    first = sees[0, 0]
    assert_near(out[:, :, ~first], want[:, :, ~first], dtype, "the others")
    assert_near(out[:, :, first], want[:, :, first], dtype, "the first")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("queries", [1, 5])
def test_large_tokens_that_lose_their_weight_on_the_way(dtype, queries):
    """Scores climb by 8 from block to block while values fall by 2^6: what came first, large as it was, ends as nothing."""
    q, k, v, n, cache = scene(1, queries, keys=640)
    block = torch.arange(640, device="cuda") // 64
    q[..., 0] = 4.0
    k[..., 0] = (block * 8 * 128 ** 0.5 / 4)[None, :, None]
    v = v * torch.exp2(10.0 - 2 * block)[None, :, None, None]
    stored(cache, k, v)
    q = q.to(dtype)
    n = n.fill_(640)
    out, lse = tpw.cache_attention(q, cache, n, return_lse=True)
    want = attended(q, cache, [640, 640])
    assert_near(out, want[0], dtype, "out")
    assert_near(lse, want[1], torch.float32, "lse")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_constant_tokens_and_storage_that_was_never_written(dtype):
    """Steps at the bottom (2^-100, all values of a token alike) and of zero, before and between others."""
    q, k, v, n, cache = scene(2, 5, keys=512)
    v[:, :130] = 3.0
    v[:, 200:230] = -1.5
    stored(cache, k, v)
    for t in (cache.v_codes, cache.v_scales):
        t[:, :, 64:100] = 0
        t[:, :, 300:310] = 0
    q = q.to(dtype)
    out = tpw.cache_attention(q, cache, n)
    assert_near(out, attended(q, cache, n.tolist())[0], dtype, "out")
    n = n.fill_(130)
    out = tpw.cache_attention(q, cache, n)
    assert_near(out, attended(q, cache, n.tolist())[0], dtype, "constant values")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("queries", [1, 4, 20])
@pytest.mark.parametrize("bits,group", [(4, 32), (4, None), (8, 32)])
def test_keys_far_from_zero_and_queries_whose_groups_cancel(dtype, queries, bits, group):
    """Scores are held in 32 bits, the sums of a group's queries that meet its zero among them: terms of about 50 * 32 that cancel, of which four truncations
    leave 2^-22, 3e-5 of a score after its scale; log-sums are about 40, so that 2^-19 of them (8e-5) is twice that."""
    q, k, v, n, cache = scene(3, queries, bits=bits, group=group)
    q = q / 2
    q[..., :32] += 1
    q[..., 32:64] -= 1
    stored(cache, k + 50, v)
    q = q.to(dtype)
    lse = tpw.cache_attention(q, cache, n, return_lse=True)[1]
    assert_near(lse, attended(q, cache, n.tolist())[1], torch.float32, "lse", times=0.25)


@pytest.mark.parametrize("queries", [1, 7, 100])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("group", [32, None])
def test_float32_scores_of_some_size_keep_their_digits(queries, bits, group):
    """Scores up to about 30, of which float32 sums leave some 2^-24 a term: 128 of them, about 1 each, 2^-20 of a probability; the bound is 8 times that."""
    q, k, v, n, cache = scene(4, queries, bits=bits, group=group)
    loud = 1 + 4 * (torch.rand(128, generator=torch.Generator().manual_seed(5)) < 0.06).cuda()
    stored(cache, k * loud, v)
    q = 2 * q
    out, lse = tpw.cache_attention(q, cache, n, causal=True, return_lse=True)
    want = attended(q, cache, n.tolist(), causal=True)
    assert_near(out, want[0], torch.float32, "out")
    assert_near(lse, want[1], torch.float32, "lse", times=0.125)


@pytest.mark.parametrize("bits,group,d", [(4, 32, 128), (4, None, 64), (8, 32, 64), (8, None, 128)])
def test_long_caches_that_are_attended_to_evenly(bits, group, d):
    """Results of tens of thousands of about equal terms are hundreds of times smaller than those: the bound of any other float16 call holds for them."""
    batch, keys, heads = 16, 65536, 8
    g = torch.Generator(device="cuda").manual_seed(6)
    cache = tpw.quantized_cache(batch, keys, heads, d, bits=bits, group=group)
    n = torch.full((batch,), keys, dtype=torch.int32, device="cuda")
    for b in range(batch):
        one = tpw.QuantizedCache(*(t[b:b + 1] for t in cache[:4]), d, bits)
        k, v = (torch.randn(1, keys, heads, d, generator=g, device="cuda") for _ in range(2))
        tpw.cache_write(one, k, v, n[:1])
    q = (0.2 * torch.randn(batch, 1, 2 * heads, d, generator=g, device="cuda")).half()
    out, lse = tpw.cache_attention(q, cache, n, return_lse=True)
    k, v = (x[0].double() for x in tpw.cache_read(one, n[:1], dtype=torch.float32))
    for h in range(2 * heads):
        s = k[:, h // 2] @ q[-1, 0, h].double() * d ** -0.5
        assert_near(out[-1, 0, h], torch.softmax(s, 0) @ v[:, h // 2], torch.float16, "out")
        assert_near(lse[-1, h], torch.logsumexp(s, 0, keepdim=True), torch.float32, "lse")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("queries", [1, 5, 40])
@pytest.mark.parametrize("weight,size", [(6, -6), (10, -9), (20, -12), (10, None), (40, -14), (80, -30)])
@pytest.mark.parametrize("options", [dict(), dict(causal=True), dict(causal=True, window=333)], ids=str)
def test_a_first_token_that_takes_the_weight_and_has_small_values(dtype, queries, weight, size, options):
    """Scores of the first token, and of one in the middle, lie far above the others', its values far below: what the rest adds keeps its digits."""
    q, k, v, n, cache = scene(7, queries, keys=640)
    q = q / 2
    q[..., 0] = 4.0
    q[:, :, 1:, 0] = 1.0   # and not for every head
    k[..., 0] = 0.0
    k[:, [0, 401], :, 0] = weight * 128 ** 0.5 / 4
    v[:, [0, 401]] *= 0.0 if size is None else 2.0 ** size
    stored(cache, k, v)
    q = q.to(dtype)
    n = torch.tensor([640, 517], dtype=torch.int32, device="cuda")
    out, lse = tpw.cache_attention(q, cache, n, return_lse=True, **options)
    want = attended(q, cache, n.tolist(), **options)
    # The large tokens' scores S have one term of about S among 128, which a sum in 32 bits cuts off by up to 2^-23 S in each of the dozen steps that follow: between two such
    # tokens (float32 results follow their ratio, 16-bit ones are coarser) that may be 24 * 2^-23 S, or 2^-18.4 S; S / 4 of the type's 2^-17, 2^-19 S, allow two thirds of it.
    times = 1 + weight / 4 if dtype == torch.float32 else 1
    for h in range(4):
        if dtype == torch.float16 and float(want[0][:, :, h].abs().max()) < 2.0 ** -14:   # below which its numbers lie 2^-24 apart
            assert bool(((out[:, :, h] - want[0][:, :, h]).abs() <= 2.0 ** -25 + 2.0 ** -10 * want[0][:, :, h].abs().max()).all())
        else:
            assert_near(out[:, :, h], want[0][:, :, h], dtype, "out", times=times)
    assert_near(lse, want[1], torch.float32, "lse")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("queries", [1, 30])
def test_scores_near_the_top(dtype, queries):
    """Scores of millions, where 32 bits hold them to a unit: finite results, of the keys that have the highest."""
    q, k, v, n, cache = scene(8, queries, keys=640)
    k[..., 0] = 0.0
    k[:, 100::7, :, 0] = 3000.0   # all the same: kept exactly, as the highest of their groups
    k[:, 100::7, :, 1:] = 0.0
    v = v * torch.exp2(torch.randint(-6, 7, v.shape[:2], generator=torch.Generator().manual_seed(9)).float()).cuda()[..., None, None]
    stored(cache, k, v)
    q[..., 0] = 40000.0 if dtype == torch.float16 else 60000.0
    q = q.to(dtype)
    out = tpw.cache_attention(q, cache, n)
    for b, length in enumerate(n.tolist()):
        want = values(cache)[1][b, 100:length:7].mean(0)   # [heads, features]
        for h in range(4):
            assert_near(out[b, :, h], want[h // 2].expand(queries, -1), dtype, "out")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("queries", [1, 5, 250])
@pytest.mark.parametrize("bits,group", [(4, 32), (4, None), (8, 32), (8, None)])
def test_values_that_are_zero_stay_zero(dtype, queries, bits, group):
    """Groups of zeros have a step all the same (2^-100): what is all zeros gives zeros, to the last bit."""
    q, k, v, n, cache = scene(9, queries, bits=bits, group=group)
    stored(cache, k, torch.zeros_like(v))
    q = q.to(dtype)
    assert not tpw.cache_attention(q, cache, n, causal=True).any()
    if group:
        v[..., 32:64] = 0
        stored(cache, k, v)
        out = tpw.cache_attention(q, cache, n, causal=True)
        assert not out[..., 32:64].any()
        assert_near(out, attended(q, cache, n.tolist(), causal=True)[0], dtype, "out")
