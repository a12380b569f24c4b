"""The quantised cache as programs use it and where kernels go wrong: masked places that hold no numbers, exponents far apart, streams and graphs, long storage,
bad arguments, and the operators one after the other."""
import math
import random

import pytest
import torch

import torchpairwise_b200 as tpw
from attention_cases import NORM_TOL, assert_near
from cache_cases import attended, filled, values

pytestmark = pytest.mark.gpu


def ints(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


def scaled_by(x, exponent):
    return torch.ldexp(x, torch.tensor(exponent, device=x.device))


def spoiled(cache, lengths, first=None):
    """The cache with all that no call may use, from a sequence's length on and before `first`, set to bits that are no numbers."""
    out = [t.clone() for t in cache[:4]]
    for b, n in enumerate(lengths):
        for codes, scales in ((out[0], out[2]), (out[1], out[3])):
            for part in (slice(n, None), slice(0, first[b] if first else 0)):
                codes[b, :, part] = 0xff
                scales[b, :, part, :, 0] = math.nan
                scales[b, :, part, :, 1] = math.inf
    return tpw.QuantizedCache(*out, cache.features, cache.bits)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("bits,group,d", [(4, 32, 128), (4, None, 64), (8, 32, 96), (8, None, 40)])
@pytest.mark.parametrize("queries,heads", [(1, 4), (5, 8), (200, 4)])
def test_what_lies_outside_is_never_used(dtype, bits, group, d, queries, heads):
    lengths = [700, 333, 0, 64]
    cache = filled(4, 900, 2, d, bits, group, seed=5)
    g = torch.Generator().manual_seed(6)
    q = torch.randn(4, queries, heads, d, generator=g).to(dtype).cuda()
    for options in (dict(causal=True), dict(), dict(causal=True, window=100)):
        want = tpw.cache_attention(q, cache, ints(*lengths), return_lse=True, **options)
        # keys before the first window are outside too, but for those of the block of 128 that it begins in
        first = [max(0, n - queries + 1 - 100) // 128 * 128 if "window" in options else 0 for n in lengths]
        got = tpw.cache_attention(q, spoiled(cache, lengths, first), ints(*lengths), return_lse=True, **options)
        assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
        assert not got[0][2].any() and bool((got[1][2] == -math.inf).all())
    a, b = tpw.cache_read(cache, ints(*lengths), dtype=dtype), tpw.cache_read(spoiled(cache, lengths), ints(*lengths), dtype=dtype)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert tpw.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("queries", [4, 300])
def test_a_key_or_value_that_is_no_number_makes_its_rows_nan(dtype, queries):
    cache = filled(1, 640, 1, 64, 4, 32, seed=7)
    q = torch.randn(1, queries, 2, 64, generator=torch.Generator().manual_seed(8)).to(dtype).cuda()
    n = ints(600)
    for which in (2, 3):
        bad = [t.clone() for t in cache[:4]]
        bad[which][0, 0, 599] = math.nan   # the last key: only the last query sees it
        out = tpw.cache_attention(q, tpw.QuantizedCache(*bad, 64, 4), n, causal=True)
        assert bool(out[0, -1].isnan().any())
        # rows of other tiles: of up to 16 rows in a line of all heads' queries, so that a head's first 15 can be with another's last, or of 128 queries of a
        # head, whose last ones see keys of the same 128 (from 512 on) from query 212 on
        assert bool(out[0, 16:128].isfinite().all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("queries", [1, 2, 250])
@pytest.mark.parametrize("keys,numbers", [(0, 0), (40, 0), (-60, 0), (0, -90), (0, 60), (20, 40)])
def test_exponents_far_from_one_another(dtype, queries, keys, numbers):
    """Keys times 2^keys with queries times 2^-keys, values times 2^numbers: the same probabilities, results times 2^numbers."""
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(2, 500, 2, 128, generator=g).cuda() for _ in range(2))
    v = v + 4   # zeros that are not small beside steps
    q = torch.randn(2, queries, 8, 128, generator=g).cuda()
    cache = tpw.quantized_cache(2, 500, 2, 128)
    n = ints(500, 321)
    tpw.cache_write(cache, scaled_by(k, keys), scaled_by(v, numbers), ints(500, 500))
    q = scaled_by(q, -keys).to(dtype)
    out, lse = tpw.cache_attention(q, cache, n, causal=True, return_lse=True)
    want = attended(q, cache, [500, 321], causal=True)
    assert_near(scaled_by(out.double(), -numbers), scaled_by(want[0], -numbers), dtype, "out")
    assert_near(lse, want[1], torch.float32 if queries < 250 else dtype, "lse")


def test_heads_of_other_magnitudes_keep_their_digits():
    """Many bfloat16 queries: a head whose values are 2^40 times another's, and a sequence with a group that is no number, cost the other nothing."""
    g = torch.Generator().manual_seed(10)
    k, v = (torch.randn(2, 640, 2, 64, generator=g).cuda() for _ in range(2))
    q = torch.randn(2, 300, 4, 64, generator=g).bfloat16().cuda()
    scaled = v.clone()
    scaled[:, :, 1] *= 2.0 ** 40
    scaled[1, 639, 1, 3] = math.nan
    cache, plain = (tpw.quantized_cache(2, 640, 2, 64) for _ in range(2))
    tpw.cache_write(cache, k, scaled, ints(640, 640))
    tpw.cache_write(plain, k, v, ints(640, 640))
    n = ints(640, 600)
    got, want = (tpw.cache_attention(q, c, n, causal=True) for c in (cache, plain))
    assert torch.equal(got[:, :, :2], want[:, :, :2])
    assert torch.equal(got[:, :, 2:], scaled_by(want[:, :, 2:].float(), 40).bfloat16())


def test_the_same_bits_each_time_whatever_the_lengths():
    rng = random.Random(11)
    for _ in range(150):
        hk = rng.choice([1, 2, 3])
        hq, batch, d = hk * rng.choice([1, 2, 5, 8]), rng.randint(1, 5), rng.choice([8, 40, 64, 72, 96, 104, 128])
        nq, cap = rng.choice([1, 1, rng.randint(2, 9), rng.randint(10, 120)]), rng.choice([rng.randint(1, 300), rng.randint(300, 3000)])
        bits, group = rng.choice([4, 8]), rng.choice([32, None])
        causal = rng.random() < 0.7
        window = rng.choice([None, rng.randint(1, 500)]) if causal else None
        dtype = rng.choice([torch.bfloat16, torch.float16, torch.float32])
        cache = filled(batch, cap, hk, d, bits, group, seed=rng.randint(0, 99))
        lengths = [rng.choice([0, rng.randint(0, cap)]) for _ in range(batch)]
        q = torch.randn(batch, nq, hq, d, device="cuda", dtype=dtype)
        runs = [tpw.cache_attention(q, cache, ints(*lengths), causal=causal, window=window, return_lse=True) for _ in range(3)]
        for other in runs[1:]:
            assert torch.equal(runs[0][0], other[0]) and torch.equal(runs[0][1], other[1])
        want = attended(q, cache, lengths, causal=causal, window=window)
        assert_near(runs[0][0], want[0], dtype, (hk, hq, batch, d, nq, cap, bits, group, causal, window, lengths))
    assert tpw.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_more_sequences_than_scratch_takes_at_once(dtype):
    """Many queries go a few sequences at a time: each as by itself."""
    cache = filled(5, 8192, 8, 128, 4, 32, seed=12)
    q = torch.randn(5, 64, 32, 128, generator=torch.Generator().manual_seed(13)).to(dtype).cuda()
    n = ints(8192, 100, 5000, 0, 7777)
    out, lse = tpw.cache_attention(q, cache, n, causal=True, return_lse=True)
    for b in range(5):
        alone = tpw.QuantizedCache(*(t[b:b + 1] for t in cache[:4]), 128, 4)
        one, l1 = tpw.cache_attention(q[b:b + 1], alone, n[b:b + 1], causal=True, return_lse=True)
        assert_near(out[b:b + 1], one.double(), dtype, "out")
        assert_near(lse[b:b + 1], l1.double(), dtype, "lse")
    alone = tpw.QuantizedCache(*(t[4:] for t in cache[:4]), 128, 4)
    assert_near(out[4:], attended(q[4:], alone, [7777], causal=True)[0], dtype, "out")


@pytest.mark.parametrize("queries,heads,features", [(1, 3, 40), (100, 4, 64)])
def test_very_many_short_sequences(queries, heads, features):
    """More sequences and heads than one grid of the many-row path takes, most of them empty, and more sequences than threads that look for a place."""
    batch = 30000
    some = filled(3, 64, heads // 2 if queries > 1 else 3, features, 4, 32, seed=21)
    pick = torch.arange(batch, device="cuda") % 3
    cache = tpw.QuantizedCache(*(t[pick].contiguous() for t in some[:4]), features, 4)
    n = torch.zeros(batch, dtype=torch.int32, device="cuda")
    for b, length in ((0, 64), (17, 5), (9999, 33), (29999, 60)):
        n[b] = length
    q = torch.randn(3, queries, heads * 2 if queries > 1 else 3, features, generator=torch.Generator().manual_seed(22)).bfloat16().cuda()
    out = tpw.cache_attention(q[pick].contiguous(), cache, n, causal=True)
    for b in (0, 17, 9999, 29999):
        alone = tpw.QuantizedCache(*(t[b:b + 1] for t in cache[:4]), features, 4)
        assert_near(out[b:b + 1], attended(q[b % 3][None], alone, [int(n[b])], causal=True)[0], torch.bfloat16, b)
    out[[0, 17, 9999, 29999]] = 0
    assert not out.any()


def test_offsets_beyond_32_bits():
    """5 GB of codes: the last sequence's rows lie past 2^32 bytes, and are those of a small cache."""
    small = filled(1, 1024, 8, 128, 8, 32, seed=14)
    cap, batch = 131072, 40
    codes = [torch.zeros(batch, 8, cap, 128, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(batch, 8, cap, 4, 2, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    big = tpw.QuantizedCache(*codes, *scales, 128, 8)
    k, v = tpw.cache_read(small, ints(1024), dtype=torch.float32)
    n = torch.zeros(batch, dtype=torch.int32, device="cuda")
    n[-1] = cap
    x = torch.zeros(batch, 1024, 8, 128, device="cuda")
    y = torch.zeros_like(x)
    x[-1], y[-1] = k[0], v[0]
    tpw.cache_write(big, x, y, n)   # what reads back exactly is stored with other steps; compare with what it reads as
    back = tpw.cache_read(big, n, tokens=1024, dtype=torch.float32)
    again = tpw.quantized_cache(1, 1024, 8, 128, bits=8)
    tpw.cache_write(again, k, v, ints(1024))
    for a, b in zip(back, tpw.cache_read(again, ints(1024), tokens=1024, dtype=torch.float32)):
        assert torch.equal(a[-1:], b) and not a[:-1].any()
    q = torch.randn(batch, 3, 16, 128, generator=torch.Generator().manual_seed(15)).bfloat16().cuda()
    out = tpw.cache_attention(q, big, n, causal=True, window=1000)
    want = attended(q[-1:], again, [1024], causal=True, window=1000)[0]
    assert_near(out[-1:], want, torch.bfloat16, "out")
    assert not out[:-1].any()


def test_streams_and_graphs():
    cache = filled(3, 2000, 2, 64, 4, 32, seed=16)
    g = torch.Generator().manual_seed(17)
    q = torch.randn(3, 2, 8, 64, generator=g).half().cuda()
    k, v = (torch.randn(3, 2, 2, 64, generator=g).half().cuda() for _ in range(2))
    long = torch.randn(3, 100, 8, 64, generator=g).half().cuda()
    n = ints(1500, 3, 2000)
    calls = [lambda: tpw.cache_attention(q, cache, n, causal=True), lambda: tpw.cache_attention(long, cache, n, causal=True), lambda: tpw.cache_read(cache, n, tokens=50)[0]]
    tpw.cache_write(cache, k, v, n)
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):   # at once, each with scratch of its own
        got = []
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(c())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # two graphs of the same calls, replayed in turn, with lengths that change in place
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            tpw.cache_write(cache, k, v, n)
            results.append([c() for c in calls])
        graphs.append(graph)
    for lengths in ((1500, 3, 2000), (7, 1999, 0), (2000, 2000, 2000)):
        n.copy_(ints(*lengths))
        tpw.cache_write(cache, k, v, n)
        want = [c() for c in calls]
        for graph in graphs + graphs[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        for result in results:
            assert all(torch.equal(a, b) for a, b in zip(result, want))
    del graphs
    assert tpw.device_status() == 0


def test_bad_arguments():
    cache = tpw.quantized_cache(2, 64, 2, 64)
    x, n = torch.zeros(2, 3, 2, 64, device="cuda"), ints(3, 3)
    q = torch.zeros(2, 1, 4, 64, device="cuda")
    R = lambda **c: cache._replace(**c)   # noqa: E731
    for call, text in (
            (lambda: tpw.cache_write(cache, x, x[:, :2], n), "same shape"), (lambda: tpw.cache_write(cache, x, x.half(), n), "type"), (lambda: tpw.cache_write(cache, x.double(), x.double(), n), "float32, float16 or bfloat16"),
            (lambda: tpw.cache_write(cache, x[:, :, :1], x[:, :, :1], n), r"must be \[2, tokens, 2, 64\]"), (lambda: tpw.cache_write(cache, x, x, n[:1]), "key_lengths"), (lambda: tpw.cache_write(cache, x, x, n.float()), "key_lengths"),
            (lambda: tpw.cache_write(cache, x, x, n.cpu()), "CUDA"), (lambda: tpw.cache_write(cache, x.clone().requires_grad_(), x, n), "gradient"),
            (lambda: tpw.cache_read(cache, n, dtype=torch.float64), "float32, float16 or bfloat16"), (lambda: tpw.cache_read(cache, n, tokens=-1), "tokens"),
            (lambda: tpw.cache_attention(q.double(), cache, n), "float32, float16 or bfloat16"), (lambda: tpw.cache_attention(q[:, :, :3], cache, n), "multiple"), (lambda: tpw.cache_attention(q[0], cache, n), "must be"),
            (lambda: tpw.cache_attention(q, cache, n, window=3), "causal"), (lambda: tpw.cache_attention(q, cache, n, causal=True, window=0), "window"), (lambda: tpw.cache_attention(q, cache, n, scale=0.0), "scale"),
            (lambda: tpw.cache_attention(q, cache, n, scale=1e-60), "scale"), (lambda: tpw.cache_attention(q.clone().requires_grad_(), cache, n), "gradient"),
            (lambda: tpw.cache_read(R(bits=5), n), "bits"), (lambda: tpw.cache_read(R(features=200), n), "features"), (lambda: tpw.cache_read(R(features=100), n), "codes must be"), (lambda: tpw.cache_read(R(bits=8), n), "codes must be"),
            (lambda: tpw.cache_read(R(k_scales=cache.k_scales[:, :, :, :1].contiguous()), n), "scales must be"), (lambda: tpw.cache_read(R(v_scales=cache.v_scales.float()), n), "scales must be"),
            (lambda: tpw.cache_read(R(v_codes=cache.k_codes), n), "must be four"), (lambda: tpw.cache_read(R(k_codes=cache.k_codes.transpose(0, 1).contiguous().transpose(0, 1)), n), "contiguous"),
            (lambda: tpw.cache_read(R(k_codes=cache.k_codes[:, :, :63].contiguous(), v_codes=cache.v_codes[:, :, :63].contiguous()), n), "multiple of 64"),
            (lambda: tpw.cache_read(cache._replace(k_codes=cache.k_codes.cpu()), n), "CUDA")):
        with pytest.raises((RuntimeError, NotImplementedError), match=text):
            call()
    with torch.no_grad():
        tpw.cache_write(cache, x.clone().requires_grad_(), x, n)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.vmap(lambda y: tpw.cache_attention(y, cache, n))(q[None])
    version = cache.k_codes._version
    tpw.cache_write(cache, x, x, n)
    assert cache.k_codes._version > version and cache.v_scales._version > 0
    # nothing to do is no error
    empty = tpw.quantized_cache(0, 64, 2, 64)
    none = ints()
    tpw.cache_write(empty, x[:0], x[:0], none)
    assert tpw.cache_read(empty, none)[0].shape == (0, 64, 2, 64) and tpw.cache_attention(q[:0], empty, none).shape == (0, 1, 4, 64)
    tpw.cache_write(cache, x[:, :0], x[:, :0], n)
    assert tpw.cache_read(cache, n, tokens=0)[1].shape == (2, 0, 2, 64) and tpw.cache_attention(q[:, :0], cache, n, return_lse=True)[1].shape == (2, 4, 0)


def test_lengths_beyond_the_capacity_and_below_zero():
    cache = filled(2, 128, 1, 64, 4, 32, seed=18)
    q = torch.randn(2, 3, 2, 64, generator=torch.Generator().manual_seed(19)).cuda()
    for many in (1, 70):
        qq = q.repeat(1, many, 1, 1)
        want = tpw.cache_attention(qq, cache, ints(128, 0), causal=True)
        for n in (ints(1000, -5), torch.tensor([2 ** 40, -(2 ** 40)], device="cuda")):
            assert torch.equal(tpw.cache_attention(qq, cache, n, causal=True), want)


@pytest.mark.parametrize("bits,group", [(4, 32), (8, None)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_serving_token_by_token(bits, group, dtype):
    """Turn, store, attend, as a decoder does it: a prompt at once, then single tokens, arrive at what attention over the values that the cache stands for gives."""
    g = torch.Generator().manual_seed(20)
    batch, prompt, steps, hq, hk, d = 3, 90, 12, 8, 2, 64
    lengths = [90, 41, 7]   # padded at their front
    total = prompt + steps
    q, k, v = (torch.randn(batch, total, h, d, generator=g).to(dtype).cuda() for h in (hq, hk, hk))
    cos, sin = tpw.rotary_table(total, d)
    cache = tpw.quantized_cache(batch, total, hk, d, bits=bits, group=group)
    n = ints(*lengths)
    outs = []

    def run(first, count):
        at = (n[:, None].long() - count + torch.arange(count, device="cuda")).clamp(min=0)
        part = slice(first, first + count)
        tq, tk = tpw.rotary_embedding(q[:, part], k[:, part], cos, sin, at)
        tpw.cache_write(cache, tk, v[:, part], n)
        outs.append(tpw.cache_attention(tq, cache, n, causal=True))
        return tq

    turned = [run(0, prompt)]
    for s in range(steps):
        n += 1
        turned.append(run(prompt + s, 1))
    got, tq = torch.cat(outs, 1), torch.cat(turned, 1)
    final = [x + steps for x in lengths]
    want = attended(tq, cache, final, causal=True)[0]
    for b, length in enumerate(lengths):
        assert not got[b, :prompt - length].any()
        assert_near(got[b:b + 1, prompt - length:], want[b:b + 1, prompt - length:], dtype, "out")
    # what the codes stand for is half a step from what was stored
    for x, (kk, vv) in ((v, values(cache)),):
        for b, length in enumerate(lengths):
            stored = x[b, prompt - length:].double()
            off = (vv[b, :final[b]] - stored).abs().amax() / (stored.max() - stored.min())
            assert float(off) <= 0.5 / (2 ** bits - 1) * (1 + 2.0 ** -6)
    assert NORM_TOL[dtype] > 0
