"""Calls of the quantised cache that its documentation allows and that once went wrong: each against what it means."""
from fractions import Fraction

import pytest
import torch

import torchpairwise_b200 as tpw
from attention_cases import assert_near
from cache_cases import attended, filled, unpacked

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def below(x):
    """The bfloat16 number before a positive one."""
    return float((torch.tensor(x).bfloat16().view(torch.int16) - 1).view(torch.bfloat16))


def above(x):
    """The bfloat16 number after x."""
    bits = torch.tensor(x).bfloat16().view(torch.int16)
    return 2.0 ** -133 if x == 0 else float((bits + (1 if x > 0 else -1)).view(torch.bfloat16))


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


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("group", [32, None])
def test_16_bit_values_whose_distance_from_the_zero_has_many_digits(dtype, bits, group):
    """Groups from a zero far below (or far above) the size of a value that lies on a middle but for it: the code is the nearest one in real arithmetic."""
    most = 2 ** bits - 1
    rows = []
    for small in (2.0 ** -14, 2.0 ** -17, 2.0 ** -20, 2.0 ** -24, 2.0 ** -30, 2.0 ** -40, 2.0 ** -90):
        for sign in (1, -1):
            # from -small (or small) to most, steps of about 1: middles stand at (c + 1/2) steps
            for step in (1.0, 1.0078125, 0.5, 4.0, 1.5):
                row = [sign * small, step * most] + [(c + 0.5) * step for c in range(most if bits == 4 else 24)]
                rows.append((row + [step] * 32)[:32])
            # a zero that is large beside values near 0
            for zero in (-1.0, -3.0, -7.0, -0.5):
                step = 2.0 if bits == 4 else 0.125
                rows.append(([zero, zero + most * step] + [sign * small * 2.0 ** -k for k in range(30)])[:32])
    x = torch.tensor(rows, dtype=torch.float64).to(dtype)
    assert torch.isfinite(x).all()
    x = torch.cat((x, x.flip(0)), 1)[None, :, None].cuda()
    n = x.shape[1]
    cache = tpw.quantized_cache(1, n, 1, 64, bits=bits, group=group)
    tpw.cache_write(cache, x, x, ints(n))
    # 64 bits do not hold all of these differences either: rational numbers do
    for code, step, zero in unpacked(cache):
        for i in range(n):
            for first in range(0, 64, group or 64):
                part = [Fraction(v) for v in x[0, i, 0, first:first + (group or 64)].double().tolist()]
                s, z = Fraction(float(step[0, 0, i, first])), Fraction(float(zero[0, 0, i, first]))
                assert z <= min(part) and z + most * s >= max(part)
                assert z + most * Fraction(below(float(s))) < max(part) and Fraction(above(float(z))) > min(part)   # the smallest and the largest that do
                assert code[0, 0, i, first:first + len(part)].tolist() == [round((v - z) / s) for v in part]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("bits", [4, 8])
def test_codes_of_16_bit_values_of_any_magnitude(dtype, bits):
    g = torch.Generator().manual_seed(34)
    top, most = 14 if dtype == torch.float16 else 90, 2 ** bits - 1
    n = 4096
    x = torch.randn(1, n, 2, 64, generator=g) * torch.exp2(torch.randint(-24 if dtype == torch.float16 else -90, top, (1, n, 2, 64), generator=g))
    x = x.to(dtype).cuda()
    cache = tpw.quantized_cache(1, n, 2, 64, bits=bits)
    tpw.cache_write(cache, x, x, ints(n))
    for code, step, zero in unpacked(cache):
        real = x.transpose(1, 2).double()
        for i, h, f in torch.randint(0, 64, (6000, 3), generator=g).tolist():
            i, h, first = 64 * f + i, h % 2, f // 32 * 32
            part = [Fraction(v) for v in real[0, h, i, first:first + 32].tolist()]
            s, z = Fraction(float(step[0, h, i, first])), Fraction(float(zero[0, h, i, first]))
            assert z <= min(part) and z + most * s >= max(part)
            assert code[0, h, i, first:first + 32].tolist() == [round((v - z) / s) for v in part]


def test_tensors_that_are_negated_when_they_are_read():
    """torch._neg_view: a tensor whose sign waits in a flag, contiguous or not."""
    g = torch.Generator().manual_seed(35)
    k, v = (torch.randn(2, 9, 2, 64, generator=g).cuda() for _ in range(2))
    n = ints(9, 20)
    got, want = (tpw.quantized_cache(2, 64, 2, 64) for _ in range(2))
    tpw.cache_write(want, -k, -v, n)
    tpw.cache_write(got, torch._neg_view(k), torch._neg_view(v.transpose(1, 2).contiguous().transpose(1, 2)), n)
    assert all(torch.equal(a, b) for a, b in zip(got[:4], want[:4]))
    for queries in (1, 300):
        q = torch.randn(2, queries, 4, 64, generator=g).half().cuda()
        assert torch.equal(tpw.cache_attention(torch._neg_view(q), want, n), tpw.cache_attention(-q, want, n))
    assert torch.equal(tpw.cache_read(want, torch._neg_view(-n))[0], tpw.cache_read(want, n)[0])


def test_lengths_far_beyond_32_bits_with_very_many_tokens():
    """Nearly 2^30 tokens (one row, repeated by its strides) of a sequence of 2^40: the last ones stand far beyond the capacity, none is stored."""
    cache = tpw.quantized_cache(1, 64, 1, 8)
    x = torch.ones(1, 1, 1, 8, device="cuda").expand(1, 2 ** 30 - 1, 1, 8)
    for n in (torch.tensor([2 ** 40], device="cuda"), torch.tensor([2 ** 62], device="cuda"), ints(2 ** 31 - 1)):
        tpw.cache_write(cache, x, x, n)
        assert not any(bool(t.any()) for t in cache[:4])
    tpw.cache_write(cache, x, x, torch.tensor([2 ** 30 - 1], device="cuda"))   # from position 0 on: the first 64 have a place
    assert bool((tpw.cache_read(cache, ints(64), dtype=torch.float32)[0] == 1).all())


def test_a_cache_that_wants_gradients_is_refused():
    """Steps and zeros are 16-bit floating-point tensors: as parameters they would silently get none."""
    cache = filled(1, 64, 1, 64, 4, 32, seed=36)
    x, q, n = torch.zeros(1, 3, 1, 64, device="cuda"), torch.zeros(1, 1, 1, 64, device="cuda"), ints(3)
    before = [t.clone() for t in cache[:4]]
    for name in ("k_scales", "v_scales"):
        wants = cache._replace(**{name: getattr(cache, name).requires_grad_()})
        for call in (lambda: tpw.cache_read(wants, n), lambda: tpw.cache_attention(q, wants, n), lambda: tpw.cache_write(wants, x, x, n)):
            with pytest.raises(RuntimeError, match="gradient"):
                call()
        with torch.no_grad():
            tpw.cache_read(wants, n)
            tpw.cache_attention(q, wants, n)
        getattr(cache, name).requires_grad_(False)
    assert all(torch.equal(a, b) for a, b in zip(cache[:4], before))


def test_a_cache_of_inference_mode():
    """Made under torch.inference_mode: written, read and attended to there; outside it is read, and a write is refused before it happens."""
    x, q, n = torch.ones(1, 3, 1, 64, device="cuda"), torch.ones(1, 1, 1, 64, device="cuda"), ints(3)
    with torch.inference_mode():
        cache = tpw.quantized_cache(1, 64, 1, 64)
        tpw.cache_write(cache, x, x, n)
        inside = tpw.cache_attention(q, cache, n)
    assert torch.equal(tpw.cache_attention(q, cache, n), inside) and bool((tpw.cache_read(cache, n)[1][:, :3] == 1).all())
    with torch.no_grad(), pytest.raises(RuntimeError, match="inference"):
        tpw.cache_write(cache, 2 * x, 2 * x, n)
    assert bool((tpw.cache_read(cache, n)[1][:, :3] == 1).all())
    # an ordinary cache may be written there
    cache = tpw.quantized_cache(1, 64, 1, 64)
    with torch.inference_mode():
        tpw.cache_write(cache, x, x, n)
    assert torch.equal(tpw.cache_attention(q, cache, n), inside)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("queries,heads,d", [(10, 8, 128), (9, 18, 64), (41, 4, 96), (48, 8, 128), (12, 32, 64), (60, 12, 40), (100, 8, 20), (70, 8, 33)])
@pytest.mark.parametrize("bits,group", [(4, 32), (8, None)])
def test_log_sums_of_rows_that_go_straight_to_the_codes(dtype, queries, heads, d, bits, group):
    """20 to 400 rows to a key head: up to 192 of them, and all of odd widths, have scores in 32 bits, whatever the type of the queries."""
    cache = filled(2, 700, 2, d, bits, group, seed=37)
    q = torch.randn(2, queries, heads, d, generator=torch.Generator().manual_seed(38)).to(dtype).cuda()
    out, lse = tpw.cache_attention(q, cache, ints(700, 333), causal=True, return_lse=True)
    want = attended(q, cache, [700, 333], causal=True)
    assert_near(out, want[0], dtype, "out")
    assert_near(lse, want[1], torch.float32, "lse")


@pytest.mark.parametrize("queries,heads", [(193, 2), (100, 4), (600, 2)])
@pytest.mark.parametrize("bits,group", [(4, 32), (8, None)])
def test_log_sums_of_many_bfloat16_rows(queries, heads, bits, group):
    """More rows go through half precision: codes' values and queries are rounded to it, and log-sums are as good as its rounding."""
    cache = filled(2, 700, 1, 64, bits, group, seed=39)
    q = torch.randn(2, queries, heads, 64, generator=torch.Generator().manual_seed(40)).bfloat16().cuda()
    out, lse = tpw.cache_attention(q, cache, ints(700, 333), causal=True, return_lse=True)
    want = attended(q, cache, [700, 333], causal=True)
    assert_near(out, want[0], torch.bfloat16, "out")
    assert_near(lse, want[1], torch.float16, "lse")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("options", [dict(causal=True), dict(), dict(causal=True, window=70)], ids=str)
def test_many_rows_with_lengths_beyond_the_capacity_and_below_zero(dtype, options):
    cache = filled(3, 512, 1, 64, 4, 32, seed=41)
    q = torch.randn(3, 300, 2, 64, generator=torch.Generator().manual_seed(42)).to(dtype).cuda()
    want = tpw.cache_attention(q, cache, ints(512, 0, 77), return_lse=True, **options)
    assert_near(want[0], attended(q, cache, [512, 0, 77], **options)[0], dtype, "out")
    for n in (ints(1000, -5, 77), ints(2 ** 31 - 1, -2 ** 31, 77), torch.tensor([2 ** 40, -(2 ** 40), 77], device="cuda")):
        got = tpw.cache_attention(q, cache, n, return_lse=True, **options)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
def test_more_key_heads_than_a_grid_has_rows(dtype):
    some = filled(1, 64, 7, 8, 4, 32, seed=43)
    heads = 70000
    pick = torch.arange(heads, device="cuda") % 7
    cache = tpw.QuantizedCache(*(t[:, pick].contiguous() for t in some[:4]), 8, 4)
    q = torch.randn(1, 193, 7, 8, generator=torch.Generator().manual_seed(44)).to(dtype).cuda()
    out = tpw.cache_attention(q[:, :, pick].contiguous(), cache, ints(60), causal=True)
    want = tpw.cache_attention(q, some, ints(60), causal=True)
    assert torch.equal(out, want[:, :, pick])
