"""The quantised cache on a B200: what is stored and read back, attention over it, and what is refused."""
import math

import pytest
import torch

import torchpairwise_b200 as tpw
from attention_cases import assert_near
from cache_cases import SHAPES, attended, filled, quantised, unpacked, values

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def ints(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


def check_stored(cache, k, v, group, where):
    """Codes, steps and zeros at where[b] = (first token, first position, count) against the definition."""
    for x, (code, step, zero) in zip((k, v), unpacked(cache)):
        want = [t.transpose(1, 2) for t in quantised(x, cache.bits, group)]   # [batch, heads, tokens, d]
        for b, (i, at, n) in enumerate(where):
            c, s, z = (t[b, :, i:i + n] for t in want)
            gc, gs, gz = (t[b, :, at:at + n] for t in (code, step, zero))
            assert torch.equal(gs.nan_to_num(-1.0), s.nan_to_num(-1.0)) and torch.equal(gz.nan_to_num(-1e30), z.nan_to_num(-1e30))
            # 16-bit values: x - zero is rounded to 32 bits, 2^-24 of at most 255 steps: such a distance from a middle decides nothing
            x64 = x[b, i:i + n].transpose(0, 1).double()
            away = ((x64 - z) / s - torch.floor((x64 - z) / s) - 0.5).abs()
            sure = (away > 255 * 2.0 ** -24) | ~torch.isfinite(s) | ((x64 - z).float().double() == x64 - z) | torch.tensor(x.dtype == torch.float32, device=x.device)
            assert torch.equal(gc[sure], c[sure]) and bool(((gc - c).abs() <= 1).all())
            fine = torch.isfinite(s)
            assert bool(((gz + gs * gc - x64).abs() <= gs / 2 * (1 + 2.0 ** -15))[fine].all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("group", [32, None])
@pytest.mark.parametrize("d", [1, 20, 33, 64, 80, 96, 120, 128])
def test_tokens_are_stored_by_the_definition_and_read_back(dtype, bits, group, d):
    g = torch.Generator().manual_seed(d)
    batch, heads, n, cap = 3, 2, 37, 130
    cache = tpw.quantized_cache(batch, cap, heads, d, bits=bits, group=group)
    k = (torch.randn(batch, n, heads, d, generator=g) * 3 + 1).to(dtype).cuda()
    v = (torch.randn(batch, n, heads, d, generator=g) * torch.exp2(torch.randint(-20, 10, (batch, n, heads, 1), generator=g))).to(dtype).cuda()
    lengths = ints(100, 37, 12)   # in the middle, at the start, longer than its sequence
    before = [t.clone() for t in cache[:4]]
    assert tpw.cache_write(cache, k, v, lengths) is None
    check_stored(cache, k, v, group, [(0, 63, 37), (0, 0, 37), (25, 0, 12)])
    for b, (lo, hi) in enumerate(((63, 100), (0, 37), (0, 12))):   # all else is as it was
        for now, then in zip(cache[:4], before):
            keep = torch.ones(cache.capacity, dtype=torch.bool, device="cuda")
            keep[lo:hi] = False
            assert torch.equal(now[b][:, keep], then[b][:, keep])
    whole = values(cache)
    for out_type in TYPES:
        for got, want in zip(tpw.cache_read(cache, lengths, dtype=out_type), whole):
            want = want.float().to(out_type)
            for b, length in enumerate((100, 37, 12)):
                want[b, length:] = 0
            assert got.dtype == out_type and torch.equal(got, want)
        for got, want in zip(tpw.cache_read(cache, lengths, tokens=n, dtype=out_type), whole):
            want = want.float().to(out_type)
            assert torch.equal(got[0], want[0, 63:100]) and torch.equal(got[1], want[1, :37])
            assert torch.equal(got[2, 25:], want[2, :12]) and not got[2, :25].any()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_values_on_a_grid_middles_and_constants(bits, dtype):
    """Whole numbers from the lowest to the highest code are kept exactly, middles between codes go to the even one, a constant row is its zero."""
    most = 2 ** bits - 1
    cache = tpw.quantized_cache(1, 64, 1, 64, bits=bits, group=None)
    grid = torch.arange(64) % (most + 1)
    grid[-1] = most
    middles = torch.cat((torch.tensor([0.0, most]), torch.arange(62) % (most if bits == 4 else 62) + 0.5))
    rows = torch.stack([grid.float() - 3, grid.float() * 0.25, middles, torch.full((64,), 0.75), torch.full((64,), -1.0), torch.zeros(64)])
    x = rows.to(dtype)[None, :, None].cuda()
    assert torch.equal(x[0, :, 0].float().cpu(), rows)
    tpw.cache_write(cache, x, x, ints(6))
    check_stored(cache, x, x, None, [(0, 0, 6)])
    for out in tpw.cache_read(cache, ints(6), tokens=6, dtype=torch.float32):
        out = out[0, :, 0].cpu()
        assert torch.equal(out[[0, 1, 3, 4, 5]], rows[[0, 1, 3, 4, 5]])
        assert torch.equal(out[2], torch.cat((rows[2, :2], torch.round(rows[2, 2:]))))


@pytest.mark.parametrize("bits", [4, 8])
def test_float32_values_beside_a_middle(bits):
    """Values a unit of the last place to either side of middles between two codes, some of whose distances from the zero are no 32-bit numbers."""
    most = 2 ** bits - 1
    for zero, step in ((-3.75, 0.5), (-1.0, 2.0 ** -7 * 1.5), (-96.0, 0.75)):
        middles = torch.tensor([zero + (c + 0.5) * step for c in range(min(most, 40))], dtype=torch.float64).float()
        near = torch.stack((torch.nextafter(middles, torch.tensor(-math.inf)), middles, torch.nextafter(middles, torch.tensor(math.inf))), -1).flatten()[:60]
        small = torch.tensor([1e-9, -1e-9])   # beside a middle at 0
        x = torch.cat((torch.tensor([zero, zero + most * step]), small, near)).float()
        x = torch.cat((x, x[:1].expand(64 - x.numel())))[None, None, None].cuda()
        cache = tpw.quantized_cache(1, 64, 1, 64, bits=bits, group=None)
        tpw.cache_write(cache, x, x, ints(1))
        # (where 0 lies above the last code, as with 15 steps from -1, the step is another one, which the definition gives too)
        want = [w[0, 0, 0] for w in quantised(x, bits, None)]
        for got in unpacked(cache):
            assert all(torch.equal(a[0, 0, 0], b) for a, b in zip(got, want))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan, 2.0 ** 100, -(2.0 ** 127)])
def test_a_group_that_does_not_fit_reads_as_nan_and_alone(bits, bad):
    g = torch.Generator().manual_seed(1)
    cache = tpw.quantized_cache(1, 64, 2, 96, bits=bits)
    x = torch.randn(1, 5, 2, 96, generator=g).cuda()
    x[0, 2, 1, 40] = bad
    x[0, 3, 0, 0] = 2.0 ** 99.5   # fits
    x[0, 4] *= 2.0 ** -120        # steps end at 2^-100
    tpw.cache_write(cache, x, x, ints(5))
    check_stored(cache, x, x, 32, [(0, 0, 5)])
    for out in tpw.cache_read(cache, ints(5), tokens=5, dtype=torch.float32):
        nan = torch.zeros_like(out, dtype=torch.bool)
        nan[0, 2, 1, 32:64] = True
        assert torch.equal(out.isnan(), nan)


def test_strides_views_and_lengths_of_either_type():
    g = torch.Generator().manual_seed(2)
    packed = torch.randn(2, 9, 6, 72, generator=g).cuda().bfloat16()
    k, v = packed[:, :, 1:3, :64], packed[:, :, 4:6, 5:69]   # the second off the 16-byte grid
    got, want = (tpw.quantized_cache(2, 64, 2, 64) for _ in range(2))
    tpw.cache_write(got, k, v, ints(9, 20))
    tpw.cache_write(want, k.contiguous(), v.contiguous(), ints(9, 20).long())
    assert all(torch.equal(a, b) for a, b in zip(got[:4], want[:4]))
    tpw.cache_write(got, k.transpose(1, 2).contiguous().transpose(1, 2), v.mT.contiguous().mT, ints(9, 20))
    assert all(torch.equal(a, b) for a, b in zip(got[:4], want[:4]))
    one = packed[:, :1, :2, :64].expand(2, 9, 2, 64)   # every token the same row
    tpw.cache_write(got, one, one, ints(9, 20))
    tpw.cache_write(want, one.contiguous(), one.contiguous(), ints(9, 20))
    assert all(torch.equal(a, b) for a, b in zip(got[:4], want[:4]))
    a, b = tpw.cache_read(got, ints(9, 20)), tpw.cache_read(got, torch.tensor([9, 20], device="cuda"))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_tokens_beyond_the_capacity_are_not_stored():
    cache = tpw.quantized_cache(2, 64, 1, 32)
    x = torch.ones(2, 10, 1, 32, device="cuda")
    for n in (ints(70, -3), torch.tensor([70, -(2 ** 40)], device="cuda")):
        tpw.cache_write(cache, x, x, n)
        got = tpw.cache_read(cache, n, dtype=torch.float32)[0]
        assert bool((got[0, 60:] == 1).all()) and not got[0, :60].any() and not got[1].any()
        tail = tpw.cache_read(cache, n, tokens=10, dtype=torch.float32)[1]
        assert bool((tail[0, :4] == 1).all()) and not tail[0, 4:].any() and not tail[1].any()
    tpw.cache_write(cache, x, x, torch.tensor([2 ** 40, 2 ** 33 + 10], device="cuda"))   # nowhere near
    assert not cache.k_codes[1].any() and not cache.k_scales[1].any()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_over_a_cache(shape, dtype):
    b, nq, cap, hq, hk, d, bits, group, causal, window, lengths = shape
    cache = filled(b, cap, hk, d, bits, group, seed=nq)
    g = torch.Generator().manual_seed(3)
    q = torch.randn(b, nq, hq, d, generator=g).to(dtype).cuda()
    n = ints(*lengths)
    out, lse = tpw.cache_attention(q, cache, n, causal=causal, window=window, return_lse=True)
    want = attended(q, cache, lengths, causal=causal, window=window)
    assert out.dtype == dtype and lse.dtype == torch.float32
    assert_near(out, want[0], dtype, "out")
    # where many rows share a key, 16-bit ones, keys may be rounded to the queries' type: scores are then as good as the type
    assert_near(lse, want[1], torch.float32 if nq * hq // hk <= 32 else dtype, "lse")
    assert torch.equal(tpw.cache_attention(q, cache, n, causal=causal, window=window), out)
    assert tpw.device_status() == 0
