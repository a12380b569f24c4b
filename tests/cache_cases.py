"""The quantised cache by its definition in 64 bits: codes, steps and zeros of a group, where they lie in storage, what they stand for."""
import math

import torch

import torchpairwise_b200 as tpw
from attention_cases import reference


def bf16_down(x):
    """The largest bfloat16 numbers not above x (float64, of magnitude 0 or 2^-110 to 2^120)."""
    ulp = torch.exp2(torch.frexp(x)[1].double() - 8)
    return torch.floor(x / ulp) * ulp


def quantised(x, bits, group):
    """Codes, step and zero of every feature of x [..., d], all in float64; NaN step and zero where a group does not fit the cache."""
    codes, steps, zeros = [], [], []
    for part in x.double().split(group or x.shape[-1], -1):
        fine = (part.abs() < 2.0 ** 100).all(-1, keepdim=True)
        part = torch.where(fine, part, torch.zeros_like(part))
        lo, hi = part.aminmax(dim=-1, keepdim=True)
        zero = bf16_down(lo)
        step = (-bf16_down((zero - hi) / (2 ** bits - 1))).clamp(min=2.0 ** -100)
        code = torch.round((part - zero) / step)
        nan = torch.where(fine, 0.0, math.nan).double()
        codes.append(code)
        steps.append((step + nan).expand_as(part))
        zeros.append((zero + nan).expand_as(part))
    return torch.cat(codes, -1), torch.cat(steps, -1), torch.cat(zeros, -1)


def place(f, d, value):
    """Where the code of feature f lies in a row of a head of d features."""
    w = max(2, -(-d // 32))
    run = 4 if value else 8
    return (f % 32 // run * w + f // 32) * run + f % run


def unpacked(cache):
    """Codes, step and zero [batch, heads, capacity, features] of keys and of values, float64, from storage feature by feature."""
    out = []
    for codes, scales, value in ((cache.k_codes, cache.k_scales, False), (cache.v_codes, cache.v_scales, True)):
        cols, steps, zeros = [], [], []
        for f in range(cache.features):
            at = place(f, cache.features, value)
            byte = codes[..., at if cache.bits == 8 else at // 2].long()
            cols.append(byte if cache.bits == 8 else byte >> 4 * (at % 2) & 15)
            g = f // 32 if scales.shape[3] > 1 else 0
            steps.append(scales[..., g, 0].double())
            zeros.append(scales[..., g, 1].double())
        out.append((torch.stack(cols, -1).double(), torch.stack(steps, -1), torch.stack(zeros, -1)))
    return out


def values(cache):
    """What a cache stands for, [batch, capacity, heads, features] in float64, keys and values."""
    return [(zero + step * code).transpose(1, 2) for code, step, zero in unpacked(cache)]


def filled(batch, capacity, heads, d, bits, group, seed=0, scale=1.0, offset=0.0):
    """A cache full of tokens, written by the operator."""
    g = torch.Generator().manual_seed(seed)
    cache = tpw.quantized_cache(batch, capacity, heads, d, bits=bits, group=group)
    k, v = ((torch.randn(batch, cache.capacity, heads, d, generator=g) * scale + offset).cuda() for _ in range(2))
    tpw.cache_write(cache, k, v, torch.full((batch,), cache.capacity, dtype=torch.int32, device="cuda"))
    return cache


def attended(q, cache, lengths, **options):
    """out and lse in float64."""
    k, v = values(cache)
    return reference(q, k, v, lengths=lengths, **options)[:2]


# batch, queries, capacity, query heads, key heads, features, bits, group, causal, window, lengths
SHAPES = [
    (1, 1, 1, 1, 1, 64, 4, 32, True, None, [1]),                 # one query, one key
    (2, 1, 300, 8, 2, 128, 4, 32, True, None, [300, 17]),        # one new token
    (2, 1, 300, 8, 2, 128, 4, None, True, None, [300, 17]),
    (2, 1, 300, 8, 2, 128, 8, 32, True, None, [300, 17]),
    (1, 1, 4097, 4, 1, 64, 8, None, True, None, [4097]),         # the same over a long odd cache
    (3, 1, 2000, 3, 3, 80, 4, 32, True, None, [2000, 0, 1]),     # every head its own keys; a sequence without any
    (2, 3, 700, 6, 2, 128, 4, 32, True, 100, [700, 2]),          # a few new tokens, the second sequence shorter than they are
    (2, 5, 1500, 8, 1, 96, 4, 32, True, None, [1500, 64]),       # 40 rows to a key head
    (1, 8, 900, 16, 2, 40, 8, 32, False, None, [899]),
    (2, 130, 130, 2, 2, 64, 4, 32, True, None, [130, 129]),      # two rows into a second tile
    (1, 127, 129, 3, 1, 128, 8, None, False, None, [129]),
    (2, 256, 640, 4, 2, 128, 4, 32, True, None, [640, 256]),     # a chunk on a cache
    (3, 77, 200, 2, 2, 64, 4, None, False, None, [200, 0, 129]),
    (1, 300, 200, 2, 1, 128, 4, 32, True, None, [200]),          # the first hundred queries see nothing
    (1, 513, 513, 2, 1, 96, 4, 32, True, 64, [513]),             # a window that moves through tiles
    (1, 200, 400, 1, 1, 80, 8, 32, True, 1, [400]),              # every query sees itself alone
    (1, 70, 90, 2, 1, 20, 4, 32, True, None, [90]),              # features off every grid
    (1, 33, 1025, 4, 4, 33, 8, 32, True, None, [1025]),
    (2, 4, 0, 2, 1, 64, 4, 32, False, None, [0, 5]),             # a cache without room
]
