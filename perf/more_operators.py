"""The work that a cache of quantised keys and values is measured on: storing tokens, reading them back, attention over it.

``listed()`` holds the cases, ``draw(rng)`` gives another of the same ranges, ``prepare`` makes what a program has in
hand before the call, ``run`` is one pass through an operator (``own``: the framework's, otherwise the plain form in
elementary torch operations), ``work`` the bytes and operations that the pass cannot do without and ``exact`` the outputs
in 64 bits.

The cache.  Keys and values of a token and head are cut into groups (of 32 features, or the whole head).  A group has a zero,
the largest bfloat16 number that is not above its lowest value, and a step, the smallest bfloat16 number (2^-100 at least) of which
2^bits - 1 reach from the zero to its highest value.  A value is held as the nearest whole number of steps above the zero, ties to
even, and stands for zero + step * code.

Storage is [batch, heads, capacity, bytes of a row] for the codes and [batch, heads, capacity, groups, 2] for step and zero.  A row has
as many features as 32s cover, 64 at least; the codes of those beyond the head are 0.  Feature 32 w + 8 t + n of a key is code (t, w, n)
of its row, feature 32 w + 4 t + n of a value code (t, w, n) of its row, where n counts to 8 and to 4; of two 4-bit codes in a byte the
first is the lower.

Tokens and queries of a call are the last ones of their sequence: i of n stands at position L - n + i of a sequence that is L long with them.
Positions below 0 do not exist: such a token is not stored and reads as zero, and such a query sees nothing.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one new token of eight sequences that are being served joins the cache and is read back: launch latency is the whole cost
        dict(name="store_step", kind="store", b=8, n=1, cap=32768, hk=8, d=128, bits=4, group=32, short=False, type="bf16"),
        # a long prompt of two sequences joins an empty cache and is read back, so that later layers see what decoding will see
        dict(name="store_prompt", kind="store", b=2, n=8192, cap=8192, hk=8, d=128, bits=4, group=32, short=False, type="bf16"),
        # single precision, an odd head in 8 bits, a ragged batch padded at its front: one sequence is shorter than the chunk
        dict(name="store_padded_f32", kind="store", b=3, n=1777, cap=4000, hk=12, d=80, bits=8, group=0, short=True, type="f32"),
        # a whole cache of ragged sequences back in 16 bits, for a layer that works on plain keys and values
        dict(name="read_long", kind="read", b=4, cap=16384, hk=8, d=128, bits=4, group=32, type="bf16"),
        # a short cache in 8 bits, one step and zero a head
        dict(name="read_short", kind="read", b=2, cap=700, hk=16, d=64, bits=8, group=0, type="f16"),
        # serving: one new token of sixteen sequences against long caches of shared key heads
        dict(name="step_long", kind="attention", b=16, nq=1, cap=16384, hq=32, hk=8, d=128, bits=4, group=32, window=0, causal=True, lse=True, type="bf16"),
        # serving, few and short sequences: latency
        dict(name="step_short", kind="attention", b=2, nq=1, cap=500, hq=16, hk=16, d=64, bits=8, group=0, window=0, causal=True, lse=True, type="f16"),
        # serving, many sequences of middling length, one step and zero a head
        dict(name="step_many", kind="attention", b=64, nq=1, cap=4096, hq=32, hk=8, d=128, bits=4, group=0, window=0, causal=True, lse=False, type="bf16"),
        # single precision, an odd head, every head with keys of its own
        dict(name="step_f32", kind="attention", b=4, nq=1, cap=8000, hq=12, hk=12, d=80, bits=8, group=32, window=0, causal=True, lse=True, type="f32"),
        # a few proposed tokens are checked at once, through a sliding window
        dict(name="propose", kind="attention", b=8, nq=5, cap=12345, hq=32, hk=8, d=128, bits=4, group=32, window=4096, causal=True, lse=False, type="bf16"),
        # a chunk of new tokens on top of a long cache
        dict(name="chunk", kind="attention", b=2, nq=256, cap=16384, hq=32, hk=8, d=128, bits=4, group=32, window=0, causal=True, lse=False, type="bf16"),
        # reading in a prompt whose keys and values are in the cache already
        dict(name="prompt", kind="attention", b=1, nq=5000, cap=5000, hq=16, hk=4, d=64, bits=4, group=32, window=0, causal=True, lse=False, type="f16"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, evenly spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    which = rng.choice(["store", "store", "read", "step", "step", "step", "propose", "chunk", "prompt"])
    hk = rng.choice([1, 2, 4, 8])
    c = dict(kind="attention", hk=hk, d=rng.choice([40, 64, 64, 80, 96, 128, 128, 128]), bits=rng.choice([4, 4, 4, 8]), group=rng.choice([32, 32, 0]),
             type=rng.choice(["bf16", "bf16", "f16", "f32"]))
    if which == "store":
        n = rng.choice([1, _log(rng, 2, 8192)])
        c.update(kind="store", b=rng.randint(1, 32) if n == 1 else rng.randint(1, 2), n=n, cap=n + rng.choice([0, _log(rng, 1, 20000)]), short=n > 8 and rng.random() < 0.3)
        return c
    if which == "read":
        c.update(kind="read", b=rng.randint(1, 4), cap=_log(rng, 60, 12000))
        return c
    c.update(hq=hk * rng.choice([1, 2, 4, 8] if hk < 8 else [1, 2, 4]), nq=1, window=0, causal=True, lse=False)
    if which == "step":
        c.update(b=rng.randint(1, 16), cap=_log(rng, 60, 16384), lse=rng.random() < 0.5)
    elif which == "propose":
        c.update(b=rng.randint(1, 8), nq=rng.randint(2, 8), cap=_log(rng, 100, 16384), window=rng.choice([0, 0, 1000]))
    elif which == "chunk":
        c.update(b=rng.randint(1, 2), nq=_log(rng, 10, 300), cap=_log(rng, 500, 12000), causal=rng.random() < 0.8)
    else:
        n = _log(rng, 60, 4000)
        c.update(b=1, nq=n, cap=n, window=rng.choice([0, 0, 512]), type=rng.choice(["bf16", "f16"]))
    return c


# ---- the cache --------------------------------------------------------------------------------------------------
def _features(c):
    """Features of a row in storage."""
    return max(64, -(-c["d"] // 32) * 32)


def _groups(c):
    return -(-c["d"] // 32) if c["group"] else 1


def _rows(c):
    """Tokens that a head's storage has room for: a multiple of 64."""
    return -(-c["cap"] // 64) * 64


def _quantise(x, c):
    """Codes [..., d] in 64 bits, step and zero [..., groups] in 32, of x [..., d]."""
    size = c["group"] or c["d"]
    groups, d = _groups(c), c["d"]
    x = x.float()
    padded = torch.nn.functional.pad(x, (0, groups * size - d), value=math.nan).unflatten(-1, (groups, size))
    hole = padded.isnan()
    lo, hi = padded.masked_fill(hole, math.inf).amin(-1), padded.masked_fill(hole, -math.inf).amax(-1)
    # towards minus infinity in the upper 16 bits
    bits = lo.view(torch.int32)
    zero = ((bits + ((bits < 0) & (bits & 0xffff != 0)).int() * 0x10000) & -0x10000).view(torch.float32)
    step = ((hi.double() - zero.double()) / (2 ** c["bits"] - 1)).clamp(min=2.0 ** -100)
    # away from zero in the upper 16 bits, from 64 bits through 32
    near = step.float()
    bits = near.view(torch.int32)
    kept = (bits & -0x10000).view(torch.float32)
    step = torch.where(kept.double() < step, ((bits & -0x10000) + 0x10000).view(torch.float32), kept)
    each = lambda t: t.repeat_interleave(size, -1)[..., :d].double()  # noqa: E731
    return ((x.double() - each(zero)) / each(step)).round_(), step, zero


def _pack(codes, c, run):
    """Codes [..., d] as rows of bytes; `run` features lie together: 8 of a key, 4 of a value."""
    codes = torch.nn.functional.pad(codes.to(torch.uint8), (0, _features(c) - c["d"]))
    codes = codes.unflatten(-1, (-1, 32 // run, run)).transpose(-3, -2).flatten(-3)
    return codes if c["bits"] == 8 else codes[..., ::2] | codes[..., 1::2] << 4


def _values(codes, scales, c, run):
    """What rows of bytes and their [step, zero] stand for: [..., d] in 32 bits."""
    if c["bits"] == 4:
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    codes = codes.unflatten(-1, (32 // run, -1, run)).transpose(-3, -2).flatten(-3)[..., :c["d"]].float()
    size = c["group"] or c["d"]
    step, zero = (scales[..., k].float().repeat_interleave(size, -1)[..., :c["d"]] for k in (0, 1))
    return codes.mul_(step).add_(zero)   # the product is exact


def _lengths(c):
    """How long each sequence is, new tokens included: they fall from the capacity to a tenth of it."""
    least = 1 if c["kind"] == "read" else c["n"] if c["kind"] == "store" else min(c["nq"], c["cap"])
    n = [max(least, round(c["cap"] * (1 - 0.9 * i / max(1, c["b"] - 1)))) for i in range(c["b"])]
    if c.get("short"):
        n[-1] = c["n"] // 3
    return n


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[c["type"]]
    b, hk, d, rows = c["b"], c["hk"], c["d"], _rows(c)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    # a few features of every key head are much larger than the others
    loud = 1 + 4 * (torch.rand(hk, d, generator=g, device="cuda") < 0.06)
    width = _features(c) * c["bits"] // 8
    s = dict(case=c, lengths=torch.tensor(_lengths(c), dtype=torch.int32, device="cuda"))
    for name in ("k", "v"):
        s[name + "_codes"] = torch.zeros(b, hk, rows, width, dtype=torch.uint8, device="cuda")
        s[name + "_scales"] = torch.zeros(b, hk, rows, _groups(c), 2, dtype=torch.bfloat16, device="cuda")
    if c["kind"] == "store":
        s["k"], s["v"] = (normal(b, c["n"], hk, d) * loud).to(dt), normal(b, c["n"], hk, d).to(dt)
        return s
    for i in range(b):   # a sequence at a time, for the memory of it
        for name, run in (("k", 8), ("v", 4)):
            x = normal(rows, hk, d).transpose(0, 1)
            codes, step, zero = _quantise(x * loud[:, None] if name == "k" else x, c)
            s[name + "_codes"][i] = _pack(codes, c, run)
            s[name + "_scales"][i] = torch.stack((step, zero), -1).bfloat16()
    if c["kind"] == "attention":
        s["q"] = normal(b, c["nq"], c["hq"], d).to(dt)
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------
def _at(s, n):
    """Positions [batch, n] of the last n tokens, and which of them exist."""
    at = s["lengths"].long()[:, None] - n + torch.arange(n, device=s["lengths"].device)
    return at, at >= 0


def _plain_store(s):
    c = s["case"]
    at, there = _at(s, c["n"])
    batch = torch.arange(c["b"], device=at.device)[:, None]
    # a token that does not exist writes what the first that does writes, at its place
    first = (c["n"] - s["lengths"].long())[:, None]
    source = torch.maximum(torch.arange(c["n"], device=at.device), first)
    at = at.clamp(min=0)
    out = []
    for name, run in (("k", 8), ("v", 4)):
        codes, step, zero = _quantise(s[name], c)
        s[name + "_codes"][batch, :, at] = _pack(codes, c, run)[batch, source]
        s[name + "_scales"][batch, :, at] = torch.stack((step, zero), -1).bfloat16()[batch, source]
        back = _values(s[name + "_codes"][batch, :, at], s[name + "_scales"][batch, :, at], c, run)
        out.append(back.masked_fill_(~there[..., None, None], 0).to(_TYPES[c["type"]]))
    return out


def _plain_read(s):
    c = s["case"]
    beyond = torch.arange(_rows(c), device=s["lengths"].device) >= s["lengths"][:, None]
    return [_values(s[name + "_codes"], s[name + "_scales"], c, run).masked_fill_(beyond[:, None, :, None], 0).to(_TYPES[c["type"]]).transpose(1, 2).contiguous()
            for name, run in (("k", 8), ("v", 4))]


def _plain_attention(s):
    c = s["case"]
    b, nq, hk, d = c["b"], c["nq"], c["hk"], c["d"]
    group = c["hq"] // hk
    n = s["lengths"].view(-1, 1, 1)
    longest = _rows(c)
    k, v = (_values(s[name + "_codes"], s[name + "_scales"], c, run) for name, run in (("k", 8), ("v", 4)))
    q = s["q"].float().view(b, nq, hk, group, d).permute(0, 2, 3, 1, 4).reshape(b, hk, group * nq, d)
    p = (q @ k.transpose(-1, -2)).mul_(1 / math.sqrt(d)).view(b, hk, group, nq, longest)
    j = torch.arange(longest, device=q.device)
    hide = (j >= n).expand(b, nq, longest)
    if c["causal"]:
        at = torch.arange(nq, device=q.device).view(1, -1, 1) + n - nq
        hide = hide | (j > at)
        if c["window"]:
            hide = hide | (j <= at - c["window"])
    p.masked_fill_(hide[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (total.log() + top).view(b, c["hq"], nq)
    p.div_(torch.where(total == 0, torch.ones_like(total), total))
    out = p.view(b, hk, group * nq, longest) @ v
    out = out.view(b, hk, group, nq, d).permute(0, 3, 1, 2, 4).reshape(b, nq, c["hq"], d).to(_TYPES[c["type"]])
    return [out, lse] if c["lse"] else [out]


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if not own:
        return (_plain_store if c["kind"] == "store" else _plain_read if c["kind"] == "read" else _plain_attention)(s)
    import torchpairwise_b200 as tpw
    cache = tpw.QuantizedCache(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"], features=c["d"], bits=c["bits"])
    if c["kind"] == "store":
        tpw.cache_write(cache, s["k"], s["v"], s["lengths"])
        return list(tpw.cache_read(cache, s["lengths"], tokens=c["n"], dtype=_TYPES[c["type"]]))
    if c["kind"] == "read":
        return list(tpw.cache_read(cache, s["lengths"], dtype=_TYPES[c["type"]]))
    out = tpw.cache_attention(s["q"], cache, s["lengths"], causal=c["causal"], window=c["window"] or None, return_lse=c["lse"])
    return list(out) if c["lse"] else [out]


def _held(c):
    """Bytes that a token and head's key and value take in the cache, what the head's own features need."""
    return 2 * (-(-c["d"] * c["bits"] // 8) + 4 * _groups(c))


def work(case):
    c = case
    e, lengths = _BYTES[c["type"]], _lengths(c)
    if c["kind"] == "store":
        stored = sum(min(c["n"], n) for n in lengths) * c["hk"]
        return dict(bytes=stored * (2 * c["d"] * e + _held(c)) + 2 * c["b"] * c["n"] * c["hk"] * c["d"] * e, flops=2 * stored * c["d"] * 6)
    if c["kind"] == "read":
        return dict(bytes=sum(lengths) * c["hk"] * _held(c) + 2 * c["b"] * _rows(c) * c["hk"] * c["d"] * e, flops=2 * sum(lengths) * c["hk"] * c["d"] * 2)
    pairs = keys = 0
    for n in lengths:
        if not c["causal"]:
            pairs, keys = pairs + c["nq"] * n, keys + n
            continue
        w = c["window"] or n
        pairs += sum(min(i, w) for i in range(max(1, n - c["nq"] + 1), n + 1))
        keys += min(n, w + c["nq"] - 1)
    q = c["b"] * c["nq"] * c["hq"]
    return dict(bytes=2 * q * c["d"] * e + (4 * q if c["lse"] else 0) + keys * c["hk"] * _held(c), flops=4 * c["d"] * pairs * c["hq"])


# ---- 64 bits ----------------------------------------------------------------------------------------------------
def _exact_values(codes, scales, c, run):
    """A lookup for every feature by itself: its byte, its place in the byte, its group."""
    f = torch.arange(c["d"], device=codes.device)
    spot = (f % 32 // run) * (_features(c) // 32) * run + f // 32 * run + f % run
    if c["bits"] == 8:
        code = codes[..., spot].double()
    else:
        code = torch.floor(codes[..., spot // 2].double() / torch.where(spot % 2 == 0, 1.0, 16.0).double()) % 16
    group = f // 32 if c["group"] else torch.zeros_like(f)
    return scales[..., 1].double()[..., group] + scales[..., 0].double()[..., group] * code


def _exact_rounded(x, c):
    """What x [..., d] reads as once it is stored."""
    out = []
    for part in x.double().split(c["group"] or c["d"], -1):
        lo, hi = part.aminmax(dim=-1, keepdim=True)
        ulp = torch.exp2(torch.frexp(lo)[1].double() - 8)
        zero = torch.floor(lo / ulp) * ulp
        step = (hi - zero) / (2 ** c["bits"] - 1)
        ulp = torch.exp2(torch.frexp(step)[1].double() - 8)
        step = (torch.ceil(step / ulp) * ulp).clamp(min=2.0 ** -100)
        out.append(zero + step * torch.round((part - zero) / step))
    return torch.cat(out, -1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    lengths = _lengths(c)
    if c["kind"] == "store":
        out = [_exact_rounded(s[name], c) for name in ("k", "v")]
        for i, n in enumerate(lengths):
            for x in out:
                x[i, :max(0, c["n"] - n)] = 0
        return out
    if c["kind"] == "read":
        out = [torch.zeros(c["b"], _rows(c), c["hk"], c["d"], dtype=torch.float64, device="cuda") for _ in "kv"]
        for i, n in enumerate(lengths):
            for x, name, run in ((out[0], "k", 8), (out[1], "v", 4)):
                x[i, :n] = _exact_values(s[name + "_codes"][i, :, :n], s[name + "_scales"][i, :, :n], c, run).transpose(0, 1)
        return out
    nq, group = c["nq"], c["hq"] // c["hk"]
    out = torch.zeros(c["b"], nq, c["hq"], c["d"], dtype=torch.float64, device="cuda")
    lse = torch.full((c["b"], c["hq"], nq), -math.inf, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lengths):
        j = torch.arange(n, device="cuda")
        at = torch.arange(n - nq, n, device="cuda")[:, None]
        seen = torch.ones(nq, n, dtype=torch.bool, device="cuda")
        if c["causal"]:
            seen = j <= at
            if c["window"]:
                seen &= j > at - c["window"]
        for h in range(c["hk"]):
            k = _exact_values(s["k_codes"][i, h, :n], s["k_scales"][i, h, :n], c, 8)
            v = _exact_values(s["v_codes"][i, h, :n], s["v_scales"][i, h, :n], c, 4)
            for m in range(h * group, (h + 1) * group):
                logits = torch.where(seen, s["q"][i, :, m].double() @ k.T * c["d"] ** -0.5, -math.inf)
                lse[i, m] = torch.logsumexp(logits, -1)
                out[i, :, m] = torch.exp(logits - lse[i, m][:, None]) @ v
    return [out, lse] if c["lse"] else [out]
