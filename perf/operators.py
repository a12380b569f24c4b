"""The work that the attention operators are measured on: rotary positions, softmax attention and its gradients.

``listed()`` holds the cases, ``draw(rng)`` gives another of the same ranges, ``prepare`` makes what a program has in
hand before the call, ``run`` is one pass through an operator (``own``: the framework's, otherwise the plain form in
elementary torch operations, in 32 bits), ``work`` the bytes and operations that the pass cannot do without and
``exact`` the outputs in 64 bits.

Tensors lie as [batch, tokens, heads, features].  Query i of a sequence with L keys stands at position L - Nq + i; with
``causal`` it sees the keys up to its own position, with ``window`` only that many of them, and no query sees keys from
L on.  A row that sees nothing is zero, its log-sum -inf.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one new token of eight sequences that are being served: launch latency is the whole cost
        dict(name="rotary_step", kind="rotary", train=False, b=8, n=1, hq=32, hk=8, d=128, rot=128, inter=False, table=32768, type="bf16"),
        # a long training batch, queries and keys in the half layout, forward and backward
        dict(name="rotary_train", kind="rotary", train=True, b=4, n=4096, hq=32, hk=8, d=128, rot=128, inter=False, table=4096, type="bf16"),
        # part of an odd head in single precision, interleaved pairs, ragged length at positions far into a long context
        dict(name="rotary_partial_f32", kind="rotary", train=True, b=3, n=1777, hq=12, hk=12, d=80, rot=32, inter=True, table=131072, type="f32"),
        # serving: one new token of sixteen sequences against long caches of shared key heads
        dict(name="step_long", kind="attention", train=False, b=16, nq=1, nk=16384, hq=32, hk=8, d=128, causal=True, window=0, ragged=True, packed=False, type="bf16"),
        # serving, few and short sequences: latency
        dict(name="step_short", kind="attention", train=False, b=2, nq=1, nk=500, hq=16, hk=16, d=64, causal=True, window=0, ragged=True, packed=False, type="f16"),
        # a chunk of new tokens on top of a long cache
        dict(name="chunk", kind="attention", train=False, b=2, nq=256, nk=16384, hq=32, hk=8, d=128, causal=True, window=0, ragged=True, packed=False, type="bf16"),
        # reading in a long prompt
        dict(name="prompt", kind="attention", train=False, b=1, nq=8192, nk=8192, hq=32, hk=8, d=128, causal=True, window=0, ragged=False, packed=True, type="bf16"),
        # training on short ragged sentences of a small model, both directions visible, one sequence with no keys at all
        dict(name="train_small", kind="attention", train=True, b=8, nq=77, nk=77, hq=8, hk=8, d=64, causal=False, window=0, ragged=True, packed=True, type="bf16"),
        # cross-attention between ragged sets in half precision, forward and backward
        dict(name="train_cross", kind="attention", train=True, b=4, nq=1500, nk=2111, hq=16, hk=16, d=64, causal=False, window=0, ragged=True, packed=False, type="f16"),
        # causal training with a sliding window and shared key heads on an odd length
        dict(name="train_window", kind="attention", train=True, b=2, nq=5001, nk=5001, hq=16, hk=4, d=96, causal=True, window=1024, ragged=False, packed=True, type="bf16"),
        # the framework's own type: single precision, forward and backward
        dict(name="train_f32", kind="attention", train=True, b=4, nq=1024, nk=1024, hq=8, hk=8, d=64, causal=False, window=0, ragged=False, packed=False, type="f32"),
        # training a long causal context with shared key heads, straight from a packed projection
        dict(name="train_long", kind="attention", train=True, b=1, nq=8192, nk=8192, hq=32, hk=8, d=128, causal=True, window=0, ragged=False, packed=True, type="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, evenly spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    which = rng.choice(["rotary", "rotary", "step", "chunk", "prompt", "train", "train", "train", "f32"])
    hk = rng.choice([1, 2, 4, 8])
    hq = hk * rng.choice([1, 2, 4])
    if which == "rotary":
        d = rng.choice([64, 80, 96, 128])
        n = rng.choice([1, _log(rng, 2, 8192)])
        b = rng.randint(1, 32) if n == 1 else rng.randint(1, 4)
        return dict(kind="rotary", train=n > 1 and rng.random() < 0.6, b=b, n=n, hq=hq, hk=hk, d=d, rot=rng.choice([d, d, d // 2, 32]),
                    inter=rng.random() < 0.4, table=max(n, rng.choice([8192, 32768, 131072])), type=rng.choice(["bf16", "f16", "f32"]))
    c = dict(kind="attention", train=False, b=rng.randint(1, 4), nq=1, nk=1, hq=hq, hk=hk, d=rng.choice([64, 64, 80, 96, 128, 128]),
             causal=True, window=0, ragged=False, packed=False, type=rng.choice(["bf16", "bf16", "f16"]))
    if which == "step":
        c.update(b=rng.randint(1, 16), nk=_log(rng, 100, 16384), ragged=True)
    elif which == "chunk":
        c.update(nq=_log(rng, 2, 400), nk=_log(rng, 500, 16384), ragged=rng.random() < 0.5)
    elif which == "prompt":
        n = _log(rng, 60, 6000)
        c.update(b=rng.randint(1, 2), nq=n, nk=n, causal=rng.random() < 0.8, window=rng.choice([0, 0, 512]), packed=rng.random() < 0.5)
    elif which == "train":
        n = _log(rng, 30, 5000)
        c.update(train=True, b=1 if n > 2000 else c["b"], nq=n, nk=n, causal=rng.random() < 0.6, packed=rng.random() < 0.5)
        if not c["causal"]:
            c.update(nk=_log(rng, 30, 5000), packed=False, ragged=rng.random() < 0.5)
        elif rng.random() < 0.3:
            c.update(window=rng.choice([100, 256, 1000]))
    else:
        c.update(train=rng.random() < 0.7, nq=_log(rng, 30, 1500), nk=_log(rng, 30, 1500), hq=hk, causal=False, ragged=rng.random() < 0.5, type="f32")
    if not c["causal"]:
        c["window"] = 0
    return c


def _lengths(c):
    """Keys that each sequence of the batch has: ragged ones fall from nk to a tenth of it; without ``causal`` the last has none."""
    if not c["ragged"]:
        return [c["nk"]] * c["b"]
    n = [max(1, round(c["nk"] * (1 - 0.9 * i / max(1, c["b"] - 1)))) for i in range(c["b"])]
    if not c["causal"] and c["b"] > 1:
        n[-1] = 0
    return n


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[c["type"]]

    def normal(*shape, dtype=dt, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    s = dict(case=c)
    if c["kind"] == "rotary":
        half = c["rot"] // 2
        # angles of the table in 64 bits, as a program makes them once for its longest context
        freq = torch.pow(torch.tensor(10000.0, dtype=torch.float64), -torch.arange(half, dtype=torch.float64) / half).cuda()
        angle = torch.arange(c["table"], dtype=torch.float64, device="cuda")[:, None] * freq
        s.update(cos=angle.cos().float(), sin=angle.sin().float())
        first = torch.randint(0, c["table"] - c["n"] + 1, (c["b"], 1), generator=g, device="cuda")
        s.update(positions=first + torch.arange(c["n"], device="cuda"))
        s.update(q=normal(c["b"], c["n"], c["hq"], c["d"]), k=normal(c["b"], c["n"], c["hk"], c["d"]))
        if c["train"]:
            s.update(gq=normal(c["b"], c["n"], c["hq"], c["d"]), gk=normal(c["b"], c["n"], c["hk"], c["d"]))
    else:
        if c["packed"]:   # views of one projection
            qkv = normal(c["b"], c["nq"], c["hq"] + 2 * c["hk"], c["d"])
            s.update(q=qkv[:, :, :c["hq"]], k=qkv[:, :, c["hq"]:c["hq"] + c["hk"]], v=qkv[:, :, c["hq"] + c["hk"]:])
        else:
            s.update(q=normal(c["b"], c["nq"], c["hq"], c["d"]), k=normal(c["b"], c["nk"], c["hk"], c["d"]), v=normal(c["b"], c["nk"], c["hk"], c["d"]))
        s["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda") if c["ragged"] else None
        if c["train"]:
            s["go"] = normal(c["b"], c["nq"], c["hq"], c["d"], scale=0.1)
    if c["train"]:
        for name in ("q", "k", "v"):
            if name in s:
                s[name] = s[name].detach().requires_grad_(True)
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------
def _turn(x, cos, sin, inter, dtype):
    """x with its first 2 * cos.size(-1) features turned by the angles, in 32 bits, rounded once."""
    r = 2 * cos.size(-1)
    x = x.float()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if inter else (x[..., :r // 2], x[..., r // 2:r])
    u, v = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, v), -1).flatten(-2) if inter else torch.cat((u, v), -1)
    return torch.cat((turned, x[..., r:]), -1).to(dtype)


def _plain_rotary(s):
    c = s["case"]
    cos, sin = s["cos"][s["positions"]][:, :, None], s["sin"][s["positions"]][:, :, None]
    dt = s["q"].dtype
    out = [_turn(s[n].detach(), cos, sin, c["inter"], dt) for n in ("q", "k")]
    if c["train"]:
        out += [_turn(s[n], cos, -sin, c["inter"], dt) for n in ("gq", "gk")]
    return out


def _hidden(c, lengths, device):
    """Truth values [B, 1, 1, Nq, Nk], or None: which keys a query does not see."""
    if not c["causal"] and lengths is None:
        return None
    j = torch.arange(c["nk"], device=device)
    n = torch.full((c["b"], 1, 1), c["nk"], device=device) if lengths is None else lengths.view(-1, 1, 1)
    hide = j >= n
    if c["causal"]:
        at = torch.arange(c["nq"], device=device).view(1, -1, 1) + n - c["nq"]
        hide = hide | (j > at)
        if c["window"]:
            hide = hide | (j <= at - c["window"])
    return hide[:, None, None].expand(-1, 1, 1, c["nq"], -1)


def _plain_attention(s):
    c = s["case"]
    b, nq, nk, hk, d = c["b"], c["nq"], c["nk"], c["hk"], c["d"]
    dt, scale, group = s["q"].dtype, 1 / math.sqrt(d), c["hq"] // hk

    def rows(x):   # [B, N, Hq, D] -> [B, Hk, group * N, D] in 32 bits
        return x.detach().float().view(b, nq, hk, group, d).permute(0, 2, 3, 1, 4).reshape(b, hk, group * nq, d)

    def back(x):
        return x.view(b, hk, group, nq, d).permute(0, 3, 1, 2, 4).reshape(b, nq, c["hq"], d).to(dt)

    q = rows(s["q"].reshape(b, nq, c["hq"], d))
    k, v = (s[n].detach().float().transpose(1, 2) for n in ("k", "v"))
    p = (q @ k.transpose(-1, -2)).mul_(scale).view(b, hk, group, nq, nk)
    hide = _hidden(c, s["lengths"], q.device)
    if hide is not None:
        p.masked_fill_(hide, -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (total.log() + top).view(b, c["hq"], nq)
    p.div_(torch.where(total == 0, torch.ones_like(total), total))
    p = p.view(b, hk, group * nq, nk)
    out = back(p @ v)
    if not c["train"]:
        return [out, lse]
    go = rows(s["go"])
    gv = p.transpose(-1, -2) @ go
    gs = go @ v.transpose(-1, -2)
    gs.sub_((gs * p).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    return [out, back(gs @ k), (gs.transpose(-1, -2) @ q).transpose(1, 2).to(dt), gv.transpose(1, 2).to(dt)]


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if not own:
        return _plain_rotary(s) if c["kind"] == "rotary" else _plain_attention(s)
    import torchpairwise_b200 as tpw
    if c["kind"] == "rotary":
        out = tpw.rotary_embedding(s["q"], s["k"], s["cos"], s["sin"], s["positions"], interleaved=c["inter"])
        if not c["train"]:
            return list(out)
        return [*(o.detach() for o in out), *torch.autograd.grad(out, (s["q"], s["k"]), (s["gq"], s["gk"]))]
    args = dict(causal=c["causal"], window=c["window"] or None, key_lengths=s["lengths"])
    if not c["train"]:
        return list(tpw.attention(s["q"], s["k"], s["v"], return_lse=True, **args))
    out = tpw.attention(s["q"], s["k"], s["v"], **args)
    return [out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["go"])]


def _pairs(c):
    """Query-key pairs that are seen, per query head."""
    total = 0
    for n in _lengths(c):
        if not c["causal"]:
            total += c["nq"] * n
            continue
        # query i sees min(n - nq + i + 1, window) keys, none where that is below one
        last, first = n, n - c["nq"] + 1
        first = max(first, 1)
        if last >= first:
            w = c["window"] or last
            ramp = min(last, w)
            total += (first + ramp) * (ramp - first + 1) // 2 if ramp >= first else 0
            total += w * (last - max(first, w + 1) + 1) if last > w else 0
    return total


def work(case):
    c = case
    e = _BYTES[c["type"]]
    if c["kind"] == "rotary":
        n = c["b"] * c["n"] * (c["hq"] + c["hk"])
        rows = min(c["b"] * c["n"], c["table"])
        passes = 2 if c["train"] else 1
        return dict(bytes=passes * n * c["d"] * e * 2 + rows * c["rot"] * 4 + c["b"] * c["n"] * 8, flops=passes * n * c["rot"] * 3)
    pairs = _pairs(c) * c["hq"]
    q = c["b"] * c["nq"] * c["hq"] * c["d"] * e
    kv = 2 * sum(min(n, c["nk"]) for n in _lengths(c)) * c["hk"] * c["d"] * e
    if not c["train"]:
        return dict(bytes=2 * q + kv + c["b"] * c["nq"] * c["hq"] * 4, flops=4 * c["d"] * pairs)
    # reads q, k, v and the gradient of the result, writes the result and three gradients; two products forward, five backward
    return dict(bytes=4 * q + kv + 2 * c["b"] * c["nk"] * c["hk"] * c["d"] * e, flops=14 * c["d"] * pairs)


# ---- 64 bits ----------------------------------------------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "rotary":
        at = s["positions"].reshape(-1)
        z = torch.complex(s["cos"][at].double(), s["sin"][at].double()).view(c["b"], c["n"], 1, -1)

        def turned(x, z):
            x = x.detach().double()
            head, rest = x[..., :c["rot"]], x[..., c["rot"]:]
            pair = head.unflatten(-1, (-1, 2)) if c["inter"] else head.unflatten(-1, (2, -1)).transpose(-1, -2)
            y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
            return torch.cat(((y if c["inter"] else y.transpose(-1, -2)).flatten(-2), rest), -1)

        out = [turned(s["q"], z), turned(s["k"], z)]
        return out + [turned(s["gq"], z.conj()), turned(s["gk"], z.conj())] if c["train"] else out
    scale, group = c["d"] ** -0.5, c["hq"] // c["hk"]
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    out = torch.zeros(c["b"], c["nq"], c["hq"], c["d"], dtype=torch.float64, device="cuda")
    lse = torch.full((c["b"], c["hq"], c["nq"]), -math.inf, dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b, n in enumerate(_lengths(c)):
        if n == 0:
            continue
        at = torch.arange(n - c["nq"], n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")
        seen = torch.ones(c["nq"], n, dtype=torch.bool, device="cuda")
        if c["causal"]:
            seen = j <= at
            if c["window"]:
                seen &= j > at - c["window"]
        for h in range(c["hq"]):
            kb, vb = k[b, :n, h // group], v[b, :n, h // group]
            logits = torch.where(seen, scale * (q[b, :, h] @ kb.T), -math.inf)
            lse[b, h] = torch.logsumexp(logits, -1)
            p = torch.where(seen, torch.exp(logits - lse[b, h][:, None]), 0.0)
            out[b, :, h] = p @ vb
            if c["train"]:
                go = s["go"][b, :, h].double()
                ds = p * (go @ vb.T - (go * out[b, :, h]).sum(-1, keepdim=True))
                dq[b, :, h] = scale * (ds @ kb)
                dk[b, :n, h // group] += scale * (ds.T @ q[b, :, h])
                dv[b, :n, h // group] += p.T @ go
    return [out, dq, dk, dv] if c["train"] else [out, lse]
