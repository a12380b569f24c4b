"""A plain float64 evaluation of attention, its gradients and rotary positions, and the sizes at which they can go wrong."""
import math

import torch

# unit roundoff of each type; float32 sums of up to a few thousand terms add about sqrt(n) of them
UNIT = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# Largest error over the norm of the result.  16-bit types: every probability (or gradient of a score) and the result are rounded
# once each, so the worst case of one term is 2 units, and the norm of many independently rounded terms is well below.  float32 and
# float64: sums over at most 2^12 terms of products rounded in the same type, 2^6 units from their random walk, times 2.
NORM_TOL = {torch.float64: 2.0 ** -46, torch.float32: 2.0 ** -17, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}


def seen_mask(nq, nk, length, causal, window, device):
    at = torch.arange(nq, device=device)[:, None] + length - nq
    j = torch.arange(nk, device=device)[None]
    m = (j < length).expand(nq, nk).clone()
    if causal:
        m &= j <= at
    if window:
        m &= j > at - window
    return m


def reference(q, k, v, *, causal=False, window=None, lengths=None, scale=None, grad=None, grad_lse=None):
    """out, lse (and dq, dk, dv) in float64 by the formulas, head by head."""
    q, k, v = q.detach().double(), k.detach().double(), v.detach().double()
    B, nq, hq, d = q.shape
    nk, hk = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    out, lse = torch.zeros_like(q), torch.full((B, hq, nq), -math.inf, dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        n = nk if lengths is None else min(max(int(lengths[b]), 0), nk)
        if n == 0 or nq == 0:
            continue
        m = seen_mask(nq, n, n, causal, window, q.device)
        some = m.any(-1)
        for h in range(hq):
            kb, vb, qb = k[b, :n, h * hk // hq], v[b, :n, h * hk // hq], q[b, :, h]
            s = (scale * qb @ kb.T).masked_fill(~m, -math.inf)
            lse[b, h] = torch.logsumexp(s, -1)
            p = torch.exp(s - torch.where(some, lse[b, h], torch.zeros_like(lse[b, h]))[:, None])
            out[b, :, h] = p @ vb
            if grad is not None or grad_lse is not None:
                g = torch.zeros_like(qb) if grad is None else grad[b, :, h].double()
                delta = (g * out[b, :, h]).sum(-1)
                if grad_lse is not None:
                    delta = delta - grad_lse[b, h].double()
                ds = p * (g @ vb.T - delta[:, None])
                dq[b, :, h] = scale * ds @ kb
                dk[b, :n, h * hk // hq] += scale * ds.T @ qb
                dv[b, :n, h * hk // hq] += p.T @ g
    return out, lse, dq, dk, dv


def assert_near(got, want, dtype, what, times=1.0):
    """Norm of the error within NORM_TOL of the norm of the result, no single value further off than 8 of them from what values of
    that size may be, and infinities and zeros of empty rows exact."""
    got = got.detach().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fin = torch.isfinite(want)
    assert torch.equal(fin, torch.isfinite(got)), f"{what}: non-finite values differ"
    assert torch.equal(got[~fin], want[~fin]), what
    if not bool(fin.any()):
        return
    g, w = got[fin], want[fin].detach()
    norm, err = float(w.norm()), float((g - w).norm())
    tol = NORM_TOL[dtype] * times
    assert err <= tol * norm + 1e-300, f"{what}: relative error {err / max(norm, 1e-300):.3g} > {tol:.3g}"
    rms = norm / math.sqrt(w.numel())
    worst = float(((g - w).abs() / (w.abs() + rms + 1e-300)).max())
    assert worst <= 8 * tol, f"{what}: a value is {worst:.3g} off, more than {8 * tol:.3g}"


# batch, queries, keys, query heads, key heads, features, causal, window, lengths
SHAPES = [
    (1, 1, 1, 1, 1, 64, False, None, None),            # one query, one key: the gradient of its score is zero
    (2, 1, 300, 8, 2, 128, True, None, [300, 17]),     # one new token
    (1, 1, 4097, 4, 1, 64, True, None, None),          # the same over a long odd cache
    (2, 3, 700, 6, 2, 128, True, 100, [700, 2]),       # a few new tokens, the second sequence shorter than they are
    (2, 130, 130, 2, 2, 64, True, None, None),         # two rows into a second tile
    (1, 127, 129, 3, 1, 128, False, None, None),
    (2, 256, 640, 4, 2, 128, True, None, [640, 256]),  # a chunk on a cache
    (3, 77, 200, 2, 2, 64, False, None, [200, 0, 129]),  # a sequence without keys
    (1, 300, 200, 2, 1, 128, True, None, None),        # the first hundred queries see nothing
    (1, 513, 513, 2, 1, 96, True, 64, None),           # a window that moves through tiles
    (1, 400, 400, 1, 1, 80, True, 1, None),            # every query sees itself alone
    (2, 385, 385, 4, 4, 32, False, None, None),
    (1, 64, 100, 2, 2, 33, False, None, [99]),         # features off the 16-byte grid
    (1, 70, 90, 2, 1, 200, True, None, None),          # wide heads
    (2, 5, 0, 2, 1, 64, False, None, None),            # no keys
    (1, 1025, 1025, 2, 2, 128, True, None, None),
]
