"""Attention where kernels go wrong that are right at ordinary sizes: long sums, batches of unequal sequences, values out of range."""
import pytest
import torch

import torchpairwise_b200 as tpw
from attention_cases import assert_near, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("keys,queries,heads", [(8192, 1024, 10), (3001, 700, 16)])
def test_float32_weights_of_early_keys_do_not_drift(causal, keys, queries, heads):
    """A row's maximum in its first tile, as heavy as all later tiles together: whatever a tile does to the sums before it adds up."""
    g = torch.Generator().manual_seed(21)
    along = torch.full((64,), 0.125)
    q = along * 4 + 0.1 * torch.randn(1, queries, heads, 64, generator=g)
    k = along * 30 + 0.5 * torch.randn(1, keys, 1, 64, generator=g)   # scores of about 15, the first key's 24
    k[:, 0] = along * 48
    v = torch.randn(1, keys, 1, 64, generator=g)
    go = torch.randn(1, queries, heads, 64, generator=g).cuda()
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    out, lse = tpw.attention(*leaves, causal=causal, return_lse=True)
    want = reference(*leaves, causal=causal, grad=go)
    assert_near(out, want[0], torch.float32, "out")
    assert_near(lse, want[1], torch.float32, "lse")
    for got, w, name in zip(torch.autograd.grad(out, leaves, go), want[2:], ("dq", "dk", "dv")):
        assert_near(got, w, torch.float32, name, 2.0)
    assert tpw.device_status() == 0


@pytest.mark.parametrize("bad", [None, float("inf"), float("nan")])
@pytest.mark.parametrize("heads", [(2, 2), (4, 2)])
def test_half_precision_gradients_of_a_sequence_are_its_own(bad, heads):
    """Sequences and heads whose gradients and values are 2^23 times another's, or not finite, change no bit of that other's gradients and cost it no
    digits."""
    g = torch.Generator().manual_seed(22)
    hq, hk = heads
    q, k, v, go = (torch.randn(2, 160, h, 64, generator=g) for h in (hq, hk, hk, hq))
    small = -9 if bad is None else 5   # with 2^5 a gradient of a score is above half precision's 65504 unless it is scaled down
    go[0] *= 2.0 ** 8
    v[0] *= 2.0 ** 6
    go[1] *= 2.0 ** small
    go[1, :, :hq // 2] *= 2.0 ** 8     # heads of the same sequence are apart too
    if bad is not None:
        go[0] = bad
    args = [t.half().cuda() for t in (q, k, v)]
    go = go.half().cuda()
    leaves = [t.requires_grad_() for t in args]
    both = torch.autograd.grad(tpw.attention(*leaves), leaves, go)
    alone = [t.detach()[1:].clone().requires_grad_() for t in args]
    single = torch.autograd.grad(tpw.attention(*alone), alone, go[1:])
    want = reference(*alone, grad=go[1:])
    for got, other, w, name in zip(both, single, want[2:], ("dq", "dk", "dv")):
        assert torch.equal(got[1:], other), name
        half = w.shape[2] // 2
        for part in (slice(0, half), slice(half, None)):
            assert_near(got[1:, :, part], w[:, :, part], torch.float16, name, 2.0)


def test_half_precision_query_heads_do_not_depend_on_one_another():
    """An infinite gradient in one query head leaves the gradient of the queries of another alone, though they share keys."""
    g = torch.Generator().manual_seed(23)
    q, k, v, go = (torch.randn(1, 200, h, 64, generator=g).half().cuda() for h in (2, 1, 1, 2))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    go = go * 2.0 ** 6
    bad = go.clone()
    bad[:, 3, 1] = float("inf")
    out = tpw.attention(*leaves)
    a, b = (torch.autograd.grad(out, q, x, retain_graph=True)[0] for x in (go, bad))
    assert torch.equal(a[:, :, 0], b[:, :, 0]) and bool(torch.isfinite(a).all())


@pytest.mark.parametrize("dtype", [torch.float64, torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("d", [33, 64, 128, 200])
@pytest.mark.parametrize("queries", [8, 300])
def test_rows_that_see_nothing_are_zero_whatever_others_see(dtype, d, queries):
    """Half of the rows are before the first key, keys before the first window are seen by no row, and what stands beside either is not finite."""
    g = torch.Generator().manual_seed(24)
    q, k, v, go = (torch.randn(1, n, 2, d, generator=g).to(dtype).cuda() for n in (queries, 200, 200, queries))
    seeing = queries // 2
    n = torch.tensor([seeing], dtype=torch.int32, device="cuda")
    empty = queries - seeing
    for bad in (float("inf"), float("nan")):
        for where in ("k", "v"):
            kk, vv = k.clone(), v.clone()
            (kk if where == "k" else vv)[:, 0] = bad
            leaves = [t.detach().requires_grad_() for t in (q, kk, vv)]
            out, lse = tpw.attention(*leaves, causal=True, key_lengths=n, return_lse=True)
            dq, = torch.autograd.grad(out, leaves[0], go)
            assert not out[:, :empty].any() and not dq[:, :empty].any() and bool((lse[:, :, :empty] == -float("inf")).all()), (bad, where)
            assert bool(torch.isnan(out[:, empty:]).any() or torch.isinf(out[:, empty:]).any())
        few = min(queries, 50)
        unseen = 200 - few - 20 + 1   # keys that end before the first query's window of 20
        for where in ("q", "go"):
            qq, gg = q[:, :few].clone(), go[:, :few].clone()
            (qq if where == "q" else gg)[:, 0] = bad
            leaves = [t.detach().requires_grad_() for t in (qq, k, v)]
            out = tpw.attention(*leaves, causal=True, window=20)
            dk, dv = torch.autograd.grad(out, leaves[1:], gg)
            assert not dk[:, :unseen].any() and not dv[:, :unseen].any(), (bad, where)
    assert tpw.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_many_walks_of_random_lengths(dtype):
    """What depends on which warp is first shows in one call of thousands: results of the same bits each time, and a clean status word."""
    import random
    rng = random.Random(31)
    for _ in range(300):
        hk = rng.choice([1, 2, 3])
        hq, batch, d = hk * rng.choice([1, 2, 5]), rng.randint(1, 3), rng.choice([8, 40, 64, 72, 104, 128])
        nq, nk = (rng.choice([rng.randint(1, 200), rng.randint(100, 900)]) for _ in range(2))
        causal = rng.random() < 0.5
        window = rng.choice([None, rng.randint(1, 300)]) if causal else None
        n = torch.tensor([rng.randint(0, nk) for _ in range(batch)], dtype=torch.int32, device="cuda")
        leaves = [torch.randn(batch, x, h, d, device="cuda", dtype=dtype).requires_grad_() for x, h in ((nq, hq), (nk, hk), (nk, hk))]
        runs = []
        for _ in range(4):
            out = tpw.attention(*leaves, causal=causal, window=window, key_lengths=n)
            runs.append([out, *torch.autograd.grad(out, leaves, leaves[0].detach())])
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))
        assert all(bool(torch.isfinite(t).all()) for t in runs[0])
    assert tpw.device_status() == 0
