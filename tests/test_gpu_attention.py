"""Attention and its gradients on a B200 against the formulas in float64 and against differences."""
import math

import pytest
import torch

import torchpairwise_b200 as tpw
from attention_cases import SHAPES, assert_near, reference

pytestmark = pytest.mark.gpu
TYPES = [torch.float64, torch.float32, torch.float16, torch.bfloat16]


def make(shape, dtype, seed=0, scale=1.0):
    B, nq, nk, hq, hk, d, causal, window, lengths = shape
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(B, n, h, d, generator=g).mul_(scale).to(dtype).cuda() for n, h in ((nq, hq), (nk, hk), (nk, hk)))
    go = torch.randn(B, nq, hq, d, generator=g).to(dtype).cuda()
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    return q, k, v, go, dict(causal=causal, window=window), n


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_gradients_follow_the_formulas(shape, dtype):
    q, k, v, go, mask, n = make(shape, dtype)
    q.requires_grad_(), k.requires_grad_(), v.requires_grad_()
    out, lse = tpw.attention(q, k, v, key_lengths=n, return_lse=True, **mask)
    assert out.dtype == dtype and lse.dtype == (torch.float64 if dtype == torch.float64 else torch.float32)
    want = reference(q, k, v, lengths=shape[-1], grad=go, **mask)
    assert_near(out, want[0], dtype, "out")
    assert_near(lse, want[1], torch.float64 if dtype == torch.float64 else torch.float32, "lse")
    grads = torch.autograd.grad(out, (q, k, v), go)
    if shape[1] > 1 or shape[2] > 1:
        for name, got, w in zip(("dq", "dk", "dv"), grads, want[2:]):
            assert got.dtype == dtype
            # ds is a difference of dO . v and delta, which carries the rounding of out: where the two cancel (rows that see one key, whose
            # gradient is zero) the bound is on what they are made of
            cancels = shape[7] == 1 or shape[8] is not None and min(shape[8]) < 3
            if name != "dv" and cancels:
                size = math.sqrt(w.numel()) * math.sqrt(shape[5])
                assert float((got.double() - w).norm()) <= 2 * size * torch.finfo(dtype).eps
            else:
                assert_near(got, w, dtype, name, 2.0)
    assert tpw.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_the_gradient_of_the_log_sum(dtype):
    shape = (2, 150, 260, 4, 2, 64, True, None, [260, 140])
    q, k, v, go, mask, n = make(shape, dtype, 3)
    q.requires_grad_(), k.requires_grad_(), v.requires_grad_()
    gl = torch.randn(2, 4, 150, generator=torch.Generator().manual_seed(4)).cuda().to(torch.float64 if dtype == torch.float64 else torch.float32)
    out, lse = tpw.attention(q, k, v, key_lengths=n, return_lse=True, **mask)
    gl = torch.where(torch.isfinite(lse.detach()), gl, torch.zeros_like(gl))
    both = reference(q, k, v, lengths=shape[-1], grad=go, grad_lse=gl, **mask)
    alone = reference(q, k, v, lengths=shape[-1], grad_lse=gl, **mask)
    for got, w in zip(torch.autograd.grad((out, lse), (q, k, v), (go, gl), retain_graph=True), both[2:]):
        assert_near(got, w, dtype, "out and lse", 2.0)
    g = torch.autograd.grad(lse, (q, k), gl)
    for got, w in zip(g, alone[2:4]):
        assert_near(got, w, dtype, "lse", 2.0)


def test_gradients_against_differences():
    torch.manual_seed(0)
    q, k, v = (torch.randn(2, n, h, 8, dtype=torch.float64, device="cuda", requires_grad=True) for n, h in ((5, 4), (7, 2), (7, 2)))
    n = torch.tensor([7, 4], device="cuda")
    for mask in (dict(), dict(causal=True), dict(causal=True, window=2), dict(key_lengths=n), dict(causal=True, key_lengths=n)):
        fn = lambda a, b, c: tpw.attention(a, b, c, scale=0.7, **mask)  # noqa: E731
        assert torch.autograd.gradcheck(fn, (q, k, v), eps=1e-6, atol=1e-7)
    assert torch.autograd.gradcheck(lambda a, b, c: tpw.attention(a, b, c, return_lse=True)[1], (q, k, v), eps=1e-6, atol=1e-7)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_views_other_streams_and_repeats(dtype):
    torch.manual_seed(1)
    qkv = torch.randn(2, 200, 8, 64, device="cuda").to(dtype)
    views = qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]
    dense = [t.contiguous() for t in views]
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in dense]
    spread = [torch.stack((t, t), -1)[..., 0] for t in dense]             # features two apart: copied
    shared = [dense[0], dense[1][:, :, :1].expand(-1, -1, 2, -1), dense[2][:, :, :1].expand(-1, -1, 2, -1)]
    first = None
    for args in (views, dense, heads_first, spread):
        leaves = [t.detach().requires_grad_() for t in args]
        out = tpw.attention(*leaves, causal=True)
        res = [out, *torch.autograd.grad(out, leaves, out.detach())]
        if first is None:
            first = res
        for a, b in zip(first, res):
            assert torch.equal(a, b)
    assert torch.equal(tpw.attention(*shared), tpw.attention(shared[0], shared[1].contiguous(), shared[2].contiguous()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = tpw.attention(*dense, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, first[0])
    # without the batch, and with lengths in 64 bits
    assert torch.equal(tpw.attention(*(t[1] for t in dense), causal=True), first[0][1])
    n = torch.tensor([150, 1 << 40], device="cuda")
    assert torch.equal(tpw.attention(*dense, key_lengths=n), tpw.attention(*dense, key_lengths=torch.tensor([150, 200], dtype=torch.int32, device="cuda")))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("nq", [1, 5, 200])
@pytest.mark.parametrize("d", [64, 128, 40])
def test_what_lies_beyond_the_keys_is_never_used(dtype, nq, d):
    torch.manual_seed(2)
    q, k, v = (torch.randn(3, n, 2, d, device="cuda").to(dtype) for n in (nq, 300, 300))
    n = torch.tensor([150, 0, 300], device="cuda")
    k2, v2 = k.clone(), v.clone()
    for bad in (math.nan, math.inf, torch.finfo(dtype).min):
        k2[0, 150:], v2[0, 150:], k2[1], v2[1] = bad, bad, bad, bad
        res = []
        for kk, vv in ((k, v), (k2, v2)):
            leaves = [t.detach().requires_grad_() for t in (q, kk, vv)]
            out, lse = tpw.attention(*leaves, key_lengths=n, return_lse=True)
            res.append([out, lse, *torch.autograd.grad(out, leaves, q)])
        for a, b in zip(*res):
            assert torch.equal(a, b) and not bool(torch.isnan(b).any())
        assert float(res[1][0][1].detach().abs().max()) == 0 and bool((res[1][1][1] == -math.inf).all())
        assert float(res[1][3][1].abs().max()) == 0 and float(res[1][4][0, 150:].abs().max()) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_large_scores_and_shifted_maxima(dtype):
    """Scores of several hundred, maxima that rise and fall by hundreds along the keys, rows whose first keys are all far below."""
    torch.manual_seed(3)
    q, k, v = (torch.randn(1, 300, 2, 64, device="cuda") for _ in range(3))
    k = k * torch.linspace(0.1, 40, 300, device="cuda")[None, :, None, None]
    k[:, 130:170] *= 3
    for kk in (k, k.flip(1)):
        args = [t.to(dtype) for t in (q, kk, v)]
        leaves = [t.detach().requires_grad_() for t in args]
        for causal in (False, True):
            out, lse = tpw.attention(*leaves, causal=causal, return_lse=True)
            want = reference(*args, causal=causal, grad=args[0])
            assert_near(out, want[0], dtype, "out", 4.0)   # scores of 500 are themselves good to 2^-24 * 500 in float32
            assert_near(lse, want[1], torch.float32, "lse")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("size", [1e-4, 1.0, 100.0])
def test_small_and_large_gradients_keep_their_digits(dtype, size):
    """Half precision ends at 65504 and thins out below 6e-5; neither may show in gradients that it can hold."""
    shape = (1, 700, 700, 2, 1, 64, False, None, None)
    q, k, v, go, mask, n = make(shape, dtype, 5, 0.5)
    go = (go.float() * size).to(dtype)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(tpw.attention(*leaves), leaves, go)
    want = reference(q, k, v, grad=go)
    for got, w, name in zip(grads, want[2:], ("dq", "dk", "dv")):
        least = torch.finfo(dtype).smallest_normal * 2.0 ** -10
        err, norm = float((got.double() - w).norm()), float(w.norm())
        # what the result's own type cannot hold (steps of 2^-24 in half precision) is no fault
        floor = math.sqrt(w.numel()) * (2.0 ** -25 if dtype == torch.float16 else least)
        assert err <= 2 * (2.0 ** -10 if dtype == torch.float16 else 2.0 ** -7) * norm + floor, name


def test_the_same_bits_each_time_and_unwanted_gradients():
    shape = (2, 500, 700, 4, 2, 128, True, None, [700, 333])
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, go, mask, n = make(shape, dtype, 6)
        leaves = [t.requires_grad_() for t in (q, k, v)]
        runs = []
        for _ in range(3):
            out = tpw.attention(*leaves, key_lengths=n, **mask)
            runs.append([out, *torch.autograd.grad(out, leaves, go)])
        for r in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], r))
        out = tpw.attention(q, k.detach(), v.detach(), key_lengths=n, **mask)
        assert torch.equal(torch.autograd.grad(out, q, go)[0], runs[0][1])
        out = tpw.attention(q.detach(), k.detach(), v, key_lengths=n, **mask)
        assert torch.equal(torch.autograd.grad(out, v, go)[0], runs[0][3])


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes and 2^31 elements, whose last sequence is the one that is looked at."""
    B, nk = 9, 1 << 20
    k = torch.empty(B, nk, 2, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    k[-1].normal_(), v[-1].normal_()
    n = torch.zeros(B, dtype=torch.int32, device="cuda")
    n[-1] = nk
    q = torch.randn(B, 1, 4, 128, dtype=torch.bfloat16, device="cuda")
    got, lse = tpw.attention(q, k, v, key_lengths=n, causal=True, return_lse=True)
    out, want_lse, *_ = reference(q[-1:], k[-1:], v[-1:], causal=True)
    assert_near(got[-1:], out, torch.bfloat16, "out")
    assert_near(lse[-1:], want_lse, torch.float32, "lse")
    assert float(got[:-1].abs().max()) == 0


def test_refusals():
    q, k = torch.zeros(2, 4, 6, 64, device="cuda"), torch.zeros(2, 5, 3, 64, device="cuda")
    bad = [
        (dict(k=k[:, :, :0], v=k[:, :, :0]), "must be a multiple"),
        (dict(q=q[:, :, :4]), "must be a multiple"),
        (dict(v=k[:, :4]), "same shape"),
        (dict(k=k.half(), v=k.half()), "has type"),
        (dict(k=k.cpu(), v=k.cpu()), "CUDA tensors only"),
        (dict(k=k[..., :32], v=k[..., :32]), "same number of features"),
        (dict(k=k[:1], v=k[:1]), "batch_size"),
        (dict(q=q[0]), "number of dimensions"),
        (dict(q=q[0, 0], k=k[0, 0], v=k[0, 0]), "3-D"),
        (dict(q=q.int(), k=k.int(), v=k.int()), "floating point"),
        (dict(window=0, causal=True), "at least 1"),
        (dict(window=4), "causal"),
        (dict(scale=0.0), "positive"),
        (dict(scale=math.nan), "positive"),
        (dict(key_lengths=torch.ones(3, dtype=torch.int32, device="cuda")), "one length"),
        (dict(key_lengths=torch.ones(2, device="cuda")), "int32 or int64"),
        (dict(q=torch.zeros(1, 2, 1, 257, device="cuda"), k=torch.zeros(1, 2, 1, 257, device="cuda"), v=torch.zeros(1, 2, 1, 257, device="cuda")), "257 features"),
    ]
    for change, text in bad:
        args = dict(dict(q=q, k=k, v=k), **change)
        with pytest.raises(RuntimeError, match=text):
            tpw.attention(args.pop("q"), args.pop("k"), args.pop("v"), **args)
    x = torch.randn(1, 4, 1, 8, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        torch.autograd.grad(tpw.attention(x, x, x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="transforms"):
        torch.vmap(lambda a: tpw.attention(a, a, a))(x)
    y = x * 1
    out = tpw.attention(y, y, y)
    y.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_a_layer_trains_and_serves_what_it_trained(dtype):
    """The example: packed projections, rotary positions, attention with gradients, and the same layer one token at a time."""
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parent.parent / "examples" / "attention_retrieval.py"
    spec = importlib.util.spec_from_file_location("attention_retrieval", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, apart = example.main(steps=6, sequences=32, dtype=dtype, report=lambda text: None)
    assert all(math.isfinite(x) for x in losses)
    # either side rounds probabilities and outputs a few times in the type: sixteen units for a sum of such terms
    assert apart < 16 * torch.finfo(dtype).eps
    assert tpw.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("d", [64, 128])
def test_lengths_of_every_size_around_the_tiles(dtype, d):
    """Each length from none to past two tiles of keys, against every number of queries that changes a kernel or fills a tile."""
    g = torch.Generator().manual_seed(11)
    sizes = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300]
    k, v = (torch.randn(len(sizes), 300, 1, d, generator=g).to(dtype).cuda() for _ in range(2))
    n = torch.tensor(sizes, dtype=torch.int32, device="cuda")
    for nq in (1, 16, 17, 33, 129, 257):
        q = torch.randn(len(sizes), nq, 2, d, generator=g).to(dtype).cuda()
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        for causal in (False, True):
            out, lse = tpw.attention(*leaves, causal=causal, key_lengths=n, return_lse=True)
            want = reference(q, k, v, causal=causal, lengths=sizes, grad=q)
            assert_near(out, want[0], dtype, f"out {nq} {causal}")
            assert_near(lse, want[1], torch.float64 if dtype == torch.float64 else torch.float32, f"lse {nq} {causal}")
            # as above: the gradients of scores cancel where a row sees a key or two
            few = [i for i, size in enumerate(sizes) if size < 3]
            rest = [i for i, size in enumerate(sizes) if size >= 3]
            for got, w, name in zip(torch.autograd.grad(out, leaves, q), want[2:], ("dq", "dk", "dv")):
                assert_near(got[rest], w[rest], dtype, f"{name} {nq} {causal}", 2.0)
                size = math.sqrt(w[few].numel()) * math.sqrt(d)
                assert float((got[few].double() - w[few]).norm()) <= 2 * size * torch.finfo(dtype).eps, f"{name} {nq} {causal}"


def test_many_blocks_of_every_kind_in_one_launch():
    """More blocks than SMs, empty ones among them, so that CTAs take over blocks with and without keys."""
    g = torch.Generator().manual_seed(12)
    lengths = [0, 700, 128, 0, 1, 333, 256, 699]
    q, k, v = (torch.randn(8, n, 12, 64, generator=g).bfloat16().cuda() for n in (600, 700, 700))
    n = torch.tensor(lengths, device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    for mask in (dict(), dict(causal=True), dict(causal=True, window=130)):
        out, lse = tpw.attention(*leaves, key_lengths=n, return_lse=True, **mask)
        want = reference(q, k, v, lengths=lengths, grad=q, **mask)
        assert_near(out, want[0], torch.bfloat16, "out")
        assert_near(lse, want[1], torch.float32, "lse")
        for got, w, name in zip(torch.autograd.grad(out, leaves, q), want[2:], ("dq", "dk", "dv")):
            assert_near(got, w, torch.bfloat16, name, 2.0)
    assert tpw.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_query_tiles_without_keys_beside_tiles_with_keys(dtype):
    """A sequence shorter than its queries: the first 192 rows see nothing, and their zeros must not be mixed up with queries on their way in."""
    g = torch.Generator().manual_seed(13)
    q, k, v = (torch.randn(64, n, 4, 64, generator=g).to(dtype).cuda() for n in (256, 160, 160))
    n = torch.full((64,), 64, dtype=torch.int32, device="cuda")
    for _ in range(10):
        out, lse = tpw.attention(q, k, v, causal=True, key_lengths=n, return_lse=True)
        assert not out[:, :192].any() and bool((lse[:, :, :192] == -math.inf).all())
        assert bool((out[:, 192:] != 0).any(-1).all())


@pytest.mark.parametrize("d", [4, 12, 20, 44, 60, 64])
@pytest.mark.parametrize("causal", [False, True])
def test_float32_widths_and_magnitudes(d, causal):
    """Widths that are no multiple of eight, views of a packed projection, and operands far from 1 whose products are not: float32 keeps all of its
    digits at every exponent."""
    g = torch.Generator().manual_seed(14)
    packed = torch.randn(2, 300, 4 + 2 + 2, d, generator=g).cuda()
    packed[:, :, :4] *= 2.0 ** 60
    packed[:, :, 4:6] *= 2.0 ** -60
    packed[:, :, 6:] *= 2.0 ** -30
    q, k, v = packed[:, :, :4], packed[:, :, 4:6], packed[:, :, 6:]
    go = torch.randn(2, 300, 4, d, generator=g).cuda() * 2.0 ** 20
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    lengths = [300, 211]
    n = torch.tensor(lengths, device="cuda")
    out, lse = tpw.attention(*leaves, causal=causal, key_lengths=n, return_lse=True)
    want = reference(q, k, v, causal=causal, lengths=lengths, grad=go)
    assert_near(out, want[0], torch.float32, f"out {d} {causal}")
    assert_near(lse, want[1], torch.float32, f"lse {d} {causal}")
    for got, w, name in zip(torch.autograd.grad(out, leaves, go), want[2:], ("dq", "dk", "dv")):
        assert_near(got, w, torch.float32, f"{name} {d} {causal}", 2.0)
    assert tpw.device_status() == 0


def test_float32_keys_that_are_not_used_may_hold_anything():
    g = torch.Generator().manual_seed(15)
    q, k, v = (torch.randn(2, 256, 2, 64, generator=g).cuda() for _ in range(3))
    n = torch.tensor([256, 130], device="cuda")
    grads = []
    for fill in (0.0, float("nan"), float("inf")):
        kk, vv = k.clone(), v.clone()
        kk[1, 130:], vv[1, 130:] = fill, fill
        leaves = [t.requires_grad_() for t in (q.clone(), kk, vv)]
        out = tpw.attention(*leaves, key_lengths=n)
        grads.append((out.detach(), *torch.autograd.grad(out, leaves, q)))
    for other in grads[1:]:
        for a, b in zip(grads[0], other):
            assert torch.equal(a, b)
    assert not grads[0][2][1, 130:].any() and not grads[0][3][1, 130:].any()
