"""Rotary positions on a B200 against complex products in float64."""
import math

import pytest
import torch

import torchpairwise_b200 as tpw

pytestmark = pytest.mark.gpu
TYPES = [torch.float64, torch.float32, torch.float16, torch.bfloat16]


def turned(x, cos, sin, at, inter):
    """x [B, N, H, D] in float64, its pairs as complex numbers times the table's."""
    r = 2 * cos.shape[1]
    z = torch.complex(cos.double(), sin.double())[at][:, :, None]
    head = x.detach().double()[..., :r]
    a, b = (head[..., 0::2], head[..., 1::2]) if inter else (head[..., :r // 2], head[..., r // 2:])
    y = torch.complex(a, b) * z
    y = torch.stack((y.real, y.imag), -1).flatten(-2) if inter else torch.cat((y.real, y.imag), -1)
    return torch.cat((y, x.detach().double()[..., r:]), -1)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("b,n,hq,hk,d,r", [(1, 1, 1, 1, 64, 64), (3, 1, 8, 2, 128, 128), (2, 77, 6, 3, 80, 32), (1, 300, 5, 5, 33, 10),
                                           (2, 40, 3, 1, 64, 36), (1, 9, 2, 2, 16, 0), (2, 1000, 16, 4, 128, 64), (2, 0, 2, 2, 8, 8)])
def test_turn_and_gradient(dtype, inter, b, n, hq, hk, d, r):
    g = torch.Generator().manual_seed(n + d)
    q, k, gq, gk = (torch.randn(b, n, h, d, generator=g).to(dtype).cuda() for h in (hq, hk, hq, hk))
    cos, sin = tpw.rotary_table(5000, r, device="cuda") if r else (torch.empty(5000, 0, device="cuda"),) * 2
    at = torch.randint(0, 5000, (b, n), generator=g).cuda()
    q.requires_grad_(), k.requires_grad_()
    out = tpw.rotary_embedding(q, k, cos, sin, at, interleaved=inter)
    grads = torch.autograd.grad(out, (q, k), (gq, gk))
    unit = {torch.float64: 2.0 ** -52, torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    for got, x, c in ((out[0], q, sin), (out[1], k, sin), (grads[0], gq, -sin), (grads[1], gk, -sin)):
        want = turned(x, cos, c, at, inter)
        assert got.dtype == dtype and got.shape == want.shape
        # two products and a sum in 32 bits, one rounding: half a unit of the result and three of the pair's length in 32 bits
        assert bool(((got.double() - want).abs() <= unit * want.abs() + 4 * 2.0 ** -24 * 8 * (dtype != torch.float64) + 1e-14).all())
        assert torch.equal(got[..., r:].detach(), x.detach()[..., r:])


def test_views_positions_and_one_tensor():
    torch.manual_seed(0)
    cos, sin = tpw.rotary_table(600, 64)
    for dtype in TYPES:
        qkv = torch.randn(2, 50, 9, 64, device="cuda").to(dtype)
        q, k = qkv[:, :, :4], qkv[:, :, 4:6]
        at = torch.arange(100, 150, device="cuda")
        a, b = tpw.rotary_embedding(q, k, cos, sin, at)
        assert torch.equal(a, tpw.rotary_embedding(q.contiguous(), None, cos, sin, at.int().expand(2, -1)))
        assert torch.equal(b, tpw.rotary_embedding(k.transpose(1, 2).contiguous().transpose(1, 2), None, cos, sin, at[None]))
        assert torch.equal(a[1], tpw.rotary_embedding(q[1], None, cos, sin, at))
        assert torch.equal(tpw.rotary_embedding(q, None, cos, sin), tpw.rotary_embedding(q, None, cos, sin, torch.arange(50, device="cuda")))
        # an odd start: rows off the 16-byte grid
        flat = torch.randn(2 * 50 * 4 * 64 + 1, device="cuda").to(dtype)[1:].view(2, 50, 4, 64)
        assert torch.equal(tpw.rotary_embedding(flat, None, cos, sin, at), tpw.rotary_embedding(flat.clone(), None, cos, sin, at))
        wide = qkv.expand(2, 50, 9, 64)[:, :, :1].expand(-1, -1, 3, -1)
        assert torch.equal(tpw.rotary_embedding(wide, None, cos, sin), tpw.rotary_embedding(wide.contiguous(), None, cos, sin))


def test_positions_outside_the_table_are_nan():
    cos, sin = tpw.rotary_table(10, 8)
    x = torch.ones(1, 4, 1, 12, device="cuda")
    y = tpw.rotary_embedding(x, None, cos, sin, torch.tensor([0, 10, -1, 1 << 40], device="cuda"))
    assert not bool(torch.isnan(y[0, 0]).any()) and bool(torch.isnan(y[0, 1:, :, :8]).all()) and bool((y[..., 8:] == 1).all())


def test_only_one_gradient_and_gradients_of_gradients():
    cos, sin = tpw.rotary_table(32, 8)
    q, k = (torch.randn(1, 5, 2, 8, dtype=torch.float64, device="cuda", requires_grad=True) for _ in range(2))
    a, b = tpw.rotary_embedding(q, k, cos, sin)
    ref = torch.autograd.grad(b.square().sum(), k, retain_graph=True)[0]
    torch.testing.assert_close(ref, 2 * k.detach(), rtol=1e-6, atol=1e-6)   # a turn keeps lengths (up to the table's 32 bits)
    assert torch.autograd.gradcheck(lambda x, y: tpw.rotary_embedding(x, y, cos, sin), (q, k), eps=1e-6, atol=1e-8)
    assert torch.autograd.gradgradcheck(lambda x: tpw.rotary_embedding(x, None, cos, sin, interleaved=True).square(), (q,), eps=1e-6, atol=1e-6)


@pytest.mark.parametrize("how", [dict(), dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
                                 dict(scaling="bands", factor=16.0, original_length=4096), dict(magnitude=1.2, base=500000.0)])
def test_table(how):
    length, r = 200000, 96
    cos, sin = tpw.rotary_table(length, r, **how)
    half, base, f = r // 2, how.get("base", 10000.0), how.get("factor", 1.0)
    i = torch.arange(half, dtype=torch.float64)
    if how.get("scaling") == "base":
        base = base * f ** (r / (r - 2))
    freq = base ** (-2 * i / r)
    if how.get("scaling") == "linear":
        freq = freq / f
    if how.get("scaling") == "bands":
        turns = 4096 * freq / (2 * math.pi)
        keep, cut = freq, freq / f
        assert how["factor"] == 16.0
        got = torch.atan2(sin[1].double().cpu(), cos[1].double().cpu())
        fast, slow = turns > 40, turns < 0.5
        torch.testing.assert_close(got[fast], keep[fast], rtol=1e-6, atol=1e-9)
        torch.testing.assert_close(got[slow], cut[slow], rtol=1e-6, atol=1e-9)
        assert bool((got <= keep * (1 + 1e-6)).all() and (got >= cut * (1 - 1e-6)).all())
        return
    angle = torch.arange(length, dtype=torch.float64)[:, None] * freq
    m = how.get("magnitude", 1.0)
    # the fraction of a turn is good to 2^-53 of 2e5 radians, then one 32-bit sine: a few units of 2^-24
    for got, want in ((cos, angle.cos() * m), (sin, angle.sin() * m)):
        assert float((got.cpu().double() - want).abs().max()) <= 6 * 2.0 ** -24 * m


def test_refusals():
    cos, sin = tpw.rotary_table(16, 8)
    x = torch.zeros(2, 4, 3, 8, device="cuda")
    for args, text in [((x, x[:, :3], cos, sin), "number of heads"), ((x, x.half(), cos, sin), "has type"), ((x[0, 0], None, cos, sin), "3-D"),
                       ((x, None, cos.double(), sin), "float32 tables"), ((x, None, cos, sin[:4]), "same shape"),
                       ((x[..., :6], None, cos, sin), "turn 8 features"), ((x, None, cos[:3], sin[:3]), "tables end"),
                       ((x, None, cos, sin, torch.zeros(5, dtype=torch.int64, device="cuda")), "positions must be"),
                       ((x, None, cos, sin, torch.zeros(4, device="cuda")), "int32 or int64"), ((x, None, cos.cpu(), sin), "CUDA tensors only"),
                       ((x.int(), None, cos, sin), "floating point"), ((x, None, cos.clone().requires_grad_(), sin), "no gradient")]:
        with pytest.raises(RuntimeError, match=text):
            tpw.rotary_embedding(*args)
