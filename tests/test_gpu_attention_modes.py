"""Attention and rotary positions under torch's ways of running an operator: forward-mode derivatives, inference mode, custom operators."""
import pytest
import torch
from torch.autograd import forward_ad

import torchpairwise_b200 as tpw

pytestmark = pytest.mark.gpu


def inputs(requires_grad=False):
    g = torch.Generator().manual_seed(0)
    x = [torch.randn(2, 20, h, 16, generator=g).cuda() for h in (4, 2, 2)]
    return [t.requires_grad_(requires_grad) for t in x], tpw.rotary_table(32, 16)


@pytest.mark.parametrize("layer", ["python", "dispatcher"])
@pytest.mark.parametrize("at", range(7))
def test_tangents_are_refused_and_not_dropped(layer, at):
    """A dual tensor in any differentiable place: no result without its tangent."""
    (q, k, v), (cos, sin) = inputs()
    ops = torch.ops.torchpairwise_b200
    attention = tpw.attention if layer == "python" else ops.attention
    rotary = tpw.rotary_embedding if layer == "python" else ops.rotary_embedding.pair
    args = [q, k, v] if at < 3 else [q, k, cos, sin]
    at = at if at < 3 else at - 3
    with forward_ad.dual_level():
        args[at] = forward_ad.make_dual(args[at], torch.ones_like(args[at]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            (attention if len(args) == 3 else rotary)(*args)


def test_tangents_of_the_gradients_are_refused():
    (q, k, v), (cos, sin) = inputs(True)
    for out in (tpw.attention(q, k, v), tpw.rotary_embedding(q, None, cos, sin)):
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, q, forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))


def test_a_dual_level_without_tangents_changes_nothing():
    (q, k, v), (cos, sin) = inputs()
    want = tpw.attention(*tpw.rotary_embedding(q, k, cos, sin), v)
    with forward_ad.dual_level():
        assert torch.equal(tpw.attention(*tpw.rotary_embedding(q, k, cos, sin), v), want)


def test_functional_jvp_is_refused():
    (q, k, v), (cos, sin) = inputs()
    for fn in (lambda a: tpw.attention(a, k, v), lambda a: tpw.rotary_embedding(a, None, cos, sin)):
        with pytest.raises(RuntimeError):
            torch.func.jvp(fn, (q,), (torch.ones_like(q),))


def test_inference_mode():
    (q, k, v), (cos, sin) = inputs(True)
    want = tpw.attention(*tpw.rotary_embedding(q, k, cos, sin), v)
    with torch.inference_mode():
        got = tpw.attention(*tpw.rotary_embedding(q, k, cos, sin), v, return_lse=True)[0]
    assert want.requires_grad and got.is_inference() and not got.requires_grad and torch.equal(got, want)


def test_the_body_of_a_custom_operator():
    @torch.library.custom_op("tpw_attention_test::layer", mutates_args=())
    def layer(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        return tpw.attention(q, k, v, causal=True)

    def backward(ctx, g):
        with torch.enable_grad():
            leaves = [t.detach().requires_grad_() for t in ctx.saved_tensors]
            out = tpw.attention(*leaves, causal=True)
        return torch.autograd.grad(out, leaves, g)

    layer.register_autograd(backward, setup_context=lambda ctx, inputs, output: ctx.save_for_backward(*inputs))
    leaves, _ = inputs(True)
    got, want = layer(*leaves), tpw.attention(*leaves, causal=True)
    g = torch.randn_like(want)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, leaves, g), torch.autograd.grad(want, leaves, g)):
        assert torch.equal(a, b)


def test_frequencies_of_a_table_receive_no_gradient():
    f = torch.ones(4, dtype=torch.float64, device="cuda", requires_grad=True)
    table = torch.ops.torchpairwise_b200.rotary_table
    with pytest.raises(RuntimeError, match="no gradient"):
        table(f, 3)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        table(forward_ad.make_dual(f.detach(), torch.ones(4, dtype=torch.float64, device="cuda")), 3)
    with torch.no_grad():
        assert torch.equal(table(f, 3)[0], table(f.detach(), 3)[0])
