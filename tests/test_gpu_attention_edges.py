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
