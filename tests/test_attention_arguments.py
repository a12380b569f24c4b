"""What the C entry points of attention make of a scale, with no GPU."""
import ctypes

import pytest

from test_attention_host import _Attention
from torchpairwise_b200 import _abi


@pytest.mark.parametrize("dtype", [_abi.F32, _abi.F64, _abi.F16, _abi.BF16])
@pytest.mark.parametrize("scale,fits", [(0.125, True), (1.2e-38, True), (2.3e38, True), (1e-46, False), (1e-40, True), (2.4e38, False), (1e300, False)])
def test_scales_that_32_bit_scores_cannot_hold_are_refused(dtype, scale, fits):
    """Below, the factor of the scores is 0 in 32 bits, and 0 times the -inf of a masked score is no probability."""
    x = ctypes.c_void_p(1 << 20)   # never followed: only sizes are asked for
    a = _Attention(dtype=dtype, B=1, Nq=2, Nk=2, Hq=2, Hk=1, D=8, scale=scale, q=x, k=x, v=x, out=x, lse=x, grad_out=x)
    for ask in (_abi.lib.tpw_attention_scratch_bytes, _abi.lib.tpw_attention_backward_scratch_bytes):
        status = ask(ctypes.byref(a))
        if dtype == _abi.F64 or fits:
            assert status >= 0, _abi.lib.tpw_last_error()
        else:
            assert status == -1 and b"32-bit scores" in _abi.lib.tpw_last_error()
