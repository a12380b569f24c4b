"""Refusals of attention and rotary positions that need no GPU: the Python functions, the schemas and the C entry points."""
import ctypes

import pytest
import torch

import torchpairwise_b200 as tpw
from torchpairwise_b200 import _abi


def test_cpu_tensors_are_rejected_loudly():
    x = torch.zeros(3, 2, 8)
    for call in (lambda: tpw.attention(x, x, x), lambda: tpw.rotary_embedding(x, None, torch.zeros(3, 4), torch.zeros(3, 4))):
        with pytest.raises((RuntimeError, NotImplementedError), match="CUDA"):
            call()


def test_table_arguments():
    for args, text in (((4, 7), "even"), ((4, 0), "even"), ((-1, 8), "negative"), ((4, 8, dict(base=1.0)), "base"), ((4, 8, dict(factor=0.0)), "factor"),
                       ((4, 8, dict(scaling="bands")), "original_length"), ((4, 8, dict(scaling="nope")), "scaling"), ((4, 2, dict(scaling="base", factor=2.0)), "more than 2"),
                       ((4, 8, dict(scaling="bands", original_length=8, fast_turns=1.0)), "turns")):
        with pytest.raises(ValueError, match=text):
            tpw.rotary_table(*args[:2], **(args[2] if len(args) > 2 else {}), device="cpu")


class _Attention(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("causal", ctypes.c_int32), ("window", ctypes.c_int64), *((n, ctypes.c_int64) for n in ("B", "Nq", "Nk", "Hq", "Hk", "D")),
                ("scale", ctypes.c_double), *((n, ctypes.c_void_p) for n in ("q", "k", "v")), *((n, ctypes.c_int64 * 3) for n in ("q_stride", "k_stride", "v_stride")),
                ("key_lengths", ctypes.c_void_p), ("out", ctypes.c_void_p), ("lse", ctypes.c_void_p), ("out_rest", ctypes.c_void_p), ("grad_out", ctypes.c_void_p), ("grad_out_stride", ctypes.c_int64 * 3),
                ("grad_lse", ctypes.c_void_p), *((n, ctypes.c_void_p) for n in ("grad_q", "grad_k", "grad_v"))]


def test_argument_errors_of_the_c_entry_points():
    lib = _abi.lib

    def call(**changes):
        a = _Attention(dtype=_abi.F32, B=1, Nq=2, Nk=2, Hq=2, Hk=1, D=8, scale=1.0)
        for name, value in changes.items():
            setattr(a, name, value)
        return lib.tpw_attention_forward(ctypes.byref(a), None, 0, None), lib.tpw_last_error()

    for changes, text in ((dict(dtype=2), b"dtype"), (dict(D=257), b"257 features"), (dict(D=0), b"0 features"), (dict(Hk=0), b"multiple"), (dict(Hq=3, Hk=2), b"multiple"),
                          (dict(window=4), b"causal"), (dict(window=-1), b"window"), (dict(scale=0.0), b"scale"), (dict(Nq=-1), b"negative"), (dict(), b"NULL")):
        status, message = call(**changes)
        assert status == 1 and text in message, (changes, message)
    assert call(B=0)[0] == 0 and call(Nq=0, Nk=0)[0] == 0
    a = _Attention(dtype=_abi.F32, B=1, Nq=2, Nk=2, Hq=2, Hk=1, D=300, scale=1.0)
    assert lib.tpw_attention_scratch_bytes(ctypes.byref(a)) == -1 and lib.tpw_attention_backward_scratch_bytes(ctypes.byref(a)) == -1
    assert lib.tpw_attention_forward(None, None, 0, None) == 1
    assert lib.tpw_rotary_apply(None, None) == 1 and b"NULL" in lib.tpw_last_error()
    assert lib.tpw_rotary_table(None, 1.0, None, None, 4, 4, None) == 1 and lib.tpw_rotary_table(None, 1.0, None, None, 0, 4, None) == 0
