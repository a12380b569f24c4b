"""The quantised cache where no GPU is needed: refusals of the Python functions and the C entry points, sizes of storage, the schemas."""
import ctypes

import pytest
import torch

import torchpairwise_b200 as tpw
from torchpairwise_b200 import _abi


def test_cpu_tensors_are_rejected_loudly():
    cache = tpw.quantized_cache(2, 5, 1, 8, device="cpu")
    x, n = torch.zeros(2, 3, 1, 8), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: tpw.cache_write(cache, x, x, n), lambda: tpw.cache_read(cache, n), lambda: tpw.cache_attention(x, cache, n)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d,width,groups", [(1, 64, 1), (32, 64, 1), (33, 64, 2), (64, 64, 2), (65, 96, 3), (96, 96, 3), (100, 128, 4), (128, 128, 4)])
def test_storage_of_a_cache(bits, d, width, groups):
    cache = tpw.quantized_cache(3, 65, 2, d, bits=bits, device="cpu")
    assert cache.capacity == 128 and cache.features == d and cache.bits == bits
    assert cache.k_codes.shape == cache.v_codes.shape == (3, 2, 128, width * bits // 8) and cache.k_codes.dtype == torch.uint8
    assert cache.k_scales.shape == cache.v_scales.shape == (3, 2, 128, groups, 2) and cache.v_scales.dtype == torch.bfloat16
    assert tpw.quantized_cache(3, 65, 2, d, bits=bits, group=None, device="cpu").k_scales.shape == (3, 2, 128, 1, 2)


def test_arguments_of_a_new_cache():
    for args, options, text in (((1, 1, 1, 0), {}, "features"), ((1, 1, 1, 129), {}, "features"), ((1, 1, 1, 8), dict(bits=5), "bits"), ((1, 1, 1, 8), dict(group=64), "group"),
                                ((-1, 1, 1, 8), {}, "negative"), ((1, -1, 1, 8), {}, "negative"), ((1, 1 << 30, 1, 8), {}, "capacity")):
        with pytest.raises(ValueError, match=text):
            tpw.quantized_cache(*args, **options, device="cpu")


class _Cache(ctypes.Structure):
    _fields_ = [("bits", ctypes.c_int32), ("groups", ctypes.c_int32), *((n, ctypes.c_int64) for n in ("B", "H", "capacity", "D")),
                ("codes", ctypes.c_void_p * 2), ("scales", ctypes.c_void_p * 2), ("lengths", ctypes.c_void_p)]


class _Rows(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("from_start", ctypes.c_int32), ("N", ctypes.c_int64), ("x", ctypes.c_void_p * 2), ("stride", ctypes.c_int64 * 3 * 2)]


class _Attention(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("causal", ctypes.c_int32), ("window", ctypes.c_int64), ("Nq", ctypes.c_int64), ("Hq", ctypes.c_int64), ("scale", ctypes.c_double),
                ("q", ctypes.c_void_p), ("q_stride", ctypes.c_int64 * 3), ("out", ctypes.c_void_p), ("lse", ctypes.c_void_p)]


X = 1 << 20   # an address that is never followed


def cache_of(**changes):
    c = _Cache(bits=4, groups=1, B=1, H=2, capacity=64, D=32, codes=(ctypes.c_void_p * 2)(X, X), scales=(ctypes.c_void_p * 2)(X, X), lengths=X)
    for name, value in changes.items():
        setattr(c, name, value)
    return c


CACHE_ERRORS = [(dict(bits=3), b"3 bits"), (dict(D=0), b"0 features"), (dict(D=129), b"129 features"), (dict(groups=2), b"2 groups"), (dict(groups=0), b"0 groups"),
                (dict(capacity=65), b"multiple of 64"), (dict(capacity=1 << 30), b"below 2^30"), (dict(B=-1), b"negative"), (dict(lengths=None), b"NULL"),
                (dict(codes=(ctypes.c_void_p * 2)(X, None)), b"NULL"), (dict(scales=(ctypes.c_void_p * 2)(X + 4, X)), b"aligned"), (dict(H=(1 << 20) + 1), b"heads")]


def test_errors_of_the_entry_points_for_rows():
    lib = _abi.lib
    rows = _Rows(dtype=_abi.F32, N=1, x=(ctypes.c_void_p * 2)(X, X))
    for entry in (lib.tpw_cache_write, lib.tpw_cache_read):
        for changes, text in CACHE_ERRORS:
            assert entry(ctypes.byref(cache_of(**changes)), ctypes.byref(rows), None) == 1 and text in lib.tpw_last_error(), (changes, lib.tpw_last_error())
        for bad, text in ((_Rows(dtype=_abi.F64, N=1, x=rows.x), b"dtype"), (_Rows(dtype=_abi.F32, N=-1, x=rows.x), b"-1 tokens"), (_Rows(dtype=_abi.F32, N=1), b"NULL")):
            assert entry(ctypes.byref(cache_of()), ctypes.byref(bad), None) == 1 and text in lib.tpw_last_error()
        assert entry(None, ctypes.byref(rows), None) == 1 and entry(ctypes.byref(cache_of()), None, None) == 1
        assert entry(ctypes.byref(cache_of()), ctypes.byref(_Rows(dtype=_abi.F32, N=0)), None) == 0
        assert entry(ctypes.byref(cache_of(B=0, lengths=None)), ctypes.byref(rows), None) == 0
    assert [lib.tpw_cache_row_bytes(b, d) for b, d in ((4, 1), (4, 128), (8, 65), (5, 64), (4, 0), (4, 129))] == [32, 64, 96, 0, 0, 0]


def test_errors_of_the_entry_points_of_attention():
    lib = _abi.lib

    def attention(**changes):
        a = _Attention(dtype=_abi.BF16, Nq=1, Hq=2, scale=1.0, q=X, out=X)
        for name, value in changes.items():
            setattr(a, name, value)
        return a

    def call(c, a):
        refused = lib.tpw_cache_attention_scratch_bytes(ctypes.byref(c), ctypes.byref(a)) == -1
        message = lib.tpw_last_error()
        assert (lib.tpw_cache_attention(ctypes.byref(c), ctypes.byref(a), None, 0, None) == 1) == refused
        return refused, message

    for changes, text in CACHE_ERRORS:
        refused, message = call(cache_of(**changes), attention())
        assert refused and text in message, (changes, message)
    for changes, text in ((dict(dtype=_abi.F64), b"dtype"), (dict(Hq=3), b"multiple"), (dict(window=4), b"causal"), (dict(window=-1), b"window"), (dict(scale=0.0), b"scale"),
                          (dict(scale=1e-46), b"scale"), (dict(scale=2.4e38), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(Nq=-1), b"-1 queries"), (dict(q=None), b"NULL"), (dict(out=X + 8), b"aligned")):
        refused, message = call(cache_of(), attention(**changes))
        assert refused and text in message, (changes, message)
    assert lib.tpw_cache_attention_scratch_bytes(None, None) == -1
    for c, a in ((cache_of(B=0), attention()), (cache_of(), attention(Nq=0)), (cache_of(), attention(Hq=0))):
        assert lib.tpw_cache_attention_scratch_bytes(ctypes.byref(c), ctypes.byref(a)) == 0 and lib.tpw_cache_attention(ctypes.byref(c), ctypes.byref(a), None, 0, None) == 0


def test_schemas_say_what_is_written():
    schema = str(torch.ops.torchpairwise_b200.cache_write.default._schema)
    assert "Tensor(a!) k_codes" in schema and "Tensor(d!) v_scales" in schema and schema.endswith("-> ()")
    for name in ("cache_read", "cache_attention"):
        assert "!" not in str(getattr(torch.ops.torchpairwise_b200, name).default._schema)


def test_messages_of_the_host_layer_format_numbers():
    """The checks come before anything that touches a device, so they can be entered with CPU tensors through a dispatch key: a message, not an abort."""
    keys = torch._C.DispatchKeySet(torch._C.DispatchKey.AutogradCUDA)
    cache = tpw.quantized_cache(1, 5, 1, 8, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        torch.ops.torchpairwise_b200.cache_read.default.redispatch(keys, *cache, torch.zeros(1, dtype=torch.int32), None, torch.float32)
