"""A cache of keys and values in 4 or 8 bits: tokens go in, come out again, and are attended to as they lie.

The operators live in the dispatcher namespace ``torchpairwise_b200`` (``csrc/torch/tpw_torch_cache.cpp``), which this module loads; they
run the sm_100a kernels of ``libtpw_b200.so`` on the current stream, CUDA tensors only.  The reference has no counterpart.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch
from torch import Tensor

from ._abi import LIB_PATH, lib

CACHE_OPS_LIBRARY = LIB_PATH.parent / "libtpw_b200_cache.so"

_write = _read = _attend = None


def _load() -> None:
    global _write, _read, _attend
    if not CACHE_OPS_LIBRARY.exists():
        raise ImportError(f"{CACHE_OPS_LIBRARY} is missing; run `python torchpairwise_b200/build.py`")
    try:
        torch.ops.load_library(str(CACHE_OPS_LIBRARY))
    except OSError as e:
        raise ImportError(f"{CACHE_OPS_LIBRARY} does not load with torch {torch.__version__}; run `python torchpairwise_b200/build.py`") from e
    ops = torch.ops.torchpairwise_b200
    _write, _read, _attend = ops.cache_write.default, ops.cache_read.default, ops.cache_attention.default


# as with attention: a tree without this library imports all the same, and what is missing is said by the functions that need it
try:
    _load()
except ImportError:
    pass


def _check(name: str, first: Tensor) -> None:
    if _write is None:
        _load()
    if not first.is_cuda:
        raise RuntimeError(f"torchpairwise_b200 runs on CUDA tensors only (no CPU path); got a tensor on {first.device}")
    if torch._C._are_functorch_transforms_active():
        raise RuntimeError(f"{name}: torch.func transforms are not supported")


class QuantizedCache(NamedTuple):
    """Keys and values of ``[batch, heads, capacity]`` tokens in 4 or 8 bits; :func:`quantized_cache` makes an empty one.

    A group of features (32, or the whole head) of a token has a zero, the largest bfloat16 number that is not above its lowest value, and
    a step, the smallest bfloat16 number (2^-100 at least) of which ``2**bits - 1`` reach from the zero to its highest value.  A value is
    held as the nearest whole number of steps above the zero, ties to even (float32: nearest to the quotient in 64 bits), and reads as ``zero + step * code``, at most half a step off.

    ``k_codes`` and ``v_codes`` are uint8 ``[batch, heads, capacity, bytes of a row]``, ``k_scales`` and ``v_scales`` bfloat16
    ``[batch, heads, capacity, groups, 2]``, step and zero; all contiguous, the capacity a multiple of 64.  A row has ``W * 32``
    features, ``W = max(2, ceil(features / 32))``; feature ``32 w + 8 t + n`` of a key (``n < 8``) is code ``(t W + w) 8 + n`` of its
    row, feature ``32 w + 4 t + n`` of a value (``n < 4``) is code ``(t W + w) 4 + n``; the codes of features beyond the head are 0.
    Of two 4-bit codes in a byte the first is the lower.  How many tokens a sequence has is not part of the cache: every call is told.
    """
    k_codes: Tensor
    v_codes: Tensor
    k_scales: Tensor
    v_scales: Tensor
    features: int
    bits: int

    @property
    def capacity(self) -> int:
        return self.k_codes.size(2)


def quantized_cache(batch: int, capacity: int, heads: int, features: int, *, bits: int = 4, group: Optional[int] = 32,
                    device: Union[str, torch.device] = "cuda") -> QuantizedCache:
    """An empty :class:`QuantizedCache` for ``capacity`` tokens of each sequence, rounded up to a multiple of 64.

    ``group`` is 32 (a step and a zero for every 32 features of a head) or None (one for the head); heads of 1 to 128 features.  A key
    and value of 128 features take 160 bytes in 4 bits (group None: 136; 8 bits: 288, 264), 512 in 16-bit types.
    """
    if bits not in (4, 8):
        raise ValueError(f"quantized_cache: bits must be 4 or 8. Got {bits}")
    if not 1 <= features <= 128:
        raise ValueError(f"quantized_cache: {features} features per head: 1 to 128 are supported")
    if group not in (32, None):
        raise ValueError(f"quantized_cache: group must be 32 or None. Got {group}")
    if batch < 0 or capacity < 0 or heads < 0:
        raise ValueError(f"quantized_cache: negative size. Got batch {batch}, capacity {capacity}, heads {heads}")
    rows = -(-capacity // 64) * 64
    if rows >= 1 << 30:
        raise ValueError(f"quantized_cache: capacity {capacity}: at most 2^30 - 64 tokens")
    groups = 1 if group is None else -(-features // 32)
    codes = [torch.zeros(batch, heads, rows, lib.tpw_cache_row_bytes(bits, features), dtype=torch.uint8, device=device) for _ in range(2)]
    scales = [torch.zeros(batch, heads, rows, groups, 2, dtype=torch.bfloat16, device=device) for _ in range(2)]
    return QuantizedCache(*codes, *scales, features, bits)


def cache_write(cache: QuantizedCache, k: Tensor, v: Tensor, key_lengths: Tensor) -> None:
    """Stores tokens: ``k`` and ``v``, ``[batch, tokens, heads, features]`` in float32, float16 or bfloat16, any strides, in one launch.

    ``key_lengths`` (int32 or int64, one per sequence, on the device) says how long each sequence is with them: token i of n goes to
    position ``length - n + i``, over what lies there.  A token whose position is below 0 or not below the capacity is not stored, so a
    batch may be padded at its front.  Values are to be finite and below 2^100 in magnitude; a group with another one reads as NaN.
    Not differentiable.
    """
    _check("cache_write", k)
    _write(*cache, k, v, key_lengths)


def cache_read(cache: QuantizedCache, key_lengths: Tensor, tokens: Optional[int] = None, *,
               dtype: torch.dtype = torch.bfloat16) -> Tuple[Tensor, Tensor]:
    """The keys and values that the codes stand for, ``[batch, tokens, heads, features]`` in ``dtype`` (float32, float16 or bfloat16).

    ``tokens`` asks for the last so many of each sequence: i of n from position ``length - n + i``.  Without it all come, position 0 first
    and as many as the capacity.  Positions outside a sequence's length, or the capacity, read as zero.  ``zero + step * code`` is
    formed in 32 bits and rounded once.
    """
    _check("cache_read", cache.k_codes)
    return _read(*cache, key_lengths, tokens, dtype)


def cache_attention(q: Tensor, cache: QuantizedCache, key_lengths: Tensor, *, causal: bool = False, window: Optional[int] = None,
                    scale: Optional[float] = None, return_lse: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """:func:`attention` over the keys and values that a cache holds, which stay in their codes on the way.

    ``q`` is ``[batch, queries, heads, features]`` in float32, float16 or bfloat16, its heads a multiple of the cache's; ``key_lengths`` as
    in :func:`cache_write`, which comes first for new tokens: query i of a sequence with L keys stands at position ``L - queries + i``.
    ``causal``, ``window``, ``scale``, ``return_lse`` and rows that see nothing are as in :func:`attention`; a length beyond the capacity counts
    as the capacity.  What lies in the cache from a sequence's length on is never used.  Within it, what is not a number makes the rows of its
    tile NaN.  Not differentiable.

    Scores are to stay below 2^24 and results below 2^90 in magnitude, as are queries; results below 2^-104 may be given as zero.  Scores, statistics and sums are held in 32 bits, and a query to 2^-39 of
    the highest magnitude of its row.  Operands of products have fewer: with 16-bit queries a probability times the step of a value is rounded to half precision
    (2^-12 of it, 2^-27 of the largest that its row met in the group), with float32 queries it and the query are two such parts (2^-23).  With more than 192 16-bit queries to
    a key head (their number times the heads that share one; widths that are multiples of 8) the probabilities and what the codes stand for are rounded to half precision: up to 65504 for float16; for
    bfloat16 under a power of two of the head, which leaves 2^-28 of the highest value (2^-32 of the highest key) in any block of 128 tokens that a query sees.
    """
    _check("cache_attention", q)
    out, lse = _attend(q, *cache, key_lengths, causal, window, scale)
    return (out, lse) if return_lse else out
