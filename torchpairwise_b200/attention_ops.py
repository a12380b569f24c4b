"""Softmax attention and rotary positions: the row-normalised exponential kernel on pairwise products, applied to values.

The operators live in the dispatcher namespace ``torchpairwise_b200`` (``csrc/torch/tpw_torch_attention.cpp``), which this module
loads; they run the sm_100a kernels of ``libtpw_b200.so`` on the current stream, CUDA tensors only.  The reference has no counterpart.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from ._abi import LIB_PATH

ATTENTION_OPS_LIBRARY = LIB_PATH.parent / "libtpw_b200_attention.so"

_attention = _rotary_one = _rotary_two = _table = None


def _load() -> None:
    global _attention, _rotary_one, _rotary_two, _table
    if not ATTENTION_OPS_LIBRARY.exists():
        raise ImportError(f"{ATTENTION_OPS_LIBRARY} is missing; run `python torchpairwise_b200/build.py`")
    try:
        torch.ops.load_library(str(ATTENTION_OPS_LIBRARY))
    except OSError as e:
        raise ImportError(f"{ATTENTION_OPS_LIBRARY} does not load with torch {torch.__version__}; run `python torchpairwise_b200/build.py`") from e
    ops = torch.ops.torchpairwise_b200
    _attention, _rotary_one, _rotary_two, _table = ops.attention.default, ops.rotary_embedding.default, ops.rotary_embedding.pair, ops.rotary_table.default


# The distances need only the kernel library, so a tree without this one, or with one built against another torch, imports all the same: what is
# missing is said by the functions that need it.
try:
    _load()
except ImportError:
    pass


def _check(name: str, q: Tensor) -> None:
    if _attention is None:
        _load()
    if not q.is_cuda:
        raise RuntimeError(f"torchpairwise_b200 runs on CUDA tensors only (no CPU path); got a tensor on {q.device}")
    if torch._C._are_functorch_transforms_active():
        raise RuntimeError(f"{name}: torch.func transforms are not supported")


def attention(q: Tensor, k: Tensor, v: Tensor, *, causal: bool = False, window: Optional[int] = None,
              key_lengths: Optional[Tensor] = None, scale: Optional[float] = None,
              return_lse: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """``softmax(scale * q k^T) v`` per head, without the matrix of scores; differentiable in ``q``, ``k`` and ``v``.

    ``q`` is ``[batch, queries, heads, features]``, ``k`` and ``v`` are ``[batch, keys, key heads, features]`` (all three may lack the
    batch), float32, float64, float16 or bfloat16, 1 to 256 features.  The heads of ``q`` are a multiple of the key heads; consecutive
    query heads share one.  Views such as the parts of one packed projection are read as they lie.

    ``key_lengths`` (int32 or int64, one per sequence, on the device) ends each sequence's keys; what lies beyond is never used.
    Query i of a sequence with L keys stands at position ``L - queries + i``, so that new tokens line up with the end of a cache:
    with ``causal`` it sees keys up to its own position, with ``window`` only the last that many of them.  A row that sees
    nothing is zero, and so are its gradients.  ``scale`` defaults to ``1 / sqrt(features)``.  ``return_lse`` also returns
    ``log(sum(exp(scores)))``, ``[batch, heads, queries]`` in float32 (float64 for float64), -inf for such a row; it is differentiable too.

    Scores, statistics and sums are held in 32 bits (64 for float64); the gradients are summed in a fixed order.  A probability is as good as its
    score, 2^-24 of the score's magnitude: scores are to stay below 2^24, beyond which neighbouring 32-bit numbers are more than a factor e apart.
    Within a sequence's length operands are to be finite (float32: below 2^127); what is not makes the rows of its tile NaN, but for rows that
    see nothing.  16-bit types run on the tensor cores where the features are a multiple of 8 up to 128, float32 where they are a multiple of 4 up to 128.
    """
    _check("attention", q)
    out, lse = _attention(q, k, v, causal, window, key_lengths, scale)
    return (out, lse) if return_lse else out


def rotary_embedding(q: Tensor, k: Optional[Tensor], cos: Tensor, sin: Tensor, positions: Optional[Tensor] = None, *,
                     interleaved: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Turns pairs of features by the angles of each token's position; differentiable in ``q`` and ``k``, which share one launch.

    ``q`` and ``k`` are ``[batch, tokens, heads, features]`` (or without the batch) and may differ in their heads; ``k`` may be None, then
    only the turned ``q`` is returned.  ``cos`` and ``sin`` are float32 tables ``[length, r / 2]`` (:func:`rotary_table`): the first r features
    are turned, the pairs being ``(i, r / 2 + i)`` or, ``interleaved``, ``(2 i, 2 i + 1)``; the rest is copied.  ``positions`` (int32 or
    int64, ``[tokens]`` or ``[batch, tokens]``) picks the tables' rows, by default 0, 1, ...; a position outside the tables gives NaN.
    """
    _check("rotary_embedding", q)
    if k is None:
        return _rotary_one(q, cos, sin, positions, interleaved)
    return _rotary_two(q, k, cos, sin, positions, interleaved)


def rotary_table(length: int, features: int, *, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                 original_length: Optional[int] = None, fast_turns: float = 32.0, slow_turns: float = 1.0, magnitude: float = 1.0,
                 device: Union[str, torch.device] = "cuda") -> Tuple[Tensor, Tensor]:
    """Tables ``(cos, sin)``, float32 ``[length, features / 2]``, for :func:`rotary_embedding`.

    Pair i turns by ``base ** (-2 i / features)`` a position.  ``scaling`` stretches the context by ``factor``: "linear" divides
    every frequency; "base" raises the base to ``base * factor ** (features / (features - 2))``, which keeps the fastest pair and
    divides the slowest by ``factor``; "bands" (the interpolation by parts of the YaRN method) divides pairs that make fewer than ``slow_turns`` turns over ``original_length``
    positions, keeps those that make more than ``fast_turns`` and blends linearly in the pair's index between.  ``magnitude`` multiplies both tables.
    Angles are reduced in 64 bits, so long contexts lose nothing.
    """
    if features < 2 or features % 2 != 0:
        raise ValueError(f"rotary_table: features must be even and at least 2. Got {features}")
    if length < 0:
        raise ValueError(f"rotary_table: negative length {length}")
    if not (base > 1.0 and math.isfinite(base)):
        raise ValueError(f"rotary_table: base must be finite and above 1. Got {base}")
    if not (factor > 0.0 and math.isfinite(factor)):
        raise ValueError(f"rotary_table: factor must be positive and finite. Got {factor}")
    half = features // 2
    if scaling == "base":
        if features == 2:
            raise ValueError("rotary_table: scaling the base needs more than 2 features")
        base = base * factor ** (features / (features - 2))
    freq = [base ** (-i / half) for i in range(half)]
    if scaling == "linear":
        freq = [f / factor for f in freq]
    elif scaling == "bands":
        if original_length is None or original_length < 1:
            raise ValueError("rotary_table: scaling by bands needs original_length")
        if not 0.0 < slow_turns < fast_turns:
            raise ValueError("rotary_table: 0 < slow_turns < fast_turns is needed")

        def index_of(turns: float) -> float:   # of the pair that makes so many turns over the original length
            return half * math.log(original_length / (2.0 * math.pi * turns)) / math.log(base)
        first = max(math.floor(index_of(fast_turns)), 0)
        last = min(math.ceil(index_of(slow_turns)), features - 1)
        span = max(last - first, 1e-3)
        # a band that ends before the first pair holds none: every pair makes fewer than slow_turns turns
        blend = [1.0 if last <= 0 else min(max((i - first) / span, 0.0), 1.0) for i in range(half)]
        freq = [f * (1.0 - t) + f / factor * t for f, t in zip(freq, blend)]
    elif scaling not in (None, "base"):
        raise ValueError(f"rotary_table: scaling must be None, 'linear', 'base' or 'bands'. Got {scaling!r}")
    if _table is None:
        _load()
    return _table(torch.tensor(freq, dtype=torch.float64, device=device), length, magnitude)
