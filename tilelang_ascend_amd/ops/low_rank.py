"""Low-rank adapters of many requests beside a shared projection (no counterpart in the reference): any product of this package gives Y, and the
rows of each request get what its own adapter adds to it:

    out = low_rank_update(L, rank, N, K)(x, w4a16_gemm(...)(x, ...), ids, A, B, scaling)

Results do not depend on timing, nor a row's on what the other rows of the call hold; nothing is copied to the host: a step can be captured in a graph.
"""
from __future__ import annotations

import operator
from typing import Optional, Sequence, Union

from ..jit import ABI_DTYPE, TORCH_DTYPES, KernelSpec, NativeCall, Param, PassConfigKey, jit

_PASS_CONFIGS = {PassConfigKey.TL_ASCEND_AUTO_SYNC: True, PassConfigKey.TL_ASCEND_MEMORY_PLANNING: True}


@jit(out_idx=[-1], pass_configs=_PASS_CONFIGS)
def _low_rank_update(L, rank, parts, K, in_dtype, out_dtype):
    N = sum(parts)
    call = NativeCall("low_rank", (L, rank, *parts, *[0] * (3 - len(parts)), K, ABI_DTYPE[TORCH_DTYPES[in_dtype]], ABI_DTYPE[TORCH_DTYPES[out_dtype]]))
    return KernelSpec("low_rank_update",
                      [Param("X", ("M", K), in_dtype), Param("Y", ("M", N), out_dtype), Param("ids", ("M",), "int32"),
                       Param("A", (L, len(parts) * rank, K), in_dtype), Param("B", (L, N, rank), in_dtype), Param("scaling", (L,), "float32"),
                       Param("out", ("M", N), out_dtype)], call, {"parts": parts})


def low_rank_update(L: int, rank: int, N: Union[int, Sequence[int]], K: int, in_dtype: str = "float16", out_dtype: Optional[str] = None):
    """kernel(X [M, K], Y [M, N], ids int32 [M], A [L, parts * rank, K], B [L, N, rank], scaling float32 [L]) -> out [M, N].

    out[m, n] = Y[m, n] + scaling[l] * sum_j (X[m] . A[l, p * rank + j]) * B[l, n, j] with l = ids[m], fp32 sums, rounded once; a row whose
    id lies outside 0 .. L - 1 is Y.  N: the projection's outputs, or those of up to three projections side by side (queries, keys and values;
    gate and up), which are the parts p, each with `rank` rows of A.  rank: 8, 16, 32, 64 or 128; an adapter of a lower rank has zeros in the
    rows and columns that it lacks.  X, A and B are in_dtype, Y and out out_dtype: in_dtype (the default) or float32.

    Where rows share work, the first sums enter the second product with 16 bits (bfloat16; 24 with a float32 output) or 22 (float16)."""
    L, rank, K = operator.index(L), operator.index(rank), operator.index(K)
    parts = tuple(operator.index(n) for n in (N if isinstance(N, (tuple, list)) else (N,)))
    if not 1 <= len(parts) <= 3:
        raise ValueError(f"N must be one to three sizes (got {N})")
    for n in parts:
        if n < 16 or n % 16 or n >= 1 << 24:
            raise ValueError(f"N must be multiples of 16 below 2^24 (got {N})")
    if not 1 <= L <= 4096:
        raise ValueError(f"L must be between 1 and 4096 (got {L})")
    if rank not in (8, 16, 32, 64, 128):
        raise ValueError(f"rank must be 8, 16, 32, 64 or 128 (got {rank})")
    if K < 32 or K % 32 or K >= 1 << 24:
        raise ValueError(f"K must be a multiple of 32 below 2^24 (got {K})")
    if in_dtype not in ("float16", "bfloat16"):
        raise ValueError(f"in_dtype must be float16 or bfloat16, got {in_dtype}")
    out_dtype = in_dtype if out_dtype is None else out_dtype
    if out_dtype not in (in_dtype, "float32"):
        raise ValueError(f"out_dtype must be {in_dtype} or float32, got {out_dtype}")
    return _low_rank_update(L, rank, parts, K, in_dtype, out_dtype)
