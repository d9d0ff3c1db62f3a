"""A mixture-of-experts layer on packed 4-bit weights: the router's choice and the experts' two products.

The reference's quantised products are dense (examples/dequantize_gemm); these operators are the same products with one
weight matrix per expert, chosen on the device:

    weights, ids = moe_route(E, top_k, ...)(logits)                          logits [M, E]
    hidden = moe_gate_up_w4a16(E, top_k, N, K, ...)(x, ids, w13, s13)        x [M, K] -> [M, top_k, N]
    y = moe_down_w4a16(E, top_k, K, N, ...)(hidden, ids, weights, w2, s2)    -> [M, K]

Routing takes any number of tokens M, the products any with M * top_k below 2^24.  Nothing is copied to the host: a step can be captured in a graph.  Weights are
those of w4a16_gemm (uint8 [rows, K/2], low nibble first, W = rn(rn(u - z) * s) in the activations' type), the experts' matrices
back to back; `gate` rows come before `up` rows.  An id outside 0 .. E - 1 is a slot without an expert here (another GPU's
share, or an empty one): its hidden row is 0 and it adds nothing.  Results do not depend on timing.
"""
from __future__ import annotations

from typing import Union

from .. import _abi
from ..jit import ABI_DTYPE, TORCH_DTYPES, KernelSpec, NativeCall, Param, PassConfigKey, jit

_PASS_CONFIGS = {PassConfigKey.TL_ASCEND_AUTO_SYNC: True, PassConfigKey.TL_ASCEND_MEMORY_PLANNING: True}
_SCORING = {"softmax": _abi.MOE_SOFTMAX, "sigmoid": _abi.MOE_SIGMOID}


def _check_experts(E: int, top_k: int) -> None:
    if not 1 <= E <= 1024:
        raise ValueError(f"E must be between 1 and 1024 (got {E})")
    if not 1 <= top_k <= 64:
        raise ValueError(f"top_k must be between 1 and 64 (got {top_k})")


@jit(out_idx=[-2, -1], pass_configs=_PASS_CONFIGS)
def moe_route(E: int, top_k: int, scoring: str = "softmax", n_group: int = 1, topk_group: int = 1, renormalize: bool = True,
              scaling: float = 1.0, with_bias: bool = False, in_dtype: str = "float32"):
    """kernel(logits [M, E] in_dtype[, bias [E] float32]) -> [weights float32 [M, top_k], ids int32 [M, top_k]].

    p = softmax(logits) or sigmoid(logits); the experts are chosen by p + bias, largest first, ties to the lowest index;
    their weights are p of the chosen ones (the bias does not enter), divided by their sum with `renormalize`, times `scaling`.
    n_group > 1: only experts of the topk_group best of n_group runs of neighbouring experts are chosen, a run's value being
    the sum of its two largest p + bias.  What is compared is binary64.  A logit (or p + bias) of -infinity or NaN masks its
    expert (a logit: in the softmax too); slots for which no expert is left hold id -1 and weight 0."""
    _check_experts(E, top_k)
    if scoring not in _SCORING:
        raise ValueError(f"scoring must be softmax or sigmoid, got {scoring}")
    if not 1 <= n_group <= 64 or E % n_group:
        raise ValueError(f"n_group must divide E={E} and be at most 64 (got {n_group})")
    if not 1 <= topk_group <= n_group:
        raise ValueError(f"topk_group must be between 1 and n_group={n_group} (got {topk_group})")
    if top_k > E // n_group * topk_group:
        raise ValueError(f"top_k={top_k} is more than the {E // n_group * topk_group} experts of the chosen groups")
    if in_dtype not in ("float16", "bfloat16", "float32"):
        raise ValueError(f"in_dtype must be float16, bfloat16 or float32, got {in_dtype}")
    params = [Param("logits", ("M", E), in_dtype)]
    if with_bias:
        params.append(Param("bias", (E,), "float32"))
    params += [Param("weights", ("M", top_k), "float32"), Param("ids", ("M", top_k), "int32")]
    call = NativeCall("moe_route", (E, top_k, n_group, topk_group, _SCORING[scoring], bool(renormalize),
                                    ABI_DTYPE[TORCH_DTYPES[in_dtype]], bool(with_bias)), float(scaling))
    return KernelSpec("moe_route", params, call, {"scoring": scoring, "groups": (n_group, topk_group), "renormalize": bool(renormalize),
                                                  "scaling": float(scaling)})


def _check_products(E, top_k, N, K, group_size, in_dtype, zeros):
    """-> (with a zero-point tensor, the scalar zero point)."""
    _check_experts(E, top_k)
    if N < 16 or N % 16:
        raise ValueError(f"N must be a multiple of 16 (got {N})")
    if K < 32 or K % 32:
        raise ValueError(f"K must be a multiple of 32 (got {K})")
    if group_size < 32 or group_size % 32 or K % group_size:
        raise ValueError(f"group_size must be a multiple of 32 that divides K={K} (got {group_size})")
    if in_dtype not in ("float16", "bfloat16"):
        raise ValueError(f"in_dtype must be float16 or bfloat16, got {in_dtype}")
    if isinstance(zeros, str):
        if zeros != "tensor":
            raise ValueError('zeros must be None, a number or "tensor"')
        return True, 0.0
    return False, 0.0 if zeros is None else float(zeros)


def _weight_params(E, rows, K, group_size, in_dtype, with_scales, zeros_tensor):
    params = [Param("W_packed", (E, rows, K // 2), "uint8")]
    if with_scales:
        params.append(Param("scales", (E, rows, K // group_size), in_dtype))
    if zeros_tensor:
        params.append(Param("zeros", (E, rows, K // group_size), in_dtype))
    return params


@jit(out_idx=[-1], pass_configs=_PASS_CONFIGS)
def moe_gate_up_w4a16(E: int, top_k: int, N: int, K: int, group_size: int = 128, in_dtype: str = "float16",
                      with_scales: bool = True, zeros: Union[None, float, int, str] = None):
    """kernel(X [M, K], ids int32 [M, top_k], W_packed uint8 [E, 2N, K/2][, scales [E, 2N, K/group_size]][, zeros]) -> H [M, top_k, N].

    H[t, j] = silu(X[t] @ W[e, :N].T) * (X[t] @ W[e, N:].T) with e = ids[t, j], fp32 sums, rounded once; 0 for a slot without an
    expert.  zeros: None (no zero point), a number (one zero point for all) or "tensor" (an input shaped like the scales)."""
    zeros_tensor, zero = _check_products(E, top_k, N, K, group_size, in_dtype, zeros)
    params = [Param("X", ("M", K), in_dtype), Param("ids", ("M", top_k), "int32"),
              *_weight_params(E, 2 * N, K, group_size, in_dtype, with_scales, zeros_tensor), Param("H", ("M", top_k, N), in_dtype)]
    call = NativeCall("moe_gate_up", (E, top_k, N, K, group_size, ABI_DTYPE[TORCH_DTYPES[in_dtype]], bool(with_scales), zeros_tensor), zero)
    return KernelSpec("moe_gate_up_w4a16", params, call, {"group": group_size, "zeros": zeros})


@jit(out_idx=[-1], pass_configs=_PASS_CONFIGS)
def moe_down_w4a16(E: int, top_k: int, N: int, K: int, group_size: int = 128, in_dtype: str = "float16", out_dtype: str = "float16",
                   with_scales: bool = True, zeros: Union[None, float, int, str] = None):
    """kernel(H [M, top_k, K], ids int32 [M, top_k], weights float32 [M, top_k], W_packed uint8 [E, N, K/2][, scales [E, N, K/group_size]]
    [, zeros]) -> Y [M, N] out_dtype.

    Y[t] = sum_j weights[t, j] * (H[t, j] @ W[ids[t, j]].T), fp32 sums, rounded once; slots without an expert add nothing."""
    zeros_tensor, zero = _check_products(E, top_k, N, K, group_size, in_dtype, zeros)
    if out_dtype not in ("float16", "bfloat16", "float32"):
        raise ValueError(f"out_dtype must be float16, bfloat16 or float32, got {out_dtype}")
    params = [Param("H", ("M", top_k, K), in_dtype), Param("ids", ("M", top_k), "int32"), Param("weights", ("M", top_k), "float32"),
              *_weight_params(E, N, K, group_size, in_dtype, with_scales, zeros_tensor), Param("Y", ("M", N), out_dtype)]
    call = NativeCall("moe_down", (E, top_k, N, K, group_size, ABI_DTYPE[TORCH_DTYPES[in_dtype]], bool(with_scales), zeros_tensor,
                                   ABI_DTYPE[TORCH_DTYPES[out_dtype]]), zero)
    return KernelSpec("moe_down_w4a16", params, call, {"group": group_size, "zeros": zeros})
