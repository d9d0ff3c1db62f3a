"""What stands between two quantised products of a transformer block: the residual's addition with the root-mean-square norm, and the gated
activation of an MLP.  The reference has neither; their 8-bit outputs are those of its quantiser (examples/deepseek_v4/act_quant.py:25-92), in one pass:

    h, q, s = residual_rms_norm(N, outputs="int8")(x, residual, weight)      # then int8_gemm_kernel_corrected(q, W, s, scale_b)
    h, y    = residual_rms_norm(N)(x, residual, weight)                      # then w4a16_gemm(y, ...)
    q, s    = gated_silu(N, outputs="int8")(gate_up)

``outputs``: "float" for Y in the activations' type, "int8" for codes Q with a scale S for each token, "both" for Y, Q, S (adapters
beside an int8 product take Y).  Q is made of the fp32 values, not of Y.  Any number of tokens M, any N.
"""
from __future__ import annotations

import operator

from ..jit import ABI_DTYPE, TORCH_DTYPES, KernelSpec, NativeCall, Param, PassConfigKey, jit

_PASS_CONFIGS = {PassConfigKey.TL_ASCEND_AUTO_SYNC: True, PassConfigKey.TL_ASCEND_MEMORY_PLANNING: True}


def _check(N: int, outputs: str, in_dtype: str):
    """-> (with Y, with Q and S)."""
    if not 1 <= N < 1 << 30:
        raise ValueError(f"N must be between 1 and 2^30 - 1 (got {N})")
    if outputs not in ("float", "int8", "both"):
        raise ValueError(f'outputs must be "float", "int8" or "both", got {outputs!r}')
    if in_dtype not in ("float16", "bfloat16"):
        raise ValueError(f"in_dtype must be float16 or bfloat16, got {in_dtype}")
    return outputs != "int8", outputs != "float"


def _output_params(N, floats, codes, in_dtype):
    return ([Param("Y", ("M", N), in_dtype)] if floats else []) + ([Param("Q", ("M", N), "int8"), Param("S", ("M",), "float32")] if codes else [])


def _norm_spec(N, eps, outputs, with_residual, round_scale, in_dtype):
    floats, codes = _check(N, outputs, in_dtype)
    if not 1e-12 <= eps <= 1:
        raise ValueError(f"eps must be between 1e-12 and 1 (got {eps})")
    params = [Param("X", ("M", N), in_dtype)]
    if with_residual:
        params.append(Param("residual", ("M", N), in_dtype))
    params.append(Param("weight", (N,), in_dtype))
    if with_residual:
        params.append(Param("H", ("M", N), in_dtype))
    params += _output_params(N, floats, codes, in_dtype)
    call = NativeCall("norm", (N, ABI_DTYPE[TORCH_DTYPES[in_dtype]], bool(round_scale), bool(with_residual), floats, codes), float(eps))
    return KernelSpec("residual_rms_norm", params, call, {"eps": float(eps), "outputs": outputs, "residual": bool(with_residual), "round_scale": bool(round_scale)})


def _gated_spec(N, outputs, round_scale, in_dtype):
    floats, codes = _check(N, outputs, in_dtype)
    call = NativeCall("gated", (N, ABI_DTYPE[TORCH_DTYPES[in_dtype]], bool(round_scale), floats, codes))
    return KernelSpec("gated_silu", [Param("X", ("M", 2 * N), in_dtype), *_output_params(N, floats, codes, in_dtype)], call,
                      {"outputs": outputs, "round_scale": bool(round_scale)})


# (how many outputs there are goes by the options, and a decorated factory has a fixed number of them)
_norm = {n: jit(_norm_spec, out_idx=list(range(-n, 0)), pass_configs=_PASS_CONFIGS) for n in (1, 2, 3, 4)}
_gated = {n: jit(_gated_spec, out_idx=list(range(-n, 0)), pass_configs=_PASS_CONFIGS) for n in (1, 2, 3)}
_OUTPUTS = {"float": 1, "int8": 2, "both": 3}


def residual_rms_norm(N: int, eps: float = 1e-6, outputs: str = "float", with_residual: bool = True, round_scale: bool = False, in_dtype: str = "bfloat16"):
    """kernel(X [M, N][, residual [M, N]], weight [N]) -> [[H,] [Y,] [Q int8 [M, N], S float32 [M]]] (the tensor itself where it is one).

    H = X + residual in their type (without a residual: X, and no H);  y = H * weight / sqrt(mean(H^2) + eps) in fp32;  Y = y rounded once;
    S = max(max|y|, 1e-4) / 127 (round_scale: the next power of two), Q = int8(rint(clamp(y / S, -127, 127))).  Without round_scale, and where S
    is not the floor, Q is decided exactly: it does not depend on how the sum of squares was formed."""
    return _norm[_OUTPUTS.get(outputs, 1) + bool(with_residual)](operator.index(N), eps, outputs, bool(with_residual), bool(round_scale), in_dtype)


def gated_silu(N: int, outputs: str = "float", round_scale: bool = False, in_dtype: str = "bfloat16"):
    """kernel(X [M, 2N]) -> [[Y,] [Q int8 [M, N], S float32 [M]]] (the tensor itself where it is one).

    y = silu(X[:, :N]) * X[:, N:] in fp32, the gates first; Y, Q and S of it as residual_rms_norm makes them."""
    return _gated[_OUTPUTS.get(outputs, 1)](operator.index(N), outputs, bool(round_scale), in_dtype)
