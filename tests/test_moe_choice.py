"""The kernels of the experts' products: which one a call runs on (asked for on the host), and calls that reach the corners of each.

Tolerances are those of test_moe.py: what the fp32 sums may be off by, which the oracle returns beside the value, plus half a step of the
output type."""
import ctypes

import pytest
import torch

from helpers import DT, gen
from oracle import ref
from tilelang_ascend_amd import _abi, ops
from test_moe import assert_close64, kernel_zeros, make_experts, make_ids, operands

gpu = pytest.mark.gpu
FEW, TILES32, TILES64, TILES256 = 1, 2, 3, 4


def choice(up, M, E, k, N, K, group, zeros):
    """-> (kernel, plan of the kernel for few pairs or None)"""
    plan = (ctypes.c_int64 * 7)()
    kernel = _abi.load().tlq_debug_moe_choice(up, M, E, k, N, K, group, isinstance(zeros, str), ctypes.cast(plan, ctypes.c_void_p))
    names = ("rows", "splits", "tiles", "parts", "lds", "lds_used", "groups")
    return kernel, dict(zip(names, plan)) if kernel == FEW else None


def run_both(up, M, E, k, N, K, group, dtype, zeros, kind, out="float32", seed=20):
    """One product against the oracle; returns the output on the CPU."""
    T = DT[dtype]
    ids = make_ids(M, E, k, kind, seed)
    Wp, s, z = make_experts(E, 2 * N if up else N, K, group, T, zeros, seed + 1)
    if up:
        X = torch.randn(M, K, generator=gen(seed + 2)).to(T)
        got = ops.moe_gate_up_w4a16(E, k, N, K, group, dtype, zeros=kernel_zeros(z))(*operands(X, ids, Wp, s, z))
        want, off = ref.moe_gate_up(X, ids, Wp, s, z, group)
    else:
        H = torch.randn(M, k, K, generator=gen(seed + 2)).to(T)
        weights = torch.softmax(torch.randn(M, k, generator=gen(seed + 3)), 1)
        got = ops.moe_down_w4a16(E, k, N, K, group, dtype, out, zeros=kernel_zeros(z))(*operands(H, ids, weights, Wp, s, z))
        want, off = ref.moe_down(H, ids, weights, Wp, s, z, group)
    assert_close64(got, want, off, f"{'gate_up' if up else 'down'} {M, E, k, N, K, group, dtype, zeros, kind}")
    return got.cpu()


# ---- few pairs with one zero point that is no whole number -----------------------------------------------------------------------
# M, E, top_k, N, K, group: one token; pairs up to the experts; more pairs than experts; rows of several parts; scales of several pieces
FRACTIONAL = [(1, 8, 2, 64, 128, 64), (1, 64, 6, 176, 512, 128), (4, 16, 3, 32, 2048, 128), (3, 4, 2, 48, 256, 32), (2, 8, 1, 64, 4160, 32), (1, 3, 2, 32, 14336, 64)]


@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("M,E,k,N,K,group", FRACTIONAL)
def test_few_pairs_use_no_more_lds_than_they_ask_for(M, E, k, N, K, group, up):
    for zeros in (None, "tensor"):
        kernel, plan = choice(up, M, E, k, N, K, group, zeros)
        assert kernel == FEW and 0 < plan["lds_used"] <= plan["lds"] <= 160 * 1024


@gpu
@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("zeros,dtype", [(7.5, "float16"), (7.5, "bfloat16"), (-300.0, "bfloat16")])
@pytest.mark.parametrize("M,E,k,N,K,group", FRACTIONAL)
def test_few_pairs_with_a_zero_point_that_does_not_fold(M, E, k, N, K, group, zeros, dtype, up):
    run_both(up, M, E, k, N, K, group, dtype, zeros, "spread")
