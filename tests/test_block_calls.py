"""Calls of the block operators that their documentation allows or refuses, beside those of test_block_ops.py: more rows than the machine takes at
once, and refusals.  Tolerances as there (gated: gates up to 8 here)."""
import ctypes

import pytest
import torch

from helpers import DT, assert_bit_equal
from oracle import ref
from tilelang_ascend_amd import _abi, ops

gpu = pytest.mark.gpu
TYPES = ["float16", "bfloat16"]
HERE, THERE = ctypes.c_void_p(16), ctypes.c_void_p(1 << 20)


def test_norm_refuses_one_place_for_two_outputs():
    """H may take X's place and so may Y, but not both: the sum would be lost behind the normalised values."""
    args = dict(X=HERE, residual=THERE, weight=THERE, H=HERE, Y=HERE, Q=None, S=None, M=4, N=64, eps=1e-6, dtype=_abi.F16, round_scale=0, stream=None)
    assert _abi.load().tlq_residual_rms_norm(*args.values()) != 0
    assert "two outputs" in _abi.last_error()


# ---- rows beyond the machine's work-groups ------------------------------------------------------------------------------------------
# N, and rows of a work-group: every kernel of rows in registers, chunks that end inside of a row and rows that begin anywhere; the kernel of longer rows
ROWS = [(72, 4), (65, 4), (1000, 4), (1544, 1), (1543, 1), (2600, 1), (4104, 1), (8200, 1), (8203, 1), (16392, 1), (32776, 1)]


def at_once(rows):
    return torch.cuda.get_device_properties(0).multi_processor_count * 64 * rows


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,rows", ROWS)
def test_norm_of_more_rows_than_work_groups(N, rows, dtype):
    """A work-group's second and third row: what calls of one row a work-group give, bit for bit, also in place."""
    most = at_once(rows)
    M = 2 * most + 3
    if M * N > 1 << 29:
        M = most + 5
    g = torch.Generator(device="cuda").manual_seed(N)
    x, r = (torch.randn(M, N, generator=g, device="cuda").to(DT[dtype]) for _ in range(2))
    w = torch.rand(N, generator=g, device="cuda").to(DT[dtype])
    kernel = ops.residual_rms_norm(N, outputs="both", in_dtype=dtype)
    whole = kernel(x, r, w)
    for m in range(0, M, most):
        for got, want in zip(whole, kernel(x[m: m + most], r[m: m + most], w)):
            assert torch.equal(got[m: m + most].view(-1).view(torch.uint8), want.view(-1).view(torch.uint8)), (m, got.dtype)
    some = [0, most - 1, most, M - 1]
    hw, yw, v = ref.residual_rms_norm(x[some].cpu(), r[some].cpu(), w, 1e-6)
    assert_bit_equal(whole[0][some], hw)
    assert torch.equal(whole[2][some].cpu(), ref.norm_codes(v))
    assert ((whole[1][some].cpu().double() - yw).abs() <= yw.abs() * (((N / 64 + 32) / 2 + 8) * 2.0**-24 + torch.finfo(DT[dtype]).eps / 2) + 2.0**-25).all()
    # H over the residual, Y over X
    q, s = torch.empty_like(whole[2]), torch.empty_like(whole[3])
    P = _abi.ptr
    _abi.check(_abi.load().tlq_residual_rms_norm(P(x), P(r), P(w), P(r), P(x), P(q), P(s), M, N, 1e-6, _abi.F16 if dtype == "float16" else _abi.BF16, 0, torch.cuda.current_stream().cuda_stream))
    for got, want in zip((r, x, q, s), whole):
        assert torch.equal(got.view(-1).view(torch.uint8), want.view(-1).view(torch.uint8)), "in place"


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,rows", ROWS)
def test_gated_of_more_rows_than_work_groups(N, rows, dtype):
    most = at_once(rows)
    M = 2 * most + 3
    if M * N > 1 << 29:
        M = most + 5
    x = torch.randn(M, 2 * N, generator=torch.Generator(device="cuda").manual_seed(N), device="cuda", dtype=torch.float32).to(DT[dtype])
    kernel = ops.gated_silu(N, outputs="both", in_dtype=dtype)
    whole = kernel(x)
    for m in range(0, M, most):
        for got, want in zip(whole, kernel(x[m: m + most])):
            assert torch.equal(got[m: m + most].view(-1).view(torch.uint8), want.view(-1).view(torch.uint8)), (m, got.dtype)
    some = [0, most - 1, most, M - 1]
    yw = ref.gated_silu(x[some].cpu())
    scale = ref.row_scales(yw)
    assert ((whole[0][some].cpu().double() - yw).abs() <= yw.abs() * (12 * 2.0**-22 + torch.finfo(DT[dtype]).eps / 2) + 2.0**-25).all()
    assert ((whole[2][some].cpu().double() - scale).abs() <= scale * (12 + 1) * 2.0**-22).all()
    assert ((whole[1][some].cpu().double() - yw / scale[:, None]).abs() <= 0.5 + 127 * (2 * 12 + 4) * 2.0**-22).all()
