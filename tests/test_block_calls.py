"""Calls of the block operators that their documentation allows or refuses, beside those of test_block_ops.py."""
import ctypes

from tilelang_ascend_amd import _abi

HERE, THERE = ctypes.c_void_p(16), ctypes.c_void_p(1 << 20)


def test_norm_refuses_one_place_for_two_outputs():
    """H may take X's place and so may Y, but not both: the sum would be lost behind the normalised values."""
    args = dict(X=HERE, residual=THERE, weight=THERE, H=HERE, Y=HERE, Q=None, S=None, M=4, N=64, eps=1e-6, dtype=_abi.F16, round_scale=0, stream=None)
    assert _abi.load().tlq_residual_rms_norm(*args.values()) != 0
    assert "two outputs" in _abi.last_error()
