"""W = rn_T(rn_T(T(u) - z) * s) for whole zero points at the ends of the range that the kernels fold into the unpacking: in bfloat16 u - z is a number of
more than eight bits, and rounds, from z = -242 down and z = 257 up."""
import pytest
import torch

from helpers import DT, assert_bit_equal, gen
from oracle import ref
from tilelang_ascend_amd import _abi, ops

pytestmark = pytest.mark.gpu
ZEROS = [-241, -242, -249, -256, -258, 241, 242, 256, 257, 260]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("z", ZEROS)
def test_dequantised_weights(z, dtype):
    T = DT[dtype]
    Wp = torch.arange(256, dtype=torch.uint8).repeat(16, 1)  # [16, 512]: every pair of nibbles
    s = (torch.rand(16, 8, generator=gen(1)) * 0.015 + 0.005).to(T)
    zt = torch.full((16, 8), float(z)).to(T)
    zt[:, 1::2] = 8  # both ways beside each other
    for zeros in (zt, z):
        want = ref.dequant_w4(Wp, s, zeros, 64, T)
        got = ops.dequantize_w4(Wp.cuda(), s.cuda(), zeros.cuda() if isinstance(zeros, torch.Tensor) else zeros, 64, T).cpu()
        assert_bit_equal(got, want, f"z={z} {dtype}")


# algorithm, M: one call for each
CALLS = [("GEMV", 1), ("GEMV", 2), ("SKINNY", 8), ("DECODE", 16), ("SMALL", 48), ("STREAM", 128), ("MFMA", 64), ("MFMA", 192), ("PANELM", 256), ("PANEL", 512), ("PANEL256", 512),
         ("TWO_PASS", 512), ("AUTO", 1), ("AUTO", 16), ("AUTO", 100), ("AUTO", 300)]


@pytest.mark.parametrize("z", [-241, -250, -256, 256, 258])
@pytest.mark.parametrize("algo,M", CALLS)
def test_products(algo, M, z):
    """bfloat16, all weights 7: with z = -250 they are rn(257) = 256 times the scale, with 258 251 times.  fp32 out: K additions, 2^-24 of the sum of magnitudes each, and
    the products of a few in a matrix instruction."""
    lib, P, N, K, group = _abi.load(), _abi.ptr, 512, 2048, 128
    A = (torch.rand(M, K, generator=gen(2)) + 0.5).bfloat16()
    Wp = torch.full((N, K // 2), 0x77, dtype=torch.uint8)
    s = (torch.rand(N, K // group, generator=gen(3)) * 0.015 + 0.005).bfloat16()
    a, w, sc = A.cuda(), Wp.cuda(), s.cuda()
    ws = torch.empty(max(lib.tlq_w4a16_workspace_bytes(M, N, K), N * K * 2) + 16, dtype=torch.uint8, device="cuda")
    for zeros in (torch.full((N, K // group), float(z)).bfloat16(), float(z)):
        tensor = isinstance(zeros, torch.Tensor)
        zc = zeros.cuda() if tensor else None
        C = torch.full((M, N), float("nan"), device="cuda")
        rc = lib.tlq_gemm_w4a16_ws(P(a), P(w), P(sc), P(zc) if tensor else None, P(C), M, N, K, group, 0.0 if tensor else zeros, _abi.BF16, _abi.F32,
                                   getattr(_abi, f"ALGO_{algo}"), P(ws), ws.numel(), torch.cuda.current_stream().cuda_stream)
        _abi.check(rc)
        W = ref.dequant_w4(Wp, s, zeros, group, torch.bfloat16).double()
        want = A.double() @ W.T
        tol = (K + 8) * 2.0**-24 * (A.double().abs() @ W.abs().T) + want.abs() * 2.0**-24
        assert bool(((C.cpu().double() - want).abs() <= tol).all()), f"{algo} M={M} z={z} tensor={tensor}: {((C.cpu().double() - want).abs() / tol).max().item():.1f} x"
