"""Calls of the block operators that their documentation allows or refuses, beside those of test_block_ops.py: more rows than the machine takes at once, more
blocks of outputs than a work-group takes at once, both types through every launch, and refusals.  Tolerances as there (gated: gates up to 8 here)."""
import ctypes

import numpy
import pytest
import torch

from helpers import DT, assert_bit_equal, gen
from oracle import ref
from test_block_launches import ask, recorder  # noqa: F401
from tilelang_ascend_amd import _abi, ops

gpu = pytest.mark.gpu
TYPES = ["float16", "bfloat16"]
HERE, THERE = ctypes.c_void_p(16), ctypes.c_void_p(1 << 20)


def test_norm_refuses_one_place_for_two_outputs():
    """H may take X's place and so may Y, but not both: the sum would be lost behind the normalised values."""
    args = dict(X=HERE, residual=THERE, weight=THERE, H=HERE, Y=HERE, Q=None, S=None, M=4, N=64, eps=1e-6, dtype=_abi.F16, round_scale=0, stream=None)
    assert _abi.load().tlq_residual_rms_norm(*args.values()) != 0
    assert "two outputs" in _abi.last_error()


@pytest.mark.parametrize("make", [lambda n: ops.residual_rms_norm(n), lambda n: ops.gated_silu(n), lambda n: ops.low_rank_update(n, 16, 64, 64), lambda n: ops.low_rank_update(4, n, 64, 64),
                                  lambda n: ops.low_rank_update(4, 16, n, 64), lambda n: ops.low_rank_update(4, 16, 64, n)])
def test_factories_refuse_sizes_that_are_no_whole_numbers(make):
    """A kernel for 64 is not what a call for 64.5 asked for."""
    for n in (64.5, 64.0, "64", None):
        with pytest.raises(TypeError):
            make(n)
    assert make(numpy.int64(64)).params[0].name == "X"


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


# ---- more blocks of outputs than a work-group of the second product takes at once -------------------------------------------------------
# M, L, rank, N, K: tiles of 64 rows, then of 16; no size of these goes to single rows, nor does a part of its outputs
BLOCKS = [(6400, 3, 8, 4112, 64), (4200, 3, 16, 4368, 64), (1700, 2, 32, 9232, 8224), (900, 3, 64, 15376, 2080), (500, 3, 128, 25616, 96),
          (6000, 200, 8, 2064, 64), (5000, 200, 16, 2576, 64), (600, 300, 32, 3600, 8224), (300, 40, 64, 9232, 2080), (300, 100, 128, 4624, 96)]


def test_blocks_reach_the_second_pass(recorder):  # noqa: F811
    result = ask(recorder, f"""
result = []
for M, L, rank, N, K in {BLOCKS}:
    size = lib.tlq_low_rank_update_workspace_bytes(M, L, rank, 1, K)
    per = []
    for n in (N, 1024):
        got = launches(lambda: lib.tlq_low_rank_update(X, Y, IDS, A, B, S, H, WS, size, M, L, rank, n, 0, 0, K, 1, 1, None))
        assert "up_kernel" in got[-1][0], (M, n)
        per.append((struct.unpack("i", got[-1][3][84:88])[0], got[-1][2] // 64 // (4 if "Li4ELi" in got[-1][0] else 1)))
    result.append(per)
""")
    for case, ((per, at_a_time), (per_part, _)) in zip(BLOCKS, result):
        assert per > at_a_time >= 1 and (per_part <= at_a_time or per_part < per), (case, per, at_a_time, per_part)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,L,rank,N,K", BLOCKS)
def test_update_of_several_blocks_a_work_group(M, L, rank, N, K, dtype):
    """What calls on 1024 of the outputs give, bit for bit, with 16-bit outputs and fp32 ones, and in place."""
    T, g = DT[dtype], torch.Generator(device="cuda").manual_seed(M + N)
    x = torch.randn(M, K, generator=g, device="cuda").to(T)
    a = (torch.randn(L, rank, K, generator=g, device="cuda") * K**-0.5).to(T)
    b = (torch.randn(L, N, rank, generator=g, device="cuda") * 0.3).to(T)
    scaling = torch.rand(L, generator=g, device="cuda") + 0.5
    ids = torch.randint(-1, L, (M,), generator=g, device="cuda", dtype=torch.int32)
    some = torch.randint(0, M, (12,), generator=gen(M))
    for out in (dtype, "float32"):
        y = torch.randn(M, N, generator=g, device="cuda").to(DT[out])
        whole = ops.low_rank_update(L, rank, N, K, in_dtype=dtype, out_dtype=out)(x, y, ids, a, b, scaling)
        for n in range(0, N, 1024):
            part = slice(n, min(n + 1024, N))
            got = ops.low_rank_update(L, rank, part.stop - n, K, in_dtype=dtype, out_dtype=out)(x, y[:, part].contiguous(), ids, a, b[:, part].contiguous(), scaling)
            assert torch.equal(got, whole[:, part]), (out, n)
        want, off = ref.low_rank_update(x[some.cuda()], y[some.cuda()], ids[some.cuda()], a, b, scaling, (N,))
        assert ((whole[some.cuda()].cpu().double() - want).abs() <= off + (want.abs() + off) * (torch.finfo(DT[out]).eps / 2) + torch.finfo(DT[out]).tiny).all()
        P, lib = _abi.ptr, _abi.load()
        bytes_ = lib.tlq_low_rank_update_workspace_bytes(M, L, rank, 1, K)
        ws = torch.empty(bytes_, dtype=torch.uint8, device="cuda")
        code = _abi.F16 if dtype == "float16" else _abi.BF16
        _abi.check(lib.tlq_low_rank_update(P(x), P(y), P(ids), P(a), P(b), P(scaling), P(y), P(ws), bytes_, M, L, rank, N, 0, 0, K, code, _abi.F32 if out == "float32" else code,
                                           torch.cuda.current_stream().cuda_stream))
        assert torch.equal(y, whole), "in place"


# ---- both types through every launch ------------------------------------------------------------------------------------------------
def test_update_launches_the_kernels_of_its_types(recorder):  # noqa: F811
    result = ask(recorder, """
rng, result = random.Random(7), set()
log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))
for _ in range(2000):
    M, L, rank, parts, K = log(1, rng.choice([64, 2000, 1 << 24])), log(1, 4096), rng.choice([8, 16, 32, 64, 128]), tuple(16 * log(1, 4096) for _ in range(rng.randint(1, 3))), 32 * log(1, 2048)
    t = rng.choice([0, 1])
    out = rng.choice([t, 2])
    size = lib.tlq_low_rank_update_workspace_bytes(M, L, rank, len(parts), K)
    of_in, of_out = ("DF16_", "DF16b")[t], ("DF16_", "DF16b", "f")[out]
    for name, g, threads, data in launches(lambda: lib.tlq_low_rank_update(X, Y, IDS, A, B, S, H, WS, size, M, L, rank, *parts, *[0] * (3 - len(parts)), K, t, out, None)):
        kind = [k for k in ("row", "up", "down_tile", "down", "plan") if "low_rank_" + k + "_kernel" in name][0]
        if kind in ("row", "up"):
            assert "_kernelI" + of_in + of_out + "Li" in name, (t, out, name)
        elif kind != "plan":
            assert "_kernelI" + of_in in name and "_kernelI" + of_in + "D" not in name, (t, out, name)
        if kind in ("row", "up"):
            assert name.split("Li")[-1].startswith(str(rank) + "E"), (rank, name)
        result.add((kind, t, out if kind in ("row", "up") else -1))
result = sorted(result)
""")
    pairs = [(0, 0), (0, 2), (1, 1), (1, 2)]
    want = {("plan", t, -1) for t in (0, 1)} | {(k, t, -1) for k in ("down", "down_tile") for t in (0, 1)} | {(k, *p) for k in ("row", "up") for p in pairs}
    assert {tuple(r) for r in result} == want
