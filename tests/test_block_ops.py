"""The norm with the residual's addition, the gated activation and the low-rank adapters against their definitions in 64 bits (oracle/ref.py), at the
sizes, values and ids where they can go wrong; their refusals; a block of them with the products, captured, on other streams, from several threads.

Tolerances.  Norm: fp32 sums of N squares, each lane a 64th of them or less and a tree: (N / 64 + 32) 2^-24 of the sum, half of that of its root, eight more
roundings; half a step of the output type on top.  The scale: as much and two roundings.  Codes: exact where the definition says so, otherwise
within half a code of y / S and what y is off.  Gated: its exponential is 2^(-g log2 e) in fp32, (|g| + 4) 2^-22 of the value.  Adapters: what the
oracle returns beside the value."""
import ctypes
import threading

import pytest
import torch

from helpers import DT, assert_bit_equal, gen
from oracle import ref
from tilelang_ascend_amd import _abi, ops

gpu = pytest.mark.gpu
TYPES = ["float16", "bfloat16"]


def norm_off(N):
    return ((N / 64 + 32) / 2 + 8) * 2.0**-24


def assert_near(got, want, off, what):
    """Within off and half a step of got's type, of the value or of its smallest normal number."""
    got = got.cpu()
    fi = torch.finfo(got.dtype)
    assert torch.isfinite(got).all(), what
    worst = ((got.double() - want).abs() - off - (want.abs() + off).clamp_min(fi.tiny) * (fi.eps / 2)).max().item()
    assert worst <= 0, f"{what}: {worst:.3e} more than allowed"


def check_codes(q, s, y, rel, what, round_scale=False, v=None):
    """Codes and scales of y [M, N] (64 bits, `rel` off): q exact where v is given and the scale is not the floor."""
    q, s = q.cpu(), s.cpu().double()
    want = ref.row_scales(y)
    if round_scale:
        # a power of two that covers the scale, and half of it does not (but for what the scale is off by)
        assert (torch.frexp(s).mantissa == 0.5).all(), what
        assert (s >= want * (1 - rel - 2.0**-22)).all() and (s / 2 < want * (1 + rel + 2.0**-22)).all(), what
    else:
        assert ((s - want).abs() <= want * (rel + 2.0**-22)).all(), what
    t = (y / s[:, None]).clamp(-127, 127)
    assert ((q.double() - t).abs() <= 0.5 + 127 * (rel + 2.0**-21)).all(), what
    if v is not None:
        above = y.abs().amax(1) > 1e-4 * (1 + 1e-5)
        assert torch.equal(q[above], ref.norm_codes(v[above])), f"{what}: codes"


def norm_inputs(M, N, dtype, seed, residual=True):
    g = gen(seed)
    x = torch.randn(M, N, generator=g).to(DT[dtype])
    r = (torch.randn(M, N, generator=g) * 4 * (1 + 20 * (torch.rand(N, generator=g) < 0.02))).to(DT[dtype]) if residual else None
    w = (torch.randn(N, generator=g) * 0.3 + 0.7).to(DT[dtype])
    return x, r, w


def run_norm(x, r, w, outputs, dtype, eps=1e-6, round_scale=False):
    """-> (H or None, Y or None, Q or None, S or None)."""
    kernel = ops.residual_rms_norm(x.shape[1], eps=eps, outputs=outputs, with_residual=r is not None, round_scale=round_scale, in_dtype=dtype)
    got = kernel(*[t.cuda() for t in (x, r, w) if t is not None])
    got = list(got) if isinstance(got, (list, tuple)) else [got]
    h = got.pop(0) if r is not None else None
    y = got.pop(0) if outputs != "int8" else None
    q, s = got if outputs != "float" else (None, None)
    return h, y, q, s


def check_norm(x, r, w, outputs, dtype, eps=1e-6, round_scale=False, what="norm"):
    h, y, q, s = run_norm(x, r, w, outputs, dtype, eps, round_scale)
    hw, yw, v = ref.residual_rms_norm(x, r, w, eps)
    rel = norm_off(x.shape[1])
    if h is not None:
        assert_bit_equal(h, hw, what + " h")
    if y is not None:
        assert y.dtype == DT[dtype]
        assert_near(y, yw, yw.abs() * rel, what + " y")
    if q is not None:
        assert q.dtype == torch.int8 and s.dtype == torch.float32
        check_codes(q, s, yw, rel, what, round_scale, None if round_scale else v)


# ---- the norm ---------------------------------------------------------------------------------------------------------------
# M, N: odd lengths, rows that end inside a chunk, a wavefront, a work-group; the longest kept in registers, and longer ones
NORM_SHAPES = [(1, 1), (3, 7), (1, 8), (5, 64), (2, 100), (7, 504), (4, 512), (9, 1000), (3, 1001), (33, 1024), (2, 2047), (6, 2048), (1, 3584), (5, 4096), (3, 4104), (1, 5120),
               (2, 8192), (2, 8200), (1, 11008), (2, 16384), (1, 16392), (2, 32768), (1, 32776), (1, 40003)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N", NORM_SHAPES)
def test_norm(M, N, dtype):
    x, r, w = norm_inputs(M, N, dtype, M * N)
    for outputs in ("float", "int8", "both"):
        check_norm(x, r, w, outputs, dtype, what=f"norm {M, N, outputs}")
    check_norm(x, None, w, "both", dtype, eps=1e-5, what=f"norm {M, N} without a residual")
    check_norm(x, r, w, "both", dtype, round_scale=True, what=f"norm {M, N} with power-of-two scales")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N", [(0, 64), (600, 256), (2300, 72), (5000, 128), (4200, 513), (1030, 2048), (300, 4096), (520, 5120)])
def test_norm_many_rows(M, N, dtype):
    x, r, w = norm_inputs(M, N, dtype, 5)
    h, y, q, s = run_norm(x, r, w, "both", dtype)
    assert y.shape == q.shape == (M, N) and s.shape == (M,)
    if M == 0:
        return
    hw, yw, _ = ref.residual_rms_norm(x, r, w, 1e-6)
    assert_bit_equal(h, hw)
    assert_near(y, yw, yw.abs() * norm_off(N), "y")
    check_codes(q, s, yw, norm_off(N), "codes")
    some = torch.randint(0, M, (5,), generator=gen(M))
    _, ys, vs = ref.residual_rms_norm(x[some], r[some], w, 1e-6)
    check_codes(q.cpu()[some], s.cpu()[some], ys, norm_off(N), "codes", v=vs)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [128, 129])
def test_norm_codes_in_the_middle_of_two(N, dtype):
    """Rows whose largest value is 127 units: n + 1/2 goes to the even code, a step of the type beside it to the nearer one."""
    T = DT[dtype]
    k = torch.arange(N) % 127
    row = (k + 0.5).to(T)
    row[-1] = 127.0
    step = torch.finfo(T).eps
    x = torch.stack([row, -row, (row.float() * (1 + step)).to(T), (row.float() * (1 - step)).to(T)])
    x[:, -1] = 127.0
    w = torch.ones(N, dtype=T)
    for scale in (1.0, 2.0**-7, 2.0**6):
        z = (x.float() * scale).to(T)
        check_norm(z, None, w, "int8", dtype, what="middles")
        _, _, q, _ = run_norm(z, None, w, "int8", dtype)
        assert q.cpu()[0, :8].tolist() == [0, 2, 2, 4, 4, 6, 6, 8]
    # products with weights of many bits: middles that only whole numbers of 22 bits tell apart
    g = gen(N)
    w = (1 + torch.rand(N, generator=g)).to(T)
    check_norm(torch.randn(60, N, generator=g).to(T), None, w, "int8", dtype, what="random products")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [64, 67, 4096])
def test_norm_rows_of_zeros_tiny_large_and_not_finite_values(N, dtype):
    T = DT[dtype]
    x, r, w = norm_inputs(9, N, dtype, 3)
    x[0] = 0
    r[0] = 0
    x[1], r[1] = torch.finfo(T).tiny, -torch.finfo(T).tiny
    x[2], r[2] = torch.finfo(T).tiny, 0
    x[3, N // 2] = float("inf")
    x[4, 5] = float("nan")
    x[5], r[5] = (60000.0, -59968.0) if T == torch.float16 else (1e15, -0.99e15)
    x[6, 1], r[6, 1] = float("inf"), float("-inf")
    w2 = w.clone()
    w2[7] = 0
    for weight in (w, w2):
        h, y, q, s = run_norm(x, r, weight, "both", dtype)
        fine = [0, 1, 2, 5, 7, 8]
        hw, yw, v = ref.residual_rms_norm(x[fine], r[fine], weight, 1e-6)
        assert_bit_equal(h[fine], hw)
        assert_near(y[fine], yw, yw.abs() * norm_off(N) + 2.0**-140, "y")
        check_codes(q[fine], s[fine], yw, norm_off(N), "codes", v=v)
        assert (q[0] == 0).all() and s[0].item() == torch.tensor(1e-4 / 127).item()
        y, q, s, h = y.cpu(), q.cpu(), s.cpu(), h.cpu()
        # an infinity: NaN there and 0 elsewhere; a NaN: the row
        assert torch.isinf(h[3, N // 2]) and torch.isnan(y[3, N // 2]) and (y[3, torch.arange(N) != N // 2] == 0).all()
        assert q[3, N // 2] == -127 and (q[3, torch.arange(N) != N // 2] == 0).all() and s[3] == s[0]
        assert torch.isnan(y[4]).all() and (q[4] == -127).all() and s[4] == s[0] and torch.isnan(y[6]).all()
    if T == torch.float16:  # the sum itself leaves the type
        h, y, _, _ = run_norm(torch.full((1, N), 60000.0, dtype=T), torch.full((1, N), 60000.0, dtype=T), w, "float", dtype)
        assert torch.isinf(h).all() and torch.isnan(y).all()


@gpu
@pytest.mark.parametrize("N,offset", [(256, 1), (256, 4), (2048, 3), (72, 8)])
def test_norm_of_tensors_that_begin_anywhere(N, offset):
    x, r, w = norm_inputs(6, N, "float16", 9)

    def put(t):
        return torch.cat([torch.zeros(offset, dtype=t.dtype), t.reshape(-1)]).cuda()[offset:].view(t.shape)

    h, y, q, s = ops.residual_rms_norm(N, outputs="both", in_dtype="float16")(put(x), put(r), put(w))
    hw, yw, v = ref.residual_rms_norm(x, r, w, 1e-6)
    assert_bit_equal(h, hw)
    assert_near(y, yw, yw.abs() * norm_off(N), "y")
    check_codes(q, s, yw, norm_off(N), "codes", v=v)


@gpu
@pytest.mark.parametrize("N", [320, 321, 4096, 8192])
def test_norm_in_place(N):
    """H over the residual, Y over X: the values of the call that writes elsewhere."""
    x, r, w = (t.cuda() for t in norm_inputs(40, N, "bfloat16", 4))
    h, y, q, s = ops.residual_rms_norm(N, outputs="both")(x, r, w)
    lib, P = _abi.load(), _abi.ptr
    q2, s2 = torch.empty_like(q), torch.empty_like(s)
    st = torch.cuda.current_stream().cuda_stream
    _abi.check(lib.tlq_residual_rms_norm(P(x), P(r), P(w), P(r), P(x), P(q2), P(s2), 40, N, 1e-6, _abi.BF16, 0, st))
    assert_bit_equal(r, h), assert_bit_equal(x, y), assert_bit_equal(q2, q), assert_bit_equal(s2, s)
    # H over X, codes alone
    x, r, w = (t.cuda() for t in norm_inputs(40, N, "bfloat16", 4))
    _abi.check(lib.tlq_residual_rms_norm(P(x), P(r), P(w), P(x), None, P(q2), P(s2), 40, N, 1e-6, _abi.BF16, 0, st))
    assert_bit_equal(x, h), assert_bit_equal(q2, q)


# ---- the gated activation -----------------------------------------------------------------------------------------------------
def gated_off(x, y):
    return (x.float().double().chunk(2, 1)[0].abs() + 4) * 2.0**-22 * y.abs()


def check_gated(x, outputs, dtype, round_scale=False, what="gated"):
    got = ops.gated_silu(x.shape[1] // 2, outputs=outputs, round_scale=round_scale, in_dtype=dtype)(x.cuda())
    got = list(got) if isinstance(got, (list, tuple)) else [got]
    want = ref.gated_silu(x)
    off = gated_off(x, want)
    if outputs != "int8":
        assert got[0].dtype == DT[dtype]
        assert_near(got[0], want, off, what)
    if outputs != "float":
        q, s = got[-2:]
        rel = (off / want.abs().clamp_min(1e-300)).max().item()
        check_codes(q, s, want, rel, what, round_scale)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N", [(0, 64), (1, 1), (3, 7), (1, 8), (5, 64), (2, 100), (70, 512), (9, 1001), (3, 2048), (2, 4104), (1, 8192), (2, 11008), (1, 14336), (3, 16384), (1, 16392), (1, 32768),
                                 (1, 32776), (600, 256), (2300, 72), (5000, 128), (4200, 129), (1030, 2048)])
def test_gated(M, N, dtype):
    x = (torch.randn(M, 2 * N, generator=gen(M * N)) * 2).to(DT[dtype])
    if M == 0:
        y, q, s = ops.gated_silu(N, outputs="both", in_dtype=dtype)(x.cuda())
        assert y.shape == q.shape == (0, N) and s.shape == (0,)
        return
    for outputs in ("float", "int8", "both"):
        check_gated(x, outputs, dtype, what=f"gated {M, N, outputs}")
    check_gated(x, "both", dtype, round_scale=True, what=f"gated {M, N} with power-of-two scales")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [64, 61, 4096])
def test_gated_far_gates_and_not_finite_values(N, dtype):
    """Gates from where exp(-g) leaves fp32, and further; infinities and NaN stay in their place, and a row's scale is that of its other values."""
    T, inf, nan = DT[dtype], float("inf"), float("nan")
    x = torch.randn(6, 2 * N, generator=gen(1))
    far = torch.tensor([-79.0, -80.0, -81.0, -86.5, -87.5, -88.0, -89.0, -95.0, -103.0, -104.0, -120.0, -150.0, -300.0, 30.0, 88.0, 89.0, 1000.0])
    x[0, : len(far)], x[0, N: N + len(far)] = far, 50.0
    x[1] = 0
    x[2, :N] = -100.0
    x = x.to(T)
    want = ref.gated_silu(x)
    y, q, s = ops.gated_silu(N, outputs="both", in_dtype=dtype)(x.cuda())
    # (below the type's normal numbers half a step is that of the smallest normal one; an exponential there may also be flushed to 0 by half of that)
    assert_near(y, want, gated_off(x, want) + torch.finfo(torch.float32).tiny, "far gates")
    rel = (103 + 4) * 2.0**-22
    check_codes(q, s, want, rel, "far gates")
    assert (q[1] == 0).all()
    x[3, 2], x[3, 5], x[3, N + 7], x[4, 0], x[5, 1] = inf, -inf, inf, nan, inf
    x[5, N + 1] = 0
    y, q, s = (t.cpu() for t in ops.gated_silu(N, outputs="both", in_dtype=dtype)(x.cuda()))
    want = ref.gated_silu(x)
    at = torch.isfinite(want)
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y[torch.isinf(want)].double(), want[torch.isinf(want)])
    assert_near(y[at], want[at], gated_off(x, want)[at] + torch.finfo(torch.float32).tiny, "beside")
    assert (q[torch.isnan(want)] == -127).all()
    # an infinity: its row's scale, -127 in its place and 0 elsewhere
    assert torch.isinf(s[3]) and (q[3][torch.isinf(want[3]) | torch.isnan(want[3])] == -127).all() and (q[3][at[3]] == 0).all() and torch.isinf(want[3]).any()
    for m in (4, 5):  # NaN alone: the scale of the others
        rest = torch.where(at[m], want[m], 0.0)
        check_codes(torch.where(at[m], q[m], 0)[None], s[m: m + 1], rest[None], rel, "beside NaN")


@gpu
@pytest.mark.parametrize("N,offset", [(256, 1), (2048, 4), (72, 8)])
def test_gated_of_tensors_that_begin_anywhere(N, offset):
    x = torch.randn(6, 2 * N, generator=gen(N)).half()
    there = torch.cat([torch.zeros(offset, dtype=x.dtype), x.reshape(-1)]).cuda()[offset:].view(x.shape)
    y, q, s = ops.gated_silu(N, outputs="both", in_dtype="float16")(there)
    want = ref.gated_silu(x)
    assert_near(y, want, gated_off(x, want), "y")
    check_codes(q, s, want, 12 * 2.0**-22, "codes")


# ---- the adapters ---------------------------------------------------------------------------------------------------------------
def make_update(M, L, rank, parts, K, dtype, kind, seed, out="same"):
    T, g = DT[dtype], gen(seed)
    N = sum(parts)
    x = torch.randn(M, K, generator=g).to(T)
    y = torch.randn(M, N, generator=g).to(T if out == "same" else torch.float32)
    a = (torch.randn(L, len(parts) * rank, K, generator=g) * K**-0.5).to(T)
    b = (torch.randn(L, N, rank, generator=g) * 0.3).to(T)
    scaling = torch.rand(L, generator=g) * 2 - 0.5
    ids = torch.randint(0, L, (M,), generator=g, dtype=torch.int32)
    if kind == "one":
        ids.fill_(L - 1)
    elif kind == "runs":
        ids = ids.sort().values
    elif kind == "none":
        ids.fill_(-1)
    elif kind == "holes":
        odd = torch.tensor([-1, L, 2**31 - 1, -(2**31), -7], dtype=torch.int32)
        holes = torch.rand(M, generator=g) < 0.4
        ids[holes] = odd[torch.randint(0, 5, (int(holes.sum()),), generator=g)]
        x[(ids < 0) | (ids >= L)] = float("nan")  # nothing of such a row is looked at
    return x, y, ids, a, b, scaling


def update_kernel(L, rank, parts, K, dtype, out="same"):
    return ops.low_rank_update(L, rank, parts if len(parts) > 1 else parts[0], K, in_dtype=dtype, out_dtype=dtype if out == "same" else "float32")


def check_update(M, L, rank, parts, K, dtype, kind, seed=1, out="same"):
    t = make_update(M, L, rank, parts, K, dtype, kind, seed, out)
    got = update_kernel(L, rank, parts, K, dtype, out)(*[v.cuda() for v in t])
    assert got.dtype == t[1].dtype and got.shape == t[1].shape
    want, off = ref.low_rank_update(*t, parts)
    assert_near(got, want, off, f"update {M, L, rank, parts, K, dtype, kind}")
    without = (t[2] < 0) | (t[2] >= L)
    assert_bit_equal(got.cpu()[without], t[1][without], "rows without an adapter")
    return t, got


# M, L, rank, parts, K, ids
UPDATES = [
    (1, 1, 8, (16,), 32, "one"), (1, 3, 16, (64,), 64, "spread"), (2, 5, 32, (48,), 96, "spread"), (1, 8, 16, (4096,), 4096, "spread"), (3, 2, 64, (80, 16, 32), 160, "holes"),
    (1, 2, 128, (128, 128), 512, "one"), (5, 4, 8, (16, 16, 16), 288, "spread"), (16, 3, 16, (272,), 2048, "holes"), (17, 1, 16, (112,), 544, "one"), (33, 40, 8, (256, 64, 64), 1056, "spread"),
    (64, 7, 32, (160, 96), 1024, "holes"), (65, 2, 64, (64,), 4128, "runs"), (100, 100, 16, (208,), 256, "spread"), (130, 4, 128, (96,), 320, "holes"), (255, 3, 8, (64, 48), 128, "spread"),
    (256, 9, 16, (1040,), 96, "holes"), (257, 1, 32, (80,), 224, "one"), (300, 5, 64, (336, 16, 16), 416, "runs"), (40, 3, 16, (16,), 256, "none"), (700, 600, 8, (32,), 64, "spread"),
    (1030, 4, 16, (144,), 192, "runs"), (1100, 3, 128, (80, 48), 160, "holes"), (1500, 2, 32, (1088,), 64, "one"), (2, 4096, 8, (32,), 32, "spread"), (9, 2, 16, (32,), 16416, "spread"),
    (513, 2, 8, (16,), 8224, "holes"), (1025, 1025, 16, (48,), 32, "spread"), (600, 3, 16, (64,), 64, "none"),
    # (tiles of 64 rows: the first product in runs of 16, and by whole tiles)
    (1700, 2, 64, (80,), 416, "runs"), (900, 7, 128, (32,), 1120, "holes"), (2600, 3, 64, (48,), 352, "holes"), (5300, 2, 32, (32,), 288, "spread"), (10300, 2, 16, (16,), 160, "runs"),
    # (tiles of 16 rows: sizes beyond what single rows are for)
    (1, 1, 8, (16,), 16416, "one"), (3, 2, 64, (80, 16, 32), 2080, "holes"), (17, 1, 16, (112,), 8224, "one"), (33, 40, 8, (256, 64, 64), 16416, "spread"), (64, 1, 32, (48,), 4128, "one"),
    (63, 9, 128, (96, 32), 1056, "spread"), (40, 3, 16, (16,), 8224, "none"), (2, 4096, 16, (32,), 8224, "spread"), (100, 100, 16, (208,), 8224, "spread"), (700, 600, 32, (32,), 352, "spread"),
    # (single rows: every rank, runs of more than one block, K that ends inside of a stage)
    (1, 2, 64, (2000,), 2048, "spread"), (1, 3, 128, (48, 4096, 16), 992, "holes"), (16, 16, 32, (4112, 32), 1120, "spread"), (2, 2, 32, (22016, 16), 4096, "runs"), (600, 40, 8, (16, 1040), 736, "holes"),
    (64, 5, 8, (8208, 48), 2080, "spread"), (9, 2, 8, (528,), 16384, "spread"),
    # (longer rows, for tiles again)
    (1, 1, 8, (16,), 32800, "one"), (3, 2, 64, (80, 16, 32), 4128, "holes"), (17, 1, 16, (112,), 16416, "one"), (33, 40, 8, (256, 64, 64), 32800, "spread"), (64, 1, 32, (48,), 8224, "one"),
    (63, 9, 128, (96, 32), 2080, "spread"), (40, 3, 16, (16,), 16416, "none"), (5, 300, 32, (32,), 8224, "spread"), (100, 100, 16, (208,), 16416, "spread"), (700, 600, 64, (32,), 352, "spread"),
    # (single rows that have more than four blocks of outputs each)
    (60, 7, 16, (22016,), 96, "holes"), (4096, 9, 8, (272,), 64, "spread"), (200, 3, 32, (2048, 48), 1504, "runs"), (2, 2, 64, (4112, 16), 1952, "holes"),
]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,L,rank,parts,K,kind", UPDATES)
def test_update(M, L, rank, parts, K, kind, dtype):
    check_update(M, L, rank, parts, K, dtype, kind)
    check_update(M, L, rank, parts, K, dtype, kind, seed=2, out="float32")


@gpu
@pytest.mark.parametrize("M,L,rank,parts,K,kind", [(8192, 3, 8, (48,), 64, "runs"), (8193, 4, 16, (32, 16), 32, "holes"), (9001, 700, 8, (32,), 64, "spread"), (20000, 2, 8, (16,), 32, "one"),
                                                   (70001, 5, 8, (16,), 32, "runs"), (33000, 4096, 8, (16,), 32, "holes"),
                                                   (8192, 3, 32, (48,), 64, "runs"), (8193, 4, 32, (32, 16), 32, "holes"), (9001, 700, 32, (32,), 64, "spread"), (20000, 2, 16, (16,), 64, "one"),
                                                   (33000, 4096, 16, (16,), 32, "holes")])
def test_update_many_rows(M, L, rank, parts, K, kind):
    t = make_update(M, L, rank, parts, K, "bfloat16", kind, 3)
    got = update_kernel(L, rank, parts, K, "bfloat16")(*[v.cuda() for v in t]).cpu()
    some = torch.cat([torch.tensor([0, 1, 63, 64, M - 2, M - 1]), torch.randint(0, M, (300,), generator=gen(M))])
    want, off = ref.low_rank_update(*[v[some] for v in t[:3]], *t[3:], parts)
    assert_near(got[some], want, off, "many rows")
    # all of them, in fp32 (the sums of both sides are off by what the oracle allows at most)
    x, y, ids, a, b, s = t
    begin, whole = 0, y.float().clone()
    for e in torch.unique(ids).tolist():
        if 0 <= e < L:
            at = ids == e
            h = x[at].float() @ a[e].float().T
            for p, n in enumerate(parts):
                begin = sum(parts[:p])
                whole[at, begin: begin + n] += s[e] * (h[:, p * rank: (p + 1) * rank] @ b[e, begin: begin + n].float().T)
    assert ((got.float() - whole).abs() <= 2.0**-8 * whole.abs() + 2.0**-10).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,rank,K", [(4, 16, 128), (70, 16, 128), (400, 16, 128), (4, 32, 4128), (70, 32, 4128), (800, 64, 2080), (4, 32, 8224), (70, 32, 8224), (900, 64, 4128)])
def test_update_large_and_small_values(M, rank, K, dtype):
    """First sums far outside float16's range, and far below its normal numbers, that the second product brings back."""
    parts, L = (64,), 3
    x, y, ids, a, b, scaling = make_update(M, L, rank, parts, K, "float16", "spread", 5)
    T = DT[dtype]
    a[0] = (a[0].float() * 2000).half()
    x[ids == 0] = (x[ids == 0].float() * 500).half()  # h near 10^6 and above
    b[0] = (b[0].float() * 1e-4).half()
    a[1] = (a[1].float() * 2e-3).half()
    x[ids == 1] = (x[ids == 1].float() * 1e-3).half()  # h near 10^-6
    scaling[0], scaling[1] = 1e-2, 3e4
    t = [v.to(T) if v.dtype == torch.float16 else v for v in (x, y, ids, a, b, scaling)]
    got = update_kernel(L, rank, parts, K, dtype, "same")(*[v.cuda() for v in t])
    want, off = ref.low_rank_update(*t, parts)
    assert_near(got, want, off, "far values")


@gpu
@pytest.mark.parametrize("M,rank,K", [(300, 16, 512), (300, 64, 2080), (420, 128, 1056), (60, 32, 4128), (300, 64, 4128), (60, 32, 8224)])
def test_update_rows_do_not_depend_on_each_other(M, rank, K):
    """A row alone, in a small batch, in a large one, beside rows of NaN: the values that it has by itself, but for sums formed in another order."""
    L, parts = 6, (96, 32)
    t = make_update(M, L, rank, parts, K, "bfloat16", "spread", 8)
    kernel = update_kernel(L, rank, parts, K, "bfloat16")
    gpu_t = [v.cuda() for v in t]
    whole = kernel(*gpu_t)
    bad = gpu_t[0].clone()
    bad[::3] = float("nan")
    beside = kernel(bad, *gpu_t[1:])
    keep = torch.arange(M) % 3 != 0
    assert_bit_equal(beside.cpu()[keep], whole.cpu()[keep], "beside NaN")
    want, off = ref.low_rank_update(*t, parts)
    for rows in (slice(7, 8), slice(40, 57), slice(0, 100)):
        assert_near(kernel(*[v[rows].contiguous() for v in gpu_t[:3]], *gpu_t[3:]), want[rows], off[rows], "alone")
    # an adapter that is NaN reaches its own rows only
    a = gpu_t[3].clone()
    a[2] = float("nan")
    other = kernel(*gpu_t[:3], a, *gpu_t[4:])
    keep = t[2] != 2
    assert_bit_equal(other.cpu()[keep], whole.cpu()[keep], "beside an adapter of NaN")
    assert torch.isnan(other.cpu()[~keep]).all()
    # the order of the rows
    perm = torch.randperm(M, generator=gen(2)).cuda()
    moved = kernel(*[v[perm].contiguous() for v in gpu_t[:3]], *gpu_t[3:])
    assert_bit_equal(moved, whole[perm], "rows in another order")
    for _ in range(3):
        assert_bit_equal(kernel(*gpu_t), whole, "again")


@gpu
def test_update_of_no_row():
    t = make_update(0, 3, 16, (64,), 32, "float16", "one", 1)
    assert update_kernel(3, 16, (64,), 32, "float16")(*[v.cuda() for v in t]).shape == (0, 64)


@gpu
@pytest.mark.parametrize("M,rank,K", [(20, 32, 256), (400, 32, 256), (20, 32, 4128), (900, 64, 288), (20, 32, 8224), (400, 32, 8224)])
def test_update_in_place_and_nothing_beside_its_outputs(M, rank, K):
    L, parts = 4, (80, 16)
    N = sum(parts)
    t = [v.cuda() for v in make_update(M, L, rank, parts, K, "float16", "holes", 3)]
    want = update_kernel(L, rank, parts, K, "float16")(*t)
    lib, P = _abi.load(), _abi.ptr
    bytes_ = lib.tlq_low_rank_update_workspace_bytes(M, L, rank, 2, K)
    ws = torch.full((bytes_ + 512,), 77, dtype=torch.uint8, device="cuda")
    around = torch.full((M * N + 256,), 3.0, dtype=torch.float16, device="cuda")
    y = around[128:-128].view(M, N)
    y.copy_(t[1])
    st = torch.cuda.current_stream().cuda_stream
    _abi.check(lib.tlq_low_rank_update(P(t[0]), P(y), P(t[2]), P(t[3]), P(t[4]), P(t[5]), P(y), P(ws[256:]), bytes_, M, L, rank, *parts, 0, K, _abi.F16, _abi.F16, st))
    assert_bit_equal(y, want, "in place")
    assert (around[:128] == 3).all() and (around[-128:] == 3).all() and (ws[:256] == 77).all() and (ws[256 + bytes_:] == 77).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,times", [(5, 0), (90, 0), (5, 1), (90, 1), (5, 3), (90, 3)])
def test_update_infinities_stay_infinities(M, times, dtype):
    """An infinity among the activations, beside weights of one sign: the row is infinite, the others are what they were."""
    K = 64 + times * 8160  # (the longer rows: for tiles)
    t = list(make_update(M, 2, 16, (64,), K, dtype, "one", 4))
    t[3], t[4], t[5] = t[3].abs() + 0.01, t[4].abs() + 0.01, t[5].abs() + 0.1
    x = t[0].clone()
    x[1, 3] = float("inf")
    kernel = update_kernel(2, 16, (64,), K, dtype)
    rest = [v.cuda() for v in t[1:]]
    got, was = kernel(x.cuda(), *rest).cpu(), kernel(t[0].cuda(), *rest).cpu()
    assert (got[1] == float("inf")).all()
    keep = torch.arange(M) != 1
    assert_bit_equal(got[keep], was[keep])
    # an infinite weight in some places of a row of B: that output alone (an infinity, or NaN)
    for rank in (8, 16, 32, 64):
        K = 64 + times * (131072 // rank)
        t = make_update(M, 2, rank, (64,), K, dtype, "one", 4)
        kernel = update_kernel(2, rank, (64,), K, dtype)
        was = kernel(*[v.cuda() for v in t]).cpu()
        for j in range(0, rank, 5):
            b = t[4].clone()
            b[1, 9, j] = float("inf")
            got = kernel(*[v.cuda() for v in (*t[:4], b, t[5])]).cpu()
            assert not torch.isfinite(got[:, 9]).any()
            keep = torch.arange(64) != 9
            assert_bit_equal(got[:, keep], was[:, keep])


@gpu
def test_update_offsets_beyond_32_bits():
    """Adapters whose matrices lie more than 4 GiB behind the first."""
    L, rank, K, N = 1200, 64, 14336, 14336
    T = torch.float16
    g = torch.Generator(device="cuda").manual_seed(1)
    a = torch.zeros(L, 2 * rank, K, dtype=T, device="cuda")
    b = torch.zeros(L, 2 * N, rank, dtype=T, device="cuda")
    assert (L - 1) * 2 * rank * K * 2 > 2**32 and (L - 1) * 2 * N * rank * 2 > 2**32
    for e in (0, L - 1):
        a[e] = (torch.randn(2 * rank, K, generator=g, device="cuda") * K**-0.5).to(T)
        b[e] = (torch.randn(2 * N, rank, generator=g, device="cuda") * 0.2).to(T)
    scaling = torch.ones(L, device="cuda")
    for M in (3, 300):
        x = torch.randn(M, K, generator=g, device="cuda").to(T)
        y = torch.randn(M, 2 * N, generator=g, device="cuda").to(T)
        ids = torch.where(torch.arange(M, device="cuda") % 2 == 0, L - 1, 0).to(torch.int32)
        got = ops.low_rank_update(L, rank, (N, N), K)(x, y, ids, a, b, scaling)
        rows = [0, 1, M - 1]
        want, off = ref.low_rank_update(x[rows], y[rows], ids[rows] // (L - 1), torch.stack([a[0], a[L - 1]]), torch.stack([b[0], b[L - 1]]), scaling[:2], (N, N))
        assert_near(got[rows], want, off, "far adapters")


@gpu
def test_update_single_rows_offsets_beyond_32_bits():
    L, rank, K, N = 4096, 64, 2048, 2752
    g = torch.Generator(device="cuda").manual_seed(2)
    a = torch.zeros(L, 3 * rank, K, dtype=torch.bfloat16, device="cuda")
    b = torch.zeros(L, 3 * N, rank, dtype=torch.bfloat16, device="cuda")
    assert (L - 1) * 3 * rank * K * 2 > 2**31 and (L - 1) * 3 * N * rank * 2 > 2**32
    a[L - 1] = (torch.randn(3 * rank, K, generator=g, device="cuda") * K**-0.5).to(torch.bfloat16)
    b[L - 1] = (torch.randn(3 * N, rank, generator=g, device="cuda") * 0.2).to(torch.bfloat16)
    x, y = torch.randn(2, K, generator=g, device="cuda").to(torch.bfloat16), torch.randn(2, 3 * N, generator=g, device="cuda").to(torch.bfloat16)
    ids = torch.tensor([L - 1, 0], dtype=torch.int32, device="cuda")
    got = ops.low_rank_update(L, rank, (N, N, N), K, in_dtype="bfloat16")(x, y, ids, a, b, torch.ones(L, device="cuda"))
    want, off = ref.low_rank_update(x[:1], y[:1], torch.zeros(1, dtype=torch.int32), a[L - 1:], b[L - 1:], torch.ones(1), (N, N, N))
    assert_near(got[:1], want, off, "far adapter")
    assert_bit_equal(got[1], y[1], "an adapter of zeros")


# ---- together ---------------------------------------------------------------------------------------------------------------------
def make_block(M, hidden, inner, L, rank, dtype, seed):
    """A block's MLP with int8 weights and adapters on both products, as a function of (x, residual, ids)."""
    T, g = DT[dtype], gen(seed)
    w = (torch.randn(hidden, generator=g) * 0.2 + 0.8).to(T).cuda()
    w1 = torch.randint(-90, 91, (2 * inner, hidden), dtype=torch.int8, generator=g).cuda()
    w2 = torch.randint(-90, 91, (hidden, inner), dtype=torch.int8, generator=g).cuda()
    s1 = (torch.rand(2 * inner, generator=g) * 4e-4 + 1e-4).cuda()
    s2 = (torch.rand(hidden, generator=g) * 4e-4 + 1e-4).cuda()
    a1, b1 = ((torch.randn(L, 2 * rank, hidden, generator=g) * hidden**-0.5).to(T).cuda(), (torch.randn(L, 2 * inner, rank, generator=g) * 0.2).to(T).cuda())
    a2, b2 = ((torch.randn(L, rank, inner, generator=g) * inner**-0.5).to(T).cuda(), (torch.randn(L, hidden, rank, generator=g) * 0.2).to(T).cuda())
    scaling = (torch.rand(L, generator=g) + 0.5).cuda()
    norm = ops.residual_rms_norm(hidden, outputs="both", in_dtype=dtype)
    product1 = ops.int8_gemm_kernel_corrected(2 * inner, hidden, out_dtype=dtype)
    update1 = ops.low_rank_update(L, rank, (inner, inner), hidden, in_dtype=dtype)
    act = ops.gated_silu(inner, outputs="both", in_dtype=dtype)
    product2 = ops.int8_gemm_kernel_corrected(hidden, inner, out_dtype=dtype)
    update2 = ops.low_rank_update(L, rank, hidden, inner, in_dtype=dtype)

    def steps(x, residual, ids):
        h, y, q, s = norm(x, residual, w)
        p1 = product1(q, w1, s, s1)
        u1 = update1(y, p1, ids, a1, b1, scaling)
        z, q2, t = act(u1)
        p2 = product2(q2, w2, t, s2)
        return {"h": h, "y": y, "q": q, "s": s, "p1": p1, "u1": u1, "z": z, "q2": q2, "t": t, "p2": p2, "u2": update2(z, p2, ids, a2, b2, scaling)}

    def check(x, residual, ids, got):
        c = {k: v.cpu() for k, v in got.items()}
        hw, yw, _ = ref.residual_rms_norm(x, residual, w, 1e-6)
        assert_bit_equal(c["h"], hw)
        assert_near(c["y"], yw, yw.abs() * norm_off(hidden), "y")
        check_codes(c["q"], c["s"], yw, norm_off(hidden), "q")
        assert_bit_equal(c["p1"], ref.ref_int8_gemm_sequential(c["q"], w1.cpu(), c["s"], s1.cpu(), T))
        want, off = ref.low_rank_update(got["y"], got["p1"], ids, a1, b1, scaling, (inner, inner))
        assert_near(c["u1"], want, off, "u1")
        zw = ref.gated_silu(c["u1"])
        assert_near(c["z"], zw, gated_off(c["u1"], zw), "z")
        assert_bit_equal(c["p2"], ref.ref_int8_gemm_sequential(c["q2"], w2.cpu(), c["t"], s2.cpu(), T))
        want, off = ref.low_rank_update(got["z"], got["p2"], ids, a2, b2, scaling, (hidden,))
        assert_near(c["u2"], want, off, "u2")

    return steps, check


def block_inputs(M, hidden, L, dtype, seed):
    g = gen(seed)
    x, r = (torch.randn(M, hidden, generator=g).to(DT[dtype]).cuda() for _ in range(2))
    return x, r, torch.randint(-1, L, (M,), generator=g, dtype=torch.int32).cuda()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,rank", [(1, 16), (21, 16), (300, 16), (21, 128), (60, 128), (300, 128), (500, 128)])
def test_a_block_of_them(M, rank, dtype):
    steps, check = make_block(M, 256, 384, 5, rank, dtype, 1)
    x, r, ids = block_inputs(M, 256, 5, dtype, 2)
    check(x, r, ids, steps(x, r, ids))


@gpu
@pytest.mark.parametrize("M,rank", [(4, 16), (300, 16), (21, 128), (60, 128), (500, 128)])
def test_a_block_captured_and_replayed(M, rank):
    """Two graphs of the same weights, with eager calls between their replays and new inputs for each."""
    steps, _ = make_block(M, 256, 384, 5, rank, "bfloat16", 1)
    graphs = []
    for seed in (3, 4):
        ins = block_inputs(M, 256, 5, "bfloat16", seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            steps(*ins)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = steps(*ins)
        graphs.append((g, ins, outs))
    for k in range(4):
        for i, (g, ins, outs) in enumerate(graphs):
            for a, b in zip(ins, block_inputs(M, 256, 5, "bfloat16", 10 * k + i)):
                a.copy_(b)
            g.replay()
            want = steps(*ins)
            torch.cuda.synchronize()
            for name in want:
                assert_bit_equal(outs[name], want[name], f"replay {k} of graph {i}: {name}")


@gpu
@pytest.mark.parametrize("rank", [16, 128])
def test_on_other_streams_and_from_several_threads(rank):
    steps, _ = make_block(30, 256, 384, 5, rank, "float16", 1)
    ins = [block_inputs(M, 256, 5, "float16", M) for M in (30, 1, 280, 64)]
    want = [steps(*i) for i in ins]
    torch.cuda.synchronize()
    failed = []

    def work(n):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    got = steps(*ins[n])
            stream.synchronize()
            for name in got:
                assert_bit_equal(got[name], want[n][name], name)
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    # an explicit stream
    x, r, ids = ins[0]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    t = make_update(30, 3, 16, (64,), 128, "float16", "spread", 1)
    kernel = update_kernel(3, 16, (64,), 128, "float16")
    on_gpu = [v.cuda() for v in t]
    torch.cuda.synchronize()
    other = kernel(*on_gpu, stream=stream.cuda_stream)
    stream.synchronize()
    assert_bit_equal(other, kernel(*on_gpu))


# ---- refusals ---------------------------------------------------------------------------------------------------------------------
def test_factories_refuse():
    for bad in ({"outputs": "fp8"}, {"eps": 0.0}, {"eps": 2.0}, {"in_dtype": "float32"}, {"outputs": None}, {"eps": float("nan")}):
        with pytest.raises(ValueError):
            ops.residual_rms_norm(64, **bad)
    for bad in ({"outputs": ""}, {"in_dtype": "int8"}):
        with pytest.raises(ValueError):
            ops.gated_silu(64, **bad)
    for n in (0, -8, 1 << 30):
        with pytest.raises(ValueError):
            ops.residual_rms_norm(n)
        with pytest.raises(ValueError):
            ops.gated_silu(n)
    for args in ((0, 16, 64, 64), (4097, 16, 64, 64), (4, 12, 64, 64), (4, 256, 64, 64), (4, 16, 60, 64), (4, 16, 0, 64), (4, 16, (64, 0), 64), (4, 16, (64, 64, 64, 64), 64), (4, 16, (), 64),
                 (4, 16, 64, 48), (4, 16, 64, 0), (4, 16, 1 << 24, 64), (4, 16, 64, 1 << 24)):
        with pytest.raises(ValueError):
            ops.low_rank_update(*args)
    for kw in ({"in_dtype": "float32"}, {"in_dtype": "float16", "out_dtype": "bfloat16"}, {"out_dtype": "int8"}):
        with pytest.raises(ValueError):
            ops.low_rank_update(4, 16, 64, 64, **kw)


def test_kernels_name_what_is_wrong_with_a_call():
    norm, gated, update = ops.residual_rms_norm(64, outputs="both"), ops.gated_silu(64), ops.low_rank_update(4, 16, 64, 32)
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="Expected 3 inputs"):
        norm(x, x)
    with pytest.raises(ValueError, match="dtype mismatch"):
        norm(x, x.half(), x[0].clone())
    with pytest.raises(ValueError, match="mismatch"):
        gated(x)
    with pytest.raises(ValueError, match="must be contiguous"):
        gated(torch.zeros(128, 2, dtype=torch.bfloat16).T)
    with pytest.raises(ValueError, match="mismatch"):
        update(torch.zeros(2, 32).half(), torch.zeros(3, 64).half(), torch.zeros(2, dtype=torch.int32), torch.zeros(4, 16, 32).half(), torch.zeros(4, 64, 16).half(), torch.ones(4))
    with pytest.raises(ValueError, match="dtype mismatch"):
        update(torch.zeros(2, 32).half(), torch.zeros(2, 64).half(), torch.zeros(2, dtype=torch.int64), torch.zeros(4, 16, 32).half(), torch.zeros(4, 64, 16).half(), torch.ones(4))


P16 = ctypes.c_void_p(16)
NORM_OK = dict(X=P16, residual=P16, weight=P16, H=P16, Y=P16, Q=P16, S=P16, M=4, N=64, eps=1e-6, dtype=_abi.F16, round_scale=0, stream=None)


@pytest.mark.parametrize("change,message", [
    ({"M": -1}, "bad shape"), ({"N": 0}, "bad shape"), ({"N": 1 << 30}, "bad shape"), ({"dtype": _abi.F32}, "dtype"), ({"eps": 0.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"eps": 1.5}, "eps"),
    ({"X": None}, "null"), ({"weight": None}, "null"), ({"H": None}, "wanted together"), ({"residual": None}, "wanted together"), ({"Q": None}, "wanted together"), ({"S": None}, "wanted together"),
    ({"Y": None, "Q": None, "S": None}, "an output is wanted"), ({"X": ctypes.c_void_p(17)}, "misaligned"), ({"S": ctypes.c_void_p(18)}, "misaligned"), ({"Y": ctypes.c_void_p(17)}, "misaligned")])
def test_norm_entry_refuses(change, message):
    args = {**NORM_OK, **change}
    assert _abi.load().tlq_residual_rms_norm(*args.values()) != 0
    assert message in _abi.last_error()


@pytest.mark.parametrize("change,message", [({"M": -1}, "bad shape"), ({"N": -5}, "bad shape"), ({"dtype": 7}, "dtype"), ({"X": None}, "null"), ({"X": ctypes.c_void_p(3)}, "misaligned"),
                                            ({"Q": P16}, "wanted together"), ({"Y": None}, "an output")])
def test_gated_entry_refuses(change, message):
    args = {**dict(X=P16, Y=P16, Q=None, S=None, M=4, N=64, dtype=_abi.BF16, round_scale=0, stream=None), **change}
    assert _abi.load().tlq_gated_silu(*args.values()) != 0
    assert message in _abi.last_error()


UPDATE_OK = dict(X=P16, Y=P16, ids=P16, A=P16, B=P16, scaling=P16, out=P16, ws=P16, ws_bytes=1 << 30, M=4, L=4, rank=16, n0=64, n1=0, n2=0, K=64, in_dtype=_abi.F16, out_dtype=_abi.F16, stream=None)


@pytest.mark.parametrize("change,message", [
    ({"M": -1}, "bad shape"), ({"M": 1 << 24}, "bad shape"), ({"L": 0}, "bad shape"), ({"L": 4097}, "bad shape"), ({"rank": 24}, "bad shape"), ({"K": 48}, "bad shape"), ({"K": 0}, "bad shape"),
    ({"n0": 0}, "parts"), ({"n0": 24}, "parts"), ({"n2": 16}, "parts"), ({"n1": -16}, "parts"), ({"n1": 1 << 24}, "parts"), ({"in_dtype": _abi.F32}, "in_dtype"), ({"out_dtype": _abi.BF16}, "out_dtype"),
    ({"X": None}, "null"), ({"out": None}, "null"), ({"scaling": None}, "null"), ({"A": ctypes.c_void_p(24)}, "aligned"), ({"ids": ctypes.c_void_p(18)}, "aligned"), ({"ws": None}, "workspace"),
    ({"ws_bytes": 16}, "workspace"), ({"ws": ctypes.c_void_p(8)}, "workspace")])
def test_update_entry_refuses(change, message):
    args = {**UPDATE_OK, **change}
    assert _abi.load().tlq_low_rank_update(*args.values()) != 0
    assert message in _abi.last_error()


def test_update_workspace_sizes():
    size = _abi.load().tlq_low_rank_update_workspace_bytes
    assert size(4, 4, 24, 1, 64) == 0 and size(4, 4, 16, 4, 64) == 0 and size(-1, 4, 16, 1, 64) == 0 and size(4, 0, 16, 1, 64) == 0 and size(4, 4, 16, 1, 0) == 0
    for L, rank, parts, K in ((1, 8, 1, 32), (8, 16, 3, 4096), (300, 64, 2, 11008), (4096, 128, 3, 64)):
        last = 0
        for M in (0, 1, 2, 15, 16, 17, 63, 64, 65, 200, 255, 256, 257, 300, 511, 512, 513, 1000, 1023, 1024, 1025, 4096, 8192, 70000, 1000000):
            bytes_ = size(M, L, rank, parts, K)
            assert bytes_ >= last, (M, L, rank, parts, K)
            last = bytes_
