"""The kernels of the experts' products: which one a call runs on (asked for on the host), and calls that reach the corners of each.

Tolerances are those of test_moe.py: what the fp32 sums may be off by, which the oracle returns beside the value, plus half a step of the
output type."""
import ctypes

import pytest
import torch

from helpers import DT, assert_bit_equal, gen
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


def run_both(up, M, E, k, N, K, group, dtype, zeros, kind, out="float32", seed=20, some=None):
    """One product against the oracle (in the rows `some`, or all); returns the output on the CPU."""
    T = DT[dtype]
    ids = make_ids(M, E, k, kind, seed)
    Wp, s, z = make_experts(E, 2 * N if up else N, K, group, T, zeros, seed + 1)
    at = torch.arange(M) if some is None else torch.tensor(some)
    if up:
        X = torch.randn(M, K, generator=gen(seed + 2)).to(T)
        got = ops.moe_gate_up_w4a16(E, k, N, K, group, dtype, zeros=kernel_zeros(z))(*operands(X, ids, Wp, s, z))
        want, off = ref.moe_gate_up(X[at], ids[at], Wp, s, z, group)
    else:
        H = torch.randn(M, k, K, generator=gen(seed + 2)).to(T)
        weights = torch.softmax(torch.randn(M, k, generator=gen(seed + 3)), 1)
        got = ops.moe_down_w4a16(E, k, N, K, group, dtype, out, zeros=kernel_zeros(z))(*operands(H, ids, weights, Wp, s, z))
        want, off = ref.moe_down(H[at], ids[at], weights[at], Wp, s, z, group)
    assert_close64(got.cpu()[at], want, off, f"{'gate_up' if up else 'down'} {M, E, k, N, K, group, dtype, zeros, kind}")
    assert bool(torch.isfinite(got).all())
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


# ---- groups of millions of values -----------------------------------------------------------------------------------------------
def test_the_group_of_a_value_for_groups_of_any_size():
    group_of = _abi.load().tlq_debug_moe_group
    longest = (1 << 24) // 32
    for units in [*range(1, 70), 127, 128, 4096, 5461, 65535, 65536, 65537, 65538, 98304, 131071, 131073, 262143, longest - 1]:
        edges = {u for q in {1, 2, 3, longest // units - 1, longest // units} for u in (q * units - 1, q * units, q * units + 1)}
        for u in sorted({0, 1, longest - 1, *edges}):
            if 0 <= u < longest:
                assert group_of(units * 32, u) == u // units, (units, u)
    for group, u in ((0, 0), (31, 0), (33, 0), (-32, 0), (1 << 24, 0), (64, -1), (64, longest)):
        assert group_of(group, u) == -1


@gpu
@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("K,group", [(2097184, 2097184), (6291456, 3145728)])
def test_scales_of_groups_of_millions_of_values(K, group, up):
    """Activations other than 0 at both ends of each group alone, so that the bound of the sums (which counts K additions) is a part of these
    few products; neighbouring rows' scales are eight times apart."""
    E, N = 2, 16
    rows = 2 * N if up else N
    g = gen(41)
    Wp = torch.randint(0, 256, (E, rows, K // 2), dtype=torch.uint8, generator=g)
    s = (2.0 ** -(4 + 3 * (torch.arange(E * rows * (K // group)) % 2)).view(E, rows, K // group)).half()
    x = torch.zeros(1, K)
    for at in range(0, K, group):
        x[0, at:at + 32] = 1.0
        x[0, at + group - 32:at + group] = torch.rand(32, generator=g) + 0.5
    x, ids = x.half(), torch.tensor([[1]], dtype=torch.int32)
    small = (x[0] != 0).nonzero()[:, 0]
    d = ref.dequant_w4(Wp[1], s[1], 0, group, torch.float16)[:, small].double() @ x[0, small].double()  # (no weight is negative: the sum of magnitudes too)
    # the zeros add nothing and lose nothing: as many additions as there are other values
    off = d * (len(small) + 8) * 2.0**-24
    if up:
        got = ops.moe_gate_up_w4a16(E, 1, N, K, group)(*operands(x, ids, Wp, s))[0, 0]
        gate, u = d.chunk(2)
        dg, du = off.chunk(2)
        want = gate / (1 + torch.exp(-gate)) * u
        allowed = 1.1 * dg * (u + du) + gate * du + (gate + 4) * 2.0**-22 * want
    else:
        got = ops.moe_down_w4a16(E, 1, N, K, group, out_dtype="float32")(*operands(x[:, None], ids, torch.ones(1, 1), Wp, s))[0]
        want, allowed = d, off + (d + off) * 3 * 2.0**-24
    assert_close64(got, want, allowed, f"K={K} group={group} up={up}")


# ---- one workspace for a program's calls ------------------------------------------------------------------------------------------
WORKSPACES = [(8, 2, 4096, 14336), (8, 2, 1024, 4096), (64, 1, 4096, 14336), (128, 8, 1408, 2048), (256, 8, 512, 7168), (3, 2, 16, 64), (1, 1, 16, 8192), (1024, 5, 96, 32)]


@pytest.mark.parametrize("E,k,N,K", WORKSPACES)
def test_a_workspace_for_many_tokens_does_for_fewer(E, k, N, K):
    lib = _abi.load()
    for size in (lib.tlq_moe_gate_up_workspace_bytes, lib.tlq_moe_down_workspace_bytes):
        sizes = [size(M, E, k, N, K) for M in sorted({*range(1, 700), *range(700, 5000, 7), *range(max(1, 4096 // k - 2), 4096 // k + 3), 8192, 100000})]
        assert sizes == sorted(sizes) and sizes[0] > 0


@gpu
@pytest.mark.parametrize("E,k,N,K", [(8, 2, 256, 8192), (4, 2, 1024, 4096), (64, 1, 64, 14336)])
def test_calls_of_every_size_in_the_workspace_of_the_largest(E, k, N, K):
    """M from 1 to the largest in one workspace of the largest one's size, in both products: the rows of the definition, and nothing behind them."""
    lib, P, most = _abi.load(), _abi.ptr, 300
    st = torch.cuda.current_stream().cuda_stream
    T = torch.float16
    w1, s1, _ = make_experts(E, 2 * N, K, 64, T, 8, 61)
    X, ids = torch.randn(most, K, generator=gen(62)).to(T), make_ids(most, E, k, "spread", 63)
    g1 = operands(X, ids, w1, s1)
    size = lib.tlq_moe_gate_up_workspace_bytes(most, E, k, N, K), lib.tlq_moe_down_workspace_bytes(most, E, k, 2 * N, K)
    ws = torch.zeros(max(size), dtype=torch.uint8, device="cuda")
    H = torch.randn(most, k, K, generator=gen(64)).to(T)
    weights = torch.softmax(torch.randn(most, k, generator=gen(65)), 1)
    g2 = operands(H, weights)
    for M in (1, 2, 3, 5, 16, 31, 32, 33, 70, 140, 287, 288, 300):
        h = torch.full((most, k, N), float("nan"), dtype=T, device="cuda")
        _abi.check(lib.tlq_moe_gate_up_w4a16(P(g1[0]), P(g1[1]), P(g1[2]), P(g1[3]), None, P(h), P(ws), size[0], M, E, k, N, K, 64, 8.0, _abi.F16, st))
        some = torch.tensor(sorted({0, M // 2, M - 1}))
        assert_close64(h[some.cuda()], *ref.moe_gate_up(X[some], ids[some], w1, s1, 8, 64), f"gate_up M={M}")
        assert not bool(h[:M].isnan().any()) and bool(h[M:].isnan().all())
        y = torch.full((most, 2 * N), float("nan"), device="cuda")
        _abi.check(lib.tlq_moe_down_w4a16(P(g2[0]), P(g1[1]), P(g2[1]), P(g1[2]), P(g1[3]), None, P(y), P(ws), size[1], M, E, k, 2 * N, K, 64, 8.0, _abi.F16,
                                          _abi.F32, st))
        assert_close64(y[some.cuda()], *ref.moe_down(H[some], ids[some], weights[some], w1, s1, 8, 64), f"down M={M}")
        assert not bool(y[:M].isnan().any()) and bool(y[M:].isnan().all())


# ---- more tokens than threads of one launch -----------------------------------------------------------------------------------------
@gpu
def test_route_of_more_tokens_than_one_launch_takes():
    """2^26 tokens are 2^32 threads."""
    M = (1 << 26) + 5
    x = torch.rand(M, 2, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").bfloat16()
    weights, ids = ops.moe_route(2, 1, renormalize=False, in_dtype="bfloat16")(x)
    assert bool((ids[:, 0] == (x[:, 1] > x[:, 0])).all())  # (ties go to the lower index)
    for part in (slice(0, 9), slice(M // 2, M // 2 + 9), slice((1 << 26) - 9, M)):
        want, _ = ref.moe_route(x[part], 1, renormalize=False)
        assert bool(((weights[part].cpu().double() - want).abs() <= want * (2.0**-24 + 2.0**-40)).all())
    assert bool((weights >= 0.5).all()) and bool((weights < 1).all())
    del x, weights, ids
    torch.cuda.empty_cache()


@gpu
def test_down_of_more_rows_than_one_launch_adds():
    """2^23 tokens of 1040 outputs are 2^32 threads of the kernel that adds a token's rows (36 GB of them)."""
    E, N, K, M = 2, 1040, 32, (1 << 23) + 3
    lib, P = _abi.load(), _abi.ptr
    g = torch.Generator(device="cuda").manual_seed(2)
    Wp, s, _ = make_experts(E, N, K, 32, torch.float16, 8, 71)
    H = torch.randn(M, 1, K, generator=g, device="cuda").half()
    ids = torch.randint(0, E, (M, 1), generator=g, device="cuda", dtype=torch.int32)
    weights = torch.rand(M, 1, generator=g, device="cuda") + 0.5
    Y = torch.full((M, N), float("nan"), dtype=torch.float16, device="cuda")
    ws = torch.empty(lib.tlq_moe_down_workspace_bytes(M, E, 1, N, K), dtype=torch.uint8, device="cuda")
    w, sc = operands(Wp, s)
    _abi.check(lib.tlq_moe_down_w4a16(P(H), P(ids), P(weights), P(w), P(sc), None, P(Y), P(ws), ws.numel(), M, E, 1, N, K, 32, 8.0, _abi.F16, _abi.F16,
                                      torch.cuda.current_stream().cuda_stream))
    some = torch.cat([torch.arange(0, M, M // 40), torch.arange((1 << 23) - 4, M)])
    take = some.cuda()
    want, off = ref.moe_down(H[take], ids[take], weights[take], Wp, s, 8, 32)
    assert_close64(Y[take], want, off, "down")
    assert not any(bool(part.isnan().any()) for part in Y.split(1 << 20))
    del H, Y, ws
    torch.cuda.empty_cache()


def test_gate_up_of_more_work_groups_than_one_launch_takes_is_refused():
    lib, p = _abi.load(), ctypes.c_void_p(0x1000)
    M, k, N, K = (1 << 24) - 1, 1, 8192, 32
    rc = lib.tlq_moe_gate_up_w4a16(p, p, p, p, None, p, p, 1 << 50, M, 8, k, N, K, 32, 0.0, _abi.F16, None)
    assert rc != 0 and "fewer tokens" in _abi.last_error(), _abi.last_error()


# ---- gates far from 0 --------------------------------------------------------------------------------------------------------------
# M, E, N, K: every kernel that applies silu (few pairs; tiles of 32; of 64; of 256; the sums of parts of K)
GATES = [(64, 64, 16, 128, FEW), (40, 2, 48, 64, TILES32), (200, 2, 16, 64, TILES64), (4096, 1, 3104, 128, TILES256), (40, 2, 16, 4096, TILES32)]


@pytest.mark.parametrize("M,E,N,K,kernel", GATES)
def test_gates_far_from_zero_reach_every_kernel(M, E, N, K, kernel):
    assert choice(True, M, E, 1, N, K, K, None)[0] == kernel


@gpu
@pytest.mark.parametrize("M,E,N,K,kernel", GATES)
def test_gates_far_from_zero(M, E, N, K, kernel):
    """silu(g) * u of exact sums g and u, for g from -94 to 100 and u = 300: bfloat16 holds all of them as normal numbers, also where exp(-g) is more than
    fp32 holds or silu(g) less.  (|g| + 4) 2^-22 of the value as in the oracle, and the rounding."""
    Wp = torch.zeros(E, 2 * N, K // 2, dtype=torch.uint8)
    Wp[:, :N, 0], Wp[:, N:, 0] = 0x01, 0x10  # gate = x[0], up = x[1]
    s = torch.ones(E, 2 * N, 1, dtype=torch.bfloat16)
    X = torch.zeros(M, K, dtype=torch.bfloat16)
    X[:, 0] = torch.linspace(-94, 100, M).bfloat16()
    X[:, 1] = 300
    ids = (torch.arange(M) % E).int()[:, None]
    got = ops.moe_gate_up_w4a16(E, 1, N, K, K, "bfloat16")(*operands(X, ids, Wp, s))[:, 0].cpu()
    g = X[:, :1].double()
    want = (g / (1 + torch.exp(-g)) * 300).expand(M, N)
    assert float(want.abs().min()) > 2.0**-126
    assert_close64(got, want, (g.abs() + 4) * 2.0**-22 * want.abs(), "far gates")


@gpu
def test_a_far_gate_beside_one_that_is_no_number():
    """Outputs are independent of each other: a NaN beside a gate of -90 leaves its product as it is."""
    N, K = 16, 64
    Wp = torch.zeros(1, 2 * N, K // 2, dtype=torch.uint8)
    Wp[:, :N, 0], Wp[:, N:, 0] = 0x01, 0x10
    X = torch.zeros(1, K, dtype=torch.bfloat16)
    X[0, 0], X[0, 1] = -90, 300
    ids = torch.zeros(1, 1, dtype=torch.int32)
    for at in range(4):
        s = torch.ones(1, 2 * N, 1, dtype=torch.bfloat16)
        s[0, at] = float("nan")
        got = ops.moe_gate_up_w4a16(1, 1, N, K, K, "bfloat16")(*operands(X, ids, Wp, s))[0, 0].cpu()
        assert bool(got[at].isnan())
        rest = torch.arange(N) != at
        want = torch.full((N - 1,), -90 / (1 + torch.exp(torch.tensor(90.0, dtype=torch.float64))).item() * 300, dtype=torch.float64)
        assert_close64(got[rest], want, 94 * 2.0**-22 * want.abs(), f"beside {at}")


# ---- tiles of 256 pairs --------------------------------------------------------------------------------------------------------------
# the pairs of each expert, and those of none: whole tiles, one more and one fewer, what is left at every candidate for a last tile of 256
COUNTS = [([256, 200], 0), ([512, 256, 768], 0), ([255, 257, 513], 7), ([256, 64, 65, 320, 321], 0), ([128, 129, 192, 193, 448, 449], 3), ([1, 0, 1024, 0, 2], 500),
          ([256] * 16, 0), ([40] * 40 + [2496], 0)]


@gpu
@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("counts,none", COUNTS)
def test_tiles_of_256_pairs_by_count(counts, none, up):
    E, K = len(counts), 128
    M = sum(counts) + none
    N = (-(-192 // (M // 256)) - 1) * (128 if up else 256) + 16  # the fewest work-groups that the rule wants, the last of them with 16 outputs
    assert choice(up, M, E, 1, N, K, 128, None)[0] == TILES256
    ids = torch.cat([torch.full((n,), e) for e, n in enumerate(counts)] + [torch.full((none,), -1)]).int()
    ids = ids[torch.randperm(len(ids), generator=gen(81))][:, None]
    Wp, s, _ = make_experts(E, 2 * N if up else N, K, 128, torch.bfloat16, 8, 82)
    some = torch.tensor(sorted({int((ids[:, 0] == e).nonzero()[i, 0]) for e in range(E) for i in {0, counts[e] // 2, counts[e] - 1} if counts[e]}))[:24]
    if up:
        X = torch.randn(M, K, generator=gen(83)).bfloat16()
        got = ops.moe_gate_up_w4a16(E, 1, N, K, 128, "bfloat16", zeros=8)(*operands(X, ids, Wp, s))
        want, off = ref.moe_gate_up(X[some], ids[some], Wp, s, 8, 128)
    else:
        H, w = torch.randn(M, 1, K, generator=gen(83)).bfloat16(), torch.ones(M, 1)
        got = ops.moe_down_w4a16(E, 1, N, K, 128, "bfloat16", "bfloat16", zeros=8)(*operands(H, ids, w, Wp, s))
        want, off = ref.moe_down(H[some], ids[some], w[some], Wp, s, 8, 128)
    assert_close64(got[some.cuda()], want, off, f"{counts} {up}")
    got = got.view(M, N)
    live = (ids[:, 0] >= 0).cuda()
    assert bool(torch.isfinite(got).all()) and bool((got[~live] == 0).all()) and bool((got[live].abs().amax(1) > 0).all())


# ---- few pairs: several passes over an expert's rows, several tiles of a wavefront ---------------------------------------------------
# up, M, E, top_k, N, K, group, type, zeros, what the plan has to be; all pairs on one expert ("one"): more of them than rows of a pass, the last pass not full
PASSES = [
    (True, 35, 64, 1, 48, 256, 64, "float16", "int", dict(rows=16, splits=1)),
    (False, 35, 64, 1, 48, 256, 64, "bfloat16", "frac", dict(rows=16, splits=1)),
    (True, 35, 64, 1, 48, 1024, 64, "bfloat16", "frac", dict(rows=16, splits=4)),
    (False, 35, 64, 1, 48, 1024, 64, "float16", "int", dict(rows=16, splits=4)),
    (True, 7, 64, 3, 48, 4128, 32, "float16", "frac", dict(rows=4, splits=4)),
    (True, 5, 8, 3, 48, 4128, 96, "bfloat16", 8, dict(rows=4, splits=4)),
    (False, 7, 8, 2, 48, 6016, 32, "bfloat16", "int", dict(rows=4, splits=4, parts=2)),
    (False, 5, 64, 3, 80, 4128, 32, "float16", 7.5, dict(rows=8, splits=4, parts=2)),
    (False, 7, 16, 3, 32, 8224, 32, "float16", "frac", dict(rows=4, splits=4, parts=3)),
    (False, 8, 64, 8, 1808, 4256, 32, "float16", "int", dict(rows=8, splits=1, tiles=2, parts=2)),
    (False, 8, 64, 8, 1808, 14336, 128, "bfloat16", "frac", dict(rows=4, splits=1, tiles=4, parts=4)),
]


@pytest.mark.parametrize("up,M,E,k,N,K,group,dtype,zeros,plan", PASSES)
def test_plans_of_several_passes(up, M, E, k, N, K, group, dtype, zeros, plan):
    kernel, got = choice(up, M, E, k, N, K, group, zeros if isinstance(zeros, str) else None)
    assert kernel == FEW and {key: got[key] for key in plan} == plan, got
    assert M * k > got["rows"] and M * k % got["rows"] or got["tiles"] > 1


@gpu
@pytest.mark.parametrize("up,M,E,k,N,K,group,dtype,zeros,plan", PASSES)
def test_few_pairs_in_several_passes(up, M, E, k, N, K, group, dtype, zeros, plan):
    run_both(up, M, E, k, N, K, group, dtype, zeros, "one")
    run_both(up, M, E, k, N, K, group, dtype, zeros, "spread", some=[0, M - 1])


# ---- which kernel -------------------------------------------------------------------------------------------------------------------
# tiles of 256 pairs with few outputs: wavefronts and 16-row tiles behind the last output
FEW_OUTPUTS = [(True, 16384, 8, 8, 16, 1536), (True, 16390, 4, 8, 144, 1536), (True, 16384, 3, 8, 48, 1664), (False, 16384, 8, 8, 16, 2048), (False, 8200, 4, 16, 272, 2048)]


@pytest.mark.parametrize("up,M,E,k,N,K", FEW_OUTPUTS)
def test_few_outputs_are_on_tiles_of_256_pairs(up, M, E, k, N, K):
    assert choice(up, M, E, k, N, K, 128, "tensor")[0] == TILES256


def big_call(up, M, E, k, N, K, group, T, ids, Wp, s, z, seed):
    """A product of tensors made on the GPU -> (output, what the oracle takes for the tokens `some`, with their experts alone)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    name = {v: n for n, v in DT.items()}[T]
    extra = [z] if isinstance(z, torch.Tensor) else []
    if up:
        x = torch.randn(M, K, generator=g, device="cuda").to(T)
        got = ops.moe_gate_up_w4a16(E, k, N, K, group, name, zeros=kernel_zeros(z))(x, ids, Wp, s, *extra)
    else:
        x = torch.randn(M, k, K, generator=g, device="cuda").to(T)
        weights = torch.rand(M, k, generator=g, device="cuda") + 0.25
        got = ops.moe_down_w4a16(E, k, N, K, group, name, "float32", zeros=kernel_zeros(z))(x, ids, weights, Wp, s, *extra)

    def check(some):
        at = torch.tensor(some, device="cuda")
        mine = ids[at]
        used = torch.unique(mine[(mine >= 0) & (mine < E)]).long()
        to = torch.full((E,), -1, dtype=torch.int32, device="cuda")
        to[used] = torch.arange(len(used), dtype=torch.int32, device="cuda")
        local = torch.where((mine >= 0) & (mine < E), to[mine.clamp(0, E - 1).long()], -1).cpu()
        part = (Wp[used].cpu(), s[used].cpu(), z[used].cpu() if isinstance(z, torch.Tensor) else z, group)
        if up:
            want, off = ref.moe_gate_up(x[at].cpu(), local, *part)
        else:
            want, off = ref.moe_down(x[at].cpu(), local, weights[at].cpu(), *part)
        assert_close64(got[at], want, off, f"{up, M, E, k, N, K}")

    return got, check


def gpu_experts(E, rows, K, group, T, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    words = torch.randint(-(2**63), 2**63 - 1, (E, rows, K // 16), generator=g, device="cuda", dtype=torch.int64)
    s = (torch.rand(E, rows, K // group, generator=g, device="cuda") * 0.015 + 0.005).to(T)
    return words.view(torch.uint8), s, torch.randint(6, 10, s.shape, generator=g, device="cuda").to(T)


@gpu
@pytest.mark.parametrize("up,M,E,k,N,K", FEW_OUTPUTS)
def test_few_outputs_on_tiles_of_256_pairs(up, M, E, k, N, K):
    T = torch.bfloat16 if up else torch.float16
    g = torch.Generator(device="cuda").manual_seed(91)
    ids = torch.randint(-1, E, (M, k), generator=g, device="cuda", dtype=torch.int32)
    Wp, s, z = gpu_experts(E, 2 * N if up else N, K, 128, T, 92)
    got, check = big_call(up, M, E, k, N, K, 128, T, ids, Wp, s, z, 93)
    check([0, 1, M // 2, M - 2, M - 1])
    assert bool(torch.isfinite(got).all())
    if up:
        assert bool((got[ids < 0] == 0).all()) and bool((got[ids >= 0].abs().amax(1) > 0).all())
    else:
        assert bool((got[(ids >= 0).any(1)].abs().amax(1) > 0).all())


# ---- weights of more than 4 GiB, a thousand experts, sixty-four of them a token -------------------------------------------------------
# M and top_k: few pairs, tiles of 32, of 64, of 256
THOUSAND = [(4, 2, FEW), (200, 8, TILES32), (4096, 8, TILES64), (32768, 8, TILES256)]


@pytest.mark.parametrize("M,k,kernel", THOUSAND)
@pytest.mark.parametrize("up", [True, False])
def test_a_thousand_experts_reach_every_kernel(M, k, kernel, up):
    assert choice(up, M, 1024, k, 1024 if up else 2048, 4224, 128, "tensor")[0] == kernel


@gpu
@pytest.mark.parametrize("up", [True, False])
def test_weights_of_more_than_4_gib(up):
    """1024 experts of 2048 rows of 4224 values, 4.4e9 bytes: the first, the last and those behind 2^31 and 2^32 bytes."""
    E, rows, K, T = 1024, 2048, 4224, torch.bfloat16
    Wp, s, z = gpu_experts(E, rows, K, 128, T, 95)
    assert Wp.numel() > 2**32
    N = rows // 2 if up else rows
    for M, k, _ in THOUSAND:
        g = torch.Generator(device="cuda").manual_seed(96)
        ids = torch.randint(0, E, (M, k), generator=g, device="cuda", dtype=torch.int32)
        ids[0, 0], ids[0, 1], ids[1, 0], ids[1, 1], ids[M - 1, 0], ids[M - 1, 1] = 0, E - 1, 496, 497, 993, 994
        got, check = big_call(up, M, E, k, N, K, 128, T, ids, Wp, s, z, 97)
        check([0, 1, M - 1])
        assert bool(torch.isfinite(got).all())
        del got, check
    del Wp, s, z
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("M,E,k", [(1, 100, 64), (5, 64, 64), (70, 1024, 64)])
def test_sixty_four_experts_a_token(M, E, k, up):
    run_both(up, M, E, k, 32, 160, 32, "bfloat16", "int", "spread", some=[0, M - 1])


# ---- slots that are mostly empty -----------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("M,E,k,N,K,kernel", [(16384, 8, 8, 272, 2048, TILES256), (512, 8, 8, 3088, 128, TILES256), (300, 8, 8, 80, 256, TILES64), (20, 16, 8, 80, 256, TILES32)])
def test_slots_that_are_mostly_empty(M, E, k, N, K, kernel, up):
    """One slot in eight has an expert here, and then with none at all."""
    assert choice(up, M, E, k, N, K, 128, "tensor")[0] == kernel
    T = torch.float16
    Wp, s, z = gpu_experts(E, 2 * N if up else N, K, 128, T, 101)
    g = torch.Generator(device="cuda").manual_seed(102)
    ids = torch.randint(0, 8 * E, (M, k), generator=g, device="cuda", dtype=torch.int32)
    ids[M - 1, k - 1] = E - 1
    for round_ids in (ids, torch.full_like(ids, -1)):
        got, check = big_call(up, M, E, k, N, K, 128, T, round_ids, Wp, s, z, 103)
        check([0, 1, 2, M // 2, M - 1])
        here = (round_ids >= 0) & (round_ids < E)
        assert bool(torch.isfinite(got).all())
        if up:
            assert bool((got[~here] == 0).all()) and bool((got[here].abs().amax(1) > 0).all() if bool(here.any()) else True)
        else:
            assert bool((got[~here.any(1)] == 0).all())


# ---- a token beside others -----------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("M", [1, 4, 12, 70, 200])
def test_a_token_gets_the_same_bits_beside_other_tokens(M):  # (few pairs, tiles of 32, of 64)
    """As many tokens, the others' inputs and experts changed: the first and the last keep their bits (below the sizes of tiles of 256 pairs, where
    the counts of all experts decide which of two kernels a pair is on)."""
    E, k, N, K = 8, 2, 96, 256
    w1, s1, z1 = operands(*make_experts(E, 2 * N, K, 64, torch.bfloat16, "int", 111))
    w2, s2, z2 = operands(*make_experts(E, K, N, 96, torch.bfloat16, "frac", 112))
    up, down = ops.moe_gate_up_w4a16(E, k, N, K, 64, "bfloat16", zeros="tensor"), ops.moe_down_w4a16(E, k, K, N, 96, "bfloat16", "float32", zeros="tensor")
    kept = sorted({0, M - 1})
    x0, ids0, weights = torch.randn(M, K, generator=gen(1)).bfloat16(), make_ids(M, E, k, "spread", 2), torch.softmax(torch.randn(M, k, generator=gen(3)), 1).cuda()
    first = None
    for other in range(4):
        x, ids = torch.randn(M, K, generator=gen(10 + other)).bfloat16(), make_ids(M, E, k, ["spread", "one", "holes", "twice"][other], 20 + other)
        x[kept], ids[kept] = x0[kept], ids0[kept]
        h = up(x.cuda(), ids.cuda(), w1, s1, z1)
        y = down(h, ids.cuda(), weights, w2, s2, z2)
        mine = h[kept].cpu(), y[kept].cpu()
        first = first or mine
        assert_bit_equal(mine[0], first[0], "hidden")
        assert_bit_equal(mine[1], first[1], "y")


# ---- zero points, scales and inputs of every kind in every kernel -------------------------------------------------------------------
# M, E, top_k, N, K, group: few pairs; tiles of 32, whole rows and K in parts; of 64, the same; of 256
EVERY = [(3, 8, 2, 48, 256, 64, FEW), (12, 4, 2, 80, 224, 32, TILES32), (12, 4, 2, 48, 4096, 128, TILES32), (130, 4, 2, 80, 320, 64, TILES64), (60, 2, 2, 48, 4160, 32, TILES64),
         (2047, 4, 2, 3088, 256, 64, TILES256)]


def every_call(up, shape, dtype, scales, zeros, weights=None, x=None, ids=None, seed=121):
    """-> (the output on the CPU, the oracle's value and bound), all in the tokens that are compared; `zeros` as the kernels take them, or a tensor."""
    M, E, k, N, K, group, _ = shape
    T = DT[dtype]
    Wp, s, _ = make_experts(E, 2 * N if up else N, K, group, T, None, seed)
    s = s if scales else None
    z = zeros(s if scales else torch.empty(E, 2 * N if up else N, K // group, dtype=T)) if callable(zeros) else zeros
    ids = make_ids(M, E, k, "spread", seed + 1) if ids is None else ids
    some = torch.tensor(sorted({0, 1, 2, M // 2, M - 2, M - 1} & set(range(M))))
    X = (torch.randn(M, K, generator=gen(seed + 2)) if up else torch.randn(M, k, K, generator=gen(seed + 2))) * (1 if scales else 0.02)
    X = X.to(T) if x is None else x(X.to(T))
    args = [X, ids, Wp] if up else [X, ids, torch.rand(M, k, generator=gen(seed + 3)) + 0.25 if weights is None else weights, Wp]
    make = ops.moe_gate_up_w4a16 if up else ops.moe_down_w4a16
    kernel = make(E, k, N, K, group, dtype, zeros=kernel_zeros(z), with_scales=scales, **({} if up else {"out_dtype": "float32"}))
    got = kernel(*operands(*args, *([s] if scales else []), z)).cpu()
    if up:
        return got[some], ref.moe_gate_up(X[some], ids[some], Wp, s, z, group), some
    return got[some], ref.moe_down(X[some], ids[some], args[2][some], Wp, s, z, group), some


@pytest.mark.parametrize("shape", EVERY)
def test_every_kernel_is_among_them(shape):
    assert choice(True, *shape[:6], None)[0] == shape[6] and choice(False, *shape[:6], "tensor")[0] == shape[6]


def whole_then_not(s):
    """Zero points that are whole numbers in the first half of a row and not in the second."""
    z = torch.randint(6, 10, s.shape, generator=gen(5)).to(s.dtype)
    half = s.shape[2] // 2
    z[:, :, half:] += 0.5
    return z


def large_whole(s):
    return (torch.randint(0, 2, s.shape, generator=gen(6)) * 512 - 256).to(s.dtype)


@gpu
@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("shape", EVERY)
def test_scales_and_zero_points_of_every_kind(shape, dtype, up):
    for scales in (True, False):
        for zeros in (None, 8, 7.5, whole_then_not):
            got, want, _ = every_call(up, shape, dtype, scales, zeros)
            assert_close64(got, *want, f"{shape} {dtype} up={up} scales={scales} zeros={zeros}")
    # the ends of the zero points that bfloat16 folds into the unpacking, and those next to them: u - z rounds there
    for zeros in (255, -255, 256, -256, 257, -258, large_whole):
        got, want, _ = every_call(up, shape, dtype, True, zeros, x=lambda x: x * 0.02)
        assert_close64(got, *want, f"{shape} {dtype} up={up} zeros={zeros}")


@gpu
@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("shape", EVERY)
def test_tokens_that_are_no_numbers_leave_the_others_alone(shape, dtype, up):
    M = shape[0]

    def spoil(x):
        x = x.clone()
        x[1::3] = float("nan")
        x[1::6] = float("inf")
        return x

    plain, want, some = every_call(up, shape, dtype, True, 8)
    got, _, _ = every_call(up, shape, dtype, True, 8, x=spoil)
    clean = (some % 3) != 1
    assert_bit_equal(got[clean], plain[clean], "clean tokens")
    assert not bool(torch.isfinite(got[~clean]).any())


@gpu
@pytest.mark.parametrize("shape", EVERY)
def test_two_graphs_and_an_eager_call_of_the_same_weights(shape):
    """Gate / up and down captured twice with inputs of their own, replayed in turn and on two streams at once, with eager calls in between."""
    M, E, k, N, K, group, _ = shape
    T = torch.bfloat16
    w1, s1, z1 = operands(*make_experts(E, 2 * N, K, group, T, "int", 131))
    w2, s2, _ = make_experts(E, K, N, N, T, None, 132) if N % 32 == 0 else make_experts(E, K, N + 16, N + 16, T, None, 132)
    w2, s2 = w2.cuda(), s2.cuda()
    N2 = w2.shape[2] * 2
    up, down = ops.moe_gate_up_w4a16(E, k, N, K, group, "bfloat16", zeros="tensor"), ops.moe_down_w4a16(E, k, K, N2, N2, "bfloat16", "float32", zeros=8)

    def layer(x, ids, weights):
        h = up(x, ids, w1, s1, z1)
        return down(torch.nn.functional.pad(h, (0, N2 - N)), ids, weights, w2, s2)

    ins = [[torch.randn(M, K, generator=gen(140 + i)).to(T).cuda(), make_ids(M, E, k, "holes", 150 + i).cuda(), torch.rand(M, k, generator=gen(160 + i)).cuda()] for i in range(4)]
    want = [layer(*a) for a in ins]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(*ins[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, slots, outs = [], [], []
    for i in range(2):
        slots.append([t.clone() for t in ins[i]])
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(layer(*slots[i]))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(4):
        for i in range(2):
            for t, v in zip(slots[i], ins[(rep + 2 * i) % 4]):
                t.copy_(v)
            outs[i].fill_(float("nan"))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        beside = layer(*ins[rep])
        torch.cuda.synchronize()
        for i in range(2):
            assert_bit_equal(outs[i].cpu(), want[(rep + 2 * i) % 4].cpu(), f"graph {i}, replay {rep}")
        assert_bit_equal(beside.cpu(), want[rep].cpu(), f"eager beside replay {rep}")


@gpu
def test_calls_from_several_threads():
    import threading

    shape = EVERY[2]
    M, E, k, N, K, group, _ = shape
    w, s, z = operands(*make_experts(E, 2 * N, K, group, torch.float16, "int", 171))
    up = ops.moe_gate_up_w4a16(E, k, N, K, group, zeros="tensor")
    ins = [(torch.randn(m, K, generator=gen(172 + m)).half().cuda(), make_ids(m, E, k, "spread", 173 + m).cuda()) for m in (1, 12, 70, 200)]
    want = [up(*a, w, s, z) for a in ins]
    torch.cuda.synchronize()
    got, errors = [[] for _ in ins], []

    def work(i):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(10):
                    got[i].append(up(*ins[i], w, s, z))
            st.synchronize()
        except Exception as e:  # noqa: BLE001 (a thread's failure is the test's)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(ins))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for g, y in zip(got, want):
        for one in g:
            assert_bit_equal(one.cpu(), y.cpu(), "threads")


@gpu
@pytest.mark.parametrize("up", [True, False])
@pytest.mark.parametrize("shape", EVERY)
def test_nothing_is_written_outside_of_the_output_and_the_workspace(shape, up):
    """A workspace of exactly the size that is asked for, and 4 KB on either side of it and of the output."""
    M, E, k, N, K, group, _ = shape
    lib, P, side = _abi.load(), ctypes.c_void_p, 4096
    T = torch.bfloat16
    w, s, z = operands(*make_experts(E, 2 * N if up else N, K, group, T, "int", 181))
    ids = make_ids(M, E, k, "holes", 182).cuda()
    x = torch.randn(M, K, generator=gen(183)).to(T).cuda() if up else torch.randn(M, k, K, generator=gen(183)).to(T).cuda()
    weights = torch.rand(M, k, generator=gen(184)).cuda()
    size = (lib.tlq_moe_gate_up_workspace_bytes if up else lib.tlq_moe_down_workspace_bytes)(M, E, k, N, K)
    out_size = M * (k if up else 1) * N * 2
    ws = torch.full((size + 2 * side,), 0xAB, dtype=torch.uint8, device="cuda")
    out = torch.full((out_size + 2 * side,), 0xFF, dtype=torch.uint8, device="cuda")
    ws_at, out_at, st = P(ws.data_ptr() + side), P(out.data_ptr() + side), torch.cuda.current_stream().cuda_stream
    if up:
        rc = lib.tlq_moe_gate_up_w4a16(_abi.ptr(x), _abi.ptr(ids), _abi.ptr(w), _abi.ptr(s), _abi.ptr(z), out_at, ws_at, size, M, E, k, N, K, group, 0.0, _abi.BF16, st)
    else:
        rc = lib.tlq_moe_down_w4a16(_abi.ptr(x), _abi.ptr(ids), _abi.ptr(weights), _abi.ptr(w), _abi.ptr(s), _abi.ptr(z), out_at, ws_at, size, M, E, k, N, K, group, 0.0,
                                    _abi.BF16, _abi.BF16, st)
    _abi.check(rc)
    torch.cuda.synchronize()
    for buffer, n, fill in ((ws, size, 0xAB), (out, out_size, 0xFF)):
        assert bool((buffer[:side] == fill).all()) and bool((buffer[side + n:] == fill).all())
    assert bool(torch.isfinite(out[side:side + out_size].view(T)).all())  # (0xFFFF is a NaN: every output was written)
