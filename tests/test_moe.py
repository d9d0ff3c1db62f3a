"""The mixture-of-experts operators against the definitions in 64 bits (oracle/ref.py: moe_*), at the sizes, masks and ids where
they can go wrong; their refusals; the three together, captured, on other streams and at the same time.

Tolerances.  Expert ids are equal.  Router weights are binary64 up to the last step: one rounding to fp32 (2^-24 of the value)
plus the 64-bit arithmetic of both sides (below 2^-40).  Products: what the fp32 sums may be off by, which the oracle returns
beside the value, plus half a step of the output type, finfo.eps / 2 of the value, or of its smallest normal number below that."""
import ctypes

import pytest
import torch

from helpers import DT, assert_bit_equal, gen
from oracle import ref
from tilelang_ascend_amd import _abi, ops

gpu = pytest.mark.gpu


# ---- helpers ------------------------------------------------------------------------------------------------------------
def make_experts(E, rows, K, group, dtype, zeros, seed):
    """(packed, scales or None, zeros as the reference takes them) on the CPU."""
    g = gen(seed)
    Wp = torch.randint(0, 256, (E, rows, K // 2), dtype=torch.uint8, generator=g)
    G = K // group
    s = (torch.rand(E, rows, G, generator=g) * 0.015 + 0.005).to(dtype)
    if zeros == "int":
        z = torch.randint(6, 10, (E, rows, G), generator=g).to(dtype)
    elif zeros == "frac":
        z = (torch.rand(E, rows, G, generator=g) * 3 + 6).to(dtype)
    else:
        z = zeros  # None or a number
    return Wp, s, z


def kernel_zeros(z):
    return "tensor" if isinstance(z, torch.Tensor) else z


def operands(*ts):
    return [t.cuda() for t in ts if isinstance(t, torch.Tensor)]


def assert_close64(got, want, off, what):
    got = got.cpu()
    fi = torch.finfo(got.dtype)
    allowed = off + (want.abs() + off).clamp_min(fi.tiny) * (fi.eps / 2)
    assert torch.isfinite(got).all(), what
    worst = ((got.to(torch.float64) - want).abs() - allowed).max().item()
    assert worst <= 0, f"{what}: {worst:.3e} more than allowed"


def check_route(logits, top_k, **kw):
    bias = kw.pop("bias", None)
    E = logits.shape[1]
    name = {v: k for k, v in DT.items()}[logits.dtype]
    kernel = ops.moe_route(E, top_k, with_bias=bias is not None, in_dtype=name, **kw)
    weights, ids = kernel(logits.cuda(), bias.cuda()) if bias is not None else kernel(logits.cuda())
    want_w, want_ids = ref.moe_route(logits, top_k, bias=bias, **kw)
    assert weights.dtype == torch.float32 and ids.dtype == torch.int32
    assert torch.equal(ids.cpu().long(), want_ids)
    err = (weights.cpu().double() - want_w).abs()
    assert (err <= want_w.abs() * (2.0**-24 + 2.0**-40) + 2.0**-149).all(), err.max()
    return weights, ids


# ---- routing --------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("M,E,k,n_group,topk_group", [
    (1, 64, 6, 1, 1), (5, 8, 2, 1, 1), (1, 1, 1, 1, 1), (7, 3, 3, 1, 1), (130, 60, 4, 4, 2), (33, 65, 8, 1, 1), (19, 160, 6, 8, 3),
    (64, 256, 8, 8, 4), (9, 256, 64, 64, 20), (6, 320, 9, 64, 7), (4, 1000, 10, 1, 1), (3, 1024, 64, 2, 1), (12, 96, 5, 3, 3)])
def test_route(M, E, k, n_group, topk_group, scoring, dtype):
    logits = (torch.randn(M, E, generator=gen(M * E + k)) * 3).to(DT[dtype])
    check_route(logits, k, scoring=scoring, n_group=n_group, topk_group=topk_group)
    bias = torch.randn(E, generator=gen(E)) * 0.1
    check_route(logits, k, scoring=scoring, n_group=n_group, topk_group=topk_group, bias=bias, renormalize=False, scaling=2.5)


@gpu
@pytest.mark.parametrize("M,E,k,n_group,topk_group", [(5, 16, 4, 16, 5), (3, 64, 7, 64, 7), (3, 60, 3, 12, 4), (5, 96, 9, 3, 2), (2, 45, 4, 15, 4), (7, 130, 5, 2, 1)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_groups_of_one_expert_and_of_odd_sizes(scoring, M, E, k, n_group, topk_group):
    logits = torch.randn(M, E, generator=gen(M + E)) * 2
    check_route(logits, k, scoring=scoring, n_group=n_group, topk_group=topk_group)
    check_route(logits - 705.0, k, scoring=scoring, n_group=n_group, topk_group=topk_group)  # sigmoid: where 64 bits run out


@gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_near_ties_are_told_apart_in_64_bits(scoring):
    x = torch.full((3, 256), 1.0)
    x[0, 77], x[0, 200], x[0, 3] = 1.0 + 2.0**-23, 1.0 + 2.0**-22, 1.0 - 2.0**-24
    x[1] = 20.0
    x[1, ::7] = 20.0 + 2.0**-19
    x[2] = 1e-12
    x[2, 5], x[2, 250] = 2e-12, 3e-12
    check_route(x, 20, scoring=scoring)
    check_route(x, 20, scoring=scoring, n_group=8, topk_group=4)


@gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_ties_go_to_the_lowest_index(scoring):
    x = torch.zeros(4, 192)
    x[1, 100:] = 1.0
    x[2, ::3] = 2.0
    x[3] = torch.tensor([0.25, -0.25]).repeat(96)
    check_route(x, 10, scoring=scoring)
    check_route(x, 10, scoring=scoring, n_group=8, topk_group=2)
    assert ops.moe_route(192, 3, scoring=scoring)(x.cuda())[1].cpu()[0].tolist() == [0, 1, 2]


@gpu
@pytest.mark.parametrize("n_group,topk_group", [(1, 1), (4, 2)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_route_masked_and_extreme_logits(scoring, n_group, topk_group):
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    E, k = 32, 5
    x = torch.randn(10, E, generator=gen(3))
    x[0] = -inf                       # nothing is left
    x[1, 2:] = -inf                   # two are left for five slots
    x[2] = nan
    x[3, ::2] = nan
    x[4] = low                        # the type's lowest value is a value like any other
    x[5, 1:] = low
    x[6, 7], x[6, 9] = inf, inf       # they share the softmax
    x[7] = torch.linspace(-2000, 2000, E)  # all but a few scores are 0 in 64 bits
    x[8, :30] = -inf
    x[9] = -800.0 + torch.arange(E)   # sigmoid: scores down to 0
    weights, ids = check_route(x, k, scoring=scoring, n_group=n_group, topk_group=topk_group)
    assert (ids[0] == -1).all() and (weights[0] == 0).all()
    assert sorted(ids[1].tolist()) == [-1, -1, -1, 0, 1]
    bias = torch.zeros(E)
    bias[0], bias[1], bias[5] = -inf, nan, 7.0
    check_route(x, k, scoring=scoring, n_group=n_group, topk_group=topk_group, bias=bias)


@gpu
def test_route_one_wavefront_of_a_work_group_left_over_and_no_token():
    for M in (0, 1, 2, 3, 4, 5):
        w, ids = ops.moe_route(16, 2)(torch.randn(M, 16, generator=gen(M)).cuda())
        assert tuple(w.shape) == tuple(ids.shape) == (M, 2)
    big = torch.randn(4099, 72, generator=gen(1))
    w, ids = ops.moe_route(72, 3)(big.cuda())
    wr, ir = ref.moe_route(big[-7:], 3)
    assert torch.equal(ids[-7:].cpu().long(), ir)


# ---- the experts' products -------------------------------------------------------------------------------------------------
# M, E, top_k, N, K, group, type, zeros, how ids are spread
SHAPES = [
    (1, 8, 2, 64, 128, 64, "float16", "int", "spread"),
    (1, 64, 6, 176, 512, 128, "bfloat16", "int", "spread"),
    (1, 4, 1, 16, 32, 32, "float16", None, "spread"),
    (2, 4, 4, 48, 96, 96, "bfloat16", 8, "spread"),
    (3, 16, 3, 32, 2048, 128, "float16", "frac", "holes"),
    (5, 8, 8, 112, 160, 32, "bfloat16", "frac", "spread"),
    (17, 3, 2, 80, 320, 64, "float16", 7.5, "one"),
    (16, 32, 4, 272, 384, 128, "bfloat16", "int", "spread"),
    (33, 5, 2, 128, 1408, 128, "float16", "int", "holes"),
    (40, 128, 8, 64, 256, 128, "bfloat16", 8, "spread"),
    (63, 2, 1, 96, 192, 64, "float16", None, "one"),
    (100, 4, 2, 144, 448, 64, "bfloat16", "int", "holes"),
    (130, 7, 3, 208, 288, 96, "float16", "frac", "spread"),
    (257, 8, 2, 64, 640, 128, "bfloat16", 8, "spread"),
    (300, 2, 2, 320, 256, 256, "float16", "int", "twice"),
    (520, 16, 2, 32, 64, 32, "float16", "int", "spread"),
    (1, 3, 2, 32, 14336, 64, "float16", "int", "spread"),
    (2, 2, 2, 16, 16448, 64, "bfloat16", "frac", "spread"),
    (9, 4, 3, 48, 4128, 32, "bfloat16", "int", "holes"),
    (24, 6, 2, 80, 992, 32, "float16", "frac", "spread"),
    # (the down product's K in parts that begin inside a window of scales)
    (40, 4, 2, 32, 4096, 128, "float16", "int", "spread"),
    (12, 4, 2, 48, 2208, 96, "bfloat16", "frac", "holes"),
    (20, 4, 2, 32, 2208, 736, "float16", 8, "spread"),
    (64, 2, 2, 16, 8192, 64, "bfloat16", 3.25, "one"),
    # (gate / up in parts of K, with outputs and pairs left over)
    (40, 3, 2, 80, 8224, 32, "float16", "frac", "holes"),
    (90, 2, 1, 176, 10240, 128, "bfloat16", 8, "spread"),
    (70, 2, 2, 1040, 2048, 64, "bfloat16", "int", "twice"),
    # (tiles of 256 pairs, and what is left of an expert's pairs)
    (700, 3, 2, 272, 384, 64, "bfloat16", "frac", "holes"),
    (1100, 2, 1, 144, 128, 32, "float16", None, "one"),
    (515, 4, 2, 160, 256, 128, "bfloat16", 8, "spread"),
    (641, 2, 1, 48, 512, 256, "float16", "int", "spread"),
    (450, 2, 2, 16, 640, 128, "float16", 7.5, "twice"),
]


def make_ids(M, E, k, kind, seed):
    g = gen(seed)
    ids = torch.rand(M, max(E, k), generator=g).argsort(1)[:, :k].remainder(E).int()
    if kind == "one":
        ids.fill_(E - 1)
    elif kind == "twice":
        ids[:, 1:] = ids[:, :1]
    elif kind == "holes":
        odd = torch.tensor([-1, E, 2**31 - 1, -(2**31), -7], dtype=torch.int32)
        holes = torch.rand(M, k, generator=g) < 0.4
        ids[holes] = odd[torch.randint(0, 5, (int(holes.sum()),), generator=g)]
        ids[0] = -1  # a token without any expert
    return ids


@gpu
@pytest.mark.parametrize("M,E,k,N,K,group,dtype,zeros,kind", SHAPES)
def test_gate_up(M, E, k, N, K, group, dtype, zeros, kind):
    T = DT[dtype]
    X = torch.randn(M, K, generator=gen(7)).to(T)
    ids = make_ids(M, E, k, kind, 11)
    Wp, s, z = make_experts(E, 2 * N, K, group, T, zeros, 13)
    got = ops.moe_gate_up_w4a16(E, k, N, K, group, dtype, zeros=kernel_zeros(z))(*operands(X, ids, Wp, s, z))
    assert got.dtype == T and tuple(got.shape) == (M, k, N)
    want, off = ref.moe_gate_up(X, ids, Wp, s, z, group)
    assert_close64(got, want, off, f"gate_up {M, E, k, N, K}")
    empty = (ids < 0) | (ids >= E)
    assert (got.cpu()[empty] == 0).all()


@gpu
@pytest.mark.parametrize("out", ["same", "float32"])
@pytest.mark.parametrize("M,E,k,N,K,group,dtype,zeros,kind", SHAPES)
def test_down(M, E, k, N, K, group, dtype, zeros, kind, out):
    T = DT[dtype]
    H = torch.randn(M, k, K, generator=gen(8)).to(T)
    ids = make_ids(M, E, k, kind, 12)
    if kind == "holes":
        H[(ids < 0) | (ids >= E)] = float("nan")  # nothing of a slot without an expert is looked at
    weights = torch.softmax(torch.randn(M, k, generator=gen(9)), 1)
    Wp, s, z = make_experts(E, N, K, group, T, zeros, 14)
    out_dtype = dtype if out == "same" else "float32"
    got = ops.moe_down_w4a16(E, k, N, K, group, dtype, out_dtype, zeros=kernel_zeros(z))(*operands(H, ids, weights, Wp, s, z))
    assert got.dtype == DT[out_dtype] and tuple(got.shape) == (M, N)
    want, off = ref.moe_down(H, ids, weights, Wp, s, z, group)
    assert_close64(got, want, off, f"down {M, E, k, N, K}")


# M, E, top_k, N, K, group, type, zeros, how ids are spread: tiles of 256 pairs beside tiles of 64 where the counts of all experts are known
# (up to 4096 pairs) and where they are not, and tiles of 32 and 64 of many pairs
MANY = [
    (2048, 5, 2, 3104, 256, 128, "bfloat16", "frac", "spread"),
    (2047, 4, 2, 3104, 128, 32, "float16", 8, "holes"),
    (1365, 3, 3, 4112, 256, 64, "float16", "int", "twice"),
    (4096, 2, 1, 3104, 128, 128, "bfloat16", 7.5, "one"),
    (4100, 7, 2, 4112, 2048, 128, "bfloat16", "frac", "holes"),
    (4200, 6, 2, 4112, 2048, 2048, "float16", 7.5, "spread"),
    (8200, 3, 1, 4112, 2048, 64, "float16", "int", "one"),
    (2100, 9, 2, 48, 96, 96, "bfloat16", "int", "holes"),
    (1100, 300, 4, 32, 64, 32, "float16", "frac", "spread"),
    (2500, 4, 2, 80, 448, 64, "float16", 8, "one"),
]


def some_tokens(M):
    return torch.cat([torch.tensor([0, 1, M - 2, M - 1]), torch.randint(0, M, (60,), generator=gen(M))])


@gpu
@pytest.mark.parametrize("M,E,k,N,K,group,dtype,zeros,kind", MANY)
def test_gate_up_of_many_pairs(M, E, k, N, K, group, dtype, zeros, kind):
    T = DT[dtype]
    X = torch.randn(M, K, generator=gen(7)).to(T)
    ids = make_ids(M, E, k, kind, 11)
    Wp, s, z = make_experts(E, 2 * N, K, group, T, zeros, 13)
    got = ops.moe_gate_up_w4a16(E, k, N, K, group, dtype, zeros=kernel_zeros(z))(*operands(X, ids, Wp, s, z)).cpu()
    some = some_tokens(M)
    want, off = ref.moe_gate_up(X[some], ids[some], Wp, s, z, group)
    assert_close64(got[some], want, off, f"gate_up {M, E, k, N, K}")
    empty = (ids < 0) | (ids >= E)
    assert (got[empty] == 0).all() and torch.isfinite(got).all()
    assert (got[~empty].abs().amax(-1) > 0).all()  # every row was written


@gpu
@pytest.mark.parametrize("M,E,k,N,K,group,dtype,zeros,kind", MANY)
def test_down_of_many_pairs(M, E, k, N, K, group, dtype, zeros, kind):
    T = DT[dtype]
    H = torch.randn(M, k, K, generator=gen(7)).to(T)
    ids = make_ids(M, E, k, kind, 11)
    weights = torch.rand(M, k, generator=gen(5)) + 0.25
    Wp, s, z = make_experts(E, N, K, group, T, zeros, 13)
    got = ops.moe_down_w4a16(E, k, N, K, group, dtype, "float32", zeros=kernel_zeros(z))(*operands(H, ids, weights, Wp, s, z)).cpu()
    some = some_tokens(M)
    want, off = ref.moe_down(H[some], ids[some], weights[some], Wp, s, z, group)
    assert_close64(got[some], want, off, f"down {M, E, k, N, K}")
    empty = ((ids < 0) | (ids >= E)).all(1)
    assert (got[empty] == 0).all() and torch.isfinite(got).all()
    assert (got[~empty].abs().amax(-1) > 0).all()


@gpu
@pytest.mark.parametrize("M", [1, 9, 40, 300])
def test_weights_that_overflow_at_the_end_of_a_row_that_is_no_multiple_of_128(M):
    """15 * 6000 is infinite in binary16: with positive activations so is every sum, and nothing behind the end of a row makes it NaN."""
    E, k, N, K = 4, 2, 32, 160
    ids = make_ids(M, E, k, "spread", 3)
    for zeros in (None, "tensor"):
        z = None if zeros is None else torch.zeros(E, 2 * N, K // 32, dtype=torch.float16)
        Wp = torch.full((E, 2 * N, K // 2), 0xFF, dtype=torch.uint8)
        s = torch.full((E, 2 * N, K // 32), 2.0**-10, dtype=torch.float16)
        s[..., -1] = 6000.0
        X = torch.rand(M, K, generator=gen(1)).half() + 0.5
        got = ops.moe_gate_up_w4a16(E, k, N, K, 32, "float16", zeros=zeros)(*operands(X, ids, Wp, s, z))
        assert (got == float("inf")).all()
        H = torch.rand(M, k, K, generator=gen(2)).half() + 0.5
        got = ops.moe_down_w4a16(E, k, 2 * N, K, 32, "float16", "float32", zeros=zeros)(*operands(H, ids, torch.ones(M, k), Wp, s, z))
        assert (got == float("inf")).all()


@gpu
def test_products_without_scales_and_without_any_expert():
    E, k, N, K = 4, 2, 32, 64
    X = (torch.randn(6, K, generator=gen(1)) * 0.02).half()
    ids = make_ids(6, E, k, "spread", 2)
    Wp, _, _ = make_experts(E, 2 * N, K, 64, torch.float16, None, 3)
    got = ops.moe_gate_up_w4a16(E, k, N, K, 64, with_scales=False, zeros=8)(*operands(X, ids, Wp))
    assert_close64(got, *ref.moe_gate_up(X, ids, Wp, None, 8, 64), "no scales")
    none = torch.full((6, k), -1, dtype=torch.int32)
    h = ops.moe_gate_up_w4a16(E, k, N, K, 64, with_scales=False, zeros=8)(*operands(X, none, Wp))
    assert (h == 0).all()
    w = torch.full((6, k), float("nan"))
    y = ops.moe_down_w4a16(E, k, 2 * N, K, 64, with_scales=False, zeros=8)(*operands(X[:, None].expand(6, k, K).contiguous(), none, w, Wp))
    assert (y == 0).all()


@gpu
@pytest.mark.parametrize("top_k", [1, 3])
def test_no_token(top_k):
    z = torch.empty
    ids = z(0, top_k, dtype=torch.int32, device="cuda")
    Wp = torch.zeros(2, 64, 32, dtype=torch.uint8, device="cuda")
    s = torch.ones(2, 64, 1, dtype=torch.float16, device="cuda")
    assert ops.moe_gate_up_w4a16(2, top_k, 32, 64, 64)(z(0, 64, dtype=torch.float16, device="cuda"), ids, Wp, s).shape == (0, top_k, 32)
    y = ops.moe_down_w4a16(2, top_k, 64, 64, 64)(z(0, top_k, 64, dtype=torch.float16, device="cuda"), ids, z(0, top_k, device="cuda"), Wp, s)
    assert y.shape == (0, 64)


@gpu
@pytest.mark.parametrize("M", [1, 4, 70, 600])
def test_a_token_gets_the_same_bits_whatever_runs_beside_it_and_every_time(M):
    """Within one call and from call to call: no sum depends on timing."""
    E, k, N, K = 8, 2, 96, 256
    X = torch.randn(M, K, generator=gen(1)).bfloat16()
    ids = make_ids(M, E, k, "spread", 2)
    weights = torch.softmax(torch.randn(M, k, generator=gen(9)), 1)
    w1, s1, z1 = make_experts(E, 2 * N, K, 64, torch.bfloat16, "int", 3)
    w2, s2, z2 = make_experts(E, K, N, 96, torch.bfloat16, "frac", 4)
    up, down = ops.moe_gate_up_w4a16(E, k, N, K, 64, "bfloat16", zeros="tensor"), ops.moe_down_w4a16(E, k, K, N, 96, "bfloat16", "float32", zeros="tensor")
    a, b = operands(X, ids, w1, s1, z1), operands(ids, weights, w2, s2, z2)
    h = up(*a)
    y = down(h, *b)
    for _ in range(3):
        h2 = up(*a)
        assert_bit_equal(h2.cpu(), h.cpu(), "hidden")
        assert_bit_equal(down(h2, *b).cpu(), y.cpu(), "y")


# ---- the three together ----------------------------------------------------------------------------------------------------
class Layer:
    def __init__(self, E=16, k=3, N=96, K=192, dtype="bfloat16", seed=0):
        T = DT[dtype]
        self.E, self.k, self.N, self.K, self.T = E, k, N, K, T
        self.bias = torch.randn(E, generator=gen(seed)) * 0.1
        self.w1, self.s1, self.z1 = make_experts(E, 2 * N, K, 64, T, "int", seed + 1)
        self.w2, self.s2, self.z2 = make_experts(E, K, N, 32, T, "int", seed + 2)
        self.route = ops.moe_route(E, k, scoring="sigmoid", n_group=4, topk_group=2, with_bias=True, scaling=1.5)
        self.up = ops.moe_gate_up_w4a16(E, k, N, K, 64, dtype, zeros="tensor")
        self.down = ops.moe_down_w4a16(E, k, K, N, 32, dtype, dtype, zeros="tensor")

    def inputs(self, M, seed):
        return torch.randn(M, self.K, generator=gen(seed)).to(self.T), torch.randn(M, self.E, generator=gen(seed + 1))

    def to_gpu(self):
        self.gpu = [t.cuda() for t in (self.bias, self.w1, self.s1, self.z1, self.w2, self.s2, self.z2)]
        return self

    def __call__(self, x, logits):
        bias, w1, s1, z1, w2, s2, z2 = self.gpu
        weights, ids = self.route(logits, bias)
        return self.down(self.up(x, ids, w1, s1, z1), ids, weights, w2, s2, z2)

    def check(self, y, x, logits):
        weights, ids = ref.moe_route(logits, self.k, "sigmoid", self.bias, 4, 2, True, 1.5)
        h, off = ref.moe_gate_up(x, ids, self.w1, self.s1, self.z1, 64)
        hidden = h.to(self.T)
        want, off2 = ref.moe_down(hidden, ids, weights.float(), self.w2, self.s2, self.z2, 32)
        # the hidden row may have been rounded to either neighbour: off by `off` and half a step
        _, mags = ref._moe_products(lambda t, j: (off + h.abs() * torch.finfo(self.T).eps / 2)[t, j].to(self.T), ids, self.w2, self.s2, self.z2, 32, self.T)
        slack = (weights[:, :, None] * mags).sum(1) * 1.02 + 1e-6  # (`mags` is made of slacks rounded to the type: 1 % is more than two of its steps)
        assert_close64(y, want, off2 + slack, "layer")


@gpu
@pytest.mark.parametrize("M", [1, 9, 70, 333])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_layer(M, dtype):
    layer = Layer(dtype=dtype).to_gpu()
    x, logits = layer.inputs(M, 5)
    layer.check(layer(x.cuda(), logits.cuda()), x, logits)


@gpu
@pytest.mark.parametrize("M", [1, 12, 200])
def test_layer_captured_and_replayed_with_other_inputs(M):
    layer = Layer().to_gpu()
    x, logits = (t.cuda() for t in layer.inputs(M, 5))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x, logits)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x, logits)
    for rep in range(4):
        xr, lr = (t.cuda() for t in layer.inputs(M, 20 + rep))
        x.copy_(xr), logits.copy_(lr)
        want = layer(xr, lr)
        y.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert_bit_equal(y.cpu(), want.cpu(), f"replay {rep}")
        want.sort()


@gpu
def test_layers_on_several_streams_at_once():
    layer = Layer().to_gpu()
    sizes = [1, 40, 300, 7]
    ins = [tuple(t.cuda() for t in layer.inputs(M, 30 + i)) for i, M in enumerate(sizes)]
    want = [layer(*a) for a in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sizes]
    for _ in range(3):
        got = []
        for st, a in zip(streams, ins):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(layer(*a))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert_bit_equal(g.cpu(), w.cpu(), "streams")


@gpu
def test_an_explicit_stream():
    layer = Layer().to_gpu()
    x, logits = (t.cuda() for t in layer.inputs(33, 5))
    want = layer(x, logits)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    bias, w1, s1, z1, w2, s2, z2 = layer.gpu
    weights, ids = layer.route(logits, bias, stream=st.cuda_stream)
    h = layer.up(x, ids, w1, s1, z1, stream=st.cuda_stream)
    y = layer.down(h, ids, weights, w2, s2, z2, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert_bit_equal(y.cpu(), want.cpu(), "explicit stream")


# ---- refusals (no GPU: arguments are checked before anything is launched) ------------------------------------------------------
FAKE, ODD, NULL = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1002), ctypes.c_void_p(0)


def _rejected(rc, *needles):
    assert rc != 0
    msg = _abi.last_error()
    for n in needles:
        assert n in msg, msg


def test_route_refuses():
    f = _abi.load().tlq_moe_route

    def call(logits=FAKE, bias=NULL, w=FAKE, ids=FAKE, M=4, E=64, k=6, g=1, kept=1, scoring=0, dtype=_abi.F32):
        return f(logits, bias, w, ids, M, E, k, g, kept, scoring, 1, 1.0, dtype, NULL)

    _rejected(call(M=-1), "bad shape")
    _rejected(call(E=0), "bad shape")
    _rejected(call(E=1025), "1024")
    _rejected(call(g=3), "n_group=3")
    _rejected(call(g=0), "n_group=0")
    _rejected(call(E=1024, g=128), "n_group=128")
    _rejected(call(g=8, kept=9), "topk_group=9")
    _rejected(call(g=8, kept=0), "topk_group=0")
    _rejected(call(k=0), "top_k=0")
    _rejected(call(k=65, E=128), "top_k=65")
    _rejected(call(k=9, g=8, kept=1), "top_k=9", "8 experts")
    _rejected(call(scoring=2), "scoring 2")
    _rejected(call(dtype=_abi.I8), "in_dtype")
    for name in ("logits", "w", "ids"):
        _rejected(call(**{name: NULL}), "null pointer")
        _rejected(call(**{name: ODD}), "misaligned")
    _rejected(call(bias=ODD), "misaligned")
    assert call(M=0, logits=NULL, w=NULL, ids=NULL) == 0


def test_products_refuse():
    lib = _abi.load()
    plenty = 1 << 40

    def up(x=FAKE, ids=FAKE, w=FAKE, s=NULL, z=NULL, h=FAKE, ws=FAKE, n=plenty, M=4, E=8, k=2, N=64, K=128, group=64, dtype=_abi.F16):
        return lib.tlq_moe_gate_up_w4a16(x, ids, w, s, z, h, ws, n, M, E, k, N, K, group, 0.0, dtype, NULL)

    def down(x=FAKE, ids=FAKE, w=FAKE, s=NULL, z=NULL, h=FAKE, ws=FAKE, n=plenty, M=4, E=8, k=2, N=64, K=128, group=64, dtype=_abi.F16, weights=FAKE, out=_abi.F16):
        return lib.tlq_moe_down_w4a16(x, ids, weights, w, s, z, h, ws, n, M, E, k, N, K, group, 0.0, dtype, out, NULL)

    for f in (up, down):
        _rejected(f(M=-1), "bad shape")
        _rejected(f(E=1025), "bad shape")
        _rejected(f(k=65), "bad shape")
        _rejected(f(k=0), "bad shape")
        _rejected(f(M=1 << 23, k=2), "2^24")
        _rejected(f(N=24), "N=24")
        _rejected(f(N=0), "N=0")
        _rejected(f(K=48), "K=48")
        _rejected(f(K=0), "K=0")
        _rejected(f(group=16), "group=16")
        _rejected(f(group=96), "group=96")
        _rejected(f(dtype=_abi.F32), "in_dtype")
        for name in ("x", "ids", "w", "h"):
            _rejected(f(**{name: NULL}), "null pointer")
            _rejected(f(**{name: ODD}), "aligned")
        _rejected(f(s=ctypes.c_void_p(0x1008)), "aligned")
        _rejected(f(z=ctypes.c_void_p(0x1008)), "aligned")
        _rejected(f(ws=NULL), "workspace")
        _rejected(f(ws=ODD), "workspace")
        assert f(M=0) == 0
    _rejected(up(n=lib.tlq_moe_gate_up_workspace_bytes(4, 8, 2, 64, 128) - 1), "workspace")
    _rejected(down(n=lib.tlq_moe_down_workspace_bytes(4, 8, 2, 64, 128) - 1), "workspace")
    _rejected(down(weights=NULL), "null pointer")
    _rejected(down(weights=ODD), "aligned")
    _rejected(down(out=_abi.I32), "out_dtype")


def test_workspace_sizes():
    lib = _abi.load()
    up, down = lib.tlq_moe_gate_up_workspace_bytes, lib.tlq_moe_down_workspace_bytes
    assert up(0, 8, 2, 64, 64) == up(4, 0, 2, 64, 64) == up(4, 8, 0, 64, 64) == up(4, 2000, 2, 64, 64) == up(4, 8, 2, 0, 64) == up(4, 8, 2, 64, 0) == 0
    assert down(0, 8, 2, 64, 64) == down(4, 8, 2, 0, 64) == down(4, 8, 2, 64, 0) == 0
    for M in (1, 3, 64, 1000, 100000):
        assert 0 < up(M, 8, 2, 64, 64) and up(M, 8, 2, 64, 64) <= up(M + 1, 8, 2, 64, 64) and up(M, 8, 2, 64, 64) % 16 == 0
        assert down(M, 8, 2, 64, 64) >= up(M, 8, 2, 64, 64)
    assert up(16, 8, 2, 64, 8192) >= up(16, 8, 2, 64, 64) + 2 * 32 * 128 * 4  # parts of K


@pytest.mark.parametrize("kwargs,message", [
    (dict(E=0, top_k=1), "E must"), (dict(E=2000, top_k=1), "E must"), (dict(E=8, top_k=0), "top_k"), (dict(E=8, top_k=9), "top_k"),
    (dict(E=8, top_k=2, scoring="max"), "scoring"), (dict(E=8, top_k=2, n_group=3), "n_group"), (dict(E=8, top_k=2, n_group=4, topk_group=5), "topk_group"),
    (dict(E=8, top_k=5, n_group=4, topk_group=2), "chosen groups"), (dict(E=8, top_k=2, in_dtype="int8"), "in_dtype")])
def test_route_factory_refuses(kwargs, message):
    with pytest.raises(ValueError, match=message):
        ops.moe_route(**kwargs)


@pytest.mark.parametrize("kwargs,message", [
    (dict(E=0, top_k=1, N=64, K=64), "E must"), (dict(E=8, top_k=65, N=64, K=64), "top_k"), (dict(E=8, top_k=2, N=40, K=64), "N must"),
    (dict(E=8, top_k=2, N=64, K=80), "K must"), (dict(E=8, top_k=2, N=64, K=64, group_size=128), "group_size"),
    (dict(E=8, top_k=2, N=64, K=96, group_size=48), "group_size"), (dict(E=8, top_k=2, N=64, K=64, group_size=64, in_dtype="float32"), "in_dtype"),
    (dict(E=8, top_k=2, N=64, K=64, group_size=64, zeros="yes"), "zeros")])
def test_product_factories_refuse(kwargs, message):
    for factory in (ops.moe_gate_up_w4a16, ops.moe_down_w4a16):
        with pytest.raises(ValueError, match=message):
            factory(**kwargs)
    with pytest.raises(ValueError, match="out_dtype"):
        ops.moe_down_w4a16(8, 2, 64, 64, 64, out_dtype="int8")


@gpu
def test_calls_refuse_what_does_not_fit():
    layer = Layer().to_gpu()
    x, logits = (t.cuda() for t in layer.inputs(4, 5))
    bias, w1, s1, z1, w2, s2, z2 = layer.gpu
    weights, ids = layer.route(logits, bias)
    with pytest.raises(ValueError, match="dtype"):
        layer.up(x, ids.long(), w1, s1, z1)
    with pytest.raises(ValueError, match="shape"):
        layer.up(x, ids[:3], w1, s1, z1)
    with pytest.raises(ValueError, match="shape"):
        layer.up(x, ids, w1[:, :-2].contiguous(), s1, z1)
    with pytest.raises(ValueError, match="contiguous"):
        layer.up(x.t().contiguous().t(), ids, w1, s1, z1)
    with pytest.raises(ValueError, match="device"):
        layer.up(x, ids.cpu(), w1, s1, z1)
    with pytest.raises(ValueError, match="shape"):
        layer.down(layer.up(x, ids, w1, s1, z1), ids, weights[:, :2].contiguous(), w2, s2, z2)
    odd = torch.empty(4 * layer.K + 1, dtype=layer.T, device="cuda")[1:].view(4, layer.K)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        layer.up(odd, ids, w1, s1, z1)
