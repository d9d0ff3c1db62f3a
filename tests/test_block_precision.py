"""What the block operators' sums hold: first sums of adapters that are small beside their row's largest, and their last bits; squares of very long rows."""
import pytest
import torch

from helpers import DT, gen
from oracle import ref
from tilelang_ascend_amd import ops

gpu = pytest.mark.gpu
TYPES = ["float16", "bfloat16"]


def update(L, rank, parts, K, dtype, out_dtype):
    return ops.low_rank_update(L, rank, parts, K, in_dtype=dtype, out_dtype=out_dtype)


def not_more(got, want, off, what):
    got = got.cpu()
    fi = torch.finfo(got.dtype)
    assert torch.isfinite(got).all(), what
    worst = ((got.double() - want).abs() - off - (want.abs() + off).clamp_min(fi.tiny) * (fi.eps / 2)).max().item()
    assert worst <= 0, f"{what}: {worst:.3e} more than allowed"


# M, L, rank, parts, K: single rows; tiles of 16 rows without and with a plan, of 64 in runs of 16 and whole
SIZES = [(3, 2, 16, (64,), 256), (20, 3, 32, (64,), 8224), (20, 3, 128, (64, 32), 512), (300, 3, 16, (48,), 16416), (500, 3, 128, (48,), 256), (900, 3, 64, (64,), 4128), (5300, 2, 32, (32,), 288), (6400, 3, 8, (32,), 64)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("quiet", [12, 20, 28])
@pytest.mark.parametrize("M,L,rank,parts,K", SIZES)
def test_first_sums_far_below_their_rows_largest(M, L, rank, parts, K, quiet, dtype):
    """Every other row of A is 2^-quiet of the others, and half of the outputs have weights of 0 for the loud ones: they are made of the quiet sums alone, and are
    as exact as any."""
    T, g, N = DT[dtype], gen(quiet + M), sum(parts)
    x = torch.randn(M, K, generator=g).to(T)
    a = torch.randn(L, len(parts) * rank, K, generator=g)
    a[:, 0::2] *= 2.0 ** (quiet // 2 - 4)
    a[:, 1::2] *= 2.0 ** (quiet // 2 - 4 - quiet)
    b = torch.randn(L, N, rank, generator=g)
    b[:, : N // 2, 0::2] = 0
    b[:, N // 2:, 0::2] *= 2.0**-6
    a, b = a.to(T), b.to(T)
    scaling = torch.rand(L, generator=g) + 0.5
    ids = torch.randint(0, L, (M,), generator=g, dtype=torch.int32)
    some = torch.arange(M) if M <= 100 else torch.cat([torch.tensor([0, M - 1]), torch.randint(0, M, (40,), generator=g)])
    for out in (dtype, "float32"):
        y = torch.zeros(M, N, dtype=DT[out])
        got = update(L, rank, parts, K, dtype, out)(*[v.cuda() for v in (x, y, ids, a, b, scaling)])
        want, off = ref.low_rank_update(x[some], y[some], ids[some], a, b, scaling, parts)
        not_more(got[some.cuda()], want, off, f"quiet sums {out}")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,L,rank,parts,K", SIZES)
def test_first_sums_enter_the_second_product_whole(M, L, rank, parts, K, dtype):
    """Whole numbers whose first sums fp32 holds exactly, in any order (below 2^24), and one power of two a row of B: fp32 sums rounded once are those sums, bit for
    bit; of float16 22 bits are handed on, each piece rounded to 11 (2^-11 of what it is made of)."""
    T, g, N = DT[dtype], gen(M), sum(parts)
    top = min(2047 if T == torch.float16 else 255, int((2**24 / K) ** 0.5))
    x = torch.randint(0, top + 1, (M, K), generator=g).to(T)
    a = torch.randint(-top, top + 1, (L, len(parts) * rank, K), generator=g).to(T)
    a[:, ::2] = a[:, ::2].abs()
    chosen = torch.randint(0, rank, (L, N), generator=g)
    b = torch.zeros(L, N, rank).scatter_(2, chosen[:, :, None], torch.randint(-8, 5, (L, N, 1), generator=g).float().exp2()).to(T)
    scaling = torch.randint(-3, 4, (L,), generator=g).float().exp2()
    ids = torch.randint(0, L, (M,), generator=g, dtype=torch.int32)
    y = torch.zeros(M, N)
    got = update(L, rank, parts, K, dtype, "float32")(*[v.cuda() for v in (x, y, ids, a, b, scaling)]).cpu()
    want = torch.zeros(M, N, dtype=torch.float64)
    for e in range(L):
        rows, begin = ids == e, 0
        h = x[rows].double() @ a[e].double().T
        assert h.abs().max() < 2**24
        for p, n in enumerate(parts):
            want[rows, begin: begin + n] = scaling[e].double() * (h[:, p * rank: (p + 1) * rank] @ b[e, begin: begin + n].double().T)
            begin += n
    assert (want.abs() > 2**16).any()
    off = want.abs() * (2.0**-22 + 2.0**-24) if T == torch.float16 else 0
    assert ((got.double() - want).abs() <= off).all(), f"{((got.double() - want).abs() / want.abs().clamp_min(2.0**-30)).max().item():.3e}"


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [32769 + 7, (1 << 22) + 5, 1 << 24])
@pytest.mark.parametrize("value", [1.1, 0.7])
def test_norm_of_very_long_rows(N, value, dtype):
    """Equal values, whose squares all round a growing sum the same way: sums of at most 64 in fp32, those in more, a tree of 256."""
    x = torch.full((2, N), value).to(DT[dtype])
    x[1, ::3] *= -0.5
    w = torch.ones(N, dtype=DT[dtype])
    y, q, s = ops.residual_rms_norm(N, outputs="both", with_residual=False, in_dtype=dtype)(x.cuda(), w.cuda())
    _, want, _ = ref.residual_rms_norm(x, None, w, 1e-6)
    rel = ((64 + 16) / 2 + 8) * 2.0**-24
    not_more(y, want, want.abs() * rel, "y")
    assert ((s.cpu().double() - ref.row_scales(want)).abs() <= ref.row_scales(want) * (rel + 2.0**-22)).all(), (s, ref.row_scales(want))
    assert (q[0] == 127).all() and (q[1, ::3].abs() == 64).all()  # (127 / 2: the even one)
