"""What the norm, the gated activation and the adapters would launch, asked without a GPU (tests/launch_arguments.c): grids within the limits, every row and
output with a work-group of its own, the adapters' plan and sums inside of the workspace; and their kernels without spilled registers."""
import json
import os
import re
import shutil
import subprocess
import sys

import pytest

from tilelang_ascend_amd import _abi, build

HERE = os.path.dirname(os.path.abspath(__file__))
PRELUDE = """
import ctypes, json, random, struct, sys
rec = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
lib = ctypes.CDLL(sys.argv[2])
i64, i32, f32, p = ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_void_p
rec.recorder_name.restype = lib.tlq_last_error.restype = ctypes.c_char_p
lib.tlq_residual_rms_norm.argtypes = [p] * 7 + [i64] * 2 + [f32, i32, i32, p]
lib.tlq_gated_silu.argtypes = [p] * 4 + [i64] * 2 + [i32, i32, p]
lib.tlq_low_rank_update_workspace_bytes.argtypes, lib.tlq_low_rank_update_workspace_bytes.restype = [i64] * 5, i64
lib.tlq_low_rank_update.argtypes = [p] * 8 + [i64] * 8 + [i32, i32, p]
X, R, W, H, Y, Q, S, IDS, A, B, WS = (i << 40 for i in range(1, 12))  # (addresses that nothing reads)
def launches(call):
    rec.recorder_clear()
    rc = call()
    assert rc == 0, lib.tlq_last_error()
    out = []
    for i in range(rec.recorder_count()):
        sizes, data = (ctypes.c_uint32 * 6)(), (ctypes.c_ubyte * 112)()
        rec.recorder_get(i, sizes, data)
        name = rec.recorder_name(i).decode()
        g, b = list(sizes[:3]), list(sizes[3:])
        assert b[1] == b[2] == 1 and b[0] <= 1024 and b[0] % 64 == 0 and g[0] * b[0] < 2**32 and 0 < g[1] <= 65535 and g[2] == 1 and g[0] > 0, (name, g, b)
        out.append((name, g, b[0], bytes(data)))
    return out
"""


@pytest.fixture(scope="module")
def recorder(tmp_path_factory):
    if not shutil.which("gcc"):
        pytest.skip("a C compiler wanted")
    out = str(tmp_path_factory.mktemp("recorder") / "launch_arguments.so")
    subprocess.run(["gcc", "-O1", "-Wall", "-Wextra", "-shared", "-fPIC", os.path.join(HERE, "launch_arguments.c"), "-o", out], check=True)
    return out


def ask(recorder, code):
    done = subprocess.run([sys.executable, "-c", PRELUDE + code + "\nprint(json.dumps(result))", recorder, _abi.library_path()], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-3000:]
    return json.loads(done.stdout)


def test_update_stays_inside_of_its_workspace(recorder):
    """Random sizes of every range: the second product reads the parts that the first writes, sums and plan end inside of the workspace, and all tiles and
    blocks of outputs have a work-group."""
    result = ask(recorder, """
rng, result = random.Random(5), set()
log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))
cases = [(64, 1, 8, (16,), 32), (65, 4096, 128, (16, 16, 16), 32), (1, 1, 8, (16,), 32), ((1 << 24) - 1, 1, 8, (16,), 32), ((1 << 24) - 1, 4096, 8, (16,), 32), (64, 1, 16, ((1 << 24) - 16,) * 3, 64),
         (2000, 4096, 16, ((1 << 24) - 16,) * 3, 64), (8192, 256, 32, (14336,), 4096), (8192, 257, 32, (14336,), 4096)]
while len(cases) < 3000:
    cases.append((log(1, rng.choice([64, 2000, 1 << 24])), log(1, 4096), rng.choice([8, 16, 32, 64, 128]), tuple(16 * log(1, 4096) for _ in range(rng.randint(1, 3))), 32 * log(1, 2048)))
for M, L, rank, parts, K in cases:
    rows, N = rank * len(parts), sum(parts)
    size = lib.tlq_low_rank_update_workspace_bytes(M, L, rank, len(parts), K)
    got = launches(lambda: lib.tlq_low_rank_update(X, Y, IDS, A, B, S, H, WS, size, M, L, rank, *parts, *[0] * (3 - len(parts)), K, rng.choice([0, 1]) if 0 else 1, rng.choice([1, 2]), None))
    what = (M, L, rank, parts, K)
    names = [n for n, _, _, _ in got]
    if len(got) == 1:  # a work-group a row and run of outputs: nothing in the workspace
        name, g, threads, data = got[0]
        x, y, a, b = struct.unpack("QQQQ", data[8:40])
        l, n, k, r, end0, end1, per_group, all_groups, groups0, groups1 = struct.unpack("iiiiiiiiii", data[56:96])
        assert struct.unpack("i", data[96:100]) == (M,), what
        assert "low_rank_row_kernel" in name and (x, y, a, b) == (X, Y, A, B) and (l, n, k, r, end0, end1) == (L, N, K, rows, parts[0], sum(parts[:2])), what
        outputs = 512 * 8 // rank * per_group
        need = [-(-n // outputs) for n in parts] + [0, 0]
        assert threads == 512 and g[0] == (M if M < 8 else -(-M // 8) * 8) * all_groups and (groups0, groups1 - groups0, all_groups - groups1) == tuple(need[:3]) and 512 * per_group < 2**31, what
        result.add((1, 0, False))
        continue
    assert len(got) == (2 if M <= 64 else 3), what
    down, up = got[-2], got[-1]
    ids, plan, m, l, x, a, sums, k, r, part_k, groups, total, subs = struct.unpack("QQiiQQQiiiiii", down[3][:72])
    by_tiles = "down_tile" in down[0]
    tile_rows = 64 if by_tiles else 16 * subs
    result.add((len(got), tile_rows, by_tiles))
    most = M if M <= 64 else M // tile_rows + min(L + 1, M)  # tiles, at most
    assert (ids, m, l, x, a, k, r, total) == (IDS, M, L, X, A, K, rows, most * subs) and subs in ((1,) if by_tiles or M <= 64 else (1, 4)), what
    assert ("Li4E" in up[0].split("up_kernel")[1].split("Li8E")[0].split("Li16E")[0].split("Li32E")[0].split("Li64E")[0].split("Li128E")[0]) == (tile_rows == 64), (what, up[0])
    cut = down[1][1]
    assert part_k % 64 == 0 and (cut - 1) * part_k < K <= cut * part_k, what
    assert down[1][0] == (-(-total // 8)) * 8 * groups, what
    per = 16 if not by_tiles else 16 * int(down[0].split("down_tile_kernel")[1].split("Li")[1][0])
    assert groups == -(-rows // per), (what, down[0], groups)
    assert sums % 16 == 0 and sums >= WS and sums + cut * M * rows * 4 <= WS + size, what
    if M > 64:
        assert plan == WS and WS + (64 + (M + 3) // 4 * 4 + 4 * most) * 4 <= sums, what
    ids, plan2, m, l, y, b, scaling, sums2, out, n, r, parts2, end0, end1, per_group, all_groups, groups0, groups1 = struct.unpack("QQiiQQQQQiiiiiiiii", up[3][:100])
    assert (ids, plan2, m, l, y, b, scaling, sums2, out, n, r, parts2) == (IDS, plan, M, L, Y, B, S, sums, H, N, rows, cut), what
    assert (end0, end1) == (parts[0], sum(parts[:2])), what
    blocks = [-(-n // 128) for n in parts] + [0, 0]
    assert groups0 * per_group >= blocks[0] and (groups1 - groups0) * per_group >= blocks[1] and (all_groups - groups1) * per_group >= blocks[2], what
    assert up[1][0] == most * all_groups, what
result = sorted(result)
""")
    assert result == [[1, 0, False], [2, 16, False], [3, 16, False], [3, 64, False], [3, 64, True]]


def test_rows_have_work_groups(recorder):
    result = ask(recorder, """
rng, result = random.Random(6), set()
log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))
cases = [((1 << 31) - 1, 1), (1, (1 << 30) - 1), (5, 32768), (5, 32769), ((1 << 31) - 1, 64), (100000, 513)]
while len(cases) < 1500:
    M, N = log(1, rng.choice([100, 10000, (1 << 31) - 1])), log(1, rng.choice([600, 40000]))
    if M * N < 1 << 38:  # (what a machine could hold)
        cases.append((M, N))
for M, N in cases:
    off = rng.choice([0, 0, 2])
    out = rng.choice([(Y, None, None), (None, Q, S), (Y, Q, S)])
    got = launches(lambda: lib.tlq_residual_rms_norm(X + off, R, W, H, *out, M, N, 1e-6, 1, 0, None))
    assert len(got) == 1
    name, g, threads, data = got[0]
    m, n, _, blocks = struct.unpack("qiii", data[56:76])
    assert (m, n, blocks) == (M, N, g[0]) and g[1] == 1, (M, N, name)
    result.add("long" if "long" in name else "rows")
    if "rows" in name:
        ch, wpr, th = (int(v) for v in __import__("re").findall(r"Li(\\d+)E", name)[:3])
        assert th == threads and ch * wpr * 512 >= N and threads // 64 % wpr == 0, (M, N, name)
        assert ("Lb1" in name) == bool(off or N % 8), (M, N, name)
    got = launches(lambda: lib.tlq_gated_silu(X + off, *out, M, N, 0, 0, None))
    if out[1] is None:
        done = 0
        for name, g, threads, data in got:
            x, y, q, s, m, n = struct.unpack("QQQQqi", data[:44])
            assert x == X + off + done * 2 * N * 2 and y == Y + done * N * 2 and n == N and threads == 256
            chunks = -(-N // 8)
            segs, rows = -(-chunks // 256), 1 if chunks > 128 else 256 // chunks
            assert g[0] == -(-m // rows) * segs, (M, N, g)
            done += m
        assert done == M, (M, N)
        result.add("flat")
    else:
        assert len(got) == 1 and ("long" in got[0][0]) == (N > 32768), (M, N)
        result.add("gated rows")
result = sorted(result)
""")
    assert result == ["flat", "gated rows", "long", "rows"]


@pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"), reason="hipcc not available")
@pytest.mark.parametrize("source,kernels", [("norm_act.hip", ["norm_rows_kernel", "gated_rows_kernel", "gated_flat_kernel"]),
                                            ("low_rank.hip", ["low_rank_down_kernel", "low_rank_down_tile_kernel", "low_rank_up_kernel", "low_rank_plan_kernel", "low_rank_row_kernel"])])
def test_no_register_spills(tmp_path, source, kernels):
    cmd = [build.hipcc_path(), *build.HIPCC_FLAGS, "-Rpass-analysis=kernel-resource-usage", "-c", f"{build.CSRC_DIR}/{source}", "-o", str(tmp_path / "out.o")]
    res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert res.returncode == 0, res.stdout[-2000:]
    seen = dict.fromkeys(kernels, 0)
    for b in re.split(r"remark: Function Name: ", res.stdout)[1:]:
        of = [k for k in kernels if k in b.split()[0]]
        if of:
            seen[of[0]] += 1
            assert int(re.search(r"ScratchSize \[bytes/lane\]: (\d+)", b).group(1)) == 0 and int(re.search(r"VGPRs Spill: (\d+)", b).group(1)) == 0, b.split()[0]
    assert min(seen.values()) >= 2, seen
