"""Launches of the largest sizes that the 4-bit linears, the attention and the
bounded cache document, without a GPU (tests/host/grids.py): fewer than 2^32
threads along an axis of a grid, at most 65535 workgroups along its second."""
import json
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
HOST = ROOT / "tests" / "host"
PKG = ROOT / "spikingbrain-cpu_amd" / "sbq"
WS = 1 << 50  # (bytes of workspace claimed)


@pytest.fixture(scope="module")
def grids(tmp_path_factory):
    so = tmp_path_factory.mktemp("trace") / "launch_trace.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-std=c++17", "-Wall", str(HOST / "launch_trace.cpp"),
                    "-o", str(so)], check=True)

    def run(calls):
        r = subprocess.run([sys.executable, str(HOST / "grids.py"), str(so), str(PKG / "libsbq.so"), str(PKG)],
                           input=json.dumps(calls), capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        return json.loads(r.stdout)

    return run


def check(grids, calls):
    for call, got in zip(calls, grids(calls)):
        assert got["rc"] == 0 and got["launches"], call
        for grid, block in got["launches"]:
            assert all(1 <= g and g * b < 1 << 32 for g, b in zip(grid, block)) and max(grid[1:]) <= 65535, (call, grid, block)


BIG = [(1 << 16, 1 << 16), (1 << 20, 1 << 18), ((1 << 20) + 5, (1 << 20) + 3), (3, 1 << 30), (1 << 30, 1), (1 << 30, 1900)]


@pytest.mark.parametrize("group", [32, 64, 128])
def test_4_bit_weights(grids, group):
    check(grids, [["sbq_quantize_groups", "@0", dt, N, K, K, group, "@1", K, "@2", None] for N, K in BIG for dt in (0, 1, 2)]
          + [["sbq_repack_w4", "@0", N, K, K, "@1", group, "@2", "@3", None] for N, K in BIG]
          + [["sbq_unpack_w4", "@0", "@1", N, K, group, "@2", K, "@3", None] for N, K in BIG]
          + [["sbq_linear_w4", "@0", dt, M, K, K, "@1", "@2", "@3", N, group, "@4", dt, N, None] for N, K in BIG
             for dt in (0, 2) for M in (1, 2, 4, 8, 16, 64, 70)]
          + [["sbq_linear_w4", "@0", 0, (1 << 31) - 1, 64, 64, "@1", "@2", None, 16, group, "@4", 0, 16, None]])


def test_attention(grids):
    def call(T, heads, kv, D, slots, qt, ct, weight):
        return ["sbq_tree_attention", "@0", qt, T, heads, D, heads * D, D, "@1", "@2", ct, slots, kv, kv * D, D, "@3", "@4",
                "@5", "@6", kv * D, D, None, 0, 0, 0.1, "@7", heads * D, D, "@8" if weight else None, "@9", WS, None]

    sizes = [(1, 1, 1, 1, 1 << 30), (1, 8, 8, 128, 1 << 30), (64, 32, 8, 128, 1 << 28), (3, 4, 1, 33, 1 << 27),
             (1024, 65536, 65536, 64, 100), (1024, 65536, 1, 256, 100), (1024, 65536, 8, 128, 1 << 20),
             (1, 65536, 65536, 80, 1 << 24), (9, 16, 16, 256, (1 << 30) - 1), (256, 8, 8, 64, 1 << 30)]
    check(grids, [call(*s, qt, ct, w) for s in sizes for qt, ct in ((0, 0), (1, 1), (2, 2), (0, 2)) for w in (False, True)])


def test_bounded_cache(grids):
    def append(slots, T, kv, D, nt, ct):
        return ["sbq_kv_append", "@0", "@1", slots, "@2", "@2", slots // 3, "@3", "@4", ct, kv, D, kv * D, D, "@5", "@6", nt, T,
                kv * D, D, "@7", WS, None]

    def take(slots, capacity, kv, D, ct):
        return ["sbq_kv_take", "@0", "@1", slots, "@2", "@3", "@4", ct, kv, D, kv * D, D, capacity, 1, "@5", "@6", "@7", "@8",
                "@9", kv * D, D, "@10", WS, None]

    check(grids, [append(1 << 30, T, kv, D, nt, 2) for T in (1, 2, 512, 513, 1 << 24, (1 << 24) - 1, 1 << 30)
                  for kv, D in ((1, 1), (8, 128), (65536, 256)) for nt in (0, 2)]
          + [take(slots, cap, 8, 128, 1) for slots in (4096, 1 << 30) for cap in (1, 4096, 1 << 24, (1 << 24) + 7, 1 << 30)])
