"""Where the paged cache's calls may write: outputs in any order of their axes, and
outputs that meet an input."""
import json
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from sbq.state import DevicePagedKVBuffer

ROOT = Path(__file__).resolve().parents[1]
HOST, PKG = ROOT / "tests" / "host", ROOT / "spikingbrain-cpu_amd"


def _grids(tmp_path, calls):
    """The C ABI's answers without a GPU."""
    so = tmp_path / "launch_trace.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-std=c++17", "-Wall", str(HOST / "launch_trace.cpp"), "-o", str(so)],
                   check=True)
    r = subprocess.run([sys.executable, str(HOST / "grids.py"), str(so), str(PKG / "sbq" / "libsbq.so"), str(PKG / "sbq")],
                       input=json.dumps(calls), capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return [got["rc"] for got in json.loads(r.stdout)]


def test_orders_of_the_outputs_axes(tmp_path):
    """Every order of [sequences, tokens, heads] packed without a gap is taken, one element less in a stride refused."""
    B, T, H, D = 3, 5, 4, 24
    cache = ["@1", "@2", "@3", "@4", 3, 8, 16, H, D, "@5", B, 4, "@6"]
    n = (B, T, H)
    calls, want = [], []
    for order in ((0, 1, 2), (0, 2, 1), (1, 0, 2), (1, 2, 0), (2, 0, 1), (2, 1, 0)):  # from the outermost in
        strides, span = [0, 0, 0], D
        for axis in reversed(order):
            strides[axis], span = span, span * n[axis]
        for axis in (None, 0, 1, 2):
            s = [x - (i == axis) for i, x in enumerate(strides)]
            calls.append(["sbq_paged_attention", "@0", 0, T, H, T * H * D, H * D, D, *cache, None, None, 0, 0.1, "@8", *s, "@9",
                          1 << 40, None])
            calls.append(["sbq_paged_read", *cache, "@7", T, "@8", "@9", 0, *s, None])
            want += [0 if axis is None else -1] * 2
    for strides, rc in (((0, H * D, D), -1), ((T * H * D, 0, D), -1), ((T * H * D, H * D, 0), -1), ((1 << 40, H * D, D), 0)):
        calls.append(["sbq_paged_read", *cache, "@7", T, "@8", "@9", 0, *strides, None])
        want.append(rc)
    # an axis of one entry has any stride
    calls.append(["sbq_paged_read", *cache, "@7", 1, "@8", "@9", 0, H * D, 0, D, None])
    want.append(0)
    assert _grids(tmp_path, calls) == want


@pytest.mark.gpu
def test_outputs_in_other_orders(dev):
    B, T, H, heads, dim = 3, 4, 6, 2, 40
    g = torch.Generator().manual_seed(1)
    for room in (64, 4000):
        b = DevicePagedKVBuffer(B, heads, dim, 20, 16, room // 16, device=dev)
        for i in range(B):
            b.reserve(i, 60)
        k, v = [torch.randn(B, 50, heads, dim, generator=g).to(dev) for _ in range(2)]
        b.append(k, v)
        q = torch.randn(B, T, H, dim, generator=g).to(dev)
        want = b.attend(q)
        for order in ((1, 0, 2), (2, 1, 0), (2, 0, 1), (0, 2, 1), (1, 2, 0)):
            sizes = [(B, T, H)[i] for i in order]
            out = torch.full((*sizes, dim), 7.0, device=dev).permute(*[order.index(i) for i in range(3)], 3)
            assert out.shape == q.shape
            assert b.attend(q, out=out) is out and torch.equal(out, want)
