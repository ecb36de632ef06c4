"""Where the paged cache's calls may write: outputs in any order of their axes, and
outputs that meet an input."""
import json
import random
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from sbq import _lib, quant
from sbq.quant import _meet
from sbq.state import DevicePagedKVBuffer, _apart_rope, _plainly_apart, qk_norm_rope

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


# ---------------------------------------------------------------------------
# outputs that meet an input
# ---------------------------------------------------------------------------
def _bytes(t):
    offsets = torch.zeros(1, dtype=torch.long)
    for n, s in zip(t.shape, t.stride()):
        offsets = (offsets[:, None] + torch.arange(n) * s).reshape(-1)
    size = t.element_size()
    return {t.data_ptr() + o * size + i for o in offsets.tolist() for i in range(size)}


def test_meet_against_every_byte():
    """Memory that is shared is always found, and views of one projection's output are apart."""
    rng = random.Random(0)
    storage = torch.zeros(1 << 14)
    apart = 0
    for _ in range(4000):
        views = []
        step = rng.randrange(1, 200)
        for _ in range(2):
            x = storage.view(torch.float16) if rng.random() < 0.2 else storage
            shape = [rng.choice((0, 1, 2, 3, 5)) if rng.random() < 0.1 else rng.randrange(1, 5) for _ in range(4)]
            stride = [rng.choice((step, step, 3 * step, 4 * step, rng.randrange(0, 60))) for _ in range(3)] + [rng.choice((1, 1, 2))]
            views.append(x.as_strided(shape, stride, rng.randrange(0, 400)))
        shared = bool(_bytes(views[0]) & _bytes(views[1]))
        meet = _meet(*views)
        assert meet or not shared, [(v.shape, v.stride(), v.storage_offset()) for v in views]
        assert meet == _meet(views[1], views[0]) or not shared
        apart += not meet
    assert apart > 300
    for B, T in ((1, 1), (1, 7), (3, 1), (3, 4)):
        qkv = torch.zeros(B, T, (6 + 2 + 2) * 8)
        q, k, v = [x.unflatten(-1, (-1, 8)) for x in qkv.split([48, 16, 16], -1)]
        assert not _meet(q, k) and not _meet(k, v) and not _meet(v, q) and not _meet(q.flatten(0, 1), k.flatten(0, 1))
        assert _meet(q, q) and _meet(q, q[..., 1:, :]) and _meet(q[..., -1:, :], q)
        assert _meet(q, qkv[..., 40:56].unflatten(-1, (-1, 8)))


def test_norms_outputs_apart():
    T, H, kv, D = 5, 4, 2, 8
    others = (torch.zeros(T, dtype=torch.long), torch.zeros(4), None, torch.zeros(8))
    qkv = torch.zeros(T, (H + 2 * kv) * D)
    q, k, v = [x.unflatten(1, (-1, D)) for x in qkv.split([H * D, kv * D, kv * D], 1)]
    new_q, new_k = torch.zeros(T, H, D), torch.zeros(T, kv, D)
    both = torch.zeros(T, H + kv, D)
    for a in ((q, k, q, k), (q, k, new_q, new_k), (q, k, q, new_k), (q, k, new_q, k), (q, k, both[:, :H], both[:, H:]),
              (q, k, q, v), (q, None, q, None), (q, None, new_q, None), (q[:1], k[:1], q[:1].as_strided((1, H, D), (7, D, 1)), k[:1])):
        _apart_rope(*a, others)
    shifted = qkv[:, D:(H + 1) * D].unflatten(1, (H, D))
    for a in ((q, k, shifted, new_k), (q, None, shifted, None), (q, k, new_q, q[:, :kv]), (q, k, new_q, new_q[:, 1:3]),
              (q, k, both[:, :H], both[:, H - 1:H - 1 + kv]), (q[1:], k[1:], q[:-1], k[1:]), (q, q[:, :kv], q, q[:, :kv]),
              (new_q, k, new_q.as_strided((T, H, D), (D, T * D, 1)), k)):
        with pytest.raises(ValueError, match="apart"):
            _apart_rope(*a, others)
    # in place: the quick answer is never one that the other refuses, and is one for a projection's rows
    assert _plainly_apart(q, k, others) and _plainly_apart(q, None, others)
    rng = random.Random(1)
    room = torch.zeros(4096)
    found = 0
    for _ in range(3000):
        T1, step = rng.randrange(1, 5), rng.choice((64, 90, 200))
        a, b = [room.as_strided((T1, rng.randrange(1, 5), 8), (rng.choice((step, step, step, 70)), rng.choice((8, 8, 12, 0)), 1),
                                rng.randrange(0, 300)) for _ in range(2)]
        o = (room[rng.randrange(0, 1500):][:4], None)
        if _plainly_apart(a, b, o):
            found += 1
            assert not _bytes(a) & _bytes(b) and not (_bytes(a) | _bytes(b)) & _bytes(o[0])
            _apart_rope(a, b, a, b, o)
    assert found > 100
    # the positions or the weights as an output
    for i in (0, 1, 3):
        room = torch.zeros(T * H * D + 64)
        o = list(others)
        o[i] = room.view(torch.long)[T * H * D // 2 - 2:][:T] if i == 0 else room[T * H * D - 2:][:8 if i == 3 else 4]
        with pytest.raises(ValueError, match="apart"):
            _apart_rope(q, k, room[:T * H * D].view(T, H, D), k, tuple(o))


def test_verification_written_over_an_input(tmp_path):
    def call(V=20000, kept="@5", token="@6", ws="@7", q="@1", T=2, counts="@4"):
        return ["sbq_verify_drafts", "@0", (T + 1) * V, V, q, T * V, V, 0, 3, T, V, "@2", "@3", counts, kept, token, ws, 1 << 20, None]

    bad = [call(kept=at) for at in ("@0", "@1", "@2", "@3", "@4", "@6")] + [call(token=at) for at in ("@0", "@2", "@3", "@4")] \
        + [call(ws=at) for at in ("@0", "@1", "@2", "@3", "@4", "@5", "@6")]
    good = [call(), call(V=100, ws="@0"), call(T=0, q="@5"), call(q=None), call(counts=None)]  # (a short row takes no workspace)
    assert _grids(tmp_path, bad) == [-1] * len(bad) and _grids(tmp_path, good) == [0] * len(good)


@pytest.mark.gpu
def test_outputs_that_meet_an_input_are_refused(dev):
    B, T, H, heads, dim = 2, 3, 4, 2, 32
    b = DevicePagedKVBuffer(B, heads, dim, 8, 16, 400, device=dev)
    for i in range(B):
        b.reserve(i, 40)
    qkv = torch.randn(B, T, (H + 2 * heads) * dim, device=dev)
    q, k, v = [x.unflatten(-1, (-1, dim)) for x in qkv.split([H * dim, heads * dim, heads * dim], -1)]
    b.append(k, v)
    kept = [t.clone() for t in (qkv, b.k, b.v, b.table, b.length)]
    want = b.attend(q)
    counts = torch.full((B,), T, device=dev)
    room = torch.empty(1 << 22, device=dev)
    size = q.numel()
    pool = b.v.as_strided((B, T, H, dim), (T * H * dim, H * dim, dim, 1))
    for a in (dict(out=q), dict(out=qkv[..., dim:(H + 1) * dim].unflatten(-1, (H, dim))), dict(out=pool),
              dict(workspace=room, out=room[5:size + 5].view(q.shape)), dict(workspace=b.k.as_strided((b.k.numel(),), (1,))),
              dict(workspace=qkv), dict(workspace=counts, counts=counts)):
        with pytest.raises(ValueError, match="apart"):
            b.attend(q, **a)
    # beside the queries, in their own rows
    wide = torch.zeros(B, T, 2 * H * dim, device=dev)
    wide[..., :H * dim] = q.flatten(2)
    out = wide[..., H * dim:].unflatten(-1, (H, dim))
    assert torch.equal(b.attend(wide[..., :H * dim].unflatten(-1, (H, dim)), out=out), want)
    assert torch.equal(b.attend(q, out=room[:size].view(q.shape), workspace=room[size:]), want)
    for t, old in zip((qkv, b.k, b.v, b.table, b.length), kept):
        assert torch.equal(t, old)
    f, pos, w = torch.rand(dim // 2, device=dev), torch.arange(B * T, device=dev), torch.rand(dim, device=dev)
    q3, k3 = q.flatten(0, 1), k.flatten(0, 1)
    for a in (dict(q_out=qkv.flatten(0, 1)[:, dim:(H + 1) * dim].unflatten(1, (H, dim))), dict(k_out=q3[:, :heads]),
              dict(q_out=q3, k_out=q3[:, 1:1 + heads])):
        with pytest.raises(ValueError, match="apart"):
            qk_norm_rope(q3, k3, pos, f, w, w, **a)
    assert torch.equal(qkv, kept[0])
    new = qk_norm_rope(q3, k3, pos, f, w, w)
    qk_norm_rope(q3, k3, pos, f, w, w, q_out=q3, k_out=k3)
    assert torch.equal(q3, new[0]) and torch.equal(k3, new[1])
    # the verification's workspace
    target = torch.softmax(torch.randn(1, 2, 20000, device=dev), -1)
    tokens, u = torch.zeros(1, 1, dtype=torch.long, device=dev), torch.rand(1, 2, device=dev)
    with pytest.raises(ValueError, match="invalid argument"):
        quant.verify_drafts(target, None, tokens, u, workspace=target)


# ---------------------------------------------------------------------------
# the attention's workspace
# ---------------------------------------------------------------------------
def test_places_of_partial_results(tmp_path):
    exe = tmp_path / "paged_parts_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", str(PKG / "csrc"),
                    str(HOST / "paged_parts_check.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.stdout.strip() == "ok", r.stdout + r.stderr


def test_workspace_goes_by_the_chip_not_by_the_sequences():
    """Two partial results for each of at most 768 workgroups, 32 rows of 256 columns
    each, and a note for each of 512 sequences and 384 row tiles: 54 MB."""
    L = _lib.load()
    rng, most = random.Random(2), 0
    calls = [(512, 16, 32, 8, 128, 64, 128, 0, 3), (256, 64, 32, 8, 128, 64, 128, 0, 3), (512, 64, 32, 8, 256, 64, 128, 0, 2),
             (65536, 1, 1, 1, 256, 64, 4096, 0, 4)]
    for _ in range(4000):
        kv = rng.choice((1, 2, 8, 40))
        page = 1 << rng.randrange(4, 11)
        calls.append((rng.choice((1, 7, 64, 600, 5000)), rng.choice((1, 4, 64, 1024)), kv * rng.choice((1, 4, 7, 64)), kv,
                      rng.choice((16, 64, 128, 256)), page, rng.randrange(1, (1 << rng.randrange(8, 21)) // page + 2),
                      rng.choice((0, 0, 1000)), rng.randrange(5)))
    for call in calls:
        most = max(most, L.sbq_paged_attn_workspace_bytes(*call))
    assert 10 << 20 < most < 54 * 10 ** 6
