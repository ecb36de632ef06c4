"""Random calls of a decode step's operators for several sequences, against the
oracles of their own tests: a fixed number of a fixed seed here, more by

    python tests/test_step_random.py CALLS [SEED]

which draws CALLS of each kind, prints every hundredth, and stops at the first
mismatch.  Table rooms, rows and vocabularies are drawn on both sides of the rules
that choose a kernel (test_draws_reach_every_kernel counts them)."""
import json
import random
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

sys.path[:0] = [str(Path(__file__).resolve().parent), str(Path(__file__).resolve().parents[1] / "spikingbrain-cpu_amd")]

from sbq.state import DevicePagedKVBuffer, qk_norm_rope  # noqa: E402
from test_paged_cache import (BF16, E4M3, F16, F32, HOST, I8, LARGEST, PKG, TYPES, _buffer, _codes)  # noqa: E402
from test_qk_norm_rope import _case, _check  # noqa: E402
from test_verify_drafts import _probs, _run, _same  # noqa: E402

CALLS, SEED = 60, 20


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


# ---------------------------------------------------------------------------
# draws: plain values, made before anything is on the GPU
# ---------------------------------------------------------------------------
def draw_attend(rng):
    while True:
        kv, rep, B = rng.choice((1, 1, 2, 3, 8)), rng.choice((1, 2, 4, 7)), rng.choice((1, 1, 2, 5, 17, 70))
        T = rng.choice((1, 1, 1, 2, 5, 9, 33, 64, 150))
        if B * T * kv * rep <= 6000:
            break
    dim = rng.choice((16, 64, 64, 128, 128, 256, rng.randrange(1, 257)))
    lengths = [rng.choice((0, 1, rng.randrange(1, 40), _log(rng, 1, 700))) for _ in range(B)]
    room = max(max(lengths), T, 1) + rng.choice((0, 0, 200, 3000, 20000, 80000, 300000))
    dtype, qt = rng.choice(TYPES)
    if rng.random() < 0.12:  # sequences that fill the chip with workgroups of their own
        kv, rep, B, T, dim, room = 8, 4, 70, rng.randrange(5, 8), rng.choice((112, 128)), rng.randrange(470, 900)
        lengths = [rng.randrange(0, 60) for _ in range(B)]
        dtype, qt = rng.choice([t for t in TYPES if t[1] != F32])
    elif rng.random() < 0.1:  # drafts or a chunk over a table with much room
        kv, rep, B, T, dim, room = 8, 4, len(lengths[:2]), rng.randrange(5, 60), rng.choice((64, 72, 128)), 300000
        lengths = [rng.randrange(T, 900) for _ in range(B)]
        dtype, qt = rng.choice([t for t in TYPES if t[1] != F32])
    return dict(B=B, T=T, kv=kv, rep=rep, dim=dim, page=rng.choice((16, 16, 32, 64, 256, 1024)), lengths=lengths, room=room,
                dtype=dtype, qt=qt, window=rng.choice((None, None, 1, _log(rng, 2, 900))), counts=rng.random() < 0.4,
                start=rng.random() < 0.3, holes=rng.random() < 0.2, size=rng.choice((0.05, 1.0, 1.0, 4.0)), seed=rng.randrange(1 << 30))


def draw_store(rng):
    heads, dim = rng.choice((1, 2, 5, 8)), rng.choice((1, 8, 64, 128, 256, rng.randrange(1, 257)))
    B, T = rng.choice((1, 2, 7, 40)), _log(rng, 1, 300)
    return dict(B=min(B, 1 + 600 // T), T=T, heads=heads, dim=dim, page=rng.choice((16, 64, 128)), dtype=rng.choice((I8, E4M3, F32, F16, BF16)),
                new=rng.choice((F32, F16, BF16)), out=rng.choice((F32, F16, BF16)), held=_log(rng, 1, 100), counts=rng.random() < 0.4,
                spread=rng.choice((0, 4, 40)), seed=rng.randrange(1 << 30))


def draw_rope(rng):
    H, kv = rng.choice((1, 3, 8, 32)), rng.choice((0, 1, 2, 8))
    D = rng.choice((64, 128, 256, rng.randrange(1, 257)))
    pairs = rng.choice((D // 2, D // 2, rng.randrange(0, D // 2 + 1)))
    return dict(T=max(1, _log(rng, 1, 4000) // (1 + H * D // 512)), H=H, kv=kv, D=D, pairs=pairs, inter=rng.random() < 0.4,
                dtype=rng.choice((F32, F16, BF16)), norm=rng.random() < 0.7, wt=rng.choice((F32, F16, BF16)), offset=rng.choice((0, 0, 1, 3)),
                seed=rng.randrange(1 << 30))


def draw_verify(rng):
    V = rng.choice((_log(rng, 1, 4096), _log(rng, 4000, 16384), _log(rng, 16385, 152000)))
    T = rng.choice((0, 1, 4, 9))
    B = max(1, min(rng.choice((1, 5, 30)), 1000000 // ((T + 1) * V)))
    return dict(B=B, T=T, V=V, dtype=rng.choice((F32, F16, BF16)), draft=rng.random() < 0.7, counts=rng.random() < 0.4,
                sharp=rng.choice((0.5, 2.0, 6.0)), seed=rng.randrange(1 << 30))


# ---------------------------------------------------------------------------
# one call each
# ---------------------------------------------------------------------------
def _expect(b, q, start, counts):
    """test_paged_cache._attention's result and tolerance, a key head at a time, and the documented bound's other
    term where what is multiplied lies in fp16 pieces (fp16 and 8-bit caches): the second piece ends at 2^-25, half of
    fp16's smallest step, against 2^14 at the row's largest weight (8 bits: times its value's scale), so each of those
    is off by up to 2^-39 of the largest, times the value (the code) beside it; a query's element likewise by 2^-39 of
    its row's largest.  (Two positions, weights 1 and 9e-11, a value of 0 in the first: 2e-12 of error.)"""
    B, T, H, D = q.shape
    rep, page, width, scale = H // b.heads, b.page, b.table.shape[1], D ** -0.5
    piece, least = 2.0 ** -20, 0.0 if b.k.dtype in (F32, BF16) else 2.0 ** -39
    qd, table = q.double().cpu().numpy(), b.table.cpu().numpy()
    length, out, tol = b.length.tolist(), np.zeros(q.shape), np.zeros(q.shape)
    pools = [p.float().cpu().double().numpy() for p in (b.k, b.v)]
    scales = [None if s is None else s.cpu().double().numpy() for s in (b.k_scale, b.v_scale)]
    for i in range(B):
        n = max(0, min(length[i], width * page))
        count = T if counts is None else int(np.clip(int(counts[i]), 0, T))
        first = length[i] - count if start is None else int(start[i])
        at = np.arange(n)
        ids = table[i, at // page]
        there = (ids >= 0) & (ids < b.k.shape[0])
        at, ids = at[there], ids[there]
        k, v = [p[ids, :, at % page] * (1.0 if s is None else s[ids, :, at % page][..., None]) for p, s in zip(pools, scales)]
        codes, unit = pools[1][ids, :, at % page], np.ones(k.shape[:2]) if scales[1] is None else scales[1][ids, :, at % page]
        pos = first + np.arange(count)
        see = at[:, None] <= pos
        if b.window:
            see &= at[:, None] > pos - b.window
        some = see.any(0)
        if not some.any():
            continue
        for h in range(b.heads):
            x = qd[i, :count, h * rep:(h + 1) * rep].reshape(count * rep, D)
            sees = see.repeat(rep, 1)
            s = np.where(sees, scale * (k[:, h] @ x.T), -np.inf)
            size = np.where(sees, scale * (np.abs(k[:, h]) @ np.abs(x).T), 0).max(0)
            p = np.exp(s - np.where(some.repeat(rep), s.max(0), 0.0))
            p /= np.where(some.repeat(rep), p.sum(0), 1.0)
            delta = size * ((D + 16) * 2.0 ** -24 + 2.0 ** -21)
            delta += least * scale * np.abs(x).max(1) * np.where(sees, np.abs(k[:, h]).sum(1)[:, None], 0).max(0)
            bound = (p.T @ np.abs(v[:, h])) * (2 * delta + piece + (sees.sum(0) + 16) * 2.0 ** -24)[:, None]
            bound += least * (p * unit[:, h, None]).max(0)[:, None] * (sees.T @ np.abs(codes[:, h]))
            out[i, :count, h * rep:(h + 1) * rep] = (p.T @ v[:, h]).reshape(count, rep, D)
            tol[i, :count, h * rep:(h + 1) * rep] = bound.reshape(count, rep, D)
    tol += (np.abs(out) + tol) * (torch.finfo(q.dtype).eps / 2) * 1.001 + (2.0 ** -25 if q.dtype == F16 else 1e-38)
    return out, tol


def attend(dev, c):
    b = _buffer(dev, c["lengths"], c["kv"], c["dim"], c["page"], c["dtype"], c["window"], seed=c["seed"], room=c["room"])
    g = torch.Generator().manual_seed(c["seed"])
    B, T = c["B"], c["T"]
    q = (torch.randn(B, T, c["kv"] * c["rep"], c["dim"], generator=g) * c["size"]).to(c["qt"]).to(dev)
    counts = torch.randint(-1, T + 2, (B,), generator=g).to(dev) if c["counts"] else None
    start = torch.randint(-3, max(c["lengths"]) + 5, (B,), generator=g).to(dev) if c["start"] else None
    if c["holes"]:
        for i in range(B):
            b.table[i, int(torch.randint(0, b.table.shape[1], (1,), generator=g))] = -1
    got = b.attend(q, start, counts).double().cpu().numpy()
    want, tol = _expect(b, q, start, counts)
    assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all(), np.nanmax(np.abs(got - want) / tol)


def store(dev, c):
    B, T, n = c["B"], c["T"], c["held"]
    b = _buffer(dev, [n + T] * B, c["heads"], c["dim"], c["page"], c["dtype"], fill=False, room=n + T)
    g = torch.Generator().manual_seed(c["seed"])
    held = torch.randint(0, n + 1, (B,), generator=g)
    b.length.copy_(held)
    wide = torch.exp2(torch.randint(-c["spread"], 1, (B, T, c["heads"], 1), generator=g).float())
    k, v = [(torch.randn(B, T, c["heads"], c["dim"], generator=g) * wide).to(c["new"]) for _ in range(2)]
    counts = torch.randint(0, T + 1, (B,), generator=g) if c["counts"] else torch.full((B,), T)
    b.append(k.to(dev), v.to(dev), None, counts.to(dev) if c["counts"] else None)
    assert torch.equal(b.length.cpu(), held + counts)
    for got, x in zip(b.read(held.to(dev), T, c["out"]), (k, v)):
        if c["dtype"] in LARGEST:
            codes, s = _codes(x, c["dtype"])
            x = codes.float() * torch.from_numpy(s)[..., None]
        else:
            x = x.to(c["dtype"]).float()
        x = torch.where(torch.arange(T)[None, :, None, None] < counts[:, None, None, None], x, 0)
        assert torch.equal(got.cpu(), x.to(c["out"]))


def rope(dev, c):
    q, k, pos, f, wq, wk = _case(dev, c["T"], c["H"], c["kv"], c["D"], c["pairs"], c["inter"], c["dtype"], c["norm"], c["seed"], wt=c["wt"])
    if c["offset"]:  # heads of a row that begins anywhere
        row = torch.zeros(c["T"], (c["H"] + c["kv"]) * c["D"] + 2 * c["offset"], dtype=c["dtype"], device=dev)
        at = c["offset"] + c["H"] * c["D"]
        views = [row[:, c["offset"]:at].unflatten(1, (c["H"], c["D"]))]
        if k is not None:
            views.append(row[:, at:at + c["kv"] * c["D"]].unflatten(1, (c["kv"], c["D"])))
        for view, x in zip(views, (q, k)):
            view.copy_(x)
        q, k = views[0], views[1] if k is not None else None
    _check(qk_norm_rope(q, k, pos, f, wq, wk, interleaved=c["inter"]), q, k, pos, f, wq, wk, c["inter"])


def verify(dev, c):
    g = torch.Generator().manual_seed(c["seed"])
    B, T, V = c["B"], c["T"], c["V"]
    target = _probs(g, B, T + 1, V, c["sharp"], c["dtype"])
    near = torch.softmax(target[:, :T].float().clamp_min(1e-9).log() + 0.4 * torch.randn(B, T, V, generator=g), -1).to(c["dtype"])
    tokens = torch.multinomial(near.float().reshape(-1, V), 1, generator=g).reshape(B, T) if T else torch.zeros(B, 0, dtype=torch.long)
    u = torch.rand(B, T + 1, generator=g)
    counts = torch.randint(0, T + 1, (B,), generator=g) if c["counts"] else None
    got, want = _run(dev, target, near if c["draft"] else None, tokens, u, counts)
    assert got[0].tolist() == want[0].tolist()
    if got[1].tolist() != want[1].tolist():  # (sums in another order: a draw within a rounding of a border may go either way)
        for b in range(B):
            if int(got[1][b]) != int(want[1][b]):
                t, n = int(want[0][b]), T if counts is None else int(counts[b])
                p = target[b, t].double()
                q = torch.zeros(V, dtype=torch.float64)
                if t < n:
                    q = near[b, t].double() if c["draft"] else q.index_fill(0, tokens[b, t], 1.0)
                mass = (p - q).clamp_min(0) if t < n and float((p - q).clamp_min(0).sum()) > 0 else p
                prefix = mass.cumsum(0)
                border = float(u[b, T].double() * prefix[-1])
                x, lo = int(got[1][b]), min(int(got[1][b]), int(want[1][b]))
                assert float(mass[x]) > 0 and abs(float(prefix[lo]) - border) <= V * 2.0 ** -52 * float(prefix[-1])


KINDS = {"attend": (draw_attend, attend), "store": (draw_store, store), "rope": (draw_rope, rope), "verify": (draw_verify, verify)}


def _cases(kind, calls, seed):
    rng = random.Random(f"{kind} {seed}")
    return [KINDS[kind][0](rng) for _ in range(calls)]


# ---------------------------------------------------------------------------
# tests
# ---------------------------------------------------------------------------
def test_draws_reach_every_kernel(tmp_path):
    so = tmp_path / "launch_trace.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-std=c++17", "-Wall", str(HOST / "launch_trace.cpp"), "-o", str(so)],
                   check=True)
    calls, code, ct = [], {F32: 0, F16: 1, BF16: 2}, {F32: 0, F16: 1, BF16: 2, I8: 3, E4M3: 4}
    cases = _cases("attend", CALLS, SEED)
    for c in cases:
        heads = c["kv"] * c["rep"]
        calls.append(["sbq_paged_attention", "@0", code[c["qt"]], c["T"], heads, c["T"] * heads * c["dim"], heads * c["dim"], c["dim"],
                      "@1", "@2", "@3", "@4", ct[c["dtype"]], 9, c["page"], c["kv"], c["dim"], "@5", c["B"], -(-c["room"] // c["page"]),
                      "@6", None, None, c["window"] or 0, 0.1, "@7", c["T"] * heads * c["dim"], heads * c["dim"], c["dim"], "@8",
                      1 << 40, None])
    r = subprocess.run([sys.executable, str(HOST / "grids.py"), str(so), str(PKG / "sbq" / "libsbq.so"), str(PKG / "sbq")],
                       input=json.dumps(calls), capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    seen = {}
    for c, got in zip(cases, json.loads(r.stdout)):
        assert got["rc"] == 0
        rows = c["rep"] * c["T"]
        wide = rows > 16 and got["launches"][0][0][0] // c["kv"] < -(-rows // 16)  # two sixteens of rows a workgroup
        kind = ("joined" if len(got["launches"]) > 1 else "whole", "wide" if wide else "narrow")
        seen[kind] = seen.get(kind, 0) + 1
    assert len(seen) == 4 and min(seen.values()) >= 2, seen
    sizes = [c["V"] for c in _cases("verify", CALLS, SEED)]
    assert all(sum(lo < v <= hi for v in sizes) >= 5 for lo, hi in ((0, 4096), (4096, 16384), (16384, 1 << 23)))
    few = [c["T"] <= 512 for c in _cases("rope", CALLS, SEED)]
    assert 5 <= sum(few) <= CALLS - 5
    alone = [c["T"] * c["heads"] <= 32 for c in _cases("store", CALLS, SEED)]
    assert 5 <= sum(alone) <= CALLS - 5


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_random_calls(dev, kind):
    for i, c in enumerate(_cases(kind, CALLS, SEED)):
        print(f"[case] {kind} {i} {c}", flush=True)
        KINDS[kind][1](dev, c)


if __name__ == "__main__":
    n, seed = int(sys.argv[1]), int(sys.argv[2]) if len(sys.argv) > 2 else 0
    for name, (_, call) in KINDS.items():
        for i, case in enumerate(_cases(name, n, seed)):
            if i % 100 == 0:
                print(f"{name} {i} of {n}, seed {seed}", flush=True)
            try:
                call(torch.device("cuda", 0), case)
            except AssertionError:
                print(f"{name} {i} of seed {seed}: {case}", flush=True)
                raise
    print(f"{n} calls of each kind, seed {seed}: no mismatch")
