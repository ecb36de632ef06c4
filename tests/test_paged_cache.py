"""The paged cache of several sequences (sbq.state.DevicePagedKVBuffer): what
append stores and read gives back, the attention over the pages against the
formula in 64 bits, pages that are missing, and a whole step with drafts."""
import json
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from conftest import announce
from sbq import _lib, quant
from sbq.state import DevicePagedKVBuffer, qk_norm_rope

F32, F16, BF16, I8, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn
LARGEST = {I8: 127.0, E4M3: 448.0}
ROOT = Path(__file__).resolve().parents[1]
HOST = ROOT / "tests" / "host"
PKG = ROOT / "spikingbrain-cpu_amd"


# ---------------------------------------------------------------------------
# on the CPU: refusals, pages, index arithmetic, launches
# ---------------------------------------------------------------------------
def test_index_arithmetic(tmp_path):
    exe = tmp_path / "paged_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", str(PKG / "csrc"),
                    str(HOST / "paged_check.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.stdout.strip() == "ok", r.stdout + r.stderr


def test_c_abi_refuses_bad_arguments():
    L = _lib.load()
    p = 1 << 16  # never read: every call below is refused, or does nothing
    cache = dict(k=p, v=p, ks=p, vs=p, ct=3, pages=8, page=16, Hk=2, D=24, table=p, B=3, width=4, length=2 * p)

    def append(start=3 * p, counts=None, kn=p, vn=p, nt=0, T=1, nsb=48, nst=48, nsh=24, **kw):
        return L.sbq_paged_append(*{**cache, **kw}.values(), start, counts, kn, vn, nt, T, nsb, nst, nsh, None)

    def read(start=p, count=1, ko=p, vo=p, ot=0, osb=48, ost=48, osh=24, **kw):
        return L.sbq_paged_read(*{**cache, **kw}.values(), start, count, ko, vo, ot, osb, ost, osh, None)

    def attend(q=p, qt=0, T=1, heads=4, qsb=96, qst=96, qsh=24, start=p, counts=p, window=0, scale=1.0, out=p, osb=96, ost=96,
               osh=24, ws=p, nws=1 << 30, **kw):
        return L.sbq_paged_attention(q, qt, T, heads, qsb, qst, qsh, *{**cache, **kw}.values(), start, counts, window, scale, out,
                                     osb, ost, osh, ws, nws, None)

    for call in (append, read, attend):
        assert call(ct=5) == -2 and call(ct=-1) == -2
        for bad in (dict(D=0), dict(D=257), dict(Hk=0), dict(Hk=65537), dict(pages=0), dict(pages=(1 << 30) + 1), dict(page=8),
                    dict(page=48), dict(page=2048), dict(B=-1), dict(B=65537), dict(width=0), dict(width=(1 << 26) + 1),
                    dict(k=None), dict(v=None), dict(ks=None), dict(vs=None), dict(table=None), dict(length=None)):
            assert call(**bad) == -1, (call.__name__, bad)
        for bad in (dict(k=p + 8), dict(v=p + 4), dict(ks=p + 4), dict(vs=p + 8), dict(table=p + 2), dict(length=p + 4)):
            assert call(**bad) == -3, (call.__name__, bad)
        assert call(B=0) == 0
    assert append(T=(1 << 29) + 1) == -1 and read(count=(1 << 29) + 1) == -1
    assert append(nt=3) == -2 and append(T=-1) == -1 and append(nst=-1) == -1 and append(start=None) == -1
    assert append(kn=None) == -1 and append(vn=None) == -1
    assert append(start=2 * p + 8) == -1 and append(start=2 * p - 16) == -1  # other sequences' lengths
    assert append(counts=2 * p) == -1 and append(counts=2 * p + 16) == -1
    assert append(start=3 * p + 4) == -3 and append(counts=p + 4) == -3 and append(kn=p + 2) == -3
    assert read(ot=4) == -2 and read(count=-1) == -1 and read(start=None) == -1 and read(ko=None) == -1
    assert read(osh=23) == -1 and read(count=2, ost=47) == -1 and read(osb=47) == -1 and read(vo=p + 2) == -3
    assert read(count=0) == 0
    assert attend(qt=3) == -2 and attend(ct=1, qt=2) == -2 and attend(ct=0, qt=1) == -2
    for bad in (dict(T=-1), dict(T=_lib.SBQ_PAGED_MAX_T + 1), dict(heads=3), dict(heads=0), dict(window=-1),
                dict(scale=float("nan")), dict(q=None), dict(out=None), dict(qsb=-1), dict(osh=23), dict(osb=95),
                dict(T=2, ost=95)):
        assert attend(**bad) == -1, bad
    for bad in (dict(q=p + 2), dict(out=p + 1), dict(start=p + 4), dict(counts=p + 2)):
        assert attend(**bad) == -3, bad
    need = L.sbq_paged_attn_workspace_bytes(3, 1, 4, 2, 24, 16, 100, 0, 3)
    assert need > 256 and attend(width=100, ws=None) == -4 and attend(width=100, nws=need - 1) == -4 and attend(T=0) == 0
    for bad in ((0, 1, 4, 2, 24, 16, 100, 0, 3), (3, 0, 4, 2, 24, 16, 100, 0, 3), (3, 1, 5, 2, 24, 16, 100, 0, 3),
                (3, 1, 4, 2, 257, 16, 100, 0, 3), (3, 1, 4, 2, 24, 17, 100, 0, 3), (3, 1, 4, 2, 24, 16, 0, 0, 3),
                (3, 1, 4, 2, 24, 16, 100, -1, 3), (3, 1, 4, 2, 24, 16, 100, 0, 9), (3, 1, 4, 2, 24, 16, 4, 0, 3)):
        assert L.sbq_paged_attn_workspace_bytes(*bad) == 0
    for window in (1 << 40, (1 << 63) - 1):  # every position
        assert L.sbq_paged_attn_workspace_bytes(3, 1, 4, 2, 24, 16, 100, window, 3) >= need


def test_pages_are_given_out_and_taken_back():
    b = DevicePagedKVBuffer(3, 2, 24, 6, 16, max_pages=5, device="cpu", dtype=I8)
    assert b.k.shape == (6, 2, 16, 24) and b.k.stride(2) == 32 and b.k_scale.shape == (6, 2, 16)
    b.reserve(0, 33)
    b.reserve(1, 16)
    first = b.table.clone()
    assert (first[0] >= 0).tolist() == [True] * 3 + [False] * 2 and (first[1] >= 0).tolist() == [True] + [False] * 4
    held = [int(i) for i in first.flatten() if i >= 0]
    assert len(set(held)) == 4 and max(held) < 6
    b.reserve(0, 20)                        # fewer: nothing changes
    assert torch.equal(b.table, first)
    with pytest.raises(RuntimeError, match="free"):
        b.reserve(2, 33)
    assert torch.equal(b.table, first)      # all or none
    with pytest.raises(ValueError, match="row"):
        b.reserve(0, 81)
    for i in (-1, 3):
        with pytest.raises(ValueError, match="sequence"):
            b.reserve(i, 1)
        with pytest.raises(ValueError, match="sequence"):
            b.release(i)
    b.release(0, 31)                        # the pages that end at or below position 31
    assert int(b.table[0, 0]) == -1 and torch.equal(b.table[0, 1:], first[0, 1:])
    b.reserve(0, 80)                        # those stay given back
    assert (b.table[0] >= 0).tolist() == [False] + [True] * 4
    used = [int(i) for i in b.table.flatten() if i >= 0]
    assert len(set(used)) == 5
    b.length[0] = 70
    b.release(0)
    assert int(b.table[0].max()) == -1 and int(b.length[0]) == 0
    b.reserve(0, 80)
    assert int(b.table[0].min()) >= 0
    b.reset()
    assert int(b.table.max()) == -1
    b.reserve(2, 80)
    b.length.copy_(torch.tensor([9, 4, 70]))
    b.truncate(40)
    assert b.length.tolist() == [9, 4, 40]
    b.truncate(-3)
    assert b.length.tolist() == [0, 0, 0]


def test_buffer_refuses():
    for bad in (dict(dtype=torch.float64), dict(sequences=0), dict(heads=0), dict(dim=0), dict(dim=257), dict(pages=0),
                dict(page=8), dict(page=40), dict(page=2048), dict(max_pages=0), dict(max_pages=1 << 27), dict(window=0),
                dict(window=1 << 62)):
        a = dict(sequences=2, heads=2, dim=8, pages=4, page=16, device="cpu")
        with pytest.raises(ValueError):
            DevicePagedKVBuffer(**{**a, **bad})
    b = DevicePagedKVBuffer(2, 2, 8, 4, 16, device="cpu")
    x = torch.zeros(2, 1, 2, 8)
    for call in (lambda: b.append(x, x), lambda: b.read(0, 1), lambda: b.attend(x)):
        with pytest.raises(ValueError, match="GPU"):
            call()


@pytest.fixture(scope="module")
def grids(tmp_path_factory):
    so = tmp_path_factory.mktemp("trace") / "launch_trace.so"
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-std=c++17", "-Wall", str(HOST / "launch_trace.cpp"), "-o", str(so)],
                   check=True)

    def run(calls):
        r = subprocess.run([sys.executable, str(HOST / "grids.py"), str(so), str(PKG / "sbq" / "libsbq.so"), str(PKG / "sbq")],
                           input=json.dumps(calls), capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        return json.loads(r.stdout)

    return run


def test_largest_launches(grids):
    """Fewer than 2^32 threads along an axis of a grid, at most 65535 workgroups along its others."""
    def cache(ct, Hk, D, B, page, width):
        return ["@1", "@2", "@3", "@4", ct, 1 << 20, page, Hk, D, "@5", B, width, "@6"]

    calls = []
    for ct in (0, 1, 2, 3, 4):
        for Hk, D, B, page, width, T in ((1, 1, 1, 16, 1 << 26, 1), (8, 128, 64, 64, 1 << 24, 1), (65536, 256, 65536, 1024, 1, 1),
                                         (8, 128, 65536, 16, 4096, 64), (65536, 64, 1, 16, 16, 1024), (1, 128, 1, 64, 1 << 24, 1024),
                                         (8, 128, 513, 16, 1 << 26, 7)):
            c = cache(ct, Hk, D, B, page, width)
            row = Hk * D
            for start in ("@6", "@7"):
                calls.append(["sbq_paged_append", *c, start, None, "@8", "@9", 0, T, T * row, row, D, None])
            calls.append(["sbq_paged_read", *c, "@7", T, "@8", "@9", 0, T * row, row, D, None])
            for rep in (1, 4) if Hk < 65536 else (1,):
                calls.append(["sbq_paged_attention", "@0", 0, T, rep * Hk, rep * T * row, rep * row, D, *c, None, None, 0, 0.1,
                              "@8", rep * T * row, rep * row, D, "@9", 1 << 50, None])
        calls.append(["sbq_paged_append", *cache(ct, 8, 128, 1, 64, 1 << 24), "@7", None, "@8", "@9", 2, 1 << 27, 0, 1024, 128,
                      None])
    for B, V in ((1, 1), (65535, 1), (65535, 1 << 23), (7, 151936)):
        calls.append(["sbq_verify_drafts", "@0", 2 * V, V, "@1", V, V, 0, B, 1, V, "@2", "@3", None, "@4", "@5", "@6", 1 << 50,
                      None])
    for T, H, Hk in (((1 << 31) - 1, 1, 0), ((1 << 31) - 1, 65536, 65536), (511, 65536, 65536), (1, 1, 1)):
        calls.append(["sbq_qk_norm_rope", "@0", "@1", 0, T, H, Hk, 256, H * 256, 256, Hk * 256, 256, "@2", 1, "@3", 1, 0, "@4",
                      "@5", 0, 1e-6, "@6", "@7", H * 256, 256, Hk * 256, 256, None])
    for call, got in zip(calls, grids(calls)):
        assert got["rc"] == 0 and got["launches"], call
        for grid, block in got["launches"]:
            assert all(1 <= g and g * b < 1 << 32 for g, b in zip(grid, block)) and max(grid[1:]) <= 65535, (call, grid, block)


# ---------------------------------------------------------------------------
# storing and reading back
# ---------------------------------------------------------------------------
def _buffer(dev, lengths, heads, dim, page, dtype, window=None, extra=3, seed=0, fill=True, room=None):
    """A buffer whose sequences hold `lengths` positions in shuffled pages; what
    no sequence holds is NaN (8 bits: a NaN scale)."""
    room = max(max(lengths, default=1), 1) if room is None else room
    width = -(-room // page)
    need = [-(-n // page) for n in lengths]
    b = DevicePagedKVBuffer(len(lengths), heads, dim, sum(need) + extra, page, width, window, dev, dtype)
    g = torch.Generator().manual_seed(seed)
    free = torch.randperm(sum(need) + extra, generator=g).tolist()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    for i, n in enumerate(need):
        for j in range(n):
            table[i, j] = free.pop()
    b.table.copy_(table)
    b.length.copy_(torch.tensor(lengths))
    if fill:
        for pool, scale in ((b.k, b.k_scale), (b.v, b.v_scale)):
            x = torch.randn(pool.shape, generator=g)
            if scale is None:
                pool.copy_(x)
            else:
                codes = torch.randint(-127, 128, pool.shape, generator=g) if dtype == I8 else (x * 100).clamp(-448, 448)
                pool.copy_(codes.to(dtype))
                scale.copy_(torch.rand(scale.shape, generator=g) * 0.02 + 1e-3)
        held = torch.zeros(b.k.shape[0], page, dtype=torch.bool)
        for i, n in enumerate(lengths):
            for j in range(need[i]):
                held[int(table[i, j]), :max(0, min(page, n - j * page))] = True
        gone = ~held.to(dev)
        for pool, scale in ((b.k, b.k_scale), (b.v, b.v_scale)):
            if scale is None:
                pool.masked_fill_(gone[:, None, :, None], float("nan"))
            else:
                scale.masked_fill_(gone[:, None], float("nan"))
    return b


def _held(b, i, n):
    """Keys and values [n, heads, dim] of sequence i's first n positions, in 64 bits (pages it lacks: 0), and which there are."""
    page, ids = b.page, b.table[i].tolist()
    k = np.zeros((n, b.heads, b.dim))
    v, there = k.copy(), np.zeros(n, dtype=bool)
    pools = [p.float().cpu().double().numpy() for p in (b.k, b.v)]
    scales = [None if s is None else s.cpu().double().numpy() for s in (b.k_scale, b.v_scale)]
    for p in range(n):
        id_ = ids[p // page] if p // page < len(ids) else -1
        if 0 <= id_ < b.k.shape[0]:
            there[p] = True
            for to, pool, s in zip((k, v), pools, scales):
                to[p] = pool[id_, :, p % page] * (1.0 if s is None else s[id_, :, p % page, None])
    return k, v, there


def _codes(x, dtype):
    """The documented codes and scales of x [..., D], with IEEE divisions (numpy)."""
    x = x.float().numpy()
    scale = (np.abs(x).max(-1) / np.float32(LARGEST[dtype])).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        y = np.where(scale[..., None] > 0, x / scale[..., None], np.float32(0)).astype(np.float32)
    y = np.clip(y, -LARGEST[dtype], LARGEST[dtype])
    codes = torch.from_numpy(np.rint(y)).to(I8) if dtype == I8 else torch.from_numpy(y).to(E4M3)
    return codes, scale


def _bits(t):
    return t.contiguous().view(torch.uint8).cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [F32, F16, BF16])
@pytest.mark.parametrize("dtype", [I8, E4M3, F32, F16, BF16])
@pytest.mark.parametrize("heads,dim,page,T", [(2, 64, 16, 1), (8, 128, 64, 1), (3, 33, 16, 5), (1, 256, 32, 20), (2, 1, 16, 17),
                                              (5, 250, 128, 3), (4, 80, 64, 64), (40, 16, 16, 2), (8, 128, 64, 9)])
def test_append_stores_and_read_gives_back(dev, heads, dim, page, T, dtype, new):
    announce(f"append heads={heads} dim={dim} page={page} T={T} {dtype} new={new}")
    lengths = [0, 1, page - 1, page, 2 * page + 5]
    B = len(lengths)
    room = max(lengths) + T
    b = _buffer(dev, [n + T for n in lengths], heads, dim, page, dtype, fill=False, room=room)
    b.length.copy_(torch.tensor(lengths))
    g = torch.Generator().manual_seed(dim)
    k, v = [(torch.randn(B, T, heads, dim, generator=g) * 3).to(new) for _ in range(2)]
    k[0, 0, 0], v[1, 0, 0] = 0.0, 1e-30 if new != F16 else 1e-7
    before = [_bits(t) for t in (b.k, b.v)]
    b.append(k.to(dev), v.to(dev))
    assert b.length.tolist() == [n + T for n in lengths]
    out = {}
    for name, x, pool, scale in (("k", k, b.k, b.k_scale), ("v", v, b.v, b.v_scale)):
        if dtype in LARGEST:
            codes, s = _codes(x, dtype)
            out[name] = codes.float() * torch.from_numpy(s)[..., None]
        else:
            codes, s = x.to(dtype), None
            out[name] = codes.float()
        touched = torch.zeros(pool.shape[0], page, dtype=torch.bool)
        pool_h, scale_h = pool.cpu(), None if scale is None else scale.cpu()
        for i, n in enumerate(lengths):
            for t in range(T):
                at = int(b.table[i, (n + t) // page]), (n + t) % page
                touched[at] = True
                assert torch.equal(_bits(pool_h[at[0], :, at[1]]), _bits(codes[i, t])), (name, i, t)
                if s is not None:
                    assert scale_h[at[0], :, at[1]].numpy().tobytes() == s[i, t].tobytes()
        left = _bits(pool_h.movedim(2, 1)[~touched])
        assert int(left.sum()) == 0  # every other position as it was
    rk, rv = b.read(torch.tensor(lengths, device=dev), T)
    for got, want in ((rk, out["k"]), (rv, out["v"])):
        assert got.dtype == (F32 if dtype in LARGEST else dtype) and got.shape == (B, T, heads, dim)
        assert torch.equal(got.float().cpu(), want if dtype in LARGEST else want.to(got.dtype).float())
    for to in (F16, BF16, F32):  # rounded once to another type, from two positions earlier on: zeros before 0 and past the end
        start = torch.tensor(lengths) - 2
        rk, rv = b.read(start.to(dev), T + 5, to)
        for got, want in ((rk, out["k"]), (rv, out["v"])):
            assert torch.equal(got[:, 2:T + 2].cpu(), want.to(to))
            assert float(got[:, T + 2:].abs().sum()) == 0 and float(got[0, :2].abs().sum()) == 0
    for i in range(B):
        rk, rv = b.read(lengths[i], T, sequence=i)
        assert torch.equal(rk.float().cpu(), out["k"][i] if dtype in LARGEST else out["k"][i].to(rk.dtype).float())


@pytest.mark.gpu
def test_quotients_are_ieee_divisions(dev):
    """Codes of vectors whose scales run over the exponents, next to borders between codes."""
    n, D = 4096, 128
    g = torch.Generator().manual_seed(5)
    x = torch.randn(1, n, 1, D, generator=g) * torch.exp2(torch.randint(-146, 120, (1, n, 1, 1), generator=g).float())
    x[0, ::2] = x[0, ::2].to(BF16).float()  # few bits: quotients on the borders themselves
    m = x.abs().amax(-1, keepdim=True)
    half = (torch.randint(-127, 127, (1, n // 4, 1, D), generator=g) + 0.5) / 127
    x[0, ::4] = (half * m[0, ::4]).reshape(n // 4, 1, D)
    x = x.clamp(-3e38, 3e38)
    for dtype in (I8, E4M3):
        b = _buffer(dev, [n], 1, D, 64, dtype, fill=False)
        b.append(x.to(dev), -x.to(dev), 0)
        codes, s = _codes(x, dtype)
        ids = b.table[0].long()
        got = b.k[ids, 0].reshape(1, n, 1, D)
        assert torch.equal(_bits(got), _bits(codes))
        assert b.k_scale[ids, 0].reshape(-1).cpu().numpy().tobytes() == s.reshape(-1).tobytes()
        neg, _ = _codes(-x, dtype)
        assert torch.equal(_bits(b.v[ids, 0].reshape(1, n, 1, D)), _bits(neg))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [I8, E4M3, BF16])
def test_append_counts_starts_bad_pages_and_capacity(dev, dtype):
    B, heads, dim, page, T = 7, 2, 32, 16, 6
    b = _buffer(dev, [40] * B, heads, dim, page, dtype, fill=False, room=48)
    g = torch.Generator().manual_seed(0)
    k, v = [torch.randn(B, T, heads, dim, generator=g).to(dev) for _ in range(2)]
    b.table[2, 0], b.table[3, 0], b.table[4, 0] = -1, b.k.shape[0], 2147483647
    kept = [_bits(t) for t in (b.k, b.v)]
    start = torch.tensor([0, 14, 0, 0, 0, -3, 45], device=dev)
    counts = torch.tensor([0, 4, 6, 6, 6, 6, 100], device=dev)
    b.append(k, v, start, counts)
    assert b.length.tolist() == [0, 18, 6, 6, 6, 0, 48]  # capacity: 3 pages of 16
    rk, rv = b.read(0, 48, F32)
    seen = torch.zeros(B, 48, dtype=torch.bool)
    seen[1, 14:18] = seen[6, 45:48] = True
    want = torch.zeros(B, 48, heads, dim)
    kh = k.cpu() if dtype == BF16 else None
    for got, x in ((rk, k), (rv, v)):
        x = x.cpu()
        if dtype in LARGEST:
            codes, s = _codes(x, dtype)
            x = codes.float() * torch.from_numpy(s)[..., None]
        else:
            x = x.to(dtype).float()
        assert torch.equal(got[1, 14:18].cpu(), x[1, :4]) and torch.equal(got[6, 45:48].cpu(), x[6, :3])
        assert float(got[~seen.to(dev)].abs().sum()) == 0
    touched = torch.zeros(b.k.shape[0], page, dtype=torch.bool)
    for i, p in [(1, 14), (1, 15), (1, 16), (1, 17), (6, 45), (6, 46), (6, 47)]:
        touched[int(b.table[i, p // page]), p % page] = True
    for pool, old in zip((b.k, b.v), kept):
        assert int(_bits(pool.movedim(2, 1)[~touched.to(dev)]).sum()) == 0
    # far starts, counts below zero
    b.append(k, v, torch.full((B,), 1 << 62, device=dev), torch.full((B,), -1, device=dev, dtype=torch.long))
    assert b.length.tolist() == [48] * B
    b.append(k, v, torch.zeros(B, dtype=torch.long, device=dev), torch.full((B,), -5, device=dev, dtype=torch.long))
    assert b.length.tolist() == [0] * B
    # a call on one sequence leaves the others
    b.append(k[1], v[1], 3, None, 1)
    assert b.length.tolist() == [0, 9, 0, 0, 0, 0, 0]
    b.append(k[1, :0], v[1, :0], sequence=1)
    assert b.length.tolist() == [0, 9, 0, 0, 0, 0, 0]
    # a vector with an infinity or NaN
    if dtype in LARGEST:
        k[0, 0, 0, 3], k[0, 1, 1, 31] = float("nan"), -float("inf")
        b.append(k[0], v[0], 0, None, 0)
        rk, _ = b.read(0, T, sequence=0)
        assert torch.isnan(rk[0, 0]).all() and torch.isnan(rk[1, 1]).all()
        rk[0, 0] = rk[1, 1] = 0
        assert torch.isfinite(rk).all()


@pytest.mark.gpu
def test_append_aliases_of_the_lengths_and_the_pool(dev):
    B, heads, dim, page, T = 4, 2, 32, 16, 3
    g = torch.Generator().manual_seed(1)
    k, v = [torch.randn(B, T, heads, dim, generator=g).to(dev) for _ in range(2)]
    b = _buffer(dev, [20] * B, heads, dim, page, F32, fill=False, room=32)
    b.length.copy_(torch.tensor([1, 5, 9, 13]))
    own = b.length
    b.append(k, v, own)                                 # the lengths themselves
    assert b.length.tolist() == [4, 8, 12, 16]
    b.append(k[0], v[0], own[2:3], None, 1)             # another sequence's
    assert b.length.tolist() == [4, 15, 12, 16]
    b.append(k, v, 0, torch.tensor([1, 2, 3, 0], device=dev))
    assert b.length.tolist() == [1, 2, 3, 0]
    b.append(k, v, None, own)                           # counts that the call itself moves
    assert b.length.tolist() == [2, 4, 6, 0]
    # rows of the pool itself as new ones
    b.append(k, v, 0)
    page_of = int(b.table[0, 0])
    rows = b.k[page_of].transpose(0, 1)[:T]             # [T, heads, dim]
    want = rows.clone()
    b.append(rows, rows, 1, None, 0)
    rk, rv = b.read(1, T, sequence=0)
    assert torch.equal(rk, want) and torch.equal(rv, want)
    # long ones: the length is moved after every workgroup has read it
    n = 1000
    big = _buffer(dev, [n + 20] * 2, heads, dim, page, F32, fill=False, room=n + 20)
    big.length.copy_(torch.tensor([7, 20]))
    k, v = [torch.randn(2, n, heads, dim, generator=g).to(dev) for _ in range(2)]
    big.append(k, v)
    assert big.length.tolist() == [n + 7, n + 20]
    rk, rv = big.read(torch.tensor([7, 20], device=dev), n)
    assert torch.equal(rk, k) and torch.equal(rv, v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [I8, BF16])
def test_append_strides(dev, dtype):
    B, T, H, heads, dim, page = 3, 4, 4, 2, 40, 16
    g = torch.Generator().manual_seed(1)
    want = None
    qkv = torch.randn(B, T, (H + 2 * heads) * dim, generator=g).to(dev)
    k = qkv[..., H * dim:(H + heads) * dim].unflatten(-1, (heads, dim))
    v = qkv[..., (H + heads) * dim:].unflatten(-1, (heads, dim))
    odd = torch.randn(B, heads, T, dim + 1, generator=g).to(dev)
    odd[..., 1:] = k.transpose(1, 2)
    columns = torch.empty(B, T, dim, heads, device=dev)
    columns.copy_(k.transpose(2, 3))
    wide = k.double()
    for kk, vv in ((k, v), (odd[..., 1:].transpose(1, 2), v), (columns.transpose(2, 3), v), (wide, v.double())):
        b = _buffer(dev, [20] * B, heads, dim, page, dtype, fill=False, room=32)
        b.append(kk, vv, 2)
        got = [t.cpu() for t in b.read(2, T)]
        want = want or got
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = k[:, :1].expand(B, T, heads, dim)  # one memory for all tokens
    b.append(one, one, 2)
    rk, _ = b.read(2, T)
    assert torch.equal(rk, rk[:, :1].expand_as(rk)) and torch.equal(rk[:, 0].cpu(), want[0][:, 0])


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _attention_of(b, q, counts, tokens, sequences):
    """_attention of some tokens of the first few sequences."""
    out, tol = _attention(b, q, None, counts, None, tokens, sequences)
    return out[:sequences][:, tokens], tol[:sequences][:, tokens]


def _attention(b, q, start, counts, scale=None, tokens=None, sequences=None):
    """The documented attention and its tolerance, in 64 bits.

    With u = 2^-24: a score carries (D + 16) u of scale sum |q||k| (products and sums of D
    terms, the scales and the logarithm's factor), and 2^-21 of it for a query
    in pieces; a weight twice the largest score's absolute error, 2^-20 of its
    own for exp2, the pieces and the values' scales (one piece of fp16 with
    bf16 queries: 2^-11), and (n + 16) u for n additions; the output half a step of its type."""
    B, T, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    qd = q.float().cpu().double().numpy()
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    rep, eps = H // b.heads, torch.finfo(q.dtype).eps / 2
    piece = 2.0 ** -11 if q.dtype == BF16 and b.k_scale is not None else 2.0 ** -20
    for i in range(B if sequences is None else min(B, sequences)):
        n = max(0, min(int(b.length[i]), b.table.shape[1] * b.page))
        count = T if counts is None else int(np.clip(int(counts[i]), 0, T))
        first = int(b.length[i]) - count if start is None else int(start[i])
        k, v, there = _held(b, i, n)
        for t in range(count):
            if tokens is not None and t not in tokens:
                continue
            pos = first + t
            see = there & (np.arange(n) <= pos)
            if b.window:
                see &= np.arange(n) > pos - b.window
            if not see.any():
                continue
            for h in range(H):
                ks, vs = k[see, h // rep], v[see, h // rep]
                s = scale * (ks @ qd[i, t, h])
                size = abs(scale) * (np.abs(ks) @ np.abs(qd[i, t, h])).max()
                p = np.exp(s - s.max())
                p /= p.sum()
                out[i, t, h] = p @ vs
                delta = size * ((D + 16) * 2.0 ** -24 + 2.0 ** -21)
                tol[i, t, h] = (p @ np.abs(vs)) * (2 * delta + piece + (len(s) + 16) * 2.0 ** -24)
    tol += (np.abs(out) + tol) * eps * 1.001 + (2.0 ** -25 if q.dtype == F16 else 1e-38)
    return out, tol


def _compare(b, q, got, start=None, counts=None, scale=None):
    want, tol = _attention(b, q, start, counts, scale)
    g = got.float().cpu().double().numpy()
    assert np.isfinite(g).all()
    bad = np.abs(g - want) > tol
    assert not bad.any(), (np.abs(g - want) / tol).max()


TYPES = [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32), (I8, F32), (I8, F16), (I8, BF16), (E4M3, F32),
         (E4M3, F16), (E4M3, BF16)]
SHAPES = [  # lengths, T, heads, kv, dim, page, window
    ([1], 1, 1, 1, 64, 16, None),
    ([0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 65], 1, 4, 2, 64, 16, None),
    ([300, 5, 0, 127, 128, 129], 1, 8, 2, 128, 64, None),
    ([100, 40], 1, 7, 1, 80, 32, None),
    ([70, 3], 1, 20, 1, 128, 16, None),
    ([200, 64], 1, 4, 4, 256, 128, None),
    ([50, 9], 1, 2, 2, 33, 16, None),
    ([20], 1, 2, 1, 1, 16, None),
    ([90, 30, 4], 4, 14, 2, 80, 16, None),
    ([90, 30, 4], 4, 14, 2, 80, 16, 20),
    ([400, 33, 17], 3, 4, 2, 128, 64, 1),
    ([400, 33, 17], 9, 8, 2, 250, 16, 100),
    ([130] * 70, 1, 2, 1, 16, 16, None),
    ([1000, 1, 1, 1, 700], 2, 8, 8, 64, 16, None),
    ([1000, 60, 700], 3, 4, 2, 128, 16, 200),
    ([513, 512, 511, 600], 1, 2, 1, 256, 64, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,qt", TYPES)
@pytest.mark.parametrize("lengths,T,heads,kv,dim,page,window", SHAPES)
def test_attention(dev, lengths, T, heads, kv, dim, page, window, dtype, qt):
    announce(f"attend lengths={lengths[:6]} T={T} heads={heads} kv={kv} dim={dim} page={page} window={window} {dtype} {qt}")
    b = _buffer(dev, lengths, kv, dim, page, dtype, window, seed=dim)
    g = torch.Generator().manual_seed(T)
    q = (torch.randn(len(lengths), T, heads, dim, generator=g) * 1.5).to(qt).to(dev)
    got = b.attend(q)
    assert got.dtype == qt and got.shape == q.shape
    _compare(b, q, got)
    if T == 1:
        assert torch.equal(b.attend(q[:, 0]), got[:, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,qt", [(F32, F32), (BF16, BF16), (BF16, F32), (I8, F32), (E4M3, BF16)])
def test_attention_long_and_ragged(dev, dtype, qt):
    """Sequences that several workgroups share, beside short ones, more than one wave of lengths to scan."""
    lengths = [6000, 3, 2500, 0, 900] + [(37 * i) % 260 for i in range(75)]
    b = _buffer(dev, lengths, 2, 64, 64, dtype, seed=1, room=6500)
    g = torch.Generator().manual_seed(0)
    q = torch.randn(len(lengths), 1, 8, 64, generator=g).to(qt).to(dev)
    _compare(b, q, b.attend(q))
    b.window = 1500
    _compare(b, q, b.attend(q))


@pytest.mark.gpu
def test_attention_of_one_long_sequence(dev):
    b = _buffer(dev, [20011], 1, 128, 128, BF16, seed=2)
    q = torch.randn(1, 1, 4, 128, generator=torch.Generator().manual_seed(0)).to(BF16).to(dev)
    _compare(b, q, b.attend(q))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,qt", [(F32, F32), (BF16, BF16), (I8, BF16)])
@pytest.mark.parametrize("width", [1, 40, 400])
def test_attention_of_more_sequences_than_a_launch_takes(dev, dtype, qt, width):
    """600 sequences, some over shared pages, in tables that are not split and that are."""
    announce(f"attend 600 sequences width={width} {dtype} {qt}")
    b = _buffer(dev, [16] * 20, 1, 32, 16, dtype, seed=4)
    many = DevicePagedKVBuffer(600, 1, 32, 1, 16, width, None, dev, dtype)
    many.k, many.v, many.k_scale, many.v_scale = b.k, b.v, b.k_scale, b.v_scale
    g = torch.Generator().manual_seed(5)
    many.table.copy_(b.table.flatten()[torch.randint(0, 20, (600, width), generator=g).to(dev)])
    many.length.copy_(torch.randint(0, 16 * min(width, 40) + 1, (600,), generator=g))
    q = torch.randn(600, 1, 3, 32, generator=g).to(qt).to(dev)
    _compare(many, q, many.attend(q))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,qt", [(F16, F32), (E4M3, F16)])
def test_attention_of_many_tokens(dev, dtype, qt):
    """Row tiles that begin and end inside a token's heads, over more positions than a workgroup takes whole, pages of 1024."""
    b = _buffer(dev, [1100, 207, 40], 2, 72, 1024, dtype, seed=9, room=2048)
    g = torch.Generator().manual_seed(6)
    q = torch.randn(3, 207, 6, 72, generator=g).to(qt).to(dev)
    counts = torch.tensor([207, 207, 31], device=dev)
    _compare(b, q, b.attend(q, counts=counts), counts=counts)
    b.window = 77
    _compare(b, q, b.attend(q, counts=counts), counts=counts)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,qt", [(F16, F16), (BF16, BF16), (I8, F16), (E4M3, BF16), (E4M3, F16), (I8, F32)])
@pytest.mark.parametrize("lengths,T,heads,kv,dim,room", [
    ([1500, 330], 300, 8, 2, 128, 9000),                  # two row tiles at a time, sequences in parts
    ([700, 100], 301, 7, 1, 72, 20000),                   # ... that end inside a tile
    ([600, 290, 10], 290, 8, 2, 64, 16000),
    ([40, 33, 129, 512] * 16, 6, 32, 8, 112, 512),        # ... whole sequences
])
def test_attention_of_rows_in_twos(dev, lengths, T, heads, kv, dim, room, dtype, qt):
    announce(f"attend lengths={lengths[:4]} T={T} heads={heads} kv={kv} dim={dim} room={room} {dtype} {qt}")
    b = _buffer(dev, lengths, kv, dim, 16, dtype, seed=dim, room=room)
    g = torch.Generator().manual_seed(T)
    q = torch.randn(len(lengths), T, heads, dim, generator=g).to(qt).to(dev)
    counts = torch.tensor([min(n, T) - (i % 3) for i, n in enumerate(lengths)], device=dev)
    got = b.attend(q, counts=counts)
    few = list(range(0, T, 23)) + [T - 1]  # (the oracle for some of the tokens, of four sequences)
    want, tol = _attention_of(b, q, counts, few, 4)
    bad = np.abs(got.float().cpu().double().numpy()[:4][:, few] - want) > tol
    assert not bad.any()
    for i in range(len(lengths)):
        assert float(got[i, int(counts[i]):].float().abs().sum()) == 0
    assert torch.isfinite(got).all()
    # an infinity (a NaN scale) in the last position: the last token alone sees it
    last = lengths[0] - 1
    page, row = int(b.table[0, last // 16]), last % 16
    if b.v_scale is None:
        b.v[page, :, row, 0] = float("inf")
    else:
        b.v_scale[page, :, row] = float("nan")
    now, end = b.attend(q, counts=counts), int(counts[0]) - 1
    assert torch.equal(now[0, :end], got[0, :end]) and torch.equal(now[1:], got[1:])
    if b.v_scale is None:
        assert torch.isinf(now[0, end, :, 0]).all() and torch.equal(now[0, end, :, 1:], got[0, end, :, 1:])
    else:
        assert torch.isnan(now[0, end]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,pages", [(I8, 17000), (F32, 4300)])
def test_pools_and_inputs_past_32_bits(dev, dtype, pages):
    """Pages more than 4 GiB into the pool, sequences' inputs as far apart, against a small pool and packed inputs."""
    announce(f"pool of {pages} pages {dtype}")
    heads, dim, page, T = 2, 128, 1024, 1500
    small, large = [DevicePagedKVBuffer(2, heads, dim, n, page, 3, None, dev, dtype) for n in (6, pages)]
    assert large.k.stride(0) * (pages - 1) * large.k.element_size() > 1 << 32
    small.table.copy_(torch.arange(6).view(2, 3))
    large.table.copy_(torch.tensor([[pages - 1, 0, pages - 3], [pages - 2, pages - 6, 5]]))
    apart = torch.empty(2 * T * heads * dim + (1 << 30) + 4096, dtype=F32, device=dev)  # 2^32 bytes between the sequences
    k, v, q = [apart[i:].as_strided((2, n, h, dim), (1 << 30, h * dim, dim, 1))
               for i, n, h in ((0, T, heads), (T * heads * dim, T, heads), (2 * T * heads * dim, 2, 4))]
    g = torch.Generator().manual_seed(7)
    for x in (k, v, q):
        x.copy_(torch.randn(x.shape, generator=g))
    small.append(k.contiguous(), v.contiguous())
    large.append(k, v)
    for x, y in zip(large.read(3, T), small.read(3, T)):
        assert torch.equal(x, y)
    assert torch.equal(large.attend(q), small.attend(q.contiguous()))
    kept = small.length.clone()
    assert torch.equal(large.length, kept) and int(kept[0]) == T
    _compare(small, q[:, 1:].contiguous(), small.attend(q[:, 1:].contiguous()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,qt", [(F32, F32), (F16, F16), (I8, F32), (E4M3, BF16)])
def test_attention_starts_counts_and_missing_pages(dev, dtype, qt):
    lengths, T = [100, 100, 100, 100, 100, 100, 100, 0], 5
    b = _buffer(dev, lengths, 2, 48, 16, dtype, seed=3, room=128)
    b.table[0, 2], b.table[1, 6], b.table[2, 0] = -1, b.k.shape[0], -2147483648
    b.table[3, :] = -1
    g = torch.Generator().manual_seed(0)
    q = torch.randn(len(lengths), T, 6, 48, generator=g).to(qt).to(dev)
    _compare(b, q, b.attend(q))
    start = torch.tensor([0, 50, -2, -100, 98, 1 << 60, 95, 3], device=dev)
    counts = torch.tensor([5, 0, 9, 2, 3, 5, -4, 1], device=dev)
    announce("starts, counts, pages that are none")
    _compare(b, q, b.attend(q, start), start)
    _compare(b, q, b.attend(q, None, counts), None, counts)
    got = b.attend(q, start, counts)
    _compare(b, q, got, start, counts)
    assert float(got[1].abs().sum()) == 0 and float(got[6].abs().sum()) == 0 and float(got[3].abs().sum()) == 0
    b.window = 7
    _compare(b, q, b.attend(q, start, counts), start, counts)
    _compare(b, q, b.attend(q, 40, None, 0.5), [40] * 8, None, 0.5)
    _compare(b, q, b.attend(q, 40, None, -0.25), [40] * 8, None, -0.25)
    b.length.fill_(1 << 40)  # more than the table holds
    b.window = None
    ok = b.attend(q, torch.full((8,), 20, device=dev))
    assert torch.isfinite(ok[4:7]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,qt", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32), (I8, F32), (E4M3, BF16)])
def test_what_a_row_does_not_see_does_not_reach_it(dev, dtype, qt):
    """Infinities, NaN and the largest values in positions that other rows of the tile see."""
    T, n = 4, 37
    b = _buffer(dev, [n, n], 1, 64, 16, dtype, seed=4, room=48)
    g = torch.Generator().manual_seed(0)
    q = torch.randn(2, T, 4, 64, generator=g).to(qt).to(dev)
    want = b.attend(q).clone()
    for what in (float("nan"), float("inf"), -float("inf"), 3e4):
        for pos in (n - 1, n - 3):  # seen by the last row, by the last three
            at, row = int(b.table[0, pos // 16]), pos % 16
            keep = [None if t is None else t.clone() for t in (b.k, b.v, b.k_scale, b.v_scale)]
            if dtype in LARGEST:
                b.k_scale[at, 0, row] = b.v_scale[at, 0, row] = what
            else:
                b.k[at, 0, row, 5], b.v[at, 0, row, 9] = what, what
            announce(f"{what} at {pos} {dtype}")
            got = b.attend(q)
            first = pos - (n - T)  # rows from this one on see it
            assert torch.equal(got[0, :first], want[0, :first]) and torch.equal(got[1], want[1])
            if what != what:
                assert torch.isnan(got[0, first:]).any(-1).all()
            for t, old in zip((b.k, b.v, b.k_scale, b.v_scale), keep):
                if t is not None:
                    t.copy_(old)
    # an infinity or NaN of V alone, seen: the formula's
    if dtype not in LARGEST:
        at, row = int(b.table[0, (n - 2) // 16]), (n - 2) % 16
        b.v[at, 0, row, 3], b.v[at, 0, row, 4], b.v[at, 0, row, 5] = float("inf"), -float("inf"), float("nan")
        got = b.attend(q)
        assert torch.equal(got[0, :2], want[0, :2])
        assert (got[0, 2:, :, 3] == float("inf")).all() and (got[0, 2:, :, 4] == -float("inf")).all()
        assert torch.isnan(got[0, 2:, :, 5]).all()
        other = [i for i in range(64) if i not in (3, 4, 5)]
        assert torch.equal(got[0, :, :, other], want[0, :, :, other])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,qt", [(F16, F16), (I8, F32), (I8, BF16), (E4M3, F16), (BF16, F32)])
def test_attention_far_scales(dev, dtype, qt):
    """One position takes nearly all the weight, values and queries of very different sizes."""
    b = _buffer(dev, [500, 80], 2, 64, 16, dtype, seed=5)
    g = torch.Generator().manual_seed(0)
    q = torch.randn(2, 1, 4, 64, generator=g)
    if b.v_scale is not None:
        spread = torch.exp2(torch.randint(-20, 8, b.v_scale.shape, generator=g).float()).to(dev)
        b.v_scale.mul_(spread)
    q[0] *= 40
    q[1, 0, :, ::2] *= 1e-4
    q = q.to(qt).to(dev)
    _compare(b, q, b.attend(q))
    _compare(b, q, b.attend(q, scale=1e-30), None, None, 1e-30)


@pytest.mark.gpu
def test_attention_strides_out_and_workspace(dev):
    b = _buffer(dev, [90, 40, 7], 2, 40, 16, I8, seed=6, room=2000)
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(3, 2, (6 + 4) * 40, generator=g).to(dev)
    q = qkv[..., :240].unflatten(-1, (6, 40))
    want = b.attend(q.contiguous())
    assert torch.equal(b.attend(q), want)
    heads_first = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(b.attend(heads_first), want)
    columns = q.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(b.attend(columns), want)
    room = torch.full((3, 2, 6, 43), 7.0, device=dev)
    assert b.attend(q, out=room[..., 1:41]).data_ptr() == room[..., 1:].data_ptr()
    assert torch.equal(room[..., 1:41], want) and float(room[..., 0].sum()) == 7 * 36 and float(room[..., 41:].sum()) == 7 * 72
    ws = torch.full((1 << 22,), 255, dtype=torch.uint8, device=dev)
    assert torch.equal(b.attend(q, workspace=ws), want)
    for bad in (dict(q=q.double()), dict(q=q.cpu()), dict(q=q[:2]), dict(q=q[:, :, :5]), dict(q=q[..., :39]), dict(q=q[:, :, :0]),
                dict(q=q, out=q), dict(q=q, out=torch.empty_like(q).half()), dict(q=q, workspace=ws[:8]),
                dict(q=q, workspace=ws.cpu()), dict(q=q, start=torch.zeros(2, dtype=torch.long, device=dev)),
                dict(q=q, counts=torch.zeros(3, device=dev)), dict(q=q, scale=float("nan")),
                dict(q=q, out=torch.empty(1, 2, 6, 40, device=dev).expand(3, 2, 6, 40))):
        with pytest.raises(ValueError):
            b.attend(**bad)
    f = _buffer(dev, [9], 2, 40, 16, BF16)
    with pytest.raises(ValueError, match="dtype"):
        f.attend(torch.zeros(1, 1, 2, 40, dtype=F16, device=dev))
    assert b.attend(q[:, :0]).shape == (3, 0, 6, 40)


@pytest.mark.gpu
def test_replaced_tensors_are_checked(dev):
    b = _buffer(dev, [20, 5], 2, 24, 16, I8)
    q = torch.randn(2, 1, 2, 24, device=dev)
    want = b.attend(q)
    for name, bad in (("k", b.k.contiguous()), ("k", b.k[:1]), ("v", b.v.float()), ("k_scale", None), ("v_scale", b.v_scale[:1]),
                      ("table", b.table.long()), ("table", b.table[:1]), ("length", b.length[:1]), ("length", b.length.int()),
                      ("length", b.length.cpu())):
        old = getattr(b, name)
        setattr(b, name, bad)
        with pytest.raises(ValueError):
            b.attend(q)
        with pytest.raises(ValueError):
            b.append(q[:, :, :2].contiguous(), q)
        setattr(b, name, old)
    assert torch.equal(b.attend(q), want)
    x = torch.zeros(2, 1, 2, 24, device=dev)
    for bad in (dict(k=x[:1], v=x[:1]), dict(k=x, v=x[:, :, :1]), dict(k=x.cpu(), v=x.cpu()), dict(k=x[0], v=x[0]),
                dict(k=x[0], v=x[0], sequence=2), dict(k=x, v=x, sequence=0), dict(k=x, v=x, start=torch.zeros(2, device=dev)),
                dict(k=x, v=x, counts=torch.zeros(1, dtype=torch.long, device=dev))):
        with pytest.raises(ValueError):
            b.append(**bad)
    for bad in (dict(start=0, count=-1), dict(start=0, count=1, dtype=I8), dict(start=0, count=1, sequence=-1)):
        with pytest.raises(ValueError):
            b.read(**bad)


# ---------------------------------------------------------------------------
# the operators together
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, I8, E4M3])
def test_step_with_drafts(dev, dtype):
    """Three sequences decode: projections' outputs through step, drafts chosen by
    verify_drafts and taken back by truncate; the attention of every step
    against the formula over what was kept, the kept tokens' positions against
    those of an append of them alone."""
    B, T, H, heads, dim, page, V = 3, 4, 4, 2, 64, 16, 500
    g = torch.Generator().manual_seed(8)
    b = DevicePagedKVBuffer(B, heads, dim, 24, page, 8, None, dev, dtype)
    plain = DevicePagedKVBuffer(B, heads, dim, 24, page, 8, None, dev, dtype)
    f = (1e4 ** -(torch.arange(32) / 32)).to(dev)
    wq, wk = [(torch.rand(dim, generator=g) + 0.5).to(dev) for _ in range(2)]
    for i, n in enumerate((11, 0, 30)):  # prompts
        b.reserve(i, 100)
        plain.reserve(i, 100)
        if n:
            k, v = [torch.randn(n, heads, dim, generator=g).to(dev) for _ in range(2)]
            for x in (b, plain):
                x.append(k, v, sequence=i)
    for step in range(6):
        qkv = torch.randn(B, T, (H + 2 * heads) * dim, generator=g).to(dev)
        q, k, v = [t.unflatten(-1, (-1, dim)) for t in qkv.split([H * dim, heads * dim, heads * dim], -1)]
        start = b.length.clone()
        counts = None if step % 2 else torch.randint(1, T + 1, (B,), generator=g).to(dev)
        out = b.step(q, k, v, f, wq, wk, counts=counts)
        qr, kr = qk_norm_rope(q.flatten(0, 1), k.flatten(0, 1), (start[:, None] + torch.arange(T, device=dev)).reshape(-1), f, wq, wk)
        _compare(b, qr.view(q.shape), out, start, counts)
        target = torch.softmax(torch.randn(B, T + 1, V, generator=g) * 2, -1).to(dev)
        draft = torch.softmax(target[:, :T].log() + 0.2 * torch.randn(B, T, V, generator=g).to(dev), -1)
        tokens = torch.multinomial(draft.reshape(-1, V).cpu(), 1, generator=g).reshape(B, T).to(dev)
        kept, token = quant.verify_drafts(target, draft, tokens, torch.rand(B, T + 1, generator=g).to(dev), counts)
        assert int(token.min()) >= 0 and int(kept.min()) >= 0
        b.truncate(start + kept)
        plain.append(kr.view(k.shape), v, None, kept)
        assert torch.equal(b.length, start + kept) and torch.equal(plain.length, b.length)
        for x, y in zip(b.read(0, 100), plain.read(0, 100)):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_truncate_by_tensors(dev):
    b = DevicePagedKVBuffer(4, 1, 16, 4, 16, device=dev)
    b.length.copy_(torch.tensor([5, 9, 0, 7]))
    b.truncate(torch.tensor([6, 3, 2, -4], device=dev))
    assert b.length.tolist() == [5, 3, 0, 0]
    for bad in (torch.tensor([1, 2], device=dev), torch.tensor([1, 2, 3, 4]), torch.ones(4, device=dev)):
        with pytest.raises(ValueError, match="length"):
            b.truncate(bad)


@pytest.mark.gpu
def test_a_refused_step_stores_nothing(dev):
    B, T, H, heads, dim = 2, 3, 4, 2, 64
    b = DevicePagedKVBuffer(B, heads, dim, 8, 16, 4, None, dev, F16)
    for i in range(B):
        b.reserve(i, 40)
    f = (1e4 ** -(torch.arange(32) / 32)).to(dev)
    q, k, v = [torch.randn(B, T, n, dim, device=dev) for n in (H, heads, heads)]
    b.step(q, k, v, f)
    before = [t.clone() for t in (b.k, b.v, b.length)]
    long = [torch.zeros(B, _lib.SBQ_PAGED_MAX_T + 1, n, dim, device=dev) for n in (H, heads, heads)]
    for bad in (lambda: b.step(q.bfloat16(), k.bfloat16(), v, f), lambda: b.step(q[:, :, :3], k, v, f),
                lambda: b.step(q, k, v[:, :1], f), lambda: b.step(q, k, v, f, scale=float("nan")), lambda: b.step(*long, f),
                lambda: b.step(q, k, v, f, counts=torch.ones(3, dtype=torch.long, device=dev))):
        with pytest.raises(ValueError):
            bad()
    none = [t[:, :0] for t in (q, k, v)]
    assert b.step(*none, f).shape == (B, 0, H, dim)  # no tokens
    for x, y in zip((b.k, b.v, b.length), before):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, I8])
def test_step_captured_and_replayed(dev, dtype):
    """A captured step, replayed with other inputs and eager calls between, on another stream too."""
    B, T, H, heads, dim, page = 5, 2, 8, 2, 128, 64
    g = torch.Generator().manual_seed(3)
    f = (1e4 ** -(torch.arange(64) / 64)).to(dev)
    w = torch.ones(dim, device=dev)
    bufs = []
    for _ in range(2):
        b = DevicePagedKVBuffer(B, heads, dim, 60, page, 10, None, dev, dtype)
        for i, n in enumerate((0, 5, 64, 300, 70)):
            b.reserve(i, n + 40)
            b.length[i] = n
        bufs.append(b)
    held = [torch.randn(B, 400, heads, dim, generator=g).to(dev) for _ in range(2)]
    for b in bufs:
        n = b.length.clone()
        b.append(held[0], held[1], 0, n)
    a, e = bufs
    q, k, v = [torch.zeros(B, T, n, dim, dtype=BF16, device=dev) for n in (H, heads, heads)]
    a.step(q, k, v, f, w, w)
    e.step(q, k, v, f, w, w)
    n0 = a.length.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = a.step(q, k, v, f, w, w)
    assert torch.equal(a.length, n0)  # (recorded, not run)
    side = torch.cuda.Stream()
    for i in range(6):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g))
        torch.cuda.synchronize()
        if i % 2:
            with torch.cuda.stream(side):
                graph.replay()
                want = e.step(q, k, v, f, w, w)
        else:
            graph.replay()
            want = e.step(q, k, v, f, w, w)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(a.length, e.length) and int(a.length[0]) == 2 + 2 * (i + 1)
        for x, y in zip(a.read(0, 400), e.read(0, 400)):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_window_behind_which_pages_are_released(dev):
    B, heads, dim, page, window = 2, 2, 64, 16, 40
    b = DevicePagedKVBuffer(B, heads, dim, 12, page, 20, window, dev, F32)
    whole = DevicePagedKVBuffer(B, heads, dim, 40, page, 20, window, dev, F32)
    g = torch.Generator().manual_seed(6)
    for t in range(300):
        k, v = [torch.randn(B, 1, heads, dim, generator=g).to(dev) for _ in range(2)]
        for x in (b, whole):
            for i in range(B):
                x.reserve(i, t + 1)
            x.append(k, v)
        if t % 50 == 49:
            q = torch.randn(B, 1, 4, dim, generator=g).to(dev)
            got = b.attend(q)
            assert torch.equal(got, whole.attend(q))
            _compare(whole, q, got)
        for i in range(B):
            b.release(i, t + 1 - window)
    assert len(b._free) + sum(len(h) for h in b._held) == 12


@pytest.mark.gpu
def test_two_buffers_on_two_streams(dev):
    bufs = [_buffer(dev, [700, 30, 200], 2, 64, 32, d, seed=i, room=800) for i, d in enumerate((I8, BF16))]
    q = torch.randn(3, 1, 8, 64, device=dev)
    want = [b.attend(q) for b in bufs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in bufs]
    got = [[], []]
    for _ in range(20):
        for i, (b, s) in enumerate(zip(bufs, streams)):
            with torch.cuda.stream(s):
                got[i].append(b.attend(q))
    torch.cuda.synchronize()
    for w, results in zip(want, got):
        assert all(torch.equal(r, w) for r in results)
