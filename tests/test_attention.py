"""Attention over a cache and a tree of drafted tokens (sbq.state.
tree_attention, DeviceKVBuffer.attend) against the formula in 64 bits.

Tolerances, from the arithmetic: with x = sum of |scale q k| over dim, a
score carries at most (dim + 2) fp32 roundings, 2^-24 (dim + 2) x, and so
does the exponent of its weight; exp2, the rescalings and the sums of n
weights add at most 2^-24 (n / 16 + 64) relative (a lane group's sums run
over a quarter of the rows; 64 covers the joins); every weight error is at
most e = 2^-24 (dim + 2) max x + 2^-24 (n / 16 + 64) relative, in numerator
and denominator, so an output is off by 2 e max|v| at most.  2-byte queries
round each weight and the output by half a step of their type.  A slot's
summed attention weight is off by 2 e of itself and its additions.
"""
import ctypes

import pytest
import torch

from conftest import announce
from sbq import _lib
from sbq.state import DeviceKVBuffer, attention_workspace, tree_attention

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


# ---------------------------------------------------------------------------
# refusals (CPU)
# ---------------------------------------------------------------------------
def test_c_abi_refuses_bad_arguments():
    L = _lib.load()
    p = 1 << 16  # never read: every call below is refused

    def attn(q=p, qt=0, T=1, H=4, D=64, qst=256, qsh=64, k=p, v=p, ct=0, slots=8, Hk=2, kss=128, ksh=64, sp=p, qp=p, kn=None,
             vn=None, nss=0, nsh=0, tree=None, tld=0, window=0, scale=0.1, out=p, ost=256, osh=64, weight=None, ws=p,
             nws=1 << 30):
        return L.sbq_tree_attention(q, qt, T, H, D, qst, qsh, k, v, ct, slots, Hk, kss, ksh, sp, qp, kn, vn, nss, nsh, tree,
                                    tld, window, scale, out, ost, osh, weight, ws, nws, None)

    assert attn(qt=5) == -2 and attn(ct=-1) == -2 and attn(qt=1) == -2 and attn(qt=1, ct=2) == -2
    assert attn(T=-1) == -1 and attn(T=1025) == -1 and attn(H=5) == -1 and attn(D=0) == -1 and attn(D=257) == -1
    assert attn(slots=0) == -1 and attn(slots=(1 << 30) + 1) == -1 and attn(Hk=0) == -1 and attn(window=-1) == -1
    assert attn(scale=float("nan")) == -1
    for name in ("q", "k", "v", "sp", "qp", "out"):
        assert attn(**{name: None}) == -1
    assert attn(kn=p) == -1 and attn(vn=p) == -1 and attn(tree=p, tld=1) == -1
    assert attn(kn=p, vn=p, tree=p, tld=0) == -1 and attn(kss=-1) == -1
    assert attn(sp=p + 4) == -3 and attn(q=p + 2) == -3 and attn(weight=p + 2) == -3
    assert attn(ws=None) == -4 and attn(nws=8) == -4
    assert attn(T=0) == 0
    need = L.sbq_attn_workspace_bytes(1, 32, 8, 128, 4096, 1)
    assert need > L.sbq_attn_workspace_bytes(1, 32, 8, 128, 4096, 0) > 0
    assert attn(H=32, Hk=8, D=128, slots=4096, weight=p, nws=need - 1) == -4
    assert L.sbq_attn_workspace_bytes(1, 5, 2, 64, 8, 0) == 0 and L.sbq_attn_workspace_bytes(0, 4, 2, 64, 8, 0) == 0


def test_c_abi_refuses_outputs_that_meet():
    L = _lib.load()
    p = 1 << 16

    def attn(T, H, D, ost, osh):
        return L.sbq_tree_attention(p, 0, T, H, D, H * D, D, p, p, 0, 8, 1, D, D, p, p, None, None, 0, 0, None, 0, 0, 0.1, p,
                                    ost, osh, None, p, 1 << 30, None)

    for bad in ((2, 1, 64, 0, 64), (1, 2, 64, 128, 63), (2, 2, 64, 64, 64), (2, 2, 64, 127, 64), (3, 2, 8, 8, 23)):
        assert attn(*bad) == -1, bad


def test_python_refuses_cpu_tensors():
    buf = DeviceKVBuffer(2, 8, 16, device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        buf.attend(torch.zeros(1, 4, 8), torch.zeros(1, dtype=torch.long))


# ---------------------------------------------------------------------------
# the formula
# ---------------------------------------------------------------------------
def _formula(q, k, v, see, scale):
    """(out, p summed over heads, largest score) in 64 bits; see [T, slots]; a
    row that sees nothing is 0."""
    T, H, D = q.shape
    rep = H // k.shape[1]
    out, ps = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, k.shape[0], dtype=torch.float64)
    xmax = 0.0
    for h in range(H):
        kh, vh, qh = k[:, h // rep].double(), v[:, h // rep].double(), q[:, h].double()
        z = (qh @ kh.t()) * scale
        xmax = max(xmax, float((qh.abs() @ kh.abs().t()).max()) * abs(scale))
        p = torch.softmax(torch.where(see, z, float("-inf")), -1)
        p = torch.where(see.any(-1, keepdim=True), p, 0.0)
        ps += p
        out[:, h] = p @ vh
    return out, ps, xmax


def _compare(o, weight, weight0, q, k, v, see, scale, slots):
    """Outputs (on the CPU) against the formula; k, v hold the drafts last."""
    want, p, xmax = _formula(q, k, v, see, scale)
    D, n = q.shape[2], k.shape[0]
    e = 2.0 ** -24 * ((D + 2) * xmax + n / 16 + 64)
    half = torch.finfo(o.dtype).eps / 2
    vmax = float(v.double().abs().max())
    tol = 2 * e * vmax
    if q.dtype != F32:
        tol += half * vmax  # the weights' roundings: at most half a step of each
        if q.dtype == F16:
            tol += n * 2.0 ** -25 * vmax  # ... or of fp16's smallest step, against a sum of at least 1
    off = (o.double() - want).abs()
    bound = tol + (want.abs() + tol) * half + torch.finfo(o.dtype).tiny
    assert bool((off <= bound).all()), f"worst {float((off / bound).max()):.3g} of the bound"
    if weight is not None:
        w = p[:, :slots].sum(0)
        tol = 2 * e * w + 2.0 ** -24 * (w + weight0.double().abs()) * (q.shape[0] * q.shape[1] / 4 + 6)
        off = (weight.double() - weight0.double() - w).abs()
        assert bool((off <= tol + 1e-30).all()), f"weight: {float((off - tol).max()):.3g} over the bound"


def _tree(T, g):
    parent = [-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, T)]
    tree, depth = torch.eye(T, dtype=torch.bool), [0] * T
    for i in range(1, T):
        tree[i] |= tree[parent[i]]
        depth[i] = depth[parent[i]] + 1
    return tree, torch.tensor(depth)


def _see(slot_pos, q_pos, tree, window):
    far = window or 1 << 40
    age = q_pos[:, None] - slot_pos[None]
    see = (slot_pos[None] >= 0) & (age >= 0) & (age < far)
    if tree is not None:
        see = torch.cat([see, tree & (q_pos[:, None] - q_pos[None] < far)], 1)
    return see


def _case(dev, T, heads, kv, D, slots, filled, window, qt, ct, drafts, weight, seed=0):
    g = torch.Generator().manual_seed(seed + T * 31 + slots)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    k, v, q = r(slots, kv, D).to(ct), r(slots, kv, D).to(ct), (r(T, heads, D) * 1.5).to(qt)
    at = torch.arange(slots)
    if window:
        pos = filled - 1 - (filled - 1 - at) % slots
        pos = torch.where(pos < 0, -1, pos)
    else:
        pos = torch.where(at < filled, at, -1)
    kn = vn = tree = None
    if drafts:
        kn, vn = r(T, kv, D).to(ct), r(T, kv, D).to(ct)
        tree, depth = _tree(T, g)
        q_pos = filled + depth
    else:
        q_pos = filled - T + torch.arange(T)
    w0 = torch.rand(slots, generator=g) if weight else None
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    buf = DeviceKVBuffer(kv, D, slots, window, dev, ct)
    buf.k.copy_(k), buf.v.copy_(v), buf.slot_pos.copy_(pos)
    wd = to(w0)
    announce(f"attend T={T} heads={heads}/{kv} D={D} slots={slots} filled={filled} window={window} {qt} over {ct} "
             f"drafts={drafts} weight={weight}")
    o = buf.attend(to(q), to(q_pos), to(kn), to(vn), to(tree), weight=wd)
    assert o.dtype == qt and o.shape == q.shape
    if drafts:
        k, v = torch.cat([k, kn]), torch.cat([v, vn])
    _compare(o.cpu(), None if wd is None else wd.cpu(), w0, q, k, v, _see(pos, q_pos, tree, window), D ** -0.5, slots)
    return buf, q, q_pos, o


TYPES = [(F32, F32), (F16, F16), (BF16, BF16), (F32, F16), (F32, BF16)]
IDS = ["f32", "f16", "bf16", "f32_f16", "f32_bf16"]


@pytest.mark.gpu
@pytest.mark.parametrize("qt,ct", TYPES, ids=IDS)
@pytest.mark.parametrize("D", [64, 128, 256, 80, 1, 33, 200])
def test_attend_types_and_widths(dev, D, qt, ct):
    for T, heads, kv, slots, filled, window, drafts, weight in (
            (1, 4, 1, 1, 1, None, False, False), (1, 8, 2, 100, 77, None, False, True),
            (5, 14, 2, 257, 300, 200, True, True), (9, 8, 8, 640, 640, None, True, False),
            (3, 6, 3, 70, 90, 60, False, True)):
        _case(dev, T, heads, kv, D, slots, filled, window, qt, ct, drafts, weight)


@pytest.mark.gpu
@pytest.mark.parametrize("qt,ct", TYPES, ids=IDS)
def test_attend_long_and_many_rows(dev, qt, ct):
    for T, heads, kv, D, slots, filled, window, drafts, weight in (
            (1, 32, 8, 128, 5000, 4321, None, False, True), (16, 8, 2, 128, 3000, 2990, None, True, True),
            (64, 16, 2, 64, 1111, 1000, None, True, False), (130, 2, 1, 128, 500, 200, None, True, True),
            (64, 4, 4, 256, 1500, 1400, None, False, False), (33, 7, 1, 128, 900, 2000, 850, True, True)):
        _case(dev, T, heads, kv, D, slots, filled, window, qt, ct, drafts, weight)


FEW = [(1, 8, 1, 128, 1, 1, None, False, True), (2, 8, 2, 64, 20001, 19000, None, True, True),
       (4, 4, 2, 128, 17000, 40000, 16990, True, True), (8, 3, 3, 80, 300, 290, None, False, True),
       (1, 256, 256, 64, 130, 130, None, False, True), (1, 264, 264, 64, 130, 120, None, False, True),
       (1, 4, 1, 256, 33000, 32990, None, False, True), (2, 4, 1, 128, 70000, 100, None, True, True),
       (1, 64, 8, 128, 40000, 39999, None, True, True), (9, 1, 1, 64, 700, 650, None, False, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("qt,ct", [(F32, F32), (BF16, BF16), (F32, F16)], ids=["f32", "bf16", "f32_f16"])
@pytest.mark.parametrize("case", FEW, ids=[f"T{c[0]}_H{c[1]}_D{c[3]}_{c[4]}" for c in FEW])
def test_attend_few_rows_weight(dev, case, qt, ct):
    """The slots' weights of few rows come from scores that the attention kept; on both sides of its limits."""
    _case(dev, *case[:7], qt, ct, *case[7:])


@pytest.mark.gpu
@pytest.mark.parametrize("qt,ct", TYPES, ids=IDS)
def test_attend_few_rows_hidden_values(dev, qt, ct):
    """Slots that a row does not see (some in blocks that no row sees) get nothing from it, whatever they hold."""
    T, heads, slots, D = 3, 2, 700, 128
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(n, heads, D, generator=g) for n in (T, slots, slots))
    q, k, v = q.to(qt), k.to(ct), v.to(ct)
    pos = torch.arange(slots)
    pos[::7] = -1
    pos[256:400] = -1
    k[pos < 0] = float("nan")
    k[650:] = float("inf")
    q_pos = torch.tensor([600, -1, 640])
    for workspace in (0, 255):  # (what it held before does not count)
        ws = torch.full((attention_workspace(T, heads, heads, D, slots, True, dev).numel(),), workspace, dtype=torch.uint8,
                        device=dev)
        weight = torch.zeros(slots, device=dev)
        o = tree_attention(q.to(dev), k.to(dev), v.to(dev), pos.to(dev), q_pos.to(dev), weight=weight, workspace=ws)
        see = _see(pos, q_pos, None, None)[:, :slots]
        clean = k.clone()
        clean[(pos < 0) | (pos > 640)] = 0.0
        assert bool((o[1] == 0).all())
        _compare(o.cpu(), weight.cpu(), torch.zeros(slots), q, clean, v, see, D ** -0.5, slots)


TILES = [(64, 8, 1, 128, 8300, 8200, None, True, True), (64, 8, 1, 64, 49300, 49000, None, True, True),
         (33, 16, 2, 128, 17000, 30000, 16900, True, True), (130, 4, 2, 64, 16500, 16400, None, True, False),
         (256, 1, 1, 128, 16384, 16384, None, False, True), (64, 4, 1, 128, 65536, 20, None, True, True),
         (16, 16, 1, 128, 49152, 60000, 40000, False, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("ct", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("case", TILES, ids=[f"T{c[0]}_D{c[3]}_{c[4]}" for c in TILES])
def test_attend_tiles(dev, case, ct):
    """Sizes of the kernels for many rows (256 and more of a key head)."""
    _case(dev, *case[:7], ct, ct, *case[7:])


@pytest.mark.gpu
def test_attend_tiles_many(dev):
    """More than 64 tiles of a workgroup: 32 row tiles leave 8 splits of 33000 slots."""
    _case(dev, 1024, 8, 1, 64, 33000, 32900, None, BF16, BF16, False, False)


@pytest.mark.gpu
@pytest.mark.parametrize("ct", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_attend_tiles_hidden_values(dev, D, ct):
    """As test_attend_empty_rows_and_hidden_values, in the kernel for many rows."""
    T, heads, slots = 64, 8, 8400
    g = torch.Generator().manual_seed(D)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v = r(T, heads, D).to(ct), r(slots, 1, D).to(ct), r(slots, 1, D).to(ct)
    kn, vn = r(T, 1, D).to(ct), r(T, 1, D).to(ct)
    pos = torch.arange(slots)
    pos[::5] = -1                      # empty slots hold anything
    k[::5], v[::5] = float("nan"), float("-inf")
    q_pos = torch.full((T,), slots + 1)
    q_pos[3], q_pos[7] = -2, 4000      # row 3 sees no slot, row 7 not all
    tree = torch.eye(T, dtype=torch.bool)
    tree[3, 3] = False
    kn[9], vn[9] = float("nan"), float("inf")   # draft 9: seen by itself and row 11 alone
    tree[11, 9] = True
    v[4004] = float("inf")             # hidden from rows 3 and 7 alone
    announce(f"tiles, hidden values D={D} {ct}")
    to = lambda t: t.to(dev)           # noqa: E731
    weight = torch.zeros(slots, device=dev)
    o = tree_attention(to(q), to(k), to(v), to(pos), to(q_pos), to(kn), to(vn), to(tree), weight=weight).cpu()
    assert bool((o[3] == 0).all())
    assert bool(torch.isnan(o[9]).all()) and bool(torch.isnan(o[11]).all())
    rest = [t for t in range(T) if t not in (3, 7, 9, 11)]
    assert bool((o[rest] == float("inf")).all())
    clean = lambda t: torch.nan_to_num(t.float(), 0.0, 0.0, 0.0).to(t.dtype)  # noqa: E731
    see = _see(pos, q_pos, tree, None)
    _compare(o[[7]], None, None, q[[7]], clean(torch.cat([k, kn])), clean(torch.cat([v, vn])), see[[7]], D ** -0.5, slots)


@pytest.mark.gpu
@pytest.mark.parametrize("qt,ct", TYPES, ids=IDS)
def test_attend_empty_rows_and_hidden_values(dev, qt, ct):
    """Rows that see nothing are 0; infinities and NaN in what a row does not
    see do not reach it, in what it sees they do."""
    for D, slots in ((128, 96), (64, 33), (80, 50)):
        T, heads, kv = 6, 4, 2
        g = torch.Generator().manual_seed(D)
        r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        q, k, v = r(T, heads, D).to(qt), r(slots, kv, D).to(ct), r(slots, kv, D).to(ct)
        kn, vn = r(T, kv, D).to(ct), r(T, kv, D).to(ct)
        pos = torch.arange(slots)
        pos[::3] = -1                   # empty slots hold anything
        k[::3], v[::3] = float("nan"), float("inf")
        q_pos = torch.tensor([-5, 7, slots + 3, slots + 3, 7, slots + 4])
        tree = torch.eye(T, dtype=torch.bool)
        tree[0, 0] = False              # row 0 sees nothing at all
        tree[5, 3] = True
        v[8:11] = float("inf")          # hidden from rows 1 and 4
        k[20, 1] = float("nan")
        kn[4], vn[4] = float("nan"), float("nan")   # draft 4: seen by itself alone
        to = lambda t: t.to(dev)        # noqa: E731
        announce(f"hidden values D={D} {qt} over {ct}")
        weight = torch.zeros(slots, device=dev)
        o = tree_attention(to(q), to(k), to(v), to(pos), to(q_pos), to(kn), to(vn), to(tree), weight=weight).cpu()
        assert bool((o[0] == 0).all())
        see = _see(pos, q_pos, tree, None)
        rows = [1]
        clean = lambda t: torch.nan_to_num(t.float(), 0.0, 0.0, 0.0).to(t.dtype)  # noqa: E731
        kk, vv = torch.cat([k, kn]), torch.cat([v, vn])
        _compare(o[rows], None, None, q[rows], clean(kk), clean(vv), see[rows], D ** -0.5, slots)
        assert bool(torch.isnan(o[4]).all())
        assert bool(torch.isinf(o[2:4, :2]).all()) and bool(torch.isnan(o[2:4, 2:]).all())  # v inf; k NaN in head 1
    # a cache that nobody sees, without drafts
    o = tree_attention(torch.ones(2, 2, 64, device=dev).to(qt), torch.full((40, 1, 64), float("nan"), device=dev).to(ct),
                       torch.full((40, 1, 64), float("nan"), device=dev).to(ct),
                       torch.full((40,), -1, device=dev), torch.arange(2, device=dev))
    assert bool((o == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("qt,ct", [(F32, F32), (F16, F16), (F32, BF16)], ids=["f32", "f16", "f32_bf16"])
def test_attend_strides(dev, qt, ct):
    """Head-major caches, sliced and misaligned rows, an out of its own strides."""
    g = torch.Generator().manual_seed(3)
    T, heads, kv, D, slots = 4, 8, 2, 64, 150
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    k, v, q = r(slots, kv, D).to(ct), r(slots, kv, D).to(ct), r(T, heads, D).to(qt)
    kn, vn = r(T, kv, D).to(ct), r(T, kv, D).to(ct)
    pos, q_pos = torch.arange(slots), slots + torch.arange(T)
    tree = torch.ones(T, T, dtype=torch.bool).tril()
    see = _see(pos, q_pos, tree, None)

    def layouts(t):
        yield t.to(dev)
        yield t.transpose(0, 1).contiguous().to(dev).transpose(0, 1)             # [heads, n, dim]
        pad = torch.zeros(t.shape[0], t.shape[1], D + 3, dtype=t.dtype)
        pad[..., 1:1 + D] = t
        yield pad.to(dev)[..., 1:1 + D]                                          # off 16 bytes
        yield t.transpose(1, 2).contiguous().to(dev).transpose(1, 2)             # dim not innermost

    for i, (kd, vd) in enumerate(zip(layouts(k), layouts(v))):
        for qd, knd, vnd in zip(layouts(q), layouts(kn), layouts(vn)):
            if i == 3:
                with pytest.raises(ValueError, match="unit stride"):
                    tree_attention(qd, kd, vd, pos.to(dev), q_pos.to(dev))
                continue
            out = torch.full((T, heads + 1, D + 2), 7.0, dtype=qt, device=dev)
            announce(f"strides cache {i} q {qd.stride()}")
            o = tree_attention(qd, kd, vd, pos.to(dev), q_pos.to(dev), knd, vnd, tree.to(dev).t().contiguous().t(),
                               out=out[:, :heads, 1:1 + D])
            _compare(o.cpu(), None, None, q, torch.cat([k, kn]), torch.cat([v, vn]), see, D ** -0.5, slots)
            assert bool((out[:, heads] == 7).all()) and bool((out[..., 0] == 7).all()) and bool((out[..., -1] == 7).all())
    # no tree: a chain
    a = tree_attention(q.to(dev), k.to(dev), v.to(dev), pos.to(dev), q_pos.to(dev), kn.to(dev), vn.to(dev))
    b = tree_attention(q.to(dev), k.to(dev), v.to(dev), pos.to(dev), q_pos.to(dev), kn.to(dev), vn.to(dev), tree.to(dev))
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_attend_far_positions_and_long_cache(dev):
    """Positions past 2^31, and a cache whose offsets pass 2^31 elements."""
    buf, q, q_pos, o = _case(dev, 3, 4, 2, 64, 100, 90, None, F32, F32, True, False)
    far = 5 << 31
    pos = torch.where(buf.slot_pos >= 0, buf.slot_pos + far, -1)
    g = torch.Generator().manual_seed(3 * 31 + 100)
    # the same keys and drafts at far positions give the same result
    k2 = tree_attention(q.to(dev), buf.k, buf.v, buf.slot_pos, q_pos.to(dev))
    k3 = tree_attention(q.to(dev), buf.k, buf.v, pos, q_pos.to(dev) + far)
    assert torch.equal(k2, k3)
    slots, stride = 70, 1 << 25   # a view of few slots far apart: offsets up to 2^31 + 2^27 elements
    big = torch.empty(slots * stride, dtype=F16, device=dev)
    k, v = (big.as_strided((slots, 1, 128), (stride, 128, 1), at) for at in (0, 4096))
    for t in (k, v):
        t.copy_(torch.randn(slots, 1, 128, generator=g).to(F16))
    q = torch.randn(2, 2, 128, generator=g).to(F16)
    announce("attend, offsets past 2^31")
    o = tree_attention(q.to(dev), k, v, torch.arange(slots, device=dev), torch.tensor([slots - 1, 30], device=dev))
    _compare(o.cpu(), None, None, q, k.cpu(), v.cpu(), _see(torch.arange(slots), torch.tensor([slots - 1, 30]), None, None),
             128 ** -0.5, slots)


@pytest.mark.gpu
def test_attend_refuses(dev):
    k = torch.zeros(8, 2, 64, device=dev)
    ok = dict(q=torch.zeros(2, 4, 64, device=dev), k=k, v=k, slot_pos=torch.arange(8, device=dev),
              q_pos=torch.arange(2, device=dev))
    kn = torch.zeros(2, 2, 64, device=dev)
    for bad in (dict(q=torch.zeros(2, 5, 64, device=dev)), dict(q=torch.zeros(2, 4, 32, device=dev)),
                dict(q=ok["q"].half()), dict(k=k.half()), dict(v=k.cpu()), dict(v=k.transpose(0, 1).contiguous().transpose(0, 1)),
                dict(slot_pos=ok["slot_pos"].int()), dict(slot_pos=ok["slot_pos"][:7]), dict(q_pos=ok["q_pos"][:1]),
                dict(q_pos=ok["q_pos"].cpu()), dict(window=0), dict(k_new=kn), dict(tree=torch.ones(2, 2, device=dev).bool()),
                dict(k_new=kn, v_new=kn.half()), dict(k_new=kn[:1], v_new=kn[:1]),
                dict(k_new=kn, v_new=kn, tree=torch.ones(2, 3, device=dev).bool()),
                dict(k_new=kn, v_new=kn, tree=torch.ones(2, 2, device=dev)), dict(weight=torch.zeros(7, device=dev)),
                dict(weight=torch.zeros(8, device=dev).double()), dict(out=torch.zeros(2, 4, 64, device=dev).half()),
                dict(workspace=torch.zeros(8, device=dev)), dict(q=torch.zeros(1025, 4, 64, device=dev),
                                                                 q_pos=torch.zeros(1025, dtype=torch.long, device=dev)),
                dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            tree_attention(**{**ok, **bad})
    empty = tree_attention(ok["q"][:0], k, k, ok["slot_pos"], ok["q_pos"][:0])
    assert empty.shape == (0, 4, 64)


@pytest.mark.gpu
def test_attend_streams_and_graph(dev):
    """Repeatable; on another stream; captured and replayed with new inputs."""
    g = torch.Generator().manual_seed(4)
    slots, kv, D, T, heads = 2000, 2, 128, 7, 8
    buf = DeviceKVBuffer(kv, D, slots, device=dev, dtype=BF16)
    buf.append(torch.randn(1500, kv, D, generator=g).to(dev), torch.randn(1500, kv, D, generator=g).to(dev))
    tree, depth = _tree(T, g)
    tree, q_pos = tree.to(dev), (1500 + depth).to(dev)
    q = torch.zeros(T, heads, D, dtype=BF16, device=dev)
    kn, vn = torch.zeros(T, kv, D, dtype=BF16, device=dev), torch.zeros(T, kv, D, dtype=BF16, device=dev)
    weight = torch.zeros(slots, device=dev)

    def step():
        return buf.attend(q, q_pos, kn, vn, tree, weight=weight)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step()
    for seed in range(4):
        for t in (q, kn, vn):
            t.copy_(torch.randn(t.shape, generator=g).to(dev))
        weight.zero_()
        graph.replay()
        w = weight.clone()
        got = o.clone()
        weight.zero_()
        assert torch.equal(step(), got) and torch.equal(weight, w)
        torch.cuda.synchronize()
        assert float(w.sum()) > 0


@pytest.mark.gpu
def test_attend_out_layouts_and_alias(dev):
    """out as a part of a larger array, tokens outside or inside; never q itself, nor with elements that meet."""
    T, heads, kv, D, slots = 3, 4, 2, 64, 200
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(n, h, D, generator=g).to(dev) for n, h in ((T, heads), (slots, kv), (slots, kv)))
    pos, q_pos = torch.arange(slots, device=dev), torch.arange(T, device=dev) + 150
    want = tree_attention(q, k, v, pos, q_pos)
    wide = torch.full((T, heads + 2, D + 8), 7.0, device=dev)
    tree_attention(q, k, v, pos, q_pos, out=wide[:, 1:1 + heads, :D])
    assert torch.equal(wide[:, 1:1 + heads, :D], want)
    wide[:, 1:1 + heads, :D] = 7.0
    assert bool((wide == 7).all())
    inside = torch.empty(heads, T, D, device=dev).transpose(0, 1)
    tree_attention(q, k, v, pos, q_pos, out=inside)
    assert torch.equal(inside, want)
    for bad in (q, torch.zeros(1, heads, D, device=dev).expand(T, heads, D)):
        with pytest.raises(ValueError):
            tree_attention(q, k, v, pos, q_pos, out=bad)
    far = tree_attention(q, k, v, pos, q_pos - 1000, q[:, :kv].contiguous(), q[:, :kv].contiguous(), window=2 ** 63 - 1)
    near = tree_attention(q, k, v, torch.full_like(pos, -1), q_pos, q[:, :kv].contiguous(), q[:, :kv].contiguous())
    assert torch.equal(far, near)  # only the drafts are seen, however wide the window


@pytest.mark.gpu
@pytest.mark.parametrize("qt,ct", TYPES, ids=IDS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attend_pairs_of_row_tiles(dev, D, qt, ct):
    """Sizes from which a wave takes two row tiles, the last one not full."""
    for T, heads, kv, slots, filled, window, drafts, weight in (
            (15, 8, 2, 36001, 35000, None, True, True), (5, 14, 2, 61000, 100000, 60990, False, False)):
        _case(dev, T, heads, kv, D, slots, filled, window, qt, ct, drafts, weight)


@pytest.mark.gpu
@pytest.mark.parametrize("qt,ct", TYPES, ids=IDS)
@pytest.mark.parametrize("D", [64, 128])
def test_attend_pairs_hidden_values(dev, D, qt, ct):
    """As test_attend_tiles_hidden_values, with two row tiles a wave."""
    T, heads, slots = 24, 2, 88000
    g = torch.Generator().manual_seed(D + 1)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v = r(T, heads, D).to(qt), r(slots, 1, D).to(ct), r(slots, 1, D).to(ct)
    kn, vn = r(T, 1, D).to(ct), r(T, 1, D).to(ct)
    pos = torch.arange(slots)
    pos[::5] = -1                      # empty slots hold anything
    k[::5], v[::5] = float("nan"), float("-inf")
    q_pos = torch.full((T,), slots + 1)
    q_pos[3], q_pos[7] = -2, 4000      # row 3 sees no slot, row 7 not all
    tree = torch.eye(T, dtype=torch.bool)
    tree[3, 3] = False
    kn[9], vn[9] = float("nan"), float("inf")   # draft 9: seen by itself and row 11 alone
    tree[11, 9] = True
    v[4004] = float("inf")             # hidden from rows 3 and 7 alone
    announce(f"pairs, hidden values D={D} {qt} over {ct}")
    to = lambda t: t.to(dev)           # noqa: E731
    o = tree_attention(to(q), to(k), to(v), to(pos), to(q_pos), to(kn), to(vn), to(tree)).cpu()
    assert bool((o[3] == 0).all())
    assert bool(torch.isnan(o[9]).all()) and bool(torch.isnan(o[11]).all())
    rest = [t for t in range(T) if t not in (3, 7, 9, 11)]
    assert bool((o[rest] == float("inf")).all())
    clean = lambda t: torch.nan_to_num(t.float(), 0.0, 0.0, 0.0).to(t.dtype)  # noqa: E731
    see = _see(pos, q_pos, tree, None)
    _compare(o[[7]], None, None, q[[7]], clean(torch.cat([k, kn])), clean(torch.cat([v, vn])), see[[7]], D ** -0.5, slots)


@pytest.mark.gpu
@pytest.mark.parametrize("qt,ct", TYPES, ids=IDS)
@pytest.mark.parametrize("T,heads,kv,D,slots", [(1, 8, 1, 64, 40000), (1, 256, 256, 8, 16000), (64, 64, 64, 64, 4096),
                                                (512, 32, 32, 64, 8192), (512, 16, 16, 128, 8200), (2, 128, 64, 256, 3000)])
def test_attend_many_slots_beside_a_large_one(dev, T, heads, kv, D, slots, qt, ct):
    """One slot of value 0 takes almost all of the weight, the others some
    2^-25 of it each; so many heads or rows that a wave takes many of them.  All values and weights are >= 0, so that each weight's
    relative error, e and half a step of the type, is the output's at most;
    2^-39 of the largest weight is half of fp16's smallest step below 2^14."""
    g = torch.Generator().manual_seed(D + T)
    q, k, v = torch.zeros(T, heads, D), torch.zeros(slots, kv, D), torch.rand(slots, kv, D, generator=g) + 0.5
    q[..., :2] = 1.0
    k[..., 0] = -17.5
    k[..., 1] = torch.randint(-2, 3, (slots, kv), generator=g) / 4
    k[0], v[0] = 0.0, 0.0
    q, k, v = q.to(qt), k.to(ct), v.to(ct)
    pos, q_pos = torch.arange(slots), slots + torch.arange(T)
    weight = torch.zeros(slots, device=dev)
    announce(f"attend, many slots beside a large one T={T} heads={heads}/{kv} D={D} slots={slots} {qt} over {ct}")
    o = tree_attention(q.to(dev), k.to(dev), v.to(dev), pos.to(dev), q_pos.to(dev), scale=1.0, weight=weight).cpu()
    want, p, xmax = _formula(q[:1], k, v, torch.ones(1, slots, dtype=torch.bool), 1.0)
    e = 2.0 ** -24 * ((D + 2) * xmax + slots / 16 + 64)
    half = torch.finfo(qt).eps / 2 if qt != F32 else 0.0
    bound = want * (2 * e + half) + slots * 2.0 ** -39
    bound = bound + (want + bound) * torch.finfo(qt).eps / 2
    off = (o.double() - want).abs()
    assert bool((off <= bound).all()), f"worst {float((off / bound).max()):.3g} of the bound"
    w = p[0] * T
    off = (weight.cpu().double() - w).abs()
    assert bool((off <= (2 * e + 2.0 ** -24 * (T * heads / 4 + 6)) * w + 1e-30).all())


@pytest.mark.gpu
@pytest.mark.parametrize("T,heads,kv,slots", [(768, 64, 64, 5504), (64, 8, 1, 8300), (6, 8, 2, 700), (15, 8, 2, 36001)])
@pytest.mark.parametrize("ct", [F16, BF16], ids=["f16", "bf16"])
def test_attend_only_scores_of_minus_infinity(dev, T, heads, kv, slots, ct):
    """A row whose scores are all -infinity is 0, whatever the values; in
    kernels with and without a joining launch."""
    g = torch.Generator().manual_seed(T)
    D = 64
    q, k, v = (torch.randn(n, h, D, generator=g) for n, h in ((T, heads), (slots, kv), (slots, kv)))
    k[..., 0] = 1.0
    q[5, :, 0] = float("-inf")
    v[3, :, 1], v[slots - 2, :, 2] = float("inf"), float("nan")
    announce(f"attend, scores of -infinity T={T} heads={heads}/{kv} slots={slots} {ct}")
    o = tree_attention(q.to(dev, ct), k.to(dev, ct), v.to(dev, ct), torch.arange(slots, device=dev),
                       torch.full((T,), slots, device=dev)).cpu()
    assert bool((o[5] == 0).all())
    rest = [t for t in range(T) if t != 5]
    assert bool((o[rest][..., 1] == float("inf")).all()) and bool(torch.isnan(o[rest][..., 2]).all())
    assert bool(torch.isfinite(o[rest][..., [0] + list(range(3, D))]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("qt,ct", TYPES, ids=IDS)
def test_attend_strides_of_single_entries(dev, qt, ct):
    """The stride of an axis of one entry does not count: one key head, one slot, one column."""
    g = torch.Generator().manual_seed(13)
    for slots, kv, D in ((90, 1, 64), (1, 2, 64), (1, 1, 16), (40, 2, 1)):
        q, k, v = (torch.randn(n, h, D, generator=g) for n, h in ((2, 4), (slots, kv), (slots, kv)))
        q, k, v = q.to(qt), k.to(ct), v.to(ct)
        pos, q_pos = torch.arange(slots), torch.tensor([slots, slots + 1])
        vd, (s0, s1, s2) = v.to(dev), v.stride()
        vd = vd.as_strided(v.shape, (s0 if slots > 1 else 7, s1 if kv > 1 else 5, s2 if D > 1 else 3))
        announce(f"strides of single entries slots={slots} kv={kv} D={D} {qt} over {ct}")
        o = tree_attention(q.to(dev), k.to(dev), vd, pos.to(dev), q_pos.to(dev))
        _compare(o.cpu(), None, None, q, k, v, _see(pos, q_pos, None, None), D ** -0.5, slots)


@pytest.mark.gpu
@pytest.mark.parametrize("qt,ct", TYPES, ids=IDS)
@pytest.mark.parametrize("T,heads,kv,D,slots", [(1, 4, 2, 64, 300), (40, 2, 1, 80, 200), (8, 8, 1, 128, 70000), (64, 8, 1, 64, 8300)])
def test_attend_very_large_scores(dev, T, heads, kv, D, slots, qt, ct):
    """Scores (times log2 e) up to 2^27, of either sign, products and sums exact
    in fp32 and more than 2^12 apart or equal: a row is the mean of the values
    of its largest score, to the rounding of the mean and of the output."""
    g = torch.Generator().manual_seed(slots)
    for top in (2 ** 10, 2 ** 22, 2 ** 23, 2 ** 24, 2 ** 25, 2 ** 26):
        for sign in (1, -1):
            q, k, v = torch.zeros(T, heads, D), torch.zeros(slots, kv, D), torch.randn(slots, kv, D, generator=g)
            b = min(4096, top // 64)                 # query times key: b * (top / b) (1 - i / 16), i = 0..7
            q[..., 0] = b * sign
            k[..., 0] = (top // b) * (1 - torch.randint(0, 8, (slots, kv), generator=g) / 16)
            q, k, v = q.to(qt), k.to(ct), v.to(ct)
            pos, q_pos = torch.arange(slots), torch.full((T,), slots)
            announce(f"attend, scores {sign * top} T={T} heads={heads}/{kv} D={D} slots={slots} {qt} over {ct}")
            o = tree_attention(q.to(dev), k.to(dev), v.to(dev), pos.to(dev), q_pos.to(dev), scale=1.0).cpu().double()
            z = q[0, 0, 0].double() * k[..., 0].double()
            for h in range(heads):
                zh, vh = z[:, h // (heads // kv)], v[:, h // (heads // kv)].double()
                want = vh[zh == zh.max()].mean(0)
                tol = (slots / 16 + 64) * 2.0 ** -24 * float(vh.abs().max())
                tol = tol + (want.abs() + tol) * torch.finfo(qt).eps / 2
                if qt != F32:  # the weights' roundings
                    tol = tol + torch.finfo(qt).eps / 2 * float(vh.abs().max())
                assert bool(((o[:, h] - want).abs() <= tol).all()), (top, sign, h)
