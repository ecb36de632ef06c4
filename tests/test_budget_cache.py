"""The bounded cache (sbq.state.DeviceBudgetKVBuffer): which slots append and
take choose, what they write and what they leave, against the documented
order; and a run of drafted tokens through 4-bit projections, the attention
over the bounded cache and its eviction together."""
import numpy as np
import pytest
import torch

from conftest import announce
from sbq import _lib, quant
from sbq.state import DeviceBudgetKVBuffer, DeviceKVBuffer, new_device_state

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


# ---------------------------------------------------------------------------
# refusals and layout (CPU)
# ---------------------------------------------------------------------------
def test_c_abi_refuses_bad_arguments():
    L = _lib.load()
    p = 1 << 16  # never read: every call below is refused

    def app(sp=p, w=p, slots=8, end=p, start=p, recent=2, k=p, v=p, ct=0, Hk=2, D=4, kss=8, ksh=4, kn=p, vn=p, nt=0, T=1,
            nss=8, nsh=4, ws=p, nws=1 << 20):
        return L.sbq_kv_append(sp, w, slots, end, start, recent, k, v, ct, Hk, D, kss, ksh, kn, vn, nt, T, nss, nsh, ws, nws,
                               None)

    assert app(ct=4) == -2 and app(nt=-2) == -2
    assert app(slots=0) == -1 and app(recent=9) == -1 and app(recent=-1) == -1 and app(T=9) == -1 and app(T=-1) == -1
    assert app(Hk=0) == -1 and app(D=0) == -1 and app(kss=-1) == -1 and app(D=1 << 16, Hk=1 << 16) == -1
    for name in ("sp", "w", "end", "start", "k", "v", "kn", "vn"):
        assert app(**{name: None}) == -1
    assert app(sp=p + 4) == -3 and app(w=p + 1) == -3 and app(ct=1, k=p + 1) == -3
    assert app(ws=None) == -4 and app(nws=7) == -4 and app(T=0) == 0

    def take(sp=p, w=p, slots=8, end=p, k=p, v=p, ct=0, Hk=2, D=4, kss=8, ksh=4, cap=4, recent=2, tp=p, tw=p, te=p, tk=p,
             tv=p, tss=8, tsh=4, ws=p, nws=1 << 20):
        return L.sbq_kv_take(sp, w, slots, end, k, v, ct, Hk, D, kss, ksh, cap, recent, tp, tw, te, tk, tv, tss, tsh, ws, nws,
                             None)

    assert take(ct=3) == -2 and take(cap=0) == -1 and take(recent=5) == -1 and take(slots=0) == -1 and take(tss=-1) == -1
    for name in ("sp", "w", "end", "k", "v", "tp", "tw", "te", "tk", "tv"):
        assert take(**{name: None}) == -1
    assert take(te=p + 4) == -3 and take(ws=None) == -4 and take(nws=16) == -4
    assert L.sbq_kv_workspace_bytes(8, 0) == 0 and L.sbq_kv_workspace_bytes(0, 8) == 0
    assert L.sbq_kv_workspace_bytes(8, 12) == 4 * 12 + 20 and app(nws=L.sbq_kv_workspace_bytes(8, 1) - 1) == -4


def test_buffer_refuses_and_new_state():
    with pytest.raises(ValueError):
        DeviceBudgetKVBuffer(2, 4, 8, 9, "cpu")
    b = DeviceBudgetKVBuffer(2, 4, 8, 2, "cpu")
    with pytest.raises(ValueError, match="GPU"):
        b.append(torch.zeros(1, 2, 4), torch.zeros(1, 2, 4))
    with pytest.raises(ValueError, match="expected"):
        b.append(torch.zeros(1, 2, 5), torch.zeros(1, 2, 5))
    with pytest.raises(ValueError, match="more tokens"):
        b.append(torch.zeros(9, 2, 4), torch.zeros(9, 2, 4))
    with pytest.raises(ValueError):
        b.take(b)
    b.slot_pos.copy_(torch.tensor([5, -1, 7, 1, 2, 9, -1, 3]))
    b.weight.fill_(2.0)
    b.truncate(6)
    assert b.slot_pos.tolist() == [5, -1, -1, 1, 2, -1, -1, 3] and b.weight.tolist() == [2, 0, 0, 2, 2, 0, 0, 2]
    b.reset()
    assert float(b.weight.sum()) == 0 and int(b.slot_pos.max()) == -1
    st = new_device_state([True, False], 4, 8, 2, 3, window=5, capacity=64, device="cpu", budget=16, recent=4)
    assert isinstance(st.layers[1].kv, DeviceBudgetKVBuffer) and st.layers[1].kv.capacity == 16
    assert st.layers[1].kv.recent == 4 and not isinstance(st.layers[0].kv, DeviceBudgetKVBuffer)
    same = new_device_state([False], 4, 8, 2, 3, window=5, capacity=16, device="cpu", budget=16)
    assert not isinstance(same.layers[0].kv, DeviceBudgetKVBuffer)


# ---------------------------------------------------------------------------
# the order
# ---------------------------------------------------------------------------
def _order(pos, weight, newest, recent):
    """Slots in the order in which they are given up (numpy)."""
    rank = np.where(pos < 0, 0, np.where(pos >= newest - recent, 3, np.where(np.isnan(weight), 2, 1)))
    w = np.where(rank == 1, weight.astype(np.float64) + 0.0, 0.0)
    # -0.0 lies below 0.0
    sign = np.where((rank == 1) & (weight == 0) & np.signbit(weight), -1, 0)
    return np.lexsort((np.arange(len(pos)), sign, w, rank))


def _weights(kind, n, r):
    if kind == "ties":
        return r.integers(0, 3, n).astype(np.float32)
    if kind == "equal":
        return np.full(n, 0.25, np.float32)
    if kind == "zero":
        return np.zeros(n, np.float32)
    if kind == "odd":
        w = r.standard_normal(n).astype(np.float32) * 1e-3
        w[r.random(n) < 0.1] = np.inf
        w[r.random(n) < 0.1] = -np.inf
        w[r.random(n) < 0.1] = np.nan
        w[r.random(n) < 0.1] = -0.0
        w[r.random(n) < 0.1] = 0.0
        w[r.random(n) < 0.1] = 1e-42
        return w
    return np.exp(r.standard_normal(n) * 2).astype(np.float32)


def _filled(dev, n, kv, D, dtype, recent, kind, used, seed):
    """A buffer with `used` of its slots holding shuffled positions below 3 n."""
    r = np.random.default_rng(seed)
    b = DeviceBudgetKVBuffer(kv, D, n, recent, dev, dtype)
    pos = r.permutation(3 * n)[:n].astype(np.int64)
    pos[r.permutation(n)[used:]] = -1
    w = _weights(kind, n, r)
    g = torch.Generator().manual_seed(seed)
    b.k.copy_(torch.randn(n, kv, D, generator=g))
    b.v.copy_(torch.randn(n, kv, D, generator=g))
    b.slot_pos.copy_(torch.from_numpy(pos))
    b.weight.copy_(torch.from_numpy(w))
    b.end.fill_(3 * n)
    return b, pos, w, g


def _same(a, b):
    return torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))


APPENDS = [(1, 1, 0, 1), (5, 3, 5, 5), (64, 1, 0, 64), (64, 64, 64, 30), (1000, 7, 100, 1000), (1000, 400, 3, 700),
           (4096, 1, 512, 4096), (4097, 12, 4000, 4097), (20000, 33, 64, 19990), (32768, 1, 1, 32768), (32769, 64, 7, 32769),
           (100003, 5, 1024, 99000), (8192, 512, 100, 8192), (8195, 513, 0, 8000), (12290, 300, 4000, 12290)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "zero", "odd"])
@pytest.mark.parametrize("n,T,recent,used", APPENDS)
def test_append_takes_the_least_attended(dev, n, T, recent, used, kind):
    b, pos, w, g = _filled(dev, n, 2, 3, F32, recent, kind, used, n + T)
    k0, v0 = b.k.cpu(), b.v.cpu()
    k, v = torch.randn(T, 2, 3, generator=g), torch.randn(T, 2, 3, generator=g)
    announce(f"append n={n} T={T} recent={recent} used={used} {kind}")
    b.append(k.to(dev), v.to(dev))
    at = np.sort(_order(pos, w, 3 * n + T, recent)[:T])
    pos[at], w[at] = 3 * n + np.arange(T), 0
    k0[at], v0[at] = k, v
    assert torch.equal(b.slot_pos.cpu(), torch.from_numpy(pos))
    assert _same(b.weight, torch.from_numpy(w)) and _same(b.k, k0) and _same(b.v, v0)
    assert int(b.end) == 3 * n + T


FEW_CANDIDATES = [(8195, 12, 100, 8195), (8192, 128, 0, 8192), (8193, 127, 8000, 8193), (8192, 129, 50, 8192),
                  (32768, 2, 1024, 32768), (12289, 64, 12289, 12289), (20000, 51, 10, 19990)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("n,T,recent,used", FEW_CANDIDATES)
def test_append_few_candidates(dev, n, T, recent, used, kind):
    """Workgroups' first slots, on both sides of the number that is ranked; a last workgroup with fewer slots than tokens."""
    test_append_takes_the_least_attended(dev, n, T, recent, used, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("ct", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("nt", [F32, F16, BF16, torch.float64], ids=["f32", "f16", "bf16", "f64"])
def test_append_types_strides_and_start(dev, nt, ct):
    for T, kv, D in ((2, 4, 128), (40, 8, 128), (3, 5, 33)):
        b, pos, w, g = _filled(dev, 300, kv, D, ct, 10, "spread", 290, T)
        k0, v0 = b.k.cpu(), b.v.cpu()
        k = torch.randn(kv, T, D + 1, generator=g).to(nt)
        v = torch.randn(T, kv, D, generator=g).to(nt)
        announce(f"append {nt} into {ct} T={T} kv={kv} D={D}")
        b.append(k.to(dev).transpose(0, 1)[..., 1:], v.to(dev), start=torch.tensor([7], device=dev) if T == 2 else 5000)
        start = 7 if T == 2 else 5000
        at = np.sort(_order(pos, w, start + T, 10)[:T])
        k0[at], v0[at] = k.transpose(0, 1)[..., 1:].to(ct), v.to(ct)
        pos[at] = start + np.arange(T)
        assert torch.equal(b.slot_pos.cpu(), torch.from_numpy(pos)) and int(b.end) == start + T
        assert _same(b.k, k0) and _same(b.v, v0)
    before = b.slot_pos.clone()
    b.append(torch.zeros(0, kv, D, device=dev), torch.zeros(0, kv, D, device=dev))
    assert torch.equal(b.slot_pos, before)
    with pytest.raises(ValueError, match="GPU"):
        b.append(torch.zeros(1, kv, D), torch.zeros(1, kv, D))


TAKES = [(1, 1, 0, 1), (10, 20, 5, 7), (100, 100, 3, 100), (100, 99, 99, 100), (1000, 64, 10, 900), (1000, 800, 100, 300),
         (5000, 1024, 1024, 5000), (20000, 777, 0, 15000), (32768, 4096, 512, 30000), (32769, 4096, 512, 32769),
         (100003, 2000, 100, 100003), (50000, 60000, 9, 49000)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("n,capacity,recent,used", TAKES)
def test_take_keeps_the_most_attended(dev, n, capacity, recent, used, kind):
    kv, D, ct = (2, 8, BF16) if n % 2 else (1, 5, F32)
    src, pos, w, g = _filled(dev, n, kv, D, ct, 0, kind, used, n)
    b = DeviceBudgetKVBuffer(kv, D, capacity, recent, dev, ct)
    b.k.fill_(7.0), b.v.fill_(8.0), b.slot_pos.fill_(3), b.weight.fill_(9.0)
    announce(f"take n={n} capacity={capacity} recent={recent} used={used} {kind}")
    b.take(src)
    at = _order(pos, w, 3 * n, recent)[max(0, n - capacity):]
    at = np.sort(at[pos[at] >= 0])
    m = len(at)
    assert torch.equal(b.slot_pos.cpu()[:m], torch.from_numpy(pos[at])) and bool((b.slot_pos[m:] == -1).all())
    assert _same(b.weight[:m].contiguous(), torch.from_numpy(w[at])) and bool((b.weight[m:] == 0).all())
    for to, fro, was in ((b.k, src.k, 7.0), (b.v, src.v, 8.0)):
        assert _same(to[:m].contiguous(), fro.cpu()[at]) and bool((to[m:] == was).all())
    assert int(b.end) == 3 * n


@pytest.mark.gpu
def test_take_from_a_window_and_refusals(dev):
    src = DeviceKVBuffer(2, 4, 12, 10, dev)
    for i in range(9):
        src.append(torch.full((2, 2, 4), float(i), device=dev), torch.full((2, 2, 4), -float(i), device=dev))
    w = torch.arange(12, device=dev).float()
    b = DeviceBudgetKVBuffer(2, 4, 6, 2, dev)
    b.take(src, w)
    # ring slots 0..5 hold positions 12..17, 6..11 hold 6..11; 16 and 17 stay, then the largest weights
    assert b.slot_pos.tolist() == [16, 17, 8, 9, 10, 11] and int(b.end) == 18
    for bad in ((b, None), (src, None), (src, w[:11]), (src, w.double()), (src, w.cpu()),
                (DeviceKVBuffer(2, 5, 12, None, dev), w), (DeviceKVBuffer(2, 4, 12, None, dev, F16), w),
                (DeviceKVBuffer(2, 4, 12, None, "cpu"), w)):
        with pytest.raises(ValueError):
            b.take(*bad)


@pytest.mark.gpu
def test_append_and_attend_captured(dev):
    """A decode step of a bounded layer (append, attend) replayed from a graph
    equals the eager steps, past the point where slots are given up."""
    kv, D, heads, n = 2, 64, 4, 40
    g = torch.Generator().manual_seed(0)
    eager, graphed = (DeviceBudgetKVBuffer(kv, D, n, 8, dev, BF16) for _ in range(2))
    k, v = torch.zeros(1, kv, D, device=dev), torch.zeros(1, kv, D, device=dev)
    q = torch.zeros(1, heads, D, dtype=BF16, device=dev)
    pos = torch.zeros(1, dtype=torch.long, device=dev)

    def step(b):
        b.append(k, v, pos)
        return b.attend(q, pos)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(graphed)
    torch.cuda.current_stream().wait_stream(side)
    graphed.reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step(graphed)
    for i in range(100):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g) * 2)
        pos.fill_(i)
        graph.replay()
        assert torch.equal(step(eager), o)
        for name in ("slot_pos", "weight", "k", "v", "end"):
            assert torch.equal(getattr(eager, name), getattr(graphed, name)), (i, name)
    held = set(eager.slot_pos.tolist())
    assert len(held) == n and set(range(92, 100)) <= held


# ---------------------------------------------------------------------------
# together: drafted tokens through one layer
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["int4", "int8"])
def test_drafted_steps_through_a_bounded_layer(dev, fmt):
    """A prompt into a full buffer with its attention weights counted, reduced
    to a bounded one, then steps of a tree of drafts: projections on the
    tree's rows, attention over cache and tree, the accepted path appended.
    Every operator is checked on the inputs it got: attention and eviction
    against the definition in 64 bits, and verifying a whole tree at once
    against its accepted path token by token."""
    H, heads, kv, D, prompt, budget, recent = 256, 8, 2, 64, 300, 96, 16
    g = torch.Generator().manual_seed(1)
    mods = {n: quant.make_linear(fmt, (torch.randn(N, H, generator=g) * 0.08).to(dev))
            for n, N in (("q", heads * D), ("k", kv * D), ("v", kv * D))}
    out = quant.make_linear(fmt, (torch.randn(H, heads * D, generator=g) * 0.05).to(dev))

    def project(x):
        T = x.shape[0]
        return mods["q"](x).view(T, heads, D), mods["k"](x).view(T, kv, D), mods["v"](x).view(T, kv, D)

    def formula(q, k, v, see):
        o, w = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(k.shape[0], dtype=torch.float64)
        for h in range(heads):
            z = q[:, h].double().cpu() @ k[:, h // 4].double().cpu().t() * D ** -0.5
            p = torch.nan_to_num(torch.softmax(torch.where(see, z, float("-inf")), -1), 0.0)
            o[:, h] = p @ v[:, h // 4].double().cpu()
            w += p.sum(0)
        return o, w

    def near(a, b, scale):
        # 64-term dot products, up to 364 weights: well below 2^-24 * 4096 of the largest value
        assert float((a.double().cpu() - b).abs().max()) <= 2.0 ** -12 * scale

    full = DeviceKVBuffer(kv, D, prompt, None, dev)
    weight = torch.zeros(prompt, device=dev)
    for at in range(0, prompt, 100):  # the prompt in chunks, every query's weights counted
        x = torch.randn(100, H, generator=g).to(dev)
        q, k, v = project(x)
        full.append(k, v)
        q_pos = at + torch.arange(100, device=dev)
        before = weight.cpu().double()
        o = full.attend(q, q_pos, weight=weight)
        want, w = formula(q, full.k, full.v, (torch.arange(prompt)[None] <= q_pos.cpu()[:, None]))
        near(o, want, float(full.v.abs().max()))
        near(weight, before + w, 100 * heads)
    b = DeviceBudgetKVBuffer(kv, D, budget, recent, dev)
    b.take(full, weight)
    keep = np.sort(_order(np.arange(prompt), weight.cpu().numpy(), prompt, recent)[prompt - budget:])
    assert b.slot_pos.tolist() == keep.tolist() and torch.equal(b.k, full.k[torch.from_numpy(keep).to(dev)])

    parent = [-1, 0, 0, 1, 1, 2, 3, 5, 6]
    T, path = len(parent), [0, 1, 3, 6, 8]
    tree, depth = torch.eye(T, dtype=torch.bool), [0] * T
    for i in range(1, T):
        tree[i] |= tree[parent[i]]
        depth[i] = depth[parent[i]] + 1
    for step in range(6):
        end = int(b.end)
        x = torch.randn(T, H, generator=g).to(dev)
        q, k, v = project(x)
        q_pos = end + torch.tensor(depth, device=dev)
        held, before, slots = b.slot_pos.cpu(), b.weight.cpu(), b.k.clone()
        o = b.attend(q, q_pos, k, v, tree.to(dev))
        see = torch.cat([(held >= 0)[None].expand(T, -1), tree], 1)
        want, w = formula(q, torch.cat([b.k, k]), torch.cat([b.v, v]), see)
        near(o, want, float(torch.cat([b.v, v]).abs().max()))
        near(b.weight, before.double() + w[:budget], T * heads)
        y = out(o.reshape(T, -1))
        # the accepted path, one token at a time over a copy of the cache
        line = DeviceKVBuffer(kv, D, budget + len(path), None, dev)
        line.k[:budget], line.v[:budget], line.slot_pos[:budget] = b.k, b.v, b.slot_pos
        for i, node in enumerate(path):
            line.k[budget + i], line.v[budget + i], line.slot_pos[budget + i] = k[node], v[node], end + i
            one = line.attend(q[node:node + 1], torch.tensor([end + i], device=dev))
            near(one, want[node:node + 1], float(line.v.abs().max()))
            near(out(one.reshape(1, -1)), y[node:node + 1].double().cpu(), float(y.abs().max()) * 8)
        weights, pos = b.weight.cpu().numpy(), held.numpy().copy()
        at = np.sort(_order(pos, weights, end + len(path), recent)[:len(path)])
        b.append(k[path], v[path])
        pos[at] = end + np.arange(len(path))
        slots[torch.from_numpy(at).to(dev)] = k[path]
        assert b.slot_pos.tolist() == pos.tolist() and torch.equal(b.k, slots) and int(b.end) == end + len(path)
    assert int((b.slot_pos >= int(b.end) - recent).sum()) == recent


def test_c_abi_refuses_rows_that_meet():
    L = _lib.load()
    p = 1 << 16
    for kss, ksh in ((0, 4), (8, 3), (7, 4), (4, 4)):
        assert L.sbq_kv_append(p, p, 8, p, p, 2, p, p, 0, 2, 4, kss, ksh, p, p, 0, 1, 8, 4, p, 1 << 20, None) == -1
        assert L.sbq_kv_take(p, p, 8, p, p, p, 0, 2, 4, 8, 4, 4, 2, p, p, p, p, p, kss, ksh, p, 1 << 20, None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_append_rows_of_the_cache_itself(dev, dtype):
    """Tokens whose keys and values are the cache's own rows, which the append takes over."""
    n = 40
    g = torch.Generator().manual_seed(5)
    buf = DeviceBudgetKVBuffer(2, 64, n, 0, dev, dtype)
    k, v = (torch.randn(n, 2, 64, generator=g).to(dev, dtype) for _ in range(2))
    buf.append(k, v)
    buf.weight.copy_(torch.rand(n, generator=g).to(dev))
    slots = torch.sort(torch.argsort(buf.weight)[:6]).values
    at = int(slots[0])
    rows = min(at, n - 6)
    announce(f"append own rows {rows}..{rows + 5} {dtype}")
    buf.append(buf.k[rows:rows + 6], buf.v[rows:rows + 6])
    assert torch.equal(buf.k[slots], k[rows:rows + 6]) and torch.equal(buf.v[slots], v[rows:rows + 6])


@pytest.mark.gpu
def test_take_refuses_its_own_weight(dev):
    src, dst = DeviceBudgetKVBuffer(2, 64, 32, 0, dev), DeviceBudgetKVBuffer(2, 64, 32, 0, dev)
    with pytest.raises(ValueError, match="own"):
        dst.take(src, dst.weight)


@pytest.mark.gpu
def test_take_from_a_very_long_cache(dev):
    """More slots than stay in LDS: every pass reads the keys again."""
    n, cap, recent = 70001, 5000, 100
    g = torch.Generator().manual_seed(6)
    src, dst = DeviceBudgetKVBuffer(1, 8, n, 0, dev), DeviceBudgetKVBuffer(1, 8, cap, recent, dev)
    src.append(torch.randn(60000, 1, 8, generator=g).to(dev), torch.randn(60000, 1, 8, generator=g).to(dev))
    weight = (torch.rand(n, generator=g) * 50).round() / 50   # (many equal ones)
    announce("take 5000 of 70001 slots")
    dst.take(src, weight.to(dev))
    order = torch.where(src.slot_pos.cpu() < 0, -1.0, torch.where(src.slot_pos.cpu() >= 60000 - recent, 1e9, weight.double()))
    kept = torch.sort(torch.argsort(order, stable=True)[n - cap:]).values
    assert torch.equal(dst.slot_pos.cpu(), src.slot_pos.cpu()[kept]) and torch.equal(dst.weight.cpu(), weight[kept])
    assert torch.equal(dst.k.cpu(), src.k.cpu()[kept]) and torch.equal(dst.v.cpu(), src.v.cpu()[kept])


@pytest.mark.gpu
def test_long_steps_in_a_graph(dev):
    """The kernels for many rows and long caches captured together and replayed
    with new inputs: a 4-bit linear, the attention with its weights, a take, an append."""
    g = torch.Generator().manual_seed(8)
    slots, cap, T, heads, D = 49152, 9000, 40, 8, 64
    long = DeviceKVBuffer(1, D, slots, device=dev, dtype=torch.bfloat16)
    rows = torch.randn(2, 45000, 1, D, generator=g).to(dev)
    long.append(rows[0], rows[1])
    lin = quant.Int4Linear(torch.randn(300, 1000, generator=g).to(dev) * 0.1, group=64)
    x = torch.zeros(T, 1000, device=dev)
    q, kn, vn = (torch.zeros(T, h, D, dtype=torch.bfloat16, device=dev) for h in (heads, 1, 1))
    q_pos = torch.full((T,), 45000, device=dev)
    weight = torch.zeros(slots, device=dev)
    small = [DeviceBudgetKVBuffer(1, D, cap, 100, dev, torch.bfloat16) for _ in range(2)]

    def step(buf):
        weight.zero_()
        y = lin(x)
        o = long.attend(q, q_pos, kn, vn, weight=weight)
        buf.take(long, weight)
        buf.append(kn[:12], vn[:12])
        return y, o

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(small[0])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, o = step(small[0])
    for i in range(4):
        announce(f"long steps, replay {i}")
        for t in (x, q, kn, vn):
            t.copy_(torch.randn(t.shape, generator=g).to(dev))
        graph.replay()
        got = y.clone(), o.clone(), weight.clone()
        want = step(small[1])
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2], weight)
        for name in ("slot_pos", "weight", "end", "k", "v"):
            assert torch.equal(getattr(small[0], name), getattr(small[1], name)), (i, name)
        assert int(small[0].end) == 45012 and int((small[0].slot_pos >= 45000).sum()) == 12


@pytest.mark.gpu
@pytest.mark.parametrize("n,capacity,newest", [(8192, 256, 600), (12288, 256, 600), (12289, 300, 2040), (20480, 256, 600),
                                               (20480, 2000, 2048), (24576, 256, 2049), (32768, 100, 600),
                                               (40000, 256, 600), (28000, 4000, 28000)])
def test_take_with_more_newest_slots_than_capacity(dev, n, capacity, newest):
    """`end` moved back (an append at an earlier start): more slots than are
    kept hold one of the newest positions, and the last of them stay."""
    recent = min(capacity, 100)
    src, pos, w, g = _filled(dev, n, 1, 4, F32, 0, "spread", n, n)
    end = int(np.sort(pos)[n - newest]) + recent
    src.end.fill_(end)
    b = DeviceBudgetKVBuffer(1, 4, capacity, recent, dev, F32)
    announce(f"take n={n} capacity={capacity}, {newest} slots of the newest positions")
    b.take(src)
    at = np.sort(_order(pos, w, end, recent)[n - capacity:])
    assert torch.equal(b.slot_pos.cpu(), torch.from_numpy(pos[at])) and _same(b.weight, torch.from_numpy(w[at]))
    assert _same(b.k, src.k.cpu()[at]) and _same(b.v, src.v.cpu()[at]) and int(b.end) == end


@pytest.mark.gpu
@pytest.mark.parametrize("n,T", [(5, 1), (300, 1), (300, 100), (9000, 40), (9000, 700), (40000, 12)])
def test_zeros_of_either_sign_are_equal(dev, n, T):
    """Slots of weight 0 and -0 are given up by index; a kept one keeps its bits."""
    r = np.random.default_rng(n + T)
    w = np.where(r.random(n) < 0.5, -0.0, 0.0).astype(np.float32)
    w[0] = 0.0
    w[r.permutation(n)[:T // 2]] = -1e-45
    at = np.sort(_order(np.arange(n), np.abs(w) * -1 + 0.0, n + T, 0)[:T])
    g = torch.Generator().manual_seed(n)
    for op in ("append", "take"):
        b = DeviceBudgetKVBuffer(1, 4, n, 0, dev)
        k = torch.randn(n, 1, 4, generator=g).to(dev)
        b.append(k, k)
        b.weight.copy_(torch.from_numpy(w))
        announce(f"{op}, zeros of either sign, n={n} T={T}")
        if op == "append":
            b.append(torch.ones(T, 1, 4, device=dev), torch.ones(T, 1, 4, device=dev))
            pos, want = np.arange(n), w.copy()
            pos[at], want[at] = n + np.arange(T), 0.0
        else:
            small = DeviceBudgetKVBuffer(1, 4, n - T, 0, dev)
            small.take(b)
            b, pos = small, np.delete(np.arange(n), at)
            want = w[pos]
        assert torch.equal(b.slot_pos.cpu(), torch.from_numpy(pos)) and _same(b.weight, torch.from_numpy(want))


@pytest.mark.gpu
@pytest.mark.parametrize("ct", [F32, BF16], ids=["f32", "bf16"])
def test_prompt_weights_slot_by_slot(dev, ct):
    """A prompt in chunks with its weights counted, then drafts: every slot's
    sum against the formula in 64 bits, to its own bound, which a single query
    row of one head left out (of the formula) would pass.  A weight is off by
    2 e of itself, e = 2^-24 ((D + 2) times the largest sum of |scale q k|, n / 16
    + 64 roundings in sums of weights), a sum by 2^-24 for each of the T * heads / 4
    + 6 terms that a lane adds."""
    heads, kv, D, prompt, chunk, T = 8, 2, 64, 300, 100, 9
    g = torch.Generator().manual_seed(12)
    buf = DeviceKVBuffer(kv, D, prompt, None, dev, ct)
    weight = torch.zeros(prompt, device=dev)
    for at in list(range(0, prompt, chunk)) + [prompt]:
        n = chunk if at < prompt else T
        q, k, v = ((torch.randn(n, h, D, generator=g) * 1.5).to(dev, ct) for h in (heads, kv, kv))
        q_pos = at + torch.arange(n)
        before = weight.cpu().double()
        announce(f"prompt weights at {at} {ct}")
        if at < prompt:
            buf.append(k, v)
            buf.attend(q, q_pos.to(dev), weight=weight)
            keys, see = buf.k.cpu().double(), torch.arange(prompt)[None] <= q_pos[:, None]
        else:
            buf.attend(q, q_pos.to(dev), k, v, weight=weight)
            keys = torch.cat([buf.k, k]).cpu().double()
            see = torch.cat([torch.ones(n, prompt, dtype=torch.bool), torch.ones(n, n, dtype=torch.bool).tril()], 1)
        p, xmax = torch.zeros(n, heads, keys.shape[0], dtype=torch.float64), 0.0
        for h in range(heads):
            qh, kh = q[:, h].cpu().double(), keys[:, h // (heads // kv)]
            xmax = max(xmax, float((qh.abs() @ kh.abs().t()).max()) * D ** -0.5)
            p[:, h] = torch.softmax((qh @ kh.t() * D ** -0.5).masked_fill(~see, float("-inf")), -1)
        w = p.sum((0, 1))[:prompt]
        e = 2.0 ** -24 * ((D + 2) * xmax + keys.shape[0] / 16 + 64)
        bound = 2 * e * w + 2.0 ** -24 * (w + before) * (n * heads / 4 + 6) + 1e-30
        off = weight.cpu().double() - before - w
        assert bool((off.abs() <= bound).all()), f"worst {float((off.abs() / bound).max()):.3g} of the bound"
        without = off + p[..., :prompt]  # the distance where this row's and head's weights were not counted
        assert bool((without.abs() > bound).any(-1).all())


@pytest.mark.gpu
def test_tokens_taken_back(dev):
    """truncate, then appends from there on: every position is held once, freed
    slots go first, and the attention is that of the tokens that are left."""
    kv, D, n, heads = 2, 64, 24, 4
    g = torch.Generator().manual_seed(14)
    buf, line = DeviceBudgetKVBuffer(kv, D, n, 4, dev), DeviceKVBuffer(kv, D, 200, None, dev)
    end = 0
    for i in range(12):
        k, v = (torch.randn(5, kv, D, generator=g).to(dev) for _ in range(2))
        if i % 3 == 2:
            end -= 4
            buf.truncate(end), line.truncate(end)
        buf.append(k, v, end), line.append(k, v, end)
        end += 5
        held = sorted(p for p in buf.slot_pos.tolist() if p >= 0)
        assert len(set(held)) == len(held) and int(buf.end) == end and set(range(end - 4, end)) <= set(held)
        assert len(held) == min(n, end) or i % 3 == 2
        at = buf.slot_pos.cpu()
        for slot in (at >= 0).nonzero().flatten().tolist():
            assert torch.equal(buf.k[slot], line.k[int(at[slot])]) and torch.equal(buf.v[slot], line.v[int(at[slot])])
        q, q_pos = torch.randn(2, heads, D, generator=g).to(dev), torch.tensor([end - 2, end - 1], device=dev)
        announce(f"tokens taken back, step {i}")
        o = buf.attend(q, q_pos)
        keep = torch.full_like(line.slot_pos, -1)
        keep[held] = torch.tensor(held, device=dev)
        # each side: weights to e = 2^-24 ((D + 2) sum |scale q k| + 66), outputs to 2 e max |v|
        e = 2.0 ** -24 * ((D + 2) * float(q.abs().sum(-1).max() * line.k.abs().max()) * D ** -0.5 + 66)
        line.slot_pos, was = keep, line.slot_pos
        other = line.attend(q, q_pos)
        line.slot_pos = was
        assert torch.allclose(o, other, rtol=0, atol=4 * e * float(line.v.abs().max()))
