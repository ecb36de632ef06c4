"""Head norms and rotation (sbq.state.qk_norm_rope, sbq_qk_norm_rope) against the
formula in 64 bits.

Tolerance of a fp32 computation: a normed value x r w carries the relative error
of r, (D/2 + 4) u at most (u = 2^-24: D products and sums under a root, the
division, the root), and two products; a rotated one a cos - b sin has that of
a and b, 2 u of the cosines' (series and reduction) and three roundings.  So
each output is off by at most (|a| + |b|) (D/2 + 14) u, and half a step of its
own type."""
import numpy as np
import pytest
import torch

from conftest import announce
from sbq import _lib
from sbq.state import qk_norm_rope

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24
PI = np.longdouble("3.14159265358979323846264338327950288")


def _formula(x, w, pos, f, eps, inter):
    """(result, |a| + |b| of each output) in 64 bits; x [n, h, D] numpy."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    n = len(f)
    # the angle's product of an int64 and a float32 in extended precision, reduced there
    angle = np.asarray(pos, dtype=np.longdouble)[:, None] * f.astype(np.longdouble)
    angle = np.remainder(angle, 2 * PI).astype(np.float64)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    i, j = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if inter else (slice(0, n), slice(n, 2 * n))
    y, size = x.copy(), np.abs(x)
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    size[..., i] = size[..., j] = np.abs(x[..., i]) + np.abs(x[..., j])
    return y, size


def _near(got, want, size, D):
    t = got.dtype
    g = got.detach().cpu().double().numpy()
    tol = size * (D / 2 + 14) * U + np.abs(want) * (torch.finfo(t).eps / 2) * 1.001 + torch.finfo(t).smallest_normal * U
    if t == F16:
        tol += 2.0 ** -25  # half a step of the smallest numbers
    bad = np.abs(g - want) > tol
    assert not bad.any(), (np.abs(g - want) / tol).max()


def _freq(n, base=1e6):
    return (base ** -(np.arange(n, dtype=np.float64) / max(n, 1))).astype(np.float32)


def _case(dev, T, H, kv, D, pairs, inter, dtype, norm, seed=0, positions=None, eps=1e-6, wt=F32):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(T, H, D, generator=g) * 2).to(dtype).to(dev)
    k = (torch.randn(T, kv, D, generator=g) * 2).to(dtype).to(dev) if kv else None
    f = torch.from_numpy(_freq(pairs)).to(dev)
    pos = torch.randint(0, 200000, (T,), generator=g) if positions is None else positions
    wq, wk = [(torch.rand(D, generator=g) + 0.5).to(wt).to(dev) if norm else None for _ in range(2)]
    return q, k, pos.to(dev), f, wq, wk if kv else None


def _check(out, q, k, pos, f, wq, wk, inter, eps=1e-6):
    for got, x, w in ((out[0], q, wq), (out[1], k, wk)):
        if x is None:
            assert got is None
            continue
        assert got.dtype == x.dtype and got.shape == x.shape
        want, size = _formula(x.float().cpu().numpy(), None if w is None else w.float().cpu().numpy(),
                              pos.cpu().numpy(), f.cpu().numpy(), eps, inter)
        _near(got, want, size, x.shape[2])


# ---------------------------------------------------------------------------
# refusals (CPU)
# ---------------------------------------------------------------------------
def test_c_abi_refuses_bad_arguments():
    L = _lib.load()
    p = 1 << 16  # never read: every call below is refused, or does nothing

    def call(q=p, k=p, dt=0, T=2, H=4, kv=2, D=8, qst=32, qsh=8, kst=16, ksh=8, pos=p, per=1, f=p, pairs=4, inter=0, wq=p, wk=p,
             wt=0, eps=1e-6, qo=p, ko=p, qost=32, qosh=8, kost=16, kosh=8):
        return L.sbq_qk_norm_rope(q, k, dt, T, H, kv, D, qst, qsh, kst, ksh, pos, per, f, pairs, inter, wq, wk, wt, eps, qo, ko,
                                  qost, qosh, kost, kosh, None)

    assert call(dt=3) == -2 and call(wt=-1) == -2
    for bad in (dict(T=-1), dict(T=1 << 31), dict(H=0), dict(kv=-1), dict(D=0), dict(D=257), dict(per=0), dict(pairs=5),
                dict(pairs=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(qst=-1), dict(ksh=-8), dict(qosh=7),
                dict(qost=31), dict(kost=8), dict(H=65537), dict(kv=65537)):
        assert call(**bad) == -1, bad
    for name in ("q", "k", "pos", "f", "qo", "ko"):
        assert call(**{name: None}) == -1
    for bad in (dict(q=p + 2), dict(pos=p + 4), dict(f=p + 1), dict(dt=1, k=p + 1), dict(wq=p + 2), dict(ko=p + 1)):
        assert call(**bad) == -3, bad
    assert call(T=0) == 0


def test_python_refuses():
    x = torch.zeros(2, 4, 8)
    with pytest.raises(ValueError, match="GPU"):
        qk_norm_rope(x, None, torch.zeros(2, dtype=torch.long), torch.ones(4))


@pytest.mark.gpu
def test_python_refuses_on_the_gpu(dev):
    q, k, pos, f, wq, wk = _case(dev, 4, 4, 2, 8, 4, False, F32, True)

    def bad(match, **kw):
        a = dict(q=q, k=k, positions=pos, inv_freq=f, q_weight=wq, k_weight=wk)
        a.update(kw)
        with pytest.raises(ValueError, match=match):
            qk_norm_rope(**a)

    bad("dtype", q=q.double(), k=k.double())
    bad("one dtype", k=k.half())
    bad("one dtype", k=k[:3])
    bad("one dtype", k=k.cpu())
    bad("positions", positions=pos.int())
    bad("positions", positions=pos[:3])
    bad("positions", positions=pos[:0])
    bad("positions", positions=pos.cpu())
    bad("inv_freq", inv_freq=f.double())
    bad("inv_freq", inv_freq=torch.ones(5, device=dev))
    bad("weights", q_weight=wq[:7])
    bad("weights", k_weight=wk.double())
    bad("weights", k_weight=wk.half())
    bad("q_out", q_out=torch.empty_like(q).half())
    bad("q_out", q_out=torch.empty(4, 8, 4, device=dev).transpose(1, 2))
    bad("k_out", k_out=torch.empty_like(q))
    bad("k_out needs k", k=None, k_weight=None, k_out=torch.empty_like(k))
    bad("invalid argument", q_out=torch.empty(1, 4, 8, device=dev).expand(4, 4, 8))


# ---------------------------------------------------------------------------
# against the formula
# ---------------------------------------------------------------------------
SIZES = [(1, 1, 1, 1, 0), (1, 1, 0, 2, 1), (1, 32, 8, 128, 64), (3, 5, 2, 7, 3), (64, 32, 8, 128, 64), (17, 14, 2, 80, 20),
         (5, 4, 4, 64, 32), (2, 3, 1, 256, 128), (2, 3, 1, 256, 1), (9, 2, 2, 250, 124), (33, 7, 1, 96, 24), (1, 1, 1, 256, 0),
         (513, 6, 2, 64, 16), (1100, 4, 1, 128, 64), (2049, 3, 1, 48, 24), (9000, 2, 1, 16, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,H,kv,D,pairs", SIZES)
def test_formula(dev, T, H, kv, D, pairs, inter, dtype):
    for norm in (True, False):
        case = _case(dev, T, H, kv, D, pairs, inter, dtype, norm, seed=T + D)
        announce(f"rope T={T} H={H} kv={kv} D={D} pairs={pairs} inter={inter} {dtype} norm={norm}")
        q, k, pos, f, wq, wk = case
        out = qk_norm_rope(q, k, pos, f, wq, wk, interleaved=inter)
        _check(out, q, k, pos, f, wq, wk, inter)


@pytest.mark.gpu
def test_far_and_negative_positions(dev):
    pos = torch.tensor([0, 1, -1, 131071, 1 << 20, (1 << 31) - 1, 1 << 40, -(1 << 33) - 7, (1 << 52) + 1])
    q, k, pos, f, wq, wk = _case(dev, len(pos), 3, 2, 64, 32, False, F32, False, positions=pos)
    # (2^52 times a float32 in 64-bit extended precision is off by 2^-11: only the others are compared there)
    out = qk_norm_rope(q, k, pos, f)
    _check((out[0][:8], out[1][:8]), q[:8], k[:8], pos[:8], f, None, None, False)
    assert torch.isfinite(out[0]).all() and torch.equal(out[0][0], q[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_of_one_projection_in_place_and_strides(dev, dtype):
    T, H, kv, D = 37, 6, 2, 40
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(T, (H + 2 * kv) * D, generator=g).to(dtype).to(dev)
    f, pos = torch.from_numpy(_freq(20)).to(dev), torch.arange(T, device=dev) + 100
    w = torch.rand(D, generator=g).to(dev)
    q, k = qkv[:, :H * D].unflatten(1, (H, D)), qkv[:, H * D:(H + kv) * D].unflatten(1, (kv, D))
    want = qk_norm_rope(q, k, pos, f, w, w)
    _check(want, q, k, pos, f, w, w, False)
    keep = qkv.clone()
    out = qk_norm_rope(q, k, pos, f, w, w, q_out=q, k_out=k)  # in place: the values' part stays
    assert out[0].data_ptr() == q.data_ptr()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, (H + kv) * D:], keep[:, (H + kv) * D:])
    # heads first, an offset that no vector load takes, columns that are not side by side
    x = torch.randn(H, T, D + 1, generator=g).to(dtype).to(dev)
    q2 = x.transpose(0, 1)[:, :, 1:]
    out2 = torch.zeros(T, H, D + 3, dtype=dtype, device=dev)
    got, none = qk_norm_rope(q2, None, pos, f, w, q_out=out2[:, :, 2:D + 2])
    assert none is None
    _check((got, None), q2, None, pos, f, w, None, False)
    assert float(out2[:, :, :2].abs().sum()) == 0 and float(out2[:, :, D + 2:].abs().sum()) == 0
    q3 = torch.randn(T, D, H, generator=g).to(dtype).to(dev).transpose(1, 2)
    _check(qk_norm_rope(q3, None, pos, f, w), q3, None, pos, f, w, None, False)
    # heads of one memory (a broadcast)
    q4 = torch.randn(T, 1, D, generator=g).to(dtype).to(dev).expand(T, H, D)
    _check(qk_norm_rope(q4, None, pos, f, w), q4, None, pos, f, w, None, False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("D,pairs", [(90, 45), (128, 63), (31, 9), (33, 16), (14, 7), (250, 117)])
def test_in_place_at_no_alignment(dev, D, pairs, inter, dtype):
    """Pieces that begin early over the columns of the one before, in rows that begin anywhere."""
    T, H, kv = 530, 5, 2
    announce(f"rope in place D={D} pairs={pairs} inter={inter} {dtype}")
    g = torch.Generator().manual_seed(D)
    qkv = torch.randn(T, (H + kv) * D + 3, generator=g).to(dtype).to(dev)
    f, pos = torch.from_numpy(_freq(pairs)).to(dev), torch.arange(T, device=dev) + 7
    w = (torch.rand(D + 1, generator=g) + 0.5).to(dev)[1:]
    q, k = qkv[:, 1:1 + H * D].unflatten(1, (H, D)), qkv[:, 1 + H * D:1 + (H + kv) * D].unflatten(1, (kv, D))
    ends = qkv[:, 0].clone(), qkv[:, 1 + (H + kv) * D:].clone()
    want = qk_norm_rope(q, k, pos, f, w, w, interleaved=inter)
    _check(want, q, k, pos, f, w, w, inter)
    qk_norm_rope(q, k, pos, f, w, w, interleaved=inter, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(qkv[:, 0], ends[0]) and torch.equal(qkv[:, 1 + (H + kv) * D:], ends[1])


@pytest.mark.gpu
def test_starts_of_sequences(dev):
    q, k, _, f, wq, wk = _case(dev, 12, 4, 2, 32, 16, False, F32, True)
    starts = torch.tensor([5, 0, 1000], device=dev)
    each = (starts[:, None] + torch.arange(4, device=dev)).reshape(-1)
    for a, b in zip(qk_norm_rope(q, k, starts, f, wq, wk), qk_norm_rope(q, k, each, f, wq, wk)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_weights_of_two_bytes_zero_rows_and_specials(dev):
    q, k, pos, f, wq, wk = _case(dev, 4, 3, 2, 64, 32, False, F32, True, wt=BF16)
    _check(qk_norm_rope(q, k, pos, f, wq, wk), q, k, pos, f, wq, wk, False)
    q[1, 2] = 0.0
    q[2, 0, 5] = float("nan")
    q[3, 1, 7] = float("inf")
    out, _ = qk_norm_rope(q, k, pos, f, wq, wk)
    assert float(out[1, 2].abs().sum()) == 0                     # eps keeps a row of zeros
    assert torch.isnan(out[2, 0]).all() and torch.isnan(out[3, 1, 7])  # ... and a bad one to itself
    rest = torch.ones(4, 3, dtype=torch.bool, device=dev)
    rest[2, 0] = rest[3, 1] = False
    assert torch.isfinite(out[rest]).all()
    empty, none = qk_norm_rope(q[:0], k[:0], pos[:0], f, wq, wk)
    assert empty.shape == (0, 3, 64) and none.shape == (0, 2, 64)


@pytest.mark.gpu
def test_other_stream_and_graph(dev):
    q, k, pos, f, wq, wk = _case(dev, 8, 4, 2, 128, 64, False, BF16, True)
    want = qk_norm_rope(q, k, pos, f, wq, wk)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = qk_norm_rope(q, k, pos, f, wq, wk)
        g = torch.cuda.CUDAGraph()
    side.synchronize()
    assert torch.equal(got[0], want[0])
    with torch.cuda.graph(g):
        held = qk_norm_rope(q, k, pos, f, wq, wk)
    for i in range(3):
        pos.add_(i)
        q.mul_(-1)
        g.replay()
        torch.cuda.synchronize()
        eager = qk_norm_rope(q, k, pos, f, wq, wk)
        assert torch.equal(held[0], eager[0]) and torch.equal(held[1], eager[1])


@pytest.mark.gpu
def test_tokens_further_apart_than_32_bits(dev):
    q, k, pos, f, wq, wk = _case(dev, 3, 2, 1, 64, 32, False, BF16, True)
    apart = torch.empty(2 * (5 << 28) + 512, dtype=BF16, device=dev)  # 2.5 GiB between tokens
    views = [apart[i:].as_strided((3, n, 64), (5 << 28, 64, 1)) for i, n in ((0, 2), (128, 1), (192, 2), (320, 1))]
    views[0].copy_(q)
    views[1].copy_(k)
    want = qk_norm_rope(q, k, pos, f, wq, wk)
    got = qk_norm_rope(views[0], views[1], pos, f, wq, wk, q_out=views[2], k_out=views[3])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_two_streams(dev):
    """Two calls at once."""
    cases = [_case(dev, 2000, 8, 2, 128, 64, inter, BF16, True) for inter in (False, True)]
    want = [qk_norm_rope(q, k, pos, f, wq, wk, interleaved=bool(i)) for i, (q, k, pos, f, wq, wk) in enumerate(cases)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(10):
        for i, (s, (q, k, pos, f, wq, wk)) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(qk_norm_rope(q, k, pos, f, wq, wk, interleaved=bool(i)))
    torch.cuda.synchronize()
    for w, results in zip(want, got):
        assert all(torch.equal(r[0], w[0]) and torch.equal(r[1], w[1]) for r in results)
