"""The attention over an 8-bit paged cache (DevicePagedKVBuffer.attend) where the
values' scales differ: inputs whose scores are exact, so that the bound is that
of the weights times the values alone.

With u = 2^-24 and scores that the kernel has exactly (0, or below all weight):
a weight times its value's scale is off by two roundings and by 2^-22 of itself
(two fp16 pieces), the sum of n products by (n + 16) u of its size, the sum of
weights and the division by (n + 8) u; the output by half a step of its type."""
import pytest
import torch

from conftest import announce
from sbq.state import DevicePagedKVBuffer

F32, F16, BF16, I8, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn
U = 2.0 ** -24


def _codes(shape, dtype, g):
    """Random codes: whole numbers, exact in either type."""
    return torch.randint(-120 if dtype == I8 else -15, 121 if dtype == I8 else 16, shape, generator=g)


def _cache(dev, dtype, k_codes, v_codes, v_scale, page=16, window=None):
    """A buffer that holds codes [B, n, heads, dim] and the values' scales [B, n, heads]; the keys' are 1."""
    B, n, heads, dim = v_codes.shape
    width = -(-n // page)
    b = DevicePagedKVBuffer(B, heads, dim, B * width, page, width, window, dev, dtype)
    g = torch.Generator().manual_seed(n)
    b.table.copy_(torch.randperm(B * width, generator=g).view(B, width))
    b.length.fill_(n)
    pos = torch.arange(n)
    at = b.table.cpu().long()[:, pos // page]  # [B, n]
    for pool, scale, codes, scales in ((b.k, b.k_scale, k_codes, torch.ones(B, n, heads)), (b.v, b.v_scale, v_codes, v_scale)):
        host, s = torch.zeros(pool.shape), torch.zeros(scale.shape)
        host[at, :, pos % page] = codes.float()
        s[at, :, pos % page] = scales.float()
        pool.copy_(host.to(dtype))
        scale.copy_(s)
    return b


def _step(t, out):
    """Half a step of type t at `out`, and of its smallest numbers."""
    return out.abs() * (torch.finfo(t).eps / 2) * 1.001 + (2.0 ** -25 if t == F16 else 1e-38)


@pytest.mark.gpu
@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_weights_keep_more_bits_than_the_output(dev, dtype, qt):
    """Equal scores and different scales of values: no rounding of the weights shows in the output."""
    g = torch.Generator().manual_seed(1)
    for n in (2, 40):
        announce(f"{n} values of equal weight, {dtype} {qt}")
        B, heads, dim = 16, 2, 64
        v = _codes((B, n, heads, dim), dtype, g)
        if n == 2:
            v[:, 1] = 0  # the larger scale has no values
        scale = torch.rand(B, n, heads, generator=g) / 2 + 0.5
        scale[:, 1] = 1.0
        b = _cache(dev, dtype, torch.zeros(B, n, heads, dim), v, scale)
        q = torch.randn(B, 1, 4, dim, generator=g).to(qt).to(dev)
        got = b.attend(q)[:, 0].double().cpu()
        x = v.double() * scale.double()[..., None]
        want, size = [t.mean(1).repeat_interleave(2, 1) for t in (x, x.abs())]
        tol = size * (2.0 ** -22 + (2 * n + 28) * U)
        tol += _step(qt, want.abs() + tol)
        assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


@pytest.mark.gpu
@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("dtype", [I8, E4M3])
@pytest.mark.parametrize("n,heavy", [(2, 0), (2, 1), (30, 7), (200, 0), (200, 133), (200, 199), (3000, 17), (3000, 2900)])
def test_scales_of_values_without_weight(dev, n, heavy, dtype, qt):
    """One position takes the weight, the others have values up to 2^90 times as
    large and weights 2^-60: each sequence its own ratio, from one where the others
    are nothing to one where they are all.  The scores are 0 and -42 (a whole number
    in every type; its weight is off by 2^-18 of itself: 61 powers of two in fp32
    steps of 2^-19, and exp2).  A weight times a scale far below the row's largest is
    off by 2^-39 of that instead of 2^-22 of itself."""
    announce(f"{n} values, the weight at {heavy}, {dtype} {qt}")
    ratios = [0, 3, 14, 20, 24, 27, 30, 34, 38, 45, 55, 58, 60, 62, 66, 80, 90]
    B, heads, dim = len(ratios), 2, 64
    g = torch.Generator().manual_seed(n + heavy)
    v = _codes((B, n, heads, dim), dtype, g)
    k = torch.zeros(B, n, heads, dim)
    k[..., 5] = -1
    k[:, heavy, :, 5] = 0
    q = torch.zeros(B, 1, 4, dim)
    q[..., 5] = 42
    light = torch.exp2(torch.tensor(ratios).double())[:, None, None]
    is_heavy = (torch.arange(n) == heavy)[None, :, None]
    for unit in (1.0, 2.0 ** -100, 2.0 ** 28):
        scale = (torch.where(is_heavy, 1.0, light) * unit).expand(B, n, heads) * (1 + torch.randint(0, 128, (B, n, heads), generator=g) / 128)
        b = _cache(dev, dtype, k, v, scale)
        got = b.attend(q.to(qt).to(dev), scale=1.0)[:, 0].double().cpu()
        p = torch.where(is_heavy, 1.0, torch.tensor(-42.0).double().exp())[..., None].expand(B, n, heads, 1)
        x, total = v.double() * scale[..., None], p.sum(1)
        want, size, small = [((p * t).sum(1) / total).repeat_interleave(2, 1)
                             for t in (x, x.abs(), torch.where(is_heavy[..., None], 0.0, x.abs()))]
        top = (p * scale[..., None]).amax(1, keepdim=True) * v.abs().double()  # the unit times each code
        tol = size * (2.0 ** -22 + (2 * n + 28) * U) + small * 2.0 ** -18 + top.sum(1).repeat_interleave(2, 1) * 2.0 ** -39
        tol += _step(qt, want.abs() + tol)
        if qt == F16:  # (an output past its largest number)
            over = (want.abs() + tol) > 65504
            want, got, tol = [torch.where(over, 0.0, t) for t in (want, got, tol)]
        assert torch.isfinite(got).all()
        assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).amax((1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("qt", [F32, BF16])
@pytest.mark.parametrize("dtype", [I8, E4M3])
def test_largest_and_smallest_values(dev, dtype, qt):
    """Values up to 2^126 (their sums still below fp32's largest), down to 2^-120, of equal weight."""
    B, n, heads, dim = 2, 3, 1, 64
    g = torch.Generator().manual_seed(3)
    for e in (118, 100, -100, -113):
        announce(f"values of 2^{e} {dtype} {qt}")
        v = _codes((B, n, heads, dim), dtype, g).clamp(-80, 80)
        scale = torch.full((B, n, heads), 2.0 ** e) * (1 + torch.rand(B, n, heads, generator=g) / 8)
        b = _cache(dev, dtype, torch.zeros(B, n, heads, dim), v, scale)
        got = b.attend(torch.zeros(B, 1, 2, dim, dtype=qt, device=dev))[:, 0].double().cpu()
        x = v.double() * scale.double()[..., None]
        want, size = [t.mean(1).expand(B, 2, dim) for t in (x, x.abs())]
        tol = size * (2.0 ** -22 + (2 * n + 28) * U) + 2.0 ** -140
        tol += _step(qt, want.abs() + tol)
        assert torch.isfinite(got).all()
        assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,qt", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F16), (F16, F32), (I8, F32), (E4M3, BF16)])
@pytest.mark.parametrize("n", [1, 37, 500, 3000])
def test_means_of_large_and_small_values(dev, n, dtype, qt):
    """Values up to just below 2^127 (fp16: 65504) in every position, which add up to far more than fp32 holds, and of
    2^-100 (2^-10): equal weights, so the mean.  Tolerance as above; one product below fp32's smallest steps each."""
    B, heads, dim = 2, 2, 64
    g = torch.Generator().manual_seed(n)
    for e in ((15, -10) if dtype == F16 else (119, 0, -100) if dtype in (I8, E4M3) else (126, 0, -100)):
        announce(f"{n} values of 2^{e} {dtype} {qt}")
        if dtype in (I8, E4M3):
            codes = _codes((B, n, heads, dim), dtype, g).abs()
            b = _cache(dev, dtype, torch.zeros(B, n, heads, dim), codes, torch.full((B, n, heads), 2.0 ** e))
            x = codes.double() * 2.0 ** e
        else:
            x = ((torch.rand(B, n, heads, dim, generator=g) + 0.99) * 2.0 ** e).to(dtype)
            b = DevicePagedKVBuffer(B, heads, dim, 2 * (n // 16 + 1), 16, n // 16 + 1, device=dev, dtype=dtype)
            for i in range(B):
                b.reserve(i, n)
            b.append(torch.zeros_like(x).to(dev), x.to(dev))
            x = x.double()
        assert e != 126 or n < 3 or float(x.sum(1).max()) > 2.0 ** 128
        got = b.attend(torch.zeros(B, 1, 4, dim, dtype=qt, device=dev))[:, 0].double().cpu()
        want = x.mean(1).repeat_interleave(2, 1)
        tol = want.abs() * (2.0 ** -22 + (2 * n + 28) * U) + 2.0 ** -149
        tol += _step(qt, want.abs() + tol)
        assert torch.isfinite(got).all()
        assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,qt", [(F32, F32), (BF16, BF16), (F16, F16), (F16, F32), (I8, F32), (E4M3, BF16)])
def test_what_is_no_number_shows_at_any_weight(dev, dtype, qt):
    """An infinity or NaN among the values that a row sees is in its result, also where its weight is far below fp32's
    smallest (scores 0 and -420), in whichever wave or part of the sequence it lies; no other column changes."""
    n, heads, dim = 3000, 1, 64
    g = torch.Generator().manual_seed(4)
    b = DevicePagedKVBuffer(1, heads, dim, 200, 16, 200, device=dev, dtype=dtype)
    b.reserve(0, n)
    k = torch.zeros(1, n, heads, dim)
    k[..., 5] = -10
    k[:, 1700, :, 5] = 0
    b.append(k.to(dev), torch.randn(1, n, heads, dim, generator=g).to(dev))
    q = torch.zeros(1, 1, 2, dim, dtype=qt, device=dev)
    q[..., 5] = 42
    want = b.attend(q, scale=1.0)
    assert torch.isfinite(want).all()
    for at in (0, 33, 700, 1699, 1701, 1801, 2999):
        for what in (float("inf"), float("nan")):
            announce(f"{what} at {at} {dtype} {qt}")
            page, row = int(b.table[0, at // 16]), at % 16
            cell = b.v[page, 0, row, 9:10] if b.v_scale is None else b.v_scale[page, 0, row:row + 1]
            keep = cell.clone()
            cell.fill_(what)
            got = b.attend(q, scale=1.0)
            cell.copy_(keep)
            if b.v_scale is None:
                assert not torch.isfinite(got[..., 9]).any()
                assert torch.equal(got[..., :9], want[..., :9]) and torch.equal(got[..., 10:], want[..., 10:])
            else:
                assert not torch.isfinite(got).any()
