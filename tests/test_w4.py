"""Linears with 4-bit weights and group scales (sbq.quant.linear_w4,
Int4Linear, quantize_groups) against the formula in 64 bits.

Tolerance of an output (a bound, not a fit): every fp32 rounding on the way
of a product into its sum is at most 2^-24 of the sum of magnitudes
S = sum |s q x|; a product passes at most 32 additions inside its matrix
instruction, one per group, one per wave (8) and the bias.  fp32 activations
are carried to 22 bits (2^-22 of each value) or 2^-39 of the largest in
their 128 columns.  The output's own rounding is half a step of its type.
"""
import ctypes

import numpy as np
import pytest
import torch

from conftest import announce
from sbq import _lib, quant

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


# ---------------------------------------------------------------------------
# refusals (CPU)
# ---------------------------------------------------------------------------
def test_c_abi_refuses_bad_arguments():
    L = _lib.load()
    p = ctypes.c_void_p(4096)  # never read: every call below is refused
    odd = ctypes.c_void_p(4104)

    def lin(x=p, xt=0, M=1, K=64, ldx=64, w=p, s=p, N=16, group=128, y=p, yt=0, ldy=16):
        return L.sbq_linear_w4(x, xt, M, K, ldx, w, s, None, N, group, y, yt, ldy, None)

    assert lin(xt=7) == -2 and lin(yt=3) == -2
    assert lin(N=0) == -1 and lin(K=0) == -1 and lin(ldx=63) == -1 and lin(ldy=15) == -1 and lin(M=-1) == -1
    assert lin(group=48) == -1 and lin(group=0) == -1 and lin(group=256) == -1
    assert lin(x=None) == -1 and lin(w=None) == -1 and lin(s=None) == -1 and lin(y=None) == -1
    assert lin(w=odd) == -3 and lin(s=odd) == -3
    assert lin(M=0) == 0
    assert lin(M=1 << 31) == -1 and lin(N=1 << 31, ldy=1 << 31) == -1
    assert L.sbq_quantize_groups(p, 9, 4, 64, 64, 32, p, 64, p, None) == -2
    assert L.sbq_quantize_groups(p, 0, 4, 64, 63, 32, p, 64, p, None) == -1
    assert L.sbq_quantize_groups(p, 0, 4, 64, 64, 16, p, 64, p, None) == -1
    assert L.sbq_quantize_groups(p, 0, 4, 64, 64, 32, None, 64, p, None) == -1
    assert L.sbq_quantize_groups(None, 0, 0, 64, 64, 32, None, 64, None, None) == 0
    assert L.sbq_repack_w4(p, 4, 64, 32, p, 32, p, p, None) == -1
    assert L.sbq_repack_w4(p, 4, 64, 64, p, 32, odd, p, None) == -3
    assert L.sbq_unpack_w4(p, p, 4, 64, 96, p, 64, p, None) == -1
    assert L.sbq_w4_packed_bytes(4096, 4096) == 4096 * 4096 // 2
    assert L.sbq_w4_packed_bytes(17, 129) == 2 * 2 * 1024
    assert L.sbq_w4_scale_count(17, 129, 64) == 32 * 4
    assert L.sbq_w4_packed_bytes(0, 5) == 0 and L.sbq_w4_scale_count(16, 128, 100) == 0


def test_python_refuses_bad_arguments():
    with pytest.raises(ValueError, match="GPU"):
        quant.quantize_groups(torch.zeros(4, 64))
    with pytest.raises(ValueError, match="GPU"):
        quant.repack_w4(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 1, dtype=BF16))
    with pytest.raises(ValueError, match="GPU"):
        quant.linear_w4(torch.zeros(1, 64), torch.zeros(1024, dtype=torch.uint8), torch.zeros(16, dtype=BF16), None, 16)
    with pytest.raises(ValueError):
        quant.Int4Linear(torch.zeros(4, 4, 4))
    with pytest.raises(ValueError, match="group"):
        quant.Int4Linear(torch.zeros(4, 64), group=100)
    with pytest.raises(ValueError, match="int8"):
        quant.Int4Linear.from_quantized(torch.zeros(4, 64), torch.zeros(4, 1))


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------
def _weight(N, K, group, seed):
    """4-bit rows with every value -8..7 and bf16 scales over four decades."""
    r = np.random.default_rng(seed)
    q = torch.from_numpy(r.integers(-8, 8, (N, K)).astype(np.int8))
    s = torch.from_numpy(np.exp(r.uniform(-8, 1, (N, -(-K // group)))).astype(np.float32)).to(BF16)
    return q, s


def _x(M, K, dtype, seed):
    r = np.random.default_rng(seed)
    x = r.standard_normal((M, K)) * np.exp(r.uniform(-3, 3, (M, 1)))
    return torch.from_numpy(x.astype(np.float32)).to(dtype)


def _check(y, x, q, s, bias, group, y_dtype):
    """y against the formula; every argument on the CPU."""
    K = q.shape[1]
    w = q.double() * s.double().repeat_interleave(group, 1)[:, :K]
    x = x.double()
    want = x @ w.t()
    mag = x.abs() @ w.abs().t()
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    steps = 32 + -(-K // 32) + 8 + 1
    xmax = torch.nn.functional.pad(x.abs(), (0, -K % 128)).view(x.shape[0], -1, 128).amax(-1)
    wsum = torch.nn.functional.pad(w.abs(), (0, -K % 128)).view(w.shape[0], -1, 128).sum(-1)
    tol = mag * (steps * 2.0 ** -24 + 2.0 ** -22) + (xmax @ wsum.t()) * 2.0 ** -39
    tol = tol + (want.abs() + tol) * torch.finfo(y_dtype).eps / 2 + torch.finfo(y_dtype).tiny
    assert y.dtype == y_dtype and y.shape == want.shape
    off = (y.double() - want).abs()
    assert bool((off <= tol).all()), f"worst {float((off / tol).max()):.3g} of the bound"


SHAPES = [(1, 1), (16, 128), (13, 200), (33, 31), (130, 2500), (512, 4096)]


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,K", SHAPES)
def test_linear_w4(dev, N, K, dtype, group):
    q, s = _weight(N, K, group, N * 7 + K)
    packed, gscale = quant.repack_w4(q.to(dev), s.to(dev), group)
    for M in (1, 2, 4, 5, 8, 9, 16, 17, 32, 33, 64, 65, 130):
        y_dtype = (F32, dtype, F16, BF16)[M % 4] if dtype == F32 else (F32, dtype)[M % 2]
        if y_dtype == F16 and dtype != F16:  # outputs beyond fp16's range are infinities
            y_dtype = F32
        x = _x(M, K, dtype, M)
        bias = torch.randn(N, generator=torch.Generator().manual_seed(M)) if M % 3 == 0 else None
        announce(f"linear_w4 M={M} N={N} K={K} group={group} {dtype}->{y_dtype}")
        xd = x.to(dev) * (2.0 ** -6 if y_dtype == F16 else 1.0)
        y = quant.linear_w4(xd, packed, gscale, None if bias is None else bias.to(dev), N, group, y_dtype)
        _check(y.cpu(), xd.cpu(), q, s, bias, group, y_dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,K", [(4100, 264), (8208, 2184), (32770, 136)])
def test_linear_w4_wide(dev, N, K, dtype, group):
    """Layers wide enough for workgroups of two and three weight tiles, all K
    ends inside a tile; what lies beyond K in x's rows does not count."""
    q, s = _weight(N, K, group, N)
    packed, gscale = quant.repack_w4(q.to(dev), s.to(dev), group)
    for M in (1, 2, 3, 8, 9, 20, 40, 64, 70) if N < 32770 else (1, 2, 4, 24):
        x = _x(M, K, dtype, M)
        wide = torch.full((M, K + 24), float("nan"), dtype=dtype)
        wide[:, :K] = x
        announce(f"linear_w4 wide M={M} N={N} K={K} group={group} {dtype}")
        y = quant.linear_w4(wide.to(dev)[:, :K], packed, gscale, None, N, group)
        _check(y.cpu(), x, q, s, None, group, F32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_linear_w4_strides_and_alignment(dev, dtype):
    N, K, group = 70, 300, 64
    q, s = _weight(N, K, group, 5)
    packed, gscale = quant.repack_w4(q.to(dev), s.to(dev), group)
    for M in (1, 3, 7, 20, 50):
        x = _x(M, K + 9, dtype, M)
        xd = x.to(dev)[:, 3:3 + K]          # rows that start off 16 bytes
        out = torch.full((M + 1, N + 5), 7.0, device=dev)
        announce(f"linear_w4 strided M={M} {dtype}")
        y = quant.linear_w4(xd, packed, gscale, None, N, group, out=out[:M, 1:1 + N])
        _check(y.cpu(), x[:, 3:3 + K], q, s, None, group, F32)
        assert bool((out[:, 0] == 7).all()) and bool((out[:, 1 + N:] == 7).all()) and bool((out[M] == 7).all())
        xt = x[:, :K].t().contiguous().to(dev).t()  # column-major
        _check(quant.linear_w4(xt, packed, gscale, None, N, group).cpu(), x[:, :K], q, s, None, group, F32)
    one = _x(1, K, dtype, 9).to(dev).expand(4, K)  # broadcast rows
    y = quant.linear_w4(one, packed, gscale, None, N, group)
    assert bool((y == y[0]).all())


@pytest.mark.gpu
def test_linear_w4_wide_range_and_non_finite(dev):
    """fp32 values far apart in one tile, subnormals, zeros; an infinity or NaN
    stays in its row, of the sign that the formula has."""
    N, K, group = 48, 256, 32
    q, s = _weight(N, K, group, 11)
    q[:, 5] = torch.where(q[:, 5] == 0, 1, q[:, 5])
    packed, gscale = quant.repack_w4(q.to(dev), s.to(dev), group)
    for M in (4, 12, 40):
        x = _x(M, K, F32, M)
        x[0] = 0.0
        x[1] *= torch.from_numpy(10.0 ** np.random.default_rng(3).uniform(-12, 12, K)).float()
        x[2] *= 1e-30
        x[3] *= 1e30
        announce(f"linear_w4 wide range M={M}")
        _check(quant.linear_w4(x.to(dev), packed, gscale, None, N, group).cpu(), x, q, s, None, group, F32)
        clean = quant.linear_w4(x.to(dev), packed, gscale, None, N, group).cpu()
        x[2, 5], x[3, 9] = float("inf"), float("nan")
        y = quant.linear_w4(x.to(dev), packed, gscale, None, N, group).cpu()
        assert torch.equal(y[:2], clean[:2]) and torch.equal(y[4:], clean[4:])
        assert torch.equal(y[2], torch.sign(q[:, 5].float()) * float("inf"))
        assert bool(torch.isnan(y[3]).all())


def _quantize(w, group):
    """The documented quantization, in numpy (fp32 divisions)."""
    N, K = w.shape
    G = -(-K // group)
    p = np.zeros((N, G * group), np.float32)
    p[:, :K] = w
    p = p.reshape(N, G, group)
    s = torch.from_numpy(np.maximum(np.abs(p).max(2), np.float32(1e-8)) / np.float32(7)).to(BF16)
    q = np.clip(np.rint(p / s.float().numpy()[:, :, None]), -7, 7).astype(np.int8)
    return torch.from_numpy(q.reshape(N, G * group)[:, :K].copy()), s


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
def test_quantize_pack_round_trip(dev, dtype, group):
    for N, K in ((1, 1), (17, 130), (40, 1000), (16, 128)):
        w = (torch.randn(N, K + 3, generator=torch.Generator().manual_seed(N)) * 0.02).to(dtype)
        w[0, 1:1 + min(K, group)] = 0  # a group of zeros
        w = w[:, 1:1 + K]
        announce(f"quantize_groups {N}x{K} group={group} {dtype}")
        q, s = quant.quantize_groups(w.to(dev), group)
        q0, s0 = _quantize(w.float().numpy(), group)
        assert torch.equal(q.cpu(), q0) and torch.equal(s.cpu(), s0)
        q1, s1 = quant.unpack_w4(*quant.repack_w4(q, s, group), N, K, group)
        assert torch.equal(q1, q) and torch.equal(s1, s)


@pytest.mark.gpu
def test_int4_linear_module(dev, tmp_path):
    g = torch.Generator().manual_seed(1)
    w, b = torch.randn(100, 300, generator=g) * 0.02, torch.randn(100, generator=g)
    lin = quant.Int4Linear(w.to(BF16), b, group=64)  # a CPU weight goes to the GPU
    q, s = _quantize(w.to(BF16).float().numpy(), 64)
    assert torch.equal(lin.qweight.cpu(), q) and torch.equal(lin.scale.cpu(), s)
    x = torch.randn(2, 3, 300, generator=g)
    y = lin(x)
    assert y.device.type == "cpu" and y.shape == (2, 3, 100)
    _check(y.reshape(6, 100), x.reshape(6, 300), q, s, b, 64, F32)
    y0 = lin(x.to(dev))
    assert torch.equal(y0.cpu(), y)
    # state_dict, dtype moves, from_quantized, make_linear
    torch.save(lin.state_dict(), tmp_path / "l.pt")
    other = quant.Int4Linear(torch.zeros(100, 300), torch.zeros(100), group=64)
    other.load_state_dict(torch.load(tmp_path / "l.pt", weights_only=True))
    assert torch.equal(other.half()(x.to(dev)), y0)
    assert torch.equal(quant.Int4Linear.from_quantized(q, s, b, 64)(x.to(dev)), y0)
    assert quant.make_linear("int4", w).group == 128 and "int4" not in quant.FORMATS
    assert torch.equal(quant.grouped_forward([(lin, x.to(dev)), (lin, x.to(dev))])[1], y0)
    with pytest.raises(RuntimeError, match="in_features"):
        lin(x[..., :299])
    with pytest.raises(ValueError, match="-8..7"):
        quant.Int4Linear.from_quantized(q + 2, s, b, 64)
    with pytest.raises(ValueError, match="scale"):
        quant.Int4Linear.from_quantized(q, s, b, 32)
    with pytest.raises(ValueError):
        quant.fuse_linears([lin, lin])
    with pytest.raises(ValueError, match="int8"):
        quant.save_quantized({"a": lin}, str(tmp_path / "q"))


@pytest.mark.gpu
def test_linear_w4_refuses_short_buffers(dev):
    q, s = _weight(32, 256, 64, 1)
    packed, gscale = quant.repack_w4(q.to(dev), s.to(dev), 64)
    x = torch.zeros(2, 256, device=dev)
    for bad in (dict(packed=packed[:-1]), dict(gscale=gscale[:-1]), dict(gscale=gscale.half()), dict(group=32),
                dict(N=33), dict(bias=torch.zeros(31, device=dev)), dict(bias=torch.zeros(32)),
                dict(out=torch.zeros(2, 31, device=dev)), dict(out=torch.zeros(1, 32, device=dev).expand(2, 32)),
                dict(out_dtype=torch.float64), dict(x2=x.cpu())):
        a = dict(x2=x, packed=packed, gscale=gscale, bias=None, N=32, group=64)
        a.update(bad)
        with pytest.raises(ValueError):
            quant.linear_w4(**a)
    assert quant.linear_w4(x[:0], packed, gscale, None, 32, 64).shape == (0, 32)


@pytest.mark.gpu
def test_linear_w4_streams_and_graph(dev):
    """On another stream, and captured and replayed with new inputs."""
    q, s = _weight(256, 512, 128, 2)
    lin = quant.Int4Linear.from_quantized(q, s)
    x = torch.zeros(3, 512, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lin(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = lin(x)
    for seed in range(3):
        x.copy_(_x(3, 512, F32, seed).to(dev))
        graph.replay()
        assert torch.equal(y, lin(x))
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 2, 4, 8, 12, 24, 40, 70])
def test_linear_w4_largest_values(dev, M, group):
    """fp32 rows that hold the largest finite values, alone and beside ordinary
    ones (each other group of 128 columns), aligned and not."""
    N, K = 48, 640
    q, s = _weight(N, K, group, M)
    s = (s.float() * 2.0 ** -20).to(BF16)  # (640 columns of 8 * 2.8 * 2^-20 times the largest value stay finite)
    packed, gscale = quant.repack_w4(q.to(dev), s.to(dev), group)
    top = torch.finfo(F32).max
    for big in (top, -top, 65520 * 2.0 ** 112, 65519 * 2.0 ** 112):
        x = _x(M, K, F32, M)
        x[:, ::97] = big
        x[:, 128:256] = x[:, 128:256].clamp(-1e3, 1e3)
        if M > 1:
            x[M - 1] = big
        wide = torch.zeros(M, K + 1)
        wide[:, 1:] = x
        for xd in (x.to(dev), wide.to(dev)[:, 1:]):
            announce(f"linear_w4 largest values M={M} group={group} {big:.7g} stride {xd.stride(0)}")
            _check(quant.linear_w4(xd, packed, gscale, None, N, group).cpu(), x, q, s, None, group, F32)
