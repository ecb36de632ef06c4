"""Weights and caches that take several launches (more than 2^28 threads): the
4-bit weights' quantizing, packing and product, the slots' attention weights, the
bounded cache's rows; on both sides of the seams."""
import pytest
import torch

from conftest import announce
from sbq import quant
from sbq.state import DeviceBudgetKVBuffer, tree_attention

F32, BF16 = torch.float32, torch.bfloat16
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group,seam", [(32, 65536), (128, 262144)])
def test_quantize_groups_in_parts(dev, group, seam):
    K, N = 4096, seam + 35
    w = torch.randn(N, K, generator=torch.Generator(device=dev).manual_seed(1), device=dev, dtype=BF16)
    announce(f"quantize_groups {N}x{K} group={group}")
    q, s = quant.quantize_groups(w, group)
    for a, b in ((0, seam // 2 + 3), (seam // 2 + 3, seam + 17), (seam + 17, N)):
        qa, sa = quant.quantize_groups(w[a:b], group)
        assert torch.equal(q[a:b], qa) and torch.equal(s[a:b], sa)
    g = w[-40:].float().view(40, -1, group)
    want = (g.abs().amax(-1).clamp_min(1e-8) / 7).to(BF16)
    assert torch.equal(s[-40:], want)


def test_pack_and_unpack_in_parts(dev):
    seam, K, group = 1 << 19, 4000, 64
    N = seam + 21
    gen = torch.Generator(device=dev).manual_seed(2)
    q = torch.randint(-8, 8, (N, K), generator=gen, device=dev, dtype=torch.int8)
    s = torch.rand(N, -(-K // group), generator=gen, device=dev).to(BF16)
    announce(f"repack_w4 {N}x{K}")
    packed, gscale = quant.repack_w4(q, s, group)
    tail = quant.repack_w4(q[seam - 32:], s[seam - 32:], group)
    assert torch.equal(packed[-tail[0].numel():], tail[0]) and torch.equal(gscale[-tail[1].numel():], tail[1])
    q1, s1 = quant.unpack_w4(packed, gscale, N, K, group)
    assert torch.equal(q1, q) and torch.equal(s1, s)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_linear_w4_in_parts(dev, dtype):
    seam, K, group = 1 << 23, 40, 32
    N = seam + 21
    gen = torch.Generator(device=dev).manual_seed(3)
    q = torch.randint(-8, 8, (N, K), generator=gen, device=dev, dtype=torch.int8)
    s = (torch.rand(N, 2, generator=gen, device=dev) + 0.1).to(BF16)
    bias = torch.randn(N, generator=gen, device=dev)
    packed, gscale = quant.repack_w4(q, s, group)
    for M in (1, 6, 20):
        x = torch.randn(M, K, generator=gen, device=dev).to(dtype)
        announce(f"linear_w4 M={M} N={N} K={K} {dtype}")
        y = quant.linear_w4(x, packed, gscale, bias, N, group, dtype)
        for a in (0, seam - 64, seam, N - 64):
            rows = slice(a, a + 64)
            w = q[rows].double() * s[rows].double().repeat_interleave(group, 1)[:, :K]
            want = x.double() @ w.t().contiguous() + bias[rows].double()
            mag = x.double().abs() @ w.abs().t().contiguous() + bias[rows].double().abs()
            # 50 fp32 roundings of a sum and its products, 22 bits of x, the output's own rounding
            tol = mag * (50 * 2.0 ** -24 + 2.0 ** -22) + (want.abs() + mag * 2.0 ** -18) * torch.finfo(dtype).eps / 2
            assert bool(((y[:, rows].double() - want).abs() <= tol).all())
        # the first columns alone, one launch: the same kernel on the same rows
        head = quant.linear_w4(x, packed[: (1 << 15) * 1024], gscale, bias, 1 << 19, group, dtype)
        assert torch.equal(head, y[:, : 1 << 19])


@pytest.mark.parametrize("ct,D,seam", [(F32, 4, 1 << 23), (BF16, 8, 1 << 24)], ids=["f32", "bf16"])
def test_attention_weights_in_parts(dev, ct, D, seam):
    """9 rows, whose slots' weights are computed from the scores once more."""
    T, heads, slots = 3, 3, seam + 50
    gen = torch.Generator(device=dev).manual_seed(4)
    k, v = (torch.randn(slots, 1, D, generator=gen, device=dev).to(ct) for _ in range(2))
    q = torch.randn(T, heads, D, generator=gen, device=dev).to(ct)
    pos = torch.arange(slots, device=dev)
    pos[::11] = -1
    q_pos = torch.tensor([slots, seam + 20, 1000], device=dev)
    weight = torch.full((slots,), 0.25, device=dev)
    announce(f"attend, weights of {slots} slots {ct}")
    tree_attention(q, k, v, pos, q_pos, weight=weight, scale=0.5)
    z = (q.double().view(-1, D) @ k[:, 0].double().t().contiguous()).view(T, heads, slots) * 0.5
    see = (pos >= 0) & (pos <= q_pos[:, None])
    p = torch.softmax(z.masked_fill(~see[:, None], float("-inf")), -1)
    want = p.sum((0, 1))
    # a score's (D + 2) roundings; the sum of weights, over 1 / 512 of the slots at most one after another and
    # then 64 joins; the sum of 9 weights and its addition to 0.25
    xmax = float((q.double().abs().view(-1, D) @ k[:, 0].double().abs().t().contiguous()).max()) * 0.5
    e = 2.0 ** -24 * ((D + 2) * xmax + slots / 512 + 64)
    off = (weight.double() - 0.25 - want).abs()
    assert bool((off <= 2 * e * want + 2.0 ** -24 * (want + 0.25) * 8).all())
    assert bool((weight[pos < 0] == 0.25).all())


def test_bounded_cache_rows_in_parts(dev):
    seam, D = 1 << 20, 4
    n, T, cap = seam + 3000, seam + 10, seam + 100
    gen = torch.Generator(device=dev).manual_seed(5)
    src, dst = DeviceBudgetKVBuffer(1, D, n, 0, dev), DeviceBudgetKVBuffer(1, D, cap, 7, dev)
    k, v = (torch.randn(n, 1, D, generator=gen, device=dev) for _ in range(2))
    announce(f"append {n} tokens")
    src.append(k, v)
    assert torch.equal(src.k, k) and torch.equal(src.v, v)
    src.weight.copy_((torch.rand(n, generator=gen, device=dev) * 1000).round())
    weight = src.weight.clone()
    announce(f"take {cap} of {n} slots")
    dst.take(src)
    key = weight.clone()
    key[-7:] = float("inf")
    kept = torch.sort(torch.sort(key, stable=True).indices[n - cap:]).values
    assert torch.equal(dst.slot_pos, kept) and torch.equal(dst.weight, weight[kept])
    assert torch.equal(dst.k, k[kept]) and torch.equal(dst.v, v[kept])
    at = torch.sort(torch.sort(weight, stable=True).indices[:T]).values
    k1, v1 = (torch.randn(T, 1, D, generator=gen, device=dev) for _ in range(2))
    announce(f"append {T} tokens into {n} slots")
    src.append(k1, v1)
    k[at], v[at] = k1, v1
    assert torch.equal(src.k, k) and torch.equal(src.v, v) and int(src.end) == n + T
    assert torch.equal(src.slot_pos[at], n + torch.arange(T, device=dev))
