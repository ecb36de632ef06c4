"""Verification of drafts over rows longer than one workgroup takes (segments of
4096 tokens are summed by one launch, the token picked by a second) and shorter:
borders of tokens and segments, empty segments, rows without a token, graphs."""
import numpy as np
import pytest
import torch

from conftest import announce
from sbq import quant
from test_verify_drafts import BF16, F16, F32, _probs, _rule, _run, _same

SIZES = [5000, 16384, 16385, 20000, 151936]  # one launch up to 16384


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", SIZES + [16388, 1 << 20])
def test_borders_of_tokens_and_segments(dev, V, dtype):
    """Masses of 1/8 at the ends of segments, whole segments empty between them, every uniform a border between two tokens:
    the next token with mass is drawn."""
    announce(f"borders V={V} {dtype}")
    at = sorted({0, 4095, 4096, V - 1, V // 2, 1, 7, V - 2} | ({8191, 8192} if V > 8192 else {4097, 4098}))[:8]
    target = torch.zeros(8, 2, V)
    target[:, :, at] = 1 / 8
    u = torch.zeros(8, 2)
    u[:, 1] = torch.arange(8) / 8
    tokens = torch.full((8, 1), 3)
    got, want = _run(dev, target.to(dtype), None, tokens, u, torch.zeros(8, dtype=torch.long))
    _same(got, want)
    assert got[1].tolist() == at
    u[:, 1] = (torch.arange(8) + 1) / 8 * (1 - 2.0 ** -24)  # just below: the one before
    got, want = _run(dev, target.to(dtype), None, tokens, u, torch.zeros(8, dtype=torch.long))
    _same(got, want)
    assert got[1].tolist() == at
    # after a refusal: what is left lies in the last segment alone, or in the first
    for keep in (at[-1], at[0]):
        draft = target[:, :1].clone()
        draft[:, :, keep] = 0
        u[:, 0], u[:, 1] = 1 - 2.0 ** -24, torch.arange(8) / 8
        got, want = _run(dev, target.to(dtype), draft.to(dtype), torch.full((8, 1), 5), u)
        _same(got, want)
        assert got[0].tolist() == [0] * 8 and got[1].tolist() == [keep] * 8
    # u q == p is refused, the least below it kept
    draft = torch.zeros(4, 1, V)
    draft[:, 0, at[3]] = 0.25
    u = torch.tensor([[0.5, 0.0], [0.49999997, 0.0], [0.0, 0.9], [1 - 2.0 ** -24, 1 - 2.0 ** -24]])
    got, want = _run(dev, target[:4].to(dtype), draft.to(dtype), torch.full((4, 1), at[3]), u)
    _same(got, want)
    assert got[0].tolist() == [0, 1, 1, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("V", SIZES)
def test_nothing_left_bad_drafts_and_bad_rows(dev, V):
    announce(f"rows without a token V={V}")
    g = torch.Generator().manual_seed(3)
    target = _probs(g, 10, 3, V, 1.0, F32)
    draft = _probs(g, 10, 2, V, 1.0, F32)
    tokens = torch.randint(0, V, (10, 2), generator=g)
    u = torch.full((10, 3), 0.5)
    draft[0, 0] = 2.0                       # nothing is left of p - q: p itself
    tokens[1, 0], tokens[2, 0], tokens[3, 0] = V, -1, 1 << 62  # no tokens: refused
    target[4, 0] = 0.0                      # no mass at all
    target[5, 0, 7] = float("nan")
    target[6, 0, V - 1] = float("inf")
    target[7, 2, 3] = float("nan")          # a row that is not reached, or is
    target[8, 0, tokens[8, 0]] = float("nan")
    draft[8, 0, tokens[8, 0]] = 1e-30
    draft[9, 0] = target[9, 0]              # nothing is left, and the draft refused
    u[0, 0], u[9, 0] = 0.99, 1.0
    got, want = _run(dev, target, draft, tokens, u)
    _same(got, want)
    assert got[0][:5].tolist() == [0] * 5 and int(got[1][4]) == -1 and int(got[0][9]) == 0 and int(got[1][9]) >= 0
    for d, counts in ((draft, torch.zeros(10, dtype=torch.long)), (None, None), (draft, torch.full((10,), 1))):
        got, want = _run(dev, target, d, tokens, u, counts)
        _same(got, want)
    got, _ = _run(dev, target, draft, tokens, u, torch.zeros(10, dtype=torch.long))
    assert got[1][4:7].tolist() == [-1, -1, -1] and int(got[1][8]) == -1
    u[:, 2] = float("nan")                  # no uniform: no token
    got = quant.verify_drafts(target.to(dev), None, tokens.to(dev), u.to(dev))
    assert got[1].tolist() == [-1] * 10


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("V", [16385, 20000, 20001, 151936])
def test_graph_with_a_workspace(dev, V, dtype):
    """Captured with an allocated workspace and with the caller's, replayed between eager calls."""
    B, T = 5, 3
    announce(f"graph V={V} {dtype}")
    g = torch.Generator().manual_seed(V)
    target, draft = _probs(g, B, T + 1, V, 2.0, dtype).to(dev), _probs(g, B, T, V, 2.0, dtype).to(dev)
    tokens = torch.randint(0, V, (B, T), generator=g).to(dev)
    u = torch.rand(B, T + 1, generator=g).to(dev)
    counts = torch.full((B,), T, device=dev)
    ws = quant.verify_workspace(B, V, dev)
    quant.verify_drafts(target, draft, tokens, u, counts)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [quant.verify_drafts(target, draft, tokens, u, counts), quant.verify_drafts(target, draft, tokens, u, counts, ws)]
    for i in range(5):
        u.copy_(torch.rand(B, T + 1, generator=g))
        tokens.copy_(torch.multinomial(draft.float().reshape(-1, V).cpu(), 1, generator=g).reshape(B, T))
        counts.copy_(torch.randint(0, T + 1, (B,), generator=g))
        ws.fill_(255)
        eager = [t.cpu().numpy() for t in quant.verify_drafts(target, draft, tokens, u, counts)]
        graph.replay()
        torch.cuda.synchronize()
        want = _rule(target.float().cpu().numpy(), draft.float().cpu().numpy(), tokens.cpu().numpy(), u.cpu().numpy(),
                     counts.cpu().numpy())
        for got in (eager, *[[t.cpu().numpy() for t in h] for h in held]):
            assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
