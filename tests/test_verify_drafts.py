"""Drafted tokens against the target's probabilities (sbq.quant.verify_drafts,
sbq_verify_drafts): whole numbers, equal to the rule in 64 bits."""
import numpy as np
import pytest
import torch

from conftest import announce
from sbq import _lib, quant

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _rule(target, draft, tokens, u, counts):
    """The documented rule, one sequence and one draft at a time, in 64 bits."""
    B, T1, V = target.shape
    kept, token = [], []
    for b in range(B):
        n = T1 - 1 if counts is None else int(np.clip(counts[b], 0, T1 - 1))
        mass, t = None, 0
        while t < n:
            x = int(tokens[b, t])
            q = np.zeros(V)
            if draft is not None:
                q = draft[b, t].astype(np.float64)
            elif 0 <= x < V:
                q[x] = 1.0
            if not (0 <= x < V and np.float64(u[b, t]) * q[x] < np.float64(target[b, t, x])):
                d = target[b, t].astype(np.float64) - q
                mass = np.where(d < 0, 0.0, d)
                break
            t += 1
        if mass is None or mass.sum() == 0:
            mass = target[b, t].astype(np.float64)
        total = mass.sum()
        kept.append(t)
        if not (0 < total < np.inf):
            token.append(-1)
            continue
        prefix = np.cumsum(mass)
        token.append(int(np.argmax((prefix > np.float64(u[b, T1 - 1]) * prefix[-1]))))
    return np.array(kept), np.array(token)


def _probs(g, B, T, V, sharp, dtype):
    return torch.softmax(torch.randn(B, T, V, generator=g) * sharp, -1).to(dtype)


def _run(dev, target, draft, tokens, u, counts=None, **kw):
    got = quant.verify_drafts(target.to(dev), None if draft is None else draft.to(dev), tokens.to(dev), u.to(dev),
                              None if counts is None else counts.to(dev), **kw)
    want = _rule(target.float().numpy(), None if draft is None else draft.float().numpy(), tokens.numpy(), u.numpy(),
                 None if counts is None else counts.numpy())
    return got, want


def _same(got, want):
    assert got[0].tolist() == want[0].tolist()
    assert got[1].tolist() == want[1].tolist()


# ---------------------------------------------------------------------------
# refusals (CPU)
# ---------------------------------------------------------------------------
def test_c_abi_refuses_bad_arguments():
    L = _lib.load()
    p = 1 << 16  # never read

    def call(t=p, psb=50, pst=10, q=p, qsb=40, qst=10, dt=0, B=2, T=4, V=10, tok=p, u=p, counts=p, kept=p, token=p, ws=p,
             nws=1 << 20):
        return L.sbq_verify_drafts(t, psb, pst, q, qsb, qst, dt, B, T, V, tok, u, counts, kept, token, ws, nws, None)

    assert call(dt=3) == -2
    for bad in (dict(B=-1), dict(B=65536), dict(T=-1), dict(T=65536), dict(V=0), dict(V=(1 << 23) + 1), dict(psb=-1),
                dict(qst=-1), dict(t=None), dict(u=None), dict(kept=None), dict(token=None), dict(tok=None)):
        assert call(**bad) == -1, bad
    for bad in (dict(t=p + 2), dict(q=p + 1), dict(tok=p + 4), dict(u=p + 2), dict(counts=p + 4), dict(kept=p + 1),
                dict(token=p + 2)):
        assert call(**bad) == -3, bad
    wide = dict(V=20000, psb=100000, pst=20000, qsb=80000, qst=20000)
    assert call(ws=None, **wide) == -4 and call(nws=L.sbq_verify_workspace_bytes(2, 20000) - 1, **wide) == -4
    assert call(B=0) == 0
    assert L.sbq_verify_workspace_bytes(0, 10) == 0 and L.sbq_verify_workspace_bytes(1, 0) == 0
    assert L.sbq_verify_workspace_bytes(3, 151936) == 3 * 38 * 16 + 16 and L.sbq_verify_workspace_bytes(3, 16384) == 0


def test_python_refuses():
    with pytest.raises(ValueError, match="GPU"):
        quant.verify_drafts(torch.zeros(1, 2, 3), None, torch.zeros(1, 1, dtype=torch.long), torch.zeros(1, 2))


@pytest.mark.gpu
def test_python_refuses_on_the_gpu(dev):
    g = torch.Generator().manual_seed(0)
    a = dict(target=_probs(g, 2, 4, 9, 1, F32).to(dev), draft=_probs(g, 2, 3, 9, 1, F32).to(dev),
             tokens=torch.zeros(2, 3, dtype=torch.long, device=dev), u=torch.zeros(2, 4, device=dev))
    quant.verify_drafts(**a)
    for match, kw in (("target", dict(target=a["target"].double())), ("target", dict(target=a["target"][0])),
                      ("draft", dict(draft=a["draft"].half())), ("draft", dict(draft=a["draft"][:, :2])),
                      ("draft", dict(draft=a["draft"].cpu())), ("tokens", dict(tokens=a["tokens"].int())),
                      ("tokens", dict(tokens=a["tokens"][:, :2])), ("u must", dict(u=a["u"][:, :3])),
                      ("u must", dict(u=a["u"].double())), ("counts", dict(counts=torch.zeros(2, device=dev))),
                      ("counts", dict(counts=torch.zeros(3, dtype=torch.long, device=dev))),
                      ("workspace", dict(workspace=torch.zeros(64, dtype=torch.uint8)))):
        with pytest.raises(ValueError, match=match):
            quant.verify_drafts(**{**a, **kw})
    with pytest.raises(ValueError, match="workspace"):
        quant.verify_drafts(torch.rand(1, 1, 20000, device=dev), None, torch.zeros(1, 0, dtype=torch.long, device=dev),
                            torch.zeros(1, 1, device=dev), workspace=torch.zeros(8, dtype=torch.uint8, device=dev))


# ---------------------------------------------------------------------------
# the rule
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("V", [1, 2, 5, 63, 1000, 4095, 4096, 4097, 16384, 20001])
@pytest.mark.parametrize("T", [0, 1, 3, 70])
def test_rule(dev, T, V, dtype):
    B = 6
    g = torch.Generator().manual_seed(V * 100 + T)
    target = _probs(g, B, T + 1, V, 2.0, dtype)
    draft = torch.softmax(target[:, :T].float().clamp_min(1e-9).log() + 0.3 * torch.randn(B, T, V, generator=g), -1).to(dtype)
    tokens = torch.multinomial(draft.float().reshape(-1, V), 1, generator=g).reshape(B, T) if T else torch.zeros(B, 0, dtype=torch.long)
    u = torch.rand(B, T + 1, generator=g)
    counts = torch.randint(-2, T + 3, (B,), generator=g)
    for d, c in ((draft, None), (None, None), (draft, counts), (None, counts)):
        announce(f"verify B={B} T={T} V={V} {dtype} draft={d is not None} counts={c is not None}")
        _same(*_run(dev, target, d, tokens, u, c))


@pytest.mark.gpu
def test_borders(dev):
    """Masses of whole powers of two, uniforms on the borders between tokens: the next token is drawn."""
    V = 5000
    target = torch.zeros(4, 2, V)
    target[:, :, [10, 4200, 4999, 300]] = 0.25  # 10, 300, 4200, 4999 in vocabulary order
    tokens = torch.full((4, 1), 10)
    u = torch.tensor([[0.5, 0.0], [0.5, 0.25], [0.5, 0.5], [0.5, 0.75]])
    got, want = _run(dev, target, None, tokens, u, torch.zeros(4, dtype=torch.long))
    _same(got, want)
    assert got[1].tolist() == [10, 300, 4200, 4999]
    # u q == p is refused, the least below it kept
    draft = torch.zeros(4, 1, V)
    draft[:, 0, 10] = 0.5
    u = torch.tensor([[0.5, 0.0], [0.49999997, 0.0], [0.0, 0.9], [1 - 2.0 ** -24, 1 - 2.0 ** -24]])
    got, want = _run(dev, target, draft, tokens, u)
    _same(got, want)
    assert got[0].tolist() == [0, 1, 1, 0]


@pytest.mark.gpu
def test_nothing_left_bad_drafts_and_bad_rows(dev):
    V = 4100
    g = torch.Generator().manual_seed(3)
    target = _probs(g, 9, 3, V, 1.0, F32)
    draft = _probs(g, 9, 2, V, 1.0, F32)
    tokens = torch.randint(0, V, (9, 2), generator=g)
    u = torch.full((9, 3), 0.5)
    draft[0, 0] = 2.0                       # nothing is left of p - q: p itself
    tokens[1, 0], tokens[2, 0], tokens[3, 0] = V, -1, 1 << 62  # no tokens: refused
    target[4, 0] = 0.0                      # no mass at all
    target[5, 0, 7] = float("nan")
    target[6, 0, 4099] = float("inf")
    target[7, 2, 3] = float("nan")          # a row that is not reached, or is
    target[8, 0, tokens[8, 0]] = float("nan")
    draft[8, 0, tokens[8, 0]] = 1e-30
    u[0, 0] = 0.99
    got, want = _run(dev, target, draft, tokens, u)
    _same(got, want)
    assert got[0][:5].tolist() == [0, 0, 0, 0, 0] and int(got[1][4]) == -1
    # the same rows with no draft before them
    got, want = _run(dev, target, draft, tokens, u, torch.zeros(9, dtype=torch.long))
    _same(got, want)
    assert got[1][4:7].tolist() == [-1, -1, -1] and int(got[1][8]) == -1
    # one-hot drafts that are no tokens leave p as it is
    got, want = _run(dev, target, None, tokens, u)
    _same(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_workspace(dev, dtype):
    B, T, V = 5, 3, 17003
    g = torch.Generator().manual_seed(9)
    big = _probs(g, B, T + 1, V + 3, 1.5, dtype).to(dev)
    target = big[:, :, 1:V + 1]             # rows that no vector load takes
    draft = _probs(g, T, B, V, 1.5, dtype).to(dev).transpose(0, 1)
    tokens = torch.randint(0, V, (T, B), generator=g).to(dev).t()
    u = torch.rand(T + 1, B, generator=g).to(dev).t()
    ws = quant.verify_workspace(B, V, dev)
    for _ in range(2):
        ws.fill_(255)
        got = quant.verify_drafts(target, draft, tokens, u, workspace=ws)
        _same(got, _rule(target.float().cpu().numpy(), draft.float().cpu().numpy(), tokens.cpu().numpy(), u.cpu().numpy(), None))
    row = target[:, :1].expand(B, T + 1, V)  # rows of one memory
    got = quant.verify_drafts(row, None, tokens, u)
    _same(got, _rule(row.float().cpu().numpy(), None, tokens.cpu().numpy(), u.cpu().numpy(), None))
    column = torch.rand(B, V, T + 1, generator=g).to(dev).transpose(1, 2)  # columns that are not side by side
    got = quant.verify_drafts(column, None, tokens, u)
    _same(got, _rule(column.cpu().numpy(), None, tokens.cpu().numpy(), u.cpu().numpy(), None))


@pytest.mark.gpu
def test_whole_vocabulary(dev):
    B, T, V = 7, 2, 151936
    g = torch.Generator().manual_seed(4)
    target, draft = _probs(g, B, T + 1, V, 2.0, F32), _probs(g, B, T, V, 2.0, F32)
    tokens = torch.multinomial(draft.reshape(-1, V), 1, generator=g).reshape(B, T)
    u = torch.rand(B, T + 1, generator=g)
    u[0, T], u[1, T] = 0.0, 1 - 2.0 ** -24
    _same(*_run(dev, target, draft, tokens, u))
    flat = torch.full((B, 1, V), 1.0 / V)   # fp32 sums would be off by many tokens
    _same(*_run(dev, flat, None, torch.zeros(B, 0, dtype=torch.long), u[:, :1].contiguous()))


@pytest.mark.gpu
def test_tokens_are_distributed_as_the_target_alone(dev):
    """The first token after the prefix, over many sequences of one distribution.
    Counts of 65535 draws: |count - n p| <= 5 sqrt(n p) + 5 fails once in a
    million for a right sampler; the uniforms are fixed."""
    n, V = 65535, 13
    g = torch.Generator().manual_seed(11)
    p, q = _probs(g, 1, 1, V, 1.0, F32)[0, 0], _probs(g, 1, 1, V, 1.5, F32)[0, 0]
    tokens = torch.multinomial(q, n, replacement=True, generator=g).reshape(n, 1)
    u = torch.rand(n, 2, generator=g)
    for draft, tok in ((q.expand(n, 1, V), tokens), (None, torch.full((n, 1), 4))):
        kept, token = quant.verify_drafts(p.to(dev).expand(n, 2, V), None if draft is None else draft.to(dev), tok.to(dev),
                                          u.to(dev))
        first = torch.where(kept.cpu() > 0, tok[:, 0], token.cpu())
        count = torch.bincount(first, minlength=V).double()
        assert ((count - n * p.double()).abs() <= 5 * (n * p.double()).sqrt() + 5).all()


@pytest.mark.gpu
def test_other_stream_and_graph(dev):
    B, T, V = 4, 3, 9001
    g = torch.Generator().manual_seed(2)
    target, draft = _probs(g, B, T + 1, V, 2.0, F32).to(dev), _probs(g, B, T, V, 2.0, F32).to(dev)
    tokens = torch.randint(0, V, (B, T), generator=g).to(dev)
    u = torch.rand(B, T + 1, generator=g).to(dev)
    want = quant.verify_drafts(target, draft, tokens, u)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = quant.verify_drafts(target, draft, tokens, u)
    side.synchronize()
    _same(got, [w.cpu().numpy() for w in want])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = quant.verify_drafts(target, draft, tokens, u)
    for i in range(4):
        u.copy_(torch.rand(B, T + 1, generator=g))
        tokens.copy_(torch.randint(0, V, (B, T), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        _same(held, [w.cpu().numpy() for w in quant.verify_drafts(target, draft, tokens, u)])


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 20001])
def test_rows_further_apart_than_32_bits(dev, V):
    B, T = 2, 1
    g = torch.Generator().manual_seed(V)
    target, draft = _probs(g, B, T + 1, V, 1.5, F32), _probs(g, B, T, V, 1.5, F32)
    tokens, u = torch.randint(0, V, (B, T), generator=g), torch.rand(B, T + 1, generator=g)
    apart = torch.empty(4 * (3 << 28), device=dev)  # 3 GiB between rows, 6 between sequences
    p = apart.as_strided((B, T + 1, V), (3 << 29, 3 << 28, 1))
    q = apart[1 << 27:].as_strided((B, T, V), (3 << 29, 3 << 28, 1))
    p.copy_(target)
    q.copy_(draft)
    _same(*_run(dev, target, draft, tokens, u))
    got = quant.verify_drafts(p, q, tokens.to(dev), u.to(dev))
    _same(got, _rule(target.numpy(), draft.numpy(), tokens.numpy(), u.numpy(), None))


@pytest.mark.gpu
def test_two_streams(dev):
    """Two calls at once, each with a workspace of its own."""
    g = torch.Generator().manual_seed(11)
    cases = []
    for B, T, V in ((9, 3, 40000), (4, 2, 9000)):
        target, draft = _probs(g, B, T + 1, V, 2.0, BF16).to(dev), _probs(g, B, T, V, 2.0, BF16).to(dev)
        cases.append((target, draft, torch.randint(0, V, (B, T), generator=g).to(dev), torch.rand(B, T + 1, generator=g).to(dev)))
    want = [quant.verify_drafts(*c) for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(20):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(quant.verify_drafts(*c))
    torch.cuda.synchronize()
    for w, results in zip(want, got):
        assert all(torch.equal(r[0], w[0]) and torch.equal(r[1], w[1]) for r in results)
