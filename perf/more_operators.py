"""Operators of a decode step for several sequences, beside the int8 linears.

A server runs one step for all of its sequences at once: the projections on a
row per token, then for every softmax layer the norms of queries and keys and
their rotation to each token's position, the new keys and values into each
sequence's pages of a shared pool, and the attention of the new tokens over
those pages.  Where tokens were drafted, the step ends with the choice of the
drafts that are kept.

Kinds of case (`op`):
  rope    norms of q and k for each head (`norm`), and the rotation of the
          first 2 * `pairs` columns, halves or neighbours (`inter`) paired
  store   T new tokens of each sequence (`one`: of one sequence, a prompt)
          into a paged cache, quantised where it has 8 bits, and read back
  attend  T new tokens of each sequence over its pages
  verify  T drafted tokens of each sequence against the target's
          probabilities: how many are kept, and the token after them

`own` is set by the program that measures: false, `run` computes the operator
from elementary torch operations; true, it calls the library.
"""
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "f8": torch.float8_e4m3fn}
SIZES = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "f8": 1}
LARGEST = {"i8": 127.0, "f8": 448.0}  # what the largest value of a vector is stored as

# no drawn case does more than the largest listed ones
MOST_ROPE = 8192 * 40 * 128
MOST_STORE = 8192 * 8 * 128
MOST_SLOTS = 64 * 16384 * 8 * 128
MOST_SCORES = 64 * 16384 * 32 * 128
MOST_VERIFY = 64 * 5 * 151936


def _package():
    """The library, from the repository's root as the working folder."""
    path = os.path.join(os.getcwd(), "spikingbrain-cpu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from sbq import quant, state

    return quant, state


def listed():
    return [
        # one token's step with the reference model's fp32 activations, queries and keys as parts of one projection: latency
        {"name": "rope_token", "op": "rope", "T": 1, "heads": 32, "kv": 8, "D": 128, "pairs": 64, "inter": False, "norm": True,
         "x": "f32"},
        # a chunk of a prompt at sizes that divide nothing: half of the columns rotated, neighbours paired
        {"name": "rope_ragged", "op": "rope", "T": 333, "heads": 14, "kv": 2, "D": 80, "pairs": 20, "inter": True, "norm": True,
         "x": "f16"},
        # several prompts side by side, the largest pass
        {"name": "rope_prompt", "op": "rope", "T": 8192, "heads": 32, "kv": 8, "D": 128, "pairs": 64, "inter": False,
         "norm": True, "x": "bf16"},
        # each step of 16 sequences with an 8-bit cache, fp32 activations
        {"name": "store_step_i8", "op": "store", "B": 16, "T": 1, "kv": 8, "D": 128, "page": 64, "max": 4096, "one": False,
         "new": "f32", "cache": "i8", "ragged": False},
        # a long prompt of one of them
        {"name": "store_prompt_f8", "op": "store", "B": 4, "T": 8192, "kv": 8, "D": 128, "page": 64, "max": 16384, "one": True,
         "new": "bf16", "cache": "f8", "ragged": False},
        # one sequence's token over an fp32 cache, the reference's types: latency
        {"name": "attend_one_f32", "op": "attend", "B": 1, "T": 1, "heads": 32, "kv": 8, "D": 128, "page": 64, "max": 2048,
         "window": 0, "q": "f32", "cache": "f32"},
        # a layer with a window: 5 sequences with up to 4 drafts each, sizes that divide nothing, small pages
        {"name": "attend_drafts_window", "op": "attend", "B": 5, "T": 4, "heads": 14, "kv": 2, "D": 80, "page": 16, "max": 5000,
         "window": 1024, "q": "f16", "cache": "f16"},
        # 16 sequences of a chat service over an 8-bit cache, fp32 activations
        {"name": "attend_batch_i8", "op": "attend", "B": 16, "T": 1, "heads": 32, "kv": 8, "D": 128, "page": 64, "max": 8192,
         "window": 0, "q": "f32", "cache": "i8"},
        # one long document
        {"name": "attend_long_bf16", "op": "attend", "B": 1, "T": 1, "heads": 32, "kv": 8, "D": 128, "page": 128, "max": 65536,
         "window": 0, "q": "bf16", "cache": "bf16"},
        # 64 sequences of very different lengths, the largest attention
        {"name": "attend_batch_f8", "op": "attend", "B": 64, "T": 1, "heads": 32, "kv": 8, "D": 128, "page": 64, "max": 16384,
         "window": 0, "q": "bf16", "cache": "f8"},
        # four drafted tokens of one sequence: latency
        {"name": "verify_one", "op": "verify", "B": 1, "T": 4, "V": 151936, "p": "f32", "draft": True, "ragged": False},
        # 64 sequences, the whole vocabulary for each
        {"name": "verify_batch", "op": "verify", "B": 64, "T": 4, "V": 151936, "p": "f32", "draft": True, "ragged": True},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("rope", "store", "store", "attend", "attend", "attend", "verify"))
    kv, rep = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 4, 7, 8))
    D = rng.choice((64, 128, 128, 256, 2 * rng.randrange(4, 125)))
    if op == "rope":
        heads = kv * rep
        pairs = D // 2 if rng.random() < 0.7 else rng.randrange(1, D // 2 + 1)
        return {"op": op, "T": _log(rng, 1, max(1, MOST_ROPE // ((heads + kv) * D * 4))), "heads": heads, "kv": kv, "D": D,
                "pairs": pairs, "inter": rng.random() < 0.3, "norm": rng.random() < 0.7, "x": rng.choice(("f32", "f16", "bf16"))}
    page = rng.choice((16, 32, 64, 128))
    if op == "store":
        one = rng.random() < 0.4
        while True:
            B, T = _log(rng, 1, 64), _log(rng, 16, 8192) if one else _log(rng, 1, 8)
            if T * kv * D * (1 if one else B) <= MOST_STORE:
                break
        return {"op": op, "B": min(B, 8) if one else B, "T": T, "kv": kv, "D": D, "page": page, "max": T + _log(rng, 16, 4096),
                "one": one, "new": rng.choice(("f32", "f16", "bf16")), "cache": rng.choice(("i8", "i8", "f8", "f8", "bf16", "f16")),
                "ragged": not one and rng.random() < 0.4}
    if op == "attend":
        cache = rng.choice(("i8", "i8", "f8", "f8", "bf16", "f16", "f32"))
        while True:
            B, T, most = _log(rng, 1, 64), rng.choice((1, 1, 1, _log(rng, 1, 8))), _log(rng, 16, 65536)
            slots = B * most * kv * D
            if slots * SIZES[cache] <= MOST_SLOTS and slots * rep * T <= MOST_SCORES and T <= most:
                break
        q = rng.choice(("f32", "f16", "bf16") if cache in LARGEST else ("f32", cache))
        return {"op": op, "B": B, "T": T, "heads": kv * rep, "kv": kv, "D": D, "page": page, "max": most,
                "window": rng.choice((0, 0, 0, _log(rng, 1, most))), "q": q, "cache": cache}
    while True:
        B, T, V = _log(rng, 1, 64), _log(rng, 1, 8), _log(rng, 1000, 151936)
        if B * (T + 1) * V <= MOST_VERIFY:
            break
    return {"op": op, "B": B, "T": T, "V": V, "p": rng.choice(("f32", "f32", "bf16")), "draft": rng.random() < 0.7,
            "ragged": rng.random() < 0.4}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _spread(case, least):
    """The sequences' lengths, from `least` to the longest, on a log scale."""
    top = case["max"]
    return [top if b == 0 else int(round(least * (top / least) ** (b * 0.6180339887 % 1))) for b in range(case["B"])]


def _shortest(case):
    return max(case["T"], case["max"] // 64)


def _rope_inputs(case, seed):
    """Views of one projection's output [T, (heads + 2 kv) * D], the norms' weights, and the tokens' positions."""
    g = _gen(seed)
    T, H, kv, D, x = case["T"], case["heads"], case["kv"], case["D"], DTYPES[case["x"]]
    qkv = (torch.randn(T, (H + 2 * kv) * D, generator=g, device=DEV) * 2).to(x)
    s = {"q": qkv[:, :H * D].unflatten(1, (H, D)), "k": qkv[:, H * D:(H + kv) * D].unflatten(1, (kv, D)),
         "inter": case["inter"], "q_weight": None, "k_weight": None, "eps": 1e-6}
    if case["norm"]:
        s["q_weight"], s["k_weight"] = [torch.rand(D, generator=g, device=DEV) + 0.5 for _ in range(2)]
    # some sequences stand at the start of a context of 131072 positions, others far into it
    s["positions"] = (torch.randint(0, 131072 - T, (1,), generator=g, device=DEV) + torch.arange(T, device=DEV)) if T > 64 else \
        torch.randint(0, 131072, (T,), generator=g, device=DEV)
    s["inv_freq"] = (1e6 ** -(torch.arange(case["pairs"], device=DEV, dtype=torch.float64) / case["pairs"])).float()
    return s


def _pages(case, g, lengths):
    """Each sequence's pages, in no order among those of a pool with some to
    spare; entries behind a sequence's last page are -1."""
    page = case["page"]
    need = [-(-n // page) for n in lengths]
    pages, width = sum(need) + 3, -(-case["max"] // page)
    free = torch.randperm(pages, generator=g, device=DEV).int()
    at = torch.arange(width, device=DEV)[None, :]
    n = torch.tensor(need, device=DEV)[:, None]
    first = n.cumsum(0) - n
    return pages, torch.where(at < n, free[(first + at).clamp_max(pages - 1)], -1).int().contiguous()


def _quantise(x, cache):
    """8-bit codes of x [..., D] and a scale for each vector."""
    most = x.abs().amax(-1)
    scale = most / torch.full_like(most, LARGEST[cache])  # (by a number, torch multiplies with its reciprocal)
    y = x / torch.where(scale > 0, scale, 1.0)[..., None]
    return (torch.round(y) if cache == "i8" else y).to(DTYPES[cache]), scale


def _pool(case, g, pages, filled):
    """Keys and values [pages, kv, page, D] (rows of whole 16 elements) and, of 8 bits, the vectors' scales."""
    kv, page, D, cache = case["kv"], case["page"], case["D"], case["cache"]
    out = {}
    for name in ("k", "v"):
        t = torch.zeros(pages, kv, page, -(-D // 16) * 16, dtype=DTYPES[cache], device=DEV)[..., :D]
        scale = torch.zeros(pages, kv, page, device=DEV) if cache in LARGEST else None
        for p in range(0, pages if filled else 0, 4096):  # a part of the pool at a time
            x = torch.randn(min(4096, pages - p), kv, page, D, generator=g, device=DEV)
            if scale is None:
                t[p:p + 4096] = x.to(t.dtype)
            else:
                codes, scale[p:p + 4096] = _quantise(x, cache)
                t.view(torch.int8)[p:p + 4096] = codes.view(torch.int8)
        out[name], out[name + "_scale"] = t, scale
    return out


def _store_inputs(case, seed):
    g = _gen(seed)
    B, T, kv, D = case["B"], case["T"], case["kv"], case["D"]
    held = [n - T for n in _spread(case, T + 1)]  # before the new tokens
    pages, table = _pages(case, g, [n + T for n in held])
    s = {"table": table, "length": torch.tensor(held, device=DEV), **_pool(case, g, pages, False)}
    s["start"] = s["length"].clone()
    n = T if case["one"] else B * T
    s["k_new"], s["v_new"] = [torch.randn(n, kv, D, generator=g, device=DEV).to(DTYPES[case["new"]]) for _ in range(2)]
    if not case["one"]:
        s["k_new"], s["v_new"] = s["k_new"].view(B, T, kv, D), s["v_new"].view(B, T, kv, D)
    s["one"] = B // 2 if case["one"] else None
    s["counts"] = None
    if case["ragged"]:  # some sequences have fewer new tokens
        s["counts"] = torch.randint(0, T + 1, (B,), generator=g, device=DEV)
        s["counts"][0] = T
    s["out"] = DTYPES[case["new"]] if case["cache"] in LARGEST else DTYPES[case["cache"]]
    return s


def _attend_inputs(case, seed):
    g = _gen(seed)
    lengths = _spread(case, _shortest(case))
    pages, table = _pages(case, g, lengths)
    s = {"table": table, "length": torch.tensor(lengths, device=DEV), **_pool(case, g, pages, True)}
    q = torch.randn(case["B"], case["T"], case["heads"], case["D"], generator=g, device=DEV) * 1.5
    s["q"], s["window"] = q.to(DTYPES[case["q"]]), case["window"]
    return s


def _verify_inputs(case, seed):
    """The target's probabilities: a few likely tokens and a long tail; the
    draft model's are near them, and its tokens drawn from them (without
    probabilities: its most likely ones)."""
    g = _gen(seed)
    B, T, V, p = case["B"], case["T"], case["V"], DTYPES[case["p"]]
    z = torch.randn(B, T + 1, V, generator=g, device=DEV) * 2
    z.scatter_add_(2, torch.randint(0, V, (B, T + 1, 20), generator=g, device=DEV),
                   7 + 2 * torch.randn(B, T + 1, 20, generator=g, device=DEV))
    y = z[:, :T] + 0.6 * torch.randn(B, T, V, generator=g, device=DEV)
    s = {"target": torch.softmax(z, -1).to(p), "draft": None, "counts": None}
    if case["draft"]:
        s["draft"] = torch.softmax(y, -1).to(p)
        s["tokens"] = (y - torch.rand(B, T, V, generator=g, device=DEV).clamp_min(1e-30).log().neg().log()).argmax(-1)
    else:
        s["tokens"] = y.argmax(-1)
    s["u"] = torch.rand(B, T + 1, generator=g, device=DEV)
    if case["ragged"]:  # some sequences drafted fewer
        s["counts"] = torch.randint(0, T + 1, (B,), generator=g, device=DEV)
    return s


def prepare(case, seed):
    op = case["op"]
    s = {"rope": _rope_inputs, "store": _store_inputs, "attend": _attend_inputs, "verify": _verify_inputs}[op](case, seed)
    if own and op in ("store", "attend"):  # a program holds the cache
        _, state = _package()
        b = state.DevicePagedKVBuffer(case["B"], case["kv"], case["D"], s["k"].shape[0], case["page"], s["table"].shape[1],
                                      case.get("window") or None, DEV, DTYPES[case["cache"]])
        for name in ("k", "v", "k_scale", "v_scale", "table", "length"):
            setattr(b, name, s[name])
        s["buffer"] = b
    s["op"], s["cache"], s["page"] = op, case.get("cache"), case.get("page")
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _turn(x, cos, sin, weight, eps, inter):
    x, n = x.float(), cos.shape[-1]
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if inter else (x[..., :n], x[..., n:2 * n])
    c, d = a * cos - b * sin, b * cos + a * sin
    return torch.cat([torch.stack([c, d], -1).flatten(-2) if inter else torch.cat([c, d], -1), x[..., 2 * n:]], -1)


def _plain_rope(s):
    angle = s["positions"].double()[:, None, None] * s["inv_freq"].double()  # far positions: 32 bits lose the angle
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    return [_turn(s[n], cos, sin, s[n + "_weight"], s["eps"], s["inter"]).to(s[n].dtype) for n in ("q", "k")]


def _plain_store(s):
    one, page, cache = s["one"], s["page"], s["cache"]
    start, table = (s["start"], s["table"]) if one is None else (s["start"][one:one + 1], s["table"][one:one + 1])
    k, v = (s["k_new"], s["v_new"]) if one is None else (s["k_new"][None], s["v_new"][None])
    T = k.shape[1]
    t = torch.arange(T, device=DEV)
    pos = start[:, None] + t
    count = torch.full_like(start, T) if s["counts"] is None else s["counts"]
    is_new = t < count[:, None]
    at = torch.gather(table.long(), 1, pos // page)
    row, slot = at[is_new], (pos % page)[is_new]  # [new tokens]
    out = {}
    for name, x in (("k", k), ("v", v)):
        x, pool = x.float()[is_new], s[name]
        if cache in LARGEST:
            x, scale = _quantise(x, cache)
            s[name + "_scale"][row, :, slot] = scale
            pool.view(torch.int8)[row, :, slot] = x.view(torch.int8)
        else:
            pool[row, :, slot] = x.to(pool.dtype)
        back = pool.view(torch.int8)[at, :, pos % page].view(pool.dtype).float() if cache in LARGEST else pool[at, :, pos % page]
        if cache in LARGEST:
            back = back * s[name + "_scale"][at, :, pos % page][..., None]
        back = torch.where(is_new[..., None, None], back, 0).to(s["out"])
        out[name] = back if one is None else back[0]
    if one is None:
        s["length"].copy_(start + count)
    else:
        s["length"][one:one + 1] = start + count
    out["length"] = s["length"]
    return out


def _plain_attend(s):
    q, table, length, page, window = s["q"], s["table"].long(), s["length"], s["page"], s["window"]
    B, T, H, D = q.shape
    kv, L = s["k"].shape[1], table.shape[1] * page
    at = table.clamp_min(0)
    k, v = [(s[n].view(torch.int8)[at].view(s[n].dtype) if s["cache"] in LARGEST else s[n][at]).float() for n in ("k", "v")]
    if s["cache"] in LARGEST:
        k, v = k * s["k_scale"][at][..., None], v * s["v_scale"][at][..., None]
    k, v = [x.transpose(1, 2).reshape(B, kv, L, D) for x in (k, v)]
    pos = torch.arange(L, device=DEV)
    q_pos = length[:, None] - T + torch.arange(T, device=DEV)
    see = (pos <= q_pos[..., None]) & (table.repeat_interleave(page, 1) >= 0)[:, None]
    if window:
        see &= pos > q_pos[..., None] - window
    # query head h reads kv head h // (H / kv)
    qt = q.float().view(B, T, kv, H // kv, D).permute(0, 2, 4, 3, 1).reshape(B, kv, D, -1)
    score = torch.matmul(k, qt).transpose(2, 3).reshape(B, kv, H // kv, T, L) * D ** -0.5
    score = score.masked_fill(~see[:, None, None], float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, kv, -1, L), torch.where(see.any(1)[:, None, :, None], v, 0))
    return o.view(B, kv, H // kv, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(q.dtype)


def _plain_verify(s):
    p, q, tokens, u = s["target"], s["draft"], s["tokens"], s["u"].double()
    B, T = tokens.shape
    t = torch.arange(T, device=DEV)
    count = torch.full((B,), T, device=DEV) if s["counts"] is None else s["counts"]
    px = torch.gather(p[:, :T], 2, tokens[..., None])[..., 0].double()
    qx = 1.0 if q is None else torch.gather(q, 2, tokens[..., None])[..., 0].double()
    ok = (u[:, :T] * qx < px) & (t < count[:, None])
    kept = ok.long().cumprod(1).sum(1)
    b = torch.arange(B, device=DEV)
    row, again = p[b, kept].double(), kept.clamp_max(T - 1)  # long sums: 64 bits
    if q is None:
        rest = row.scatter(1, tokens[b, again][:, None], 0.0)
    else:
        rest = (row - q[b, again].double()).clamp_min(0)
    use = (kept < count) & (rest.sum(1) > 0)
    mass = torch.where(use[:, None], rest, row).cumsum(1)
    token = (mass > u[:, T:] * mass[:, -1:]).long().argmax(1)
    return kept, token


def run(s):
    op = s["op"]
    if not own:
        return {"rope": _plain_rope, "store": _plain_store, "attend": _plain_attend, "verify": _plain_verify}[op](s)
    quant, state = _package()
    if op == "rope":
        return list(state.qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], s["q_weight"], s["k_weight"], s["eps"],
                                       s["inter"]))
    if op == "verify":
        return quant.verify_drafts(s["target"], s["draft"], s["tokens"], s["u"], s["counts"])
    b = s["buffer"]
    if op == "attend":
        return b.attend(s["q"])
    one = s["one"]
    start = s["start"] if one is None else s["start"][one:one + 1]
    b.append(s["k_new"], s["v_new"], start, s["counts"], one)
    k, v = b.read(start, s["k_new"].shape[0 if one is not None else 1], s["out"], one)
    return {"k": k, "v": v, "length": b.length}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "rope":
        n = case["T"] * (case["heads"] + case["kv"]) * case["D"]
        extra = 8 * case["T"] + 4 * case["pairs"] + (8 * case["D"] if case["norm"] else 0)
        return {"bytes": 2 * n * SIZES[case["x"]] + extra, "flops": n * (7 if case["norm"] else 3)}
    if op == "verify":  # a row of the target's and, after a refusal, one of the draft's
        b = case["B"] * (2 if case["draft"] else 1) * case["V"] * SIZES[case["p"]]
        return {"bytes": b, "flops": 3 * case["B"] * case["V"]}
    vector = case["D"] * SIZES[case["cache"]] + (4 if case["cache"] in LARGEST else 0)  # one token's keys or values of a head
    if op == "store":
        n = 2 * case["T"] * (1 if case["one"] else case["B"]) * case["kv"]
        out = SIZES[case["new"]] if case["cache"] in LARGEST else SIZES[case["cache"]]
        return {"bytes": n * (case["D"] * (SIZES[case["new"]] + out) + vector), "flops": 4 * n * case["D"]}
    T, window = case["T"], case["window"]
    held = sum(min(n, window + T - 1) if window else n for n in _spread(case, _shortest(case)))
    b = 2 * held * case["kv"] * vector + 2 * case["B"] * T * case["heads"] * case["D"] * SIZES[case["q"]]
    return {"bytes": b + 4 * held // case["page"] + 8 * case["B"], "flops": 4 * T * case["heads"] * case["D"] * held}


# ---------------------------------------------------------------------------
# the same results in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_rope(case, seed):
    s = _rope_inputs(case, seed)
    n, out = case["pairs"], []
    first = torch.arange(n, device=DEV) * (2 if case["inter"] else 1)
    second = first + (1 if case["inter"] else n)
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()[None, :]
    z = torch.polar(torch.ones_like(angle), angle)[:, None, :]
    for name in ("q", "k"):
        x = s[name].double()
        if case["norm"]:
            x = x / (x.pow(2).sum(-1, keepdim=True) / case["D"] + s["eps"]).sqrt() * s[name + "_weight"].double()
        turned = torch.complex(x[..., first], x[..., second]) * z
        y = x.clone()
        y[..., first], y[..., second] = turned.real, turned.imag
        out.append(y)
    return out


def _near_e4m3(y):
    """The nearest e4m3 values of y, ties to even: 3 bits after the first, none below 2^-9."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _exact_store(case, seed):
    s = _store_inputs(case, seed)
    out = {}
    for name in ("k", "v"):
        x = s[name + "_new"].double()
        if case["cache"] in LARGEST:
            scale = (x.abs().amax(-1, keepdim=True) / LARGEST[case["cache"]]).float().double()  # (held in 32 bits)
            y = torch.where(scale > 0, x / scale, 0.0).float().double()  # (and so is the quotient)
            x = scale * (torch.round(y) if case["cache"] == "i8" else _near_e4m3(y))
        else:
            x = s[name + "_new"].to(DTYPES[case["cache"]]).double()
        if case["ragged"]:
            for b, n in enumerate(s["counts"].tolist()):
                x[b, n:] = 0.0
        out[name] = x
    length = s["start"].clone()
    if case["one"]:
        length[s["one"]] += case["T"]
    else:
        length += case["T"] if s["counts"] is None else s["counts"]
    out["length"] = length
    return out


def _exact_attend(case, seed):
    s = _attend_inputs(case, seed)
    T, H, D, page = case["T"], case["heads"], case["D"], case["page"]
    rep = H // case["kv"]
    out = torch.zeros(case["B"], T, H, D, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_spread(case, _shortest(case))):  # one sequence at a time
        low = max(0, n - T - case["window"] + 1) if case["window"] else 0
        first = low // page
        at = s["table"][b, first:-(-n // page)].long()
        k, v = [s[x].view(torch.int8)[at].view(s[x].dtype).double() if case["cache"] in LARGEST else s[x][at].double()
                for x in ("k", "v")]
        if case["cache"] in LARGEST:
            k, v = k * s["k_scale"][at].double()[..., None], v * s["v_scale"][at].double()[..., None]
        k, v = [x.transpose(0, 1).flatten(1, 2)[:, low - first * page:n - first * page].contiguous() for x in (k, v)]
        age = torch.arange(n - T, n, device=DEV)[:, None] - torch.arange(low, n, device=DEV)
        see = (age >= 0) & (age < (case["window"] or 1 << 60))
        for h in range(case["kv"]):
            z = torch.matmul(s["q"][b, :, h * rep:(h + 1) * rep].double().reshape(T * rep, D), k[h].t().contiguous())
            z = torch.where(see.repeat_interleave(rep, 0), z / D ** 0.5, float("-inf"))
            out[b, :, h * rep:(h + 1) * rep] = torch.matmul(torch.softmax(z, -1), v[h]).view(T, rep, D)
    return out


def _exact_verify(case, seed):
    s = _verify_inputs(case, seed)
    kept, token = [], []
    tokens, u = s["tokens"].tolist(), s["u"].double().tolist()
    counts = [case["T"]] * case["B"] if s["counts"] is None else s["counts"].tolist()
    for b in range(case["B"]):
        t, mass = 0, None
        while t < counts[b]:
            x = tokens[b][t]
            p = s["target"][b, t].double()
            if s["draft"] is None:
                q = torch.zeros_like(p)
                q[x] = 1.0
            else:
                q = s["draft"][b, t].double()
            if not u[b][t] * float(q[x]) < float(p[x]):
                mass = torch.relu(p - q)
                break
            t += 1
        if mass is None or float(mass.sum()) == 0.0:
            mass = s["target"][b, t].double()
        mass = torch.cumsum(mass, 0)
        want = torch.full((1,), u[b][case["T"]], dtype=torch.float64, device=DEV) * mass[-1]
        kept.append(t)
        token.append(int(torch.searchsorted(mass, want, right=True)))
    return torch.tensor(kept, device=DEV), torch.tensor(token, device=DEV)


def exact(case, seed):
    return {"rope": _exact_rope, "store": _exact_store, "attend": _exact_attend, "verify": _exact_verify}[case["op"]](case, seed)
