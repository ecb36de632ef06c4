"""Operators of a decode step with drafted tokens, beside the int8 linears.

A serving loop that drafts several tokens per step verifies them in one pass:
every projection runs on a handful of rows (one per node of the tree of
drafts), the attention reads the cache once for all of them, and a layer with
a bounded cache replaces the slots that earlier tokens attended to least.

Kinds of case (`op`):
  linear  one linear with 4-bit weights and group scales on [M, K] activations
  attend  T query tokens over a cache, and over each other's keys by a tree of
          drafts where `drafts` is set; `weight`: the attention weight that
          each cached slot received is added to its running sum
  append  T tokens into a full bounded cache, in the place of the slots of
          least weight (the `recent` newest positions stay)
  take    a prompt's cache reduced to a bounded one by the same rule

`own` is set by the program that measures: false, `run` computes the operator
from elementary torch operations; true, it calls the library.
"""
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}

# no drawn case does more than the largest listed ones
MOST_LINEAR = 151936 * 2560
MOST_LINEAR_FLOPS = 2 * 64 * 12288 * 4096
MOST_SCORES = 64 * 32 * 65536 * 128
MOST_CACHE = 2 * 65536 * 8 * 128 * 2


def _package():
    """The library, from the repository's root as the working folder."""
    path = os.path.join(os.getcwd(), "spikingbrain-cpu_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from sbq import quant, state

    return quant, state


def listed():
    return [
        # one small projection of a decode step with the reference model's fp32 activations: latency
        {"name": "w4_o_m1", "op": "linear", "M": 1, "N": 2560, "K": 4096, "group": 128, "x": "f32", "y": "f32"},
        # the widest projection of a decode step, fp16 activations: the weight stream
        {"name": "w4_gate_up_m1", "op": "linear", "M": 1, "N": 24576, "K": 4096, "group": 128, "x": "f16", "y": "f16"},
        # a small tree of drafts on a layer whose sizes divide nothing, fine groups
        {"name": "w4_ragged_m5", "op": "linear", "M": 5, "N": 2999, "K": 2500, "group": 32, "x": "f32", "y": "f32"},
        # a tree of 64 drafts through one part of an FFN
        {"name": "w4_tree_m64", "op": "linear", "M": 64, "N": 12288, "K": 4096, "group": 64, "x": "bf16", "y": "bf16"},
        # the vocabulary projection of one token, the largest weight of a step
        {"name": "w4_lm_head_m1", "op": "linear", "M": 1, "N": 151936, "K": 2560, "group": 128, "x": "f32", "y": "f32"},
        # a sequence's ordinary decode step over a cache of the default fp32 that also counts its attention weights
        {"name": "attend_decode_f32", "op": "attend", "T": 1, "heads": 32, "kv": 8, "D": 128, "slots": 2304, "filled": 2048,
         "window": 0, "q": "f32", "cache": "f32", "drafts": False, "weight": True},
        # a tree of 16 drafts over a chat's cache
        {"name": "attend_tree_t16", "op": "attend", "T": 16, "heads": 32, "kv": 8, "D": 128, "slots": 8192, "filled": 6000,
         "window": 0, "q": "f16", "cache": "f16", "drafts": True, "weight": False},
        # drafts in a layer with a window (a ring of slots), of odd sizes, fp32 queries over a 2-byte cache
        {"name": "attend_ring_t5", "op": "attend", "T": 5, "heads": 14, "kv": 2, "D": 80, "slots": 1100, "filled": 3001,
         "window": 1024, "q": "f32", "cache": "bf16", "drafts": True, "weight": False},
        # a tree of 64 drafts over a long document, the largest attention
        {"name": "attend_tree_t64_long", "op": "attend", "T": 64, "heads": 32, "kv": 8, "D": 128, "slots": 65536,
         "filled": 65000, "window": 0, "q": "bf16", "cache": "bf16", "drafts": True, "weight": True},
        # each decode step of a layer with a bounded cache: one token in, the least attended one out
        {"name": "append_t1", "op": "append", "T": 1, "slots": 4096, "recent": 512, "kv": 8, "D": 128, "new": "f32",
         "cache": "bf16"},
        # the accepted drafts of a step into a long bounded cache
        {"name": "append_t12_long", "op": "append", "T": 12, "slots": 32768, "recent": 1024, "kv": 8, "D": 128, "new": "f32",
         "cache": "f32"},
        # the end of a long prompt: its cache reduced to the bounded one
        {"name": "take_prompt", "op": "take", "slots": 32768, "filled": 30000, "capacity": 4096, "recent": 512, "kv": 8,
         "D": 128, "cache": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("linear", "linear", "attend", "attend", "append", "take"))
    if op == "linear":
        while True:
            M, N, K = _log(rng, 1, 64), _log(rng, 128, 151936), _log(rng, 128, 12288)
            if rng.random() < 0.7:  # a real layer's sizes; the rest stay odd
                N, K = max(128, N // 64 * 64), max(128, K // 64 * 64)
            if N * K <= MOST_LINEAR and 2 * M * N * K <= MOST_LINEAR_FLOPS:
                break
        x = rng.choice(("f32", "f32", "f16", "bf16"))
        return {"op": op, "M": M, "N": N, "K": K, "group": rng.choice((32, 64, 128, 128)), "x": x,
                "y": x if rng.random() < 0.5 else "f32", "bias": rng.random() < 0.3}
    cache = rng.choice(("f32", "f16", "bf16", "bf16"))
    if op == "attend":
        while True:
            T, kv, rep = _log(rng, 1, 64), rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 4, 7, 8))
            D, slots = rng.choice((64, 128, 128, 256, rng.randrange(8, 250))), _log(rng, 64, 65536)
            if T * kv * rep * slots * D <= MOST_SCORES and 2 * slots * kv * D * SIZES[cache] <= MOST_CACHE:
                break
        window = rng.choice((0, 0, max(1, slots - rng.randrange(1, 64))))
        drafts = rng.random() < 0.6
        if window and not drafts and T > slots - window:
            T = slots - window  # the ring holds the window beside the appended tokens
        filled = rng.randrange(max(T, slots // 4), 2 * slots if window else slots + 1)
        return {"op": op, "T": T, "heads": kv * rep, "kv": kv, "D": D, "slots": slots, "filled": filled, "window": window,
                "q": rng.choice((cache, "f32")), "cache": cache, "drafts": drafts, "weight": rng.random() < 0.4}
    kv, D = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 128, rng.randrange(8, 250)))
    if op == "append":
        slots = _log(rng, 256, 32768)
        return {"op": op, "T": _log(rng, 1, 64), "slots": slots, "recent": rng.randrange(1, slots // 2), "kv": kv, "D": D,
                "new": rng.choice(("f32", cache)), "cache": cache}
    slots = _log(rng, 512, 32768)
    capacity = rng.randrange(128, slots // 2)
    return {"op": op, "slots": slots, "filled": rng.randrange(slots // 2, slots + 1), "capacity": capacity,
            "recent": rng.randrange(1, capacity), "kv": kv, "D": D, "cache": cache}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _linear_inputs(case, seed):
    """4-bit weights q and their group scales as a quantized checkpoint holds
    them (N(0, 0.02) weights), a bias, and N(0, 1) activations with 1% of the
    channels 20 times larger."""
    g = _gen(seed)
    N, K, group = case["N"], case["K"], case["group"]
    G = -(-K // group)
    w = torch.zeros(N, G * group, device=DEV)
    w[:, :K] = torch.randn(N, K, generator=g, device=DEV) * 0.02
    w = w.view(N, G, group)
    scale = (w.abs().amax(2).clamp_min(1e-8) / 7).to(torch.bfloat16)
    q = torch.round(w / scale.float()[:, :, None]).clamp(-7, 7).to(torch.int8).view(N, G * group)[:, :K].contiguous()
    bias = torch.randn(N, generator=g, device=DEV) if case.get("bias") else None
    x = torch.randn(case["M"], K, generator=g, device=DEV)
    x *= torch.where(torch.rand(K, generator=g, device=DEV) < 0.01, 20.0, 1.0)
    return q, scale, bias, x.to(DTYPES[case["x"]])


def _cache(case, g, slots):
    shape = (slots, case["kv"], case["D"])
    dtype = DTYPES[case["cache"]]
    return [torch.randn(shape, generator=g, device=DEV).to(dtype) for _ in range(2)]


def _attend_inputs(case, seed):
    g = _gen(seed)
    T, slots, filled = case["T"], case["slots"], case["filled"]
    k, v = _cache(case, g, slots)
    at = torch.arange(slots, device=DEV)
    if case["window"]:  # a ring: slot s holds the newest position that is s modulo the slots
        slot_pos = filled - 1 - (filled - 1 - at) % slots
        slot_pos = torch.where(slot_pos < 0, -1, slot_pos)
    else:
        slot_pos = torch.where(at < filled, at, -1)
    s = {"k": k, "v": v, "slot_pos": slot_pos, "k_new": None, "v_new": None, "tree": None}
    s["q"] = (torch.randn(T, case["heads"], case["D"], generator=g, device=DEV) * 1.5).to(DTYPES[case["q"]])
    if case["drafts"]:
        s["k_new"], s["v_new"] = _cache(case, g, T)
        # each draft continues an earlier one, more often a late one
        r = torch.rand(T, generator=torch.Generator().manual_seed(seed)).tolist()
        parent = [-1] + [int(i * r[i] ** 0.5) for i in range(1, T)]
        tree, depth = torch.eye(T, dtype=torch.bool), [0] * T
        for i in range(1, T):
            tree[i] |= tree[parent[i]]
            depth[i] = depth[parent[i]] + 1
        s["tree"], s["q_pos"] = tree.to(DEV), filled + torch.tensor(depth, device=DEV)
    else:  # the tokens' own keys are in the cache already
        s["q_pos"] = filled - T + torch.arange(T, device=DEV)
    s["weight"] = torch.rand(slots, generator=g, device=DEV) if case["weight"] else None
    return s


def _slot_weights(g, slots):
    """Running sums of attention weight: a few slots with most of it, some with none at all."""
    w = torch.exp(torch.randn(slots, generator=g, device=DEV) * 2 - 3)
    return torch.where(torch.rand(slots, generator=g, device=DEV) < 0.05, 0.0, w)


def _append_inputs(case, seed):
    g = _gen(seed)
    slots, T = case["slots"], case["T"]
    k, v = _cache(case, g, slots)
    # a full cache after many replacements: positions up to four times the slots, in no order
    slot_pos = torch.randperm(4 * slots, generator=g, device=DEV)[:slots].contiguous()
    new = [torch.randn(T, case["kv"], case["D"], generator=g, device=DEV).to(DTYPES[case["new"]]) for _ in range(2)]
    return {"k": k, "v": v, "slot_pos": slot_pos, "weight": _slot_weights(g, slots), "k_new": new[0], "v_new": new[1],
            "end": torch.full((1,), 4 * slots, dtype=torch.long, device=DEV), "recent": case["recent"]}


def _take_inputs(case, seed):
    g = _gen(seed)
    slots, capacity = case["slots"], case["capacity"]
    k, v = _cache(case, g, slots)
    at = torch.arange(slots, device=DEV)
    return {"k": k, "v": v, "slot_pos": torch.where(at < case["filled"], at, -1), "weight": _slot_weights(g, slots),
            "end": torch.full((1,), case["filled"], dtype=torch.long, device=DEV), "recent": case["recent"],
            "to_k": torch.zeros((capacity,) + k.shape[1:], dtype=k.dtype, device=DEV),
            "to_v": torch.zeros((capacity,) + k.shape[1:], dtype=k.dtype, device=DEV),
            "to_pos": torch.full((capacity,), -1, dtype=torch.long, device=DEV),
            "to_weight": torch.zeros(capacity, device=DEV)}


def prepare(case, seed):
    op = case["op"]
    if op == "linear":
        q, scale, bias, x = _linear_inputs(case, seed)
        s = {"q": q, "scale": scale, "bias": bias, "x": x, "group": case["group"], "y": DTYPES[case["y"]]}
        if own:  # a program holds the layer, its weights laid out once
            quant, _ = _package()
            s["layer"] = quant.Int4Linear.from_quantized(q, scale, bias, case["group"])
            s["layer"].out_dtype = s["y"]
    elif op == "attend":
        s = _attend_inputs(case, seed)
        s["window"] = case["window"] or None
        if own:
            _, state = _package()
            s["buffer"] = state.DeviceKVBuffer(case["kv"], case["D"], case["slots"], s["window"], DEV, s["k"].dtype)
            s["buffer"].k, s["buffer"].v, s["buffer"].slot_pos = s["k"], s["v"], s["slot_pos"]
    elif op == "append":
        s = _append_inputs(case, seed)
        if own:
            _, state = _package()
            s["buffer"] = state.DeviceBudgetKVBuffer(case["kv"], case["D"], case["slots"], case["recent"], DEV, s["k"].dtype)
            for name in ("k", "v", "slot_pos", "weight", "end"):
                setattr(s["buffer"], name, s[name])
    else:
        s = _take_inputs(case, seed)
        if own:
            _, state = _package()
            s["from"] = state.DeviceKVBuffer(case["kv"], case["D"], case["slots"], None, DEV, s["k"].dtype)
            for name in ("k", "v", "slot_pos", "end"):
                setattr(s["from"], name, s[name])
            s["buffer"] = state.DeviceBudgetKVBuffer(case["kv"], case["D"], case["capacity"], case["recent"], DEV, s["k"].dtype)
            s["buffer"].k, s["buffer"].v = s["to_k"], s["to_v"]
            s["buffer"].slot_pos, s["buffer"].weight = s["to_pos"], s["to_weight"]
    s["op"] = op
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _plain_linear(s):
    q, group = s["q"], s["group"]
    w = q.float() * s["scale"].float().repeat_interleave(group, 1)[:, : q.shape[1]]
    y = torch.matmul(s["x"].float(), w.t())
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["y"])


def _plain_attend(s):
    q, k, v, q_pos, slot_pos, window = s["q"], s["k"], s["v"], s["q_pos"], s["slot_pos"], s["window"]
    T, H, D = q.shape
    slots, kv = k.shape[:2]
    see = (slot_pos >= 0) & (slot_pos <= q_pos[:, None])
    if window:
        see &= slot_pos > q_pos[:, None] - window
    k, v = k.float(), v.float()
    if s["tree"] is not None:
        new = s["tree"] & (q_pos > q_pos[:, None] - window) if window else s["tree"]
        see, k, v = torch.cat([see, new], 1), torch.cat([k, s["k_new"].float()]), torch.cat([v, s["v_new"].float()])
    # query head h reads kv head h // (H / kv)
    qh = q.float().view(T, kv, H // kv, D).permute(1, 2, 0, 3).reshape(kv, -1, D)
    score = torch.matmul(qh, k.permute(1, 2, 0).contiguous()).view(kv, H // kv, T, -1) * D ** -0.5
    score = score.masked_fill(~see, float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(kv, -1, p.shape[-1]), v.transpose(0, 1).contiguous())
    o = o.view(kv, H // kv, T, D).permute(2, 0, 1, 3).reshape(T, H, D).to(q.dtype)
    if s["weight"] is None:
        return o
    s["weight"] += p[..., :slots].sum((0, 1, 2))
    return o, s["weight"]


def _plain_order(s, newest):
    """The slots in the order in which they are given up: free ones, then by
    weight, the `recent` positions before `newest` last; ties by slot."""
    key = s["weight"].masked_fill(s["slot_pos"] >= newest - s["recent"], float("inf"))
    key = key.masked_fill(s["slot_pos"] < 0, float("-inf"))
    return torch.sort(key, stable=True).indices


def _plain_append(s):
    T = s["k_new"].shape[0]
    at = _plain_order(s, s["end"] + T)[:T].sort().values
    s["k"][at] = s["k_new"].to(s["k"].dtype)
    s["v"][at] = s["v_new"].to(s["v"].dtype)
    s["slot_pos"][at] = s["end"] + torch.arange(T, device=DEV)
    s["weight"][at] = 0.0
    s["end"] += T
    return {name: s[name] for name in ("k", "v", "slot_pos", "weight", "end")}


def _plain_take(s):
    n = s["to_pos"].shape[0]
    at = _plain_order(s, s["end"])[-n:].sort().values
    s["to_k"].copy_(s["k"][at])
    s["to_v"].copy_(s["v"][at])
    s["to_pos"].copy_(s["slot_pos"][at])
    s["to_weight"].copy_(s["weight"][at])
    return {name: s[name] for name in ("to_k", "to_v", "to_pos", "to_weight")}


def run(s):
    op = s["op"]
    if not own:
        return {"linear": _plain_linear, "attend": _plain_attend, "append": _plain_append, "take": _plain_take}[op](s)
    if op == "linear":
        return s["layer"](s["x"])
    b = s["buffer"]
    if op == "attend":
        o = b.attend(s["q"], s["q_pos"], s["k_new"], s["v_new"], s["tree"], weight=s["weight"])
        return o if s["weight"] is None else (o, s["weight"])
    if op == "append":
        b.append(s["k_new"], s["v_new"])
        return {name: s[name] for name in ("k", "v", "slot_pos", "weight", "end")}
    b.take(s["from"], s["weight"])
    return {name: s[name] for name in ("to_k", "to_v", "to_pos", "to_weight")}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        b = N * ((K + 1) // 2) + 2 * N * -(-K // case["group"]) + M * K * SIZES[case["x"]] + M * N * SIZES[case["y"]]
        return {"bytes": b + (4 * N if case.get("bias") else 0), "flops": 2 * M * N * K}
    row = case["kv"] * case["D"] * SIZES[case["cache"]]  # one token's keys
    if op == "attend":
        T, H, D, slots = case["T"], case["heads"], case["D"], case["slots"]
        held = min(slots, case["filled"], case["window"] + T if case["window"] else slots)  # what some query sees
        new = T if case["drafts"] else 0
        b = 2 * (held + new) * row + 8 * slots + 8 * T + new * T + 2 * T * H * D * SIZES[case["q"]]
        return {"bytes": b + (8 * held if case["weight"] else 0), "flops": 4 * T * H * D * (held + new)}
    if op == "append":
        T, slots = case["T"], case["slots"]
        new = 2 * T * case["kv"] * case["D"] * SIZES[case["new"]]
        return {"bytes": 12 * slots + new + T * (2 * row + 12), "flops": slots}
    return {"bytes": 12 * case["slots"] + case["capacity"] * (4 * row + 12), "flops": case["slots"]}


# ---------------------------------------------------------------------------
# the same results in 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _exact_linear(case, seed):
    q, scale, bias, x = _linear_inputs(case, seed)
    M, K, group = case["M"], case["K"], case["group"]
    y = torch.zeros(M, case["N"], dtype=torch.float64, device=DEV)
    for i, k0 in enumerate(range(0, K, group)):  # one group of columns at a time
        part = torch.matmul(x[:, k0:k0 + group].double(), q[:, k0:k0 + group].double().t().contiguous())
        y += part * scale[:, i].double()
    return y if bias is None else y + bias.double()


def _exact_attend(case, seed):
    s = _attend_inputs(case, seed)
    T, H, D, kv, slots = case["T"], case["heads"], case["D"], case["kv"], case["slots"]
    far = case["window"] or 1 << 60
    age = s["q_pos"][:, None] - s["slot_pos"][None, :]
    see = (s["slot_pos"][None, :] >= 0) & (age >= 0) & (age < far)
    k, v = s["k"], s["v"]
    if case["drafts"]:
        k, v = torch.cat([k, s["k_new"]]), torch.cat([v, s["v_new"]])
        see = torch.cat([see, s["tree"] & (s["q_pos"][:, None] - s["q_pos"][None, :] < far)], 1)
    o = torch.zeros(T, H, D, dtype=torch.float64, device=DEV)
    weight = torch.zeros(slots, dtype=torch.float64, device=DEV)
    for h in range(H):  # one head at a time
        kh, vh = (t[:, h // (H // kv)].double().contiguous() for t in (k, v))
        z = torch.matmul(s["q"][:, h].double(), kh.t().contiguous()) / D ** 0.5
        p = torch.softmax(torch.where(see, z, float("-inf")), -1)
        o[:, h] = torch.matmul(p, vh)
        weight += p[:, :slots].sum(0)
    return o if s["weight"] is None else (o, s["weight"].double() + weight)


def _exact_order(s, newest):
    pos, w = s["slot_pos"].cpu().numpy(), s["weight"].cpu().numpy()
    rank = np.where(pos < 0, 0, np.where(pos >= newest - s["recent"], 2, 1))
    return np.lexsort((np.arange(len(pos)), np.where(rank == 1, w, 0), rank))


def _exact_append(case, seed):
    s = _append_inputs(case, seed)
    T, end = case["T"], int(s["end"])
    at = np.sort(_exact_order(s, end + T)[:T])
    out = {"slot_pos": s["slot_pos"].cpu().numpy(), "weight": s["weight"].double().cpu().numpy(), "end": s["end"] + T}
    for name in ("k", "v"):
        t = s[name].double()
        for i, slot in enumerate(at):
            t[int(slot)] = s[name + "_new"][i].to(s[name].dtype).double()
        out[name] = t
    for i, slot in enumerate(at):
        out["slot_pos"][slot], out["weight"][slot] = end + i, 0.0
    return out


def _exact_take(case, seed):
    s = _take_inputs(case, seed)
    at = np.sort(_exact_order(s, case["filled"])[-case["capacity"]:])
    pick = torch.from_numpy(at).to(DEV)
    return {"to_k": s["k"].double()[pick], "to_v": s["v"].double()[pick], "to_pos": s["slot_pos"][pick],
            "to_weight": s["weight"].double()[pick]}


def exact(case, seed):
    return {"linear": _exact_linear, "attend": _exact_attend, "append": _exact_append, "take": _exact_take}[case["op"]](case, seed)
