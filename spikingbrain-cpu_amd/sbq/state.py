"""Device-resident decode state for the callers of the quantized linears.

The reference model keeps its inference state on the CPU (paths relative to
the reference repository):

* ``KVBuffer`` (model.py:61-85) grows CPU key / value tensors, or keeps the
  last ``window`` positions of a sliding-window layer;
* ``LayerState`` (model.py:94-97) adds a hybrid layer's shared [H, K, V] and
  partition [P, H, K, V] recurrent states;
* ``new_state`` (model.py:412-424) zero-initialises one of them per layer;
* ``forward_tokens`` builds the token ids as a CPU tensor (model.py:440) and
  the engine picks the next token on the CPU logits (engine.py:29-31).

With the linears on the GPU every projection then pays a host round trip.
The classes here hold the same state in HBM with fixed capacities: every
tensor keeps its address from step to step, positions are device tensors, a
key / value append is an ``index_copy_`` at slots computed on the device,
and which keys a query sees is given by the position each slot holds (a mask
for the attention) rather than by slicing.  A whole decode step, the token
feeding the next step included, can therefore be captured in a HIP graph and
replayed once per token with no host work in between.

For several sequences at once DevicePagedKVBuffer holds the keys and values in
pages of one pool, optionally in 8 bits.

Capacity: a full-attention buffer holds ``capacity`` positions (slot =
position).  A sliding-window buffer is a ring of ``capacity`` slots (slot =
position mod capacity); it must hold the window plus the tokens appended by
one call, so that no key a query of that call sees is overwritten.
"""
from __future__ import annotations

import functools
from dataclasses import dataclass, field

import torch

from . import _lib
from .quant import _DTYPE_CODE, _meet, _on_device, _reached, _span, _stream


def _as_pos(p, device: torch.device) -> torch.Tensor:
    if isinstance(p, torch.Tensor):
        return p.reshape(1).to(device=device, dtype=torch.long)
    return torch.tensor([int(p)], dtype=torch.long, device=device)


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """t [n, heads, dim] with unit stride in dim (else a contiguous copy)."""
    return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _within(t: torch.Tensor, storage: torch.Tensor) -> bool:
    """Does t begin inside the contiguous `storage`?"""
    at = t.data_ptr() - storage.data_ptr()
    return 0 <= at < storage.numel() * storage.element_size()


def attention_workspace(T: int, heads: int, kv_heads: int, dim: int, slots: int, weight: bool,
                        device: torch.device) -> torch.Tensor:
    """Scratch of tree_attention for these sizes (any content; one call at a time)."""
    n = _lib.load().sbq_attn_workspace_bytes(T, heads, kv_heads, dim, slots, int(weight))
    return torch.empty(n, dtype=torch.uint8, device=device)


def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slot_pos: torch.Tensor, q_pos: torch.Tensor,
                   k_new: torch.Tensor | None = None, v_new: torch.Tensor | None = None,
                   tree: torch.Tensor | None = None, window: int | None = None, scale: float | None = None,
                   weight: torch.Tensor | None = None, out: torch.Tensor | None = None,
                   workspace: torch.Tensor | None = None) -> torch.Tensor:
    """The attention of model.py:208-229 on the GPU for q [T, heads, dim] at
    positions q_pos [T] over a cache k, v [slots, kv_heads, dim] whose slots
    hold the positions slot_pos [slots] (-1: empty), and over the T tokens'
    own keys and values k_new, v_new [T, kv_heads, dim] where they are given:
    drafted tokens that are not in the cache, verified in one pass.  Query
    head h reads key head h // (heads / kv_heads).

    Token t sees a cached slot iff 0 <= slot_pos <= q_pos[t], and draft j iff
    tree[t, j] (bool [T, T], normally t's ancestors and itself; None: j <= t);
    with a window also only positions > q_pos[t] - window.  A row that sees
    nothing is 0; what a row does not see does not reach it.

    q has the cache's dtype or fp32 (then all products are fp32); the result
    has q's.  scale defaults to dim ** -0.5.  weight: fp32 [slots], to which
    the attention weight that each cached slot received, summed over tokens
    and heads, is added."""
    gpu, device = q.get_device(), q.device
    if gpu < 0:
        raise ValueError("tree_attention: q must be a GPU tensor")
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or k.shape[2] != q.shape[2]:
        raise ValueError("tree_attention: expected q [T, heads, dim] and k, v [slots, kv_heads, dim]")
    T, heads, dim = q.shape
    slots, kv_heads, _ = k.shape
    qt, ct = q.dtype, k.dtype
    if ct not in _DTYPE_CODE or v.dtype != ct or (qt != ct and qt != torch.float32):
        raise ValueError("tree_attention: k and v must share a dtype (float32, float16 or bfloat16), q have it or float32")
    if not 1 <= dim <= 256 or kv_heads < 1 or heads < 1 or heads % kv_heads or slots < 1:
        raise ValueError("tree_attention: 1 <= dim <= 256, heads a multiple of kv_heads, and slots >= 1")
    if T > _lib.SBQ_ATTN_MAX_T:
        raise ValueError(f"tree_attention: at most {_lib.SBQ_ATTN_MAX_T} tokens per call")
    ks = k.stride()
    if (k.get_device() != gpu or v.get_device() != gpu or (dim > 1 and ks[2] != 1)
            or (ks != v.stride() and any(n > 1 and a != b for n, a, b in zip(k.shape, ks, v.stride())))):
        raise ValueError(f"tree_attention: k and v must be on {q.device}, with the same strides and unit stride in dim")
    if (slot_pos.dtype != torch.int64 or slot_pos.get_device() != gpu or slot_pos.shape != (slots,)
            or not slot_pos.is_contiguous()):
        raise ValueError(f"tree_attention: slot_pos must be a contiguous int64 [{slots}] tensor on {q.device}")
    if q_pos.dtype != torch.int64 or q_pos.get_device() != gpu or q_pos.numel() != T or not q_pos.is_contiguous():
        raise ValueError(f"tree_attention: q_pos must be a contiguous int64 tensor of {T} positions on {q.device}")
    if window is not None and window < 1:
        raise ValueError("tree_attention: window must be >= 1")
    if (k_new is None) != (v_new is None) or (tree is not None and k_new is None):
        raise ValueError("tree_attention: k_new and v_new go together, and tree with them")
    if k_new is not None:
        if k_new.shape != (T, kv_heads, dim) or v_new.shape != k_new.shape or k_new.get_device() != gpu \
                or v_new.get_device() != gpu or k_new.dtype != k.dtype or v_new.dtype != k.dtype:
            raise ValueError(f"tree_attention: k_new and v_new must be {k.dtype} [T={T}, {kv_heads}, {dim}] on {q.device}")
        k_new, v_new = _rows_of(k_new), _rows_of(v_new)
        if k_new.stride() != v_new.stride():
            k_new, v_new = k_new.contiguous(), v_new.contiguous()
    if tree is not None:
        if tree.dtype not in (torch.bool, torch.uint8) or tree.shape != (T, T) or tree.get_device() != gpu:
            raise ValueError(f"tree_attention: tree must be a bool [T={T}, T] tensor on {q.device}")
        if not tree.is_contiguous():
            tree = tree.contiguous()
    if weight is not None and (weight.dtype != torch.float32 or weight.get_device() != gpu or weight.shape != (slots,)
                               or not weight.is_contiguous()):
        raise ValueError(f"tree_attention: weight must be a contiguous float32 [{slots}] tensor on {q.device}")
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(T, heads, dim, dtype=qt, device=device)
    elif out.shape != q.shape or out.dtype != qt or out.get_device() != gpu or (dim > 1 and out.stride(2) != 1):
        raise ValueError("tree_attention: out must have q's shape, dtype and device, with unit stride in dim")
    if T == 0:
        return out
    if out.data_ptr() == q.data_ptr():
        raise ValueError("tree_attention: out must not be q itself")
    q = _rows_of(q)
    if workspace is None:
        workspace = attention_workspace(T, heads, kv_heads, dim, slots, weight is not None, device)
    elif workspace.get_device() != gpu or not workspace.is_contiguous():
        raise ValueError(f"tree_attention: workspace must be a contiguous tensor on {q.device}")
    qs, os_ = q.stride(), out.stride()
    ns = (0, 0) if k_new is None else k_new.stride()
    with _on_device(device):
        _lib.check(_lib.load().sbq_tree_attention(
            q.data_ptr(), _DTYPE_CODE[qt], T, heads, dim, qs[0], qs[1], k.data_ptr(), v.data_ptr(), _DTYPE_CODE[ct], slots,
            kv_heads, ks[0], ks[1], slot_pos.data_ptr(), q_pos.data_ptr(),
            None if k_new is None else k_new.data_ptr(), None if v_new is None else v_new.data_ptr(), ns[0], ns[1],
            None if tree is None else tree.data_ptr(), T, window or 0, dim ** -0.5 if scale is None else scale,
            out.data_ptr(), os_[0], os_[1], None if weight is None else weight.data_ptr(), workspace.data_ptr(),
            workspace.numel() * workspace.element_size(), _stream(device)), "sbq_tree_attention")
    return out


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, inv_freq: torch.Tensor,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 interleaved: bool = False, q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The head norms and the rotation between the projections and the
    attention (model.py:260-270, rotary 46-51) in one pass: q [tokens, heads,
    dim] and k [tokens, kv_heads, dim] (or None) of one dtype, for instance
    views of a fused projection's output.  Every vector is divided by its root
    mean square (+ eps) and multiplied by q_weight / k_weight [dim] (None: no
    norm), then its first 2 * len(inv_freq) columns are rotated by position *
    inv_freq[i]: column i with i + len(inv_freq), or with `interleaved` 2i with
    2i + 1.  The angle is exact (the reference's fp32 product is not, far into
    a context), the rest fp32, rounded once.

    positions: int64 [n], tokens a multiple of n: token t stands at positions[t
    // (tokens / n)] + t % (tokens / n), so [tokens] gives each its own and the
    starts of n sequences are enough for their next tokens.  q_out, k_out: q and
    k themselves, or tensors apart from each other and every input (default: new
    ones)."""
    gpu, dtype, shape, device = q.get_device(), q.dtype, q.shape, q.device
    code, n, pairs = _DTYPE_CODE.get(dtype), positions.numel(), inv_freq.numel()
    wt = None if q_weight is None else q_weight.dtype
    if k_weight is not None:
        wt = k_weight.dtype if wt is None or wt is k_weight.dtype else False
    if gpu < 0 or code is None or len(shape) != 3 or not (
            positions.dtype is torch.int64 and positions.get_device() == gpu and positions.is_contiguous()
            and inv_freq.dtype is torch.float32 and inv_freq.get_device() == gpu and inv_freq.is_contiguous()
            and 2 * pairs <= shape[2] <= 256 and (shape[0] % n == 0 if n else shape[0] == 0)
            and (wt is None or wt in _DTYPE_CODE)
            and (q_weight is None or (q_weight.numel() == shape[2] and q_weight.get_device() == gpu and q_weight.is_contiguous()))
            and (k_weight is None or (k_weight.numel() == shape[2] and k_weight.get_device() == gpu and k_weight.is_contiguous()))):
        _refuse_rope(q, positions, inv_freq, q_weight, k_weight)
    tokens, heads, dim = shape
    qs = q.stride()
    if qs[2] != 1 and dim > 1:
        q = q.contiguous()
        qs = q.stride()
    given = q_out is not None or k_out is not None
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif q_out.shape != shape or q_out.dtype != dtype or q_out.get_device() != gpu or (dim > 1 and q_out.stride(2) != 1):
        raise ValueError("qk_norm_rope: q_out must have q's shape, dtype and device, with unit stride in dim")
    kv_heads = at_k = at_ko = 0
    ks = ko = (0, 0)
    if k is None:
        if k_out is not None:
            raise ValueError("qk_norm_rope: k_out needs k")
    else:
        kshape, ks = k.shape, k.stride()
        if len(kshape) != 3 or kshape[0] != tokens or kshape[2] != dim or k.dtype is not dtype or k.get_device() != gpu:
            raise ValueError("qk_norm_rope: expected q [tokens, heads, dim] and k [tokens, kv_heads, dim] of one dtype on one GPU")
        if ks[2] != 1 and dim > 1:
            k = k.contiguous()
            ks = k.stride()
        if k_out is None:
            k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        elif k_out.shape != kshape or k_out.dtype != dtype or k_out.get_device() != gpu or (dim > 1 and k_out.stride(2) != 1):
            raise ValueError("qk_norm_rope: k_out must have k's shape, dtype and device, with unit stride in dim")
        kv_heads, ko, at_k, at_ko = kshape[1], k_out.stride(), k.data_ptr(), k_out.data_ptr()
    if tokens == 0:
        return q_out, k_out
    if given and not (q_out is q and k_out is k and _plainly_apart(q, k, (positions, inv_freq, q_weight, k_weight))):
        _apart_rope(q, k, q_out, k_out, (positions, inv_freq, q_weight, k_weight))
    qo = q_out.stride()
    with _on_device(device):
        _lib.check(_lib.load().sbq_qk_norm_rope(
            q.data_ptr(), at_k, code, tokens, heads, kv_heads, dim, qs[0], qs[1], ks[0], ks[1], positions.data_ptr(), tokens // n,
            inv_freq.data_ptr(), pairs, interleaved, None if q_weight is None else q_weight.data_ptr(),
            None if k_weight is None else k_weight.data_ptr(), 0 if wt is None else _DTYPE_CODE[wt], eps, q_out.data_ptr(), at_ko,
            qo[0], qo[1], ko[0], ko[1], _stream(device)), "sbq_qk_norm_rope")
    return q_out, k_out


def _same_place(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Are a and b, of one shape and dtype, the same elements?"""
    return a.data_ptr() == b.data_ptr() and all(s == t for n, s, t in zip(a.shape, a.stride(), b.stride()) if n > 1)


def _plainly_apart(q: torch.Tensor, k: torch.Tensor | None, others) -> bool:
    """Are q and k, written in place, heads of one projection's rows, and the
    others elsewhere?  (The quick answer for what a step does every time.)"""
    lo, (tokens, heads, dim), (st, sh, _), size = q.data_ptr(), q.shape, q.stride(), q.element_size()
    step, of_q = st * size, ((heads - 1) * sh + dim) * size
    hi = lo + (tokens - 1) * step + of_q
    if k is not None:
        at, (kt, kh, _) = k.data_ptr() - lo, k.stride()
        of_k = ((k.shape[1] - 1) * kh + dim) * size
        if kt != st or not of_q <= at <= step - of_k:
            return False
        hi += at + of_k - of_q
    for t in others:
        if t is not None and lo - 8 * t.numel() < t.data_ptr() < hi:
            return False
    return True


def _apart_rope(q, k, q_out, k_out, others) -> None:
    """Refuses outputs that are neither an input nor apart from everything."""
    in_q, in_k = _same_place(q, q_out), k is not None and _same_place(k, k_out)
    pairs = [] if in_q else [(q_out, q)]
    if k is not None:
        pairs += [(q_out, k_out)] + ([] if in_k else [(k_out, k), (q_out, k)]) + ([] if in_q else [(k_out, q)])
    outs = [_span(t) for t in (q_out, k_out) if t is not None]
    spans = [_span(t) for t in others if t is not None]
    if any(_meet(a, b) for a, b in pairs) or any(a[0] < b[1] and b[0] < a[1] for a in outs for b in spans):
        raise ValueError("qk_norm_rope: q_out and k_out must be q and k themselves, or apart from each other and every input")


def _refuse_rope(q, positions, inv_freq, q_weight, k_weight):
    """The reason why qk_norm_rope does not take these."""
    if not q.is_cuda:
        raise ValueError("qk_norm_rope: q must be a GPU tensor")
    if q.dtype not in _DTYPE_CODE:
        raise ValueError(f"qk_norm_rope: unsupported dtype {q.dtype}; expected float32, float16 or bfloat16")
    if q.dim() != 3:
        raise ValueError("qk_norm_rope: expected q [tokens, heads, dim] and k [tokens, kv_heads, dim] of one dtype on one GPU")
    tokens, _, dim = q.shape
    n = positions.numel()
    if positions.dtype != torch.int64 or positions.device != q.device or not positions.is_contiguous() \
            or (tokens % n if n else tokens):
        raise ValueError(f"qk_norm_rope: positions must be a contiguous int64 tensor on {q.device} whose size divides {tokens} "
                         "tokens")
    if (inv_freq.dtype != torch.float32 or inv_freq.device != q.device or not inv_freq.is_contiguous()
            or 2 * inv_freq.numel() > dim or dim > 256):
        raise ValueError(f"qk_norm_rope: inv_freq must be a contiguous float32 tensor on {q.device} of at most dim / 2 entries, "
                         "dim at most 256")
    raise ValueError(f"qk_norm_rope: weights must be contiguous [{dim}] tensors of one float dtype on {q.device}")


class DeviceKVBuffer:
    """model.py:61-85 KVBuffer with its storage in device memory.

    ``append(k, v)`` stores [T, heads, dim] keys / values at the positions
    ``end .. end + T - 1`` and returns ``(keys, values, slot_pos)``: the whole
    storage [slots, heads, dim] and the position each slot holds (-1 for an
    empty slot).  ``visible(q_pos)`` is the attention mask of queries at
    positions ``q_pos`` [T]: the slots holding a position <= the query's
    and, for a window, > the query's position - window, which are the keys the
    reference's ``append`` returns together with the mask its ``attention``
    (model.py:208-229) applies to them."""

    def __init__(self, heads: int, dim: int, capacity: int, window: int | None = None,
                 device: torch.device | str | None = None, dtype: torch.dtype = torch.float32):
        if capacity < 1 or (window is not None and (window < 1 or capacity < window + 1)):
            raise ValueError("DeviceKVBuffer: capacity must be >= 1, and >= window + 1 for a window")
        self.heads, self.dim, self.window, self.capacity = heads, dim, window, capacity
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.k = torch.zeros(capacity, heads, dim, dtype=dtype, device=dev)
        self.v = torch.zeros(capacity, heads, dim, dtype=dtype, device=dev)
        self.slot_pos = torch.full((capacity,), -1, dtype=torch.long, device=dev)
        self.end = torch.zeros((1,), dtype=torch.long, device=dev)  # next position to write

    @property
    def device(self) -> torch.device:
        return self.k.device

    def reset(self) -> None:
        self.k.zero_()
        self.v.zero_()
        self.slot_pos.fill_(-1)
        self.end.zero_()

    def append(self, k: torch.Tensor, v: torch.Tensor, start=None):
        """Store k, v [T, heads, dim] at positions start .. start + T - 1
        (default: after the last append); start may be an int or a device
        tensor (graph capture).  With a window, T must be <= capacity -
        window (the ring keeps every key the new queries see)."""
        T = k.shape[0]
        if tuple(k.shape[1:]) != (self.heads, self.dim) or k.shape != v.shape:
            raise ValueError(f"DeviceKVBuffer.append: expected [T, {self.heads}, {self.dim}] keys and values")
        if self.window is not None and T > self.capacity - self.window:
            raise ValueError("DeviceKVBuffer.append: more tokens than the ring holds beside the window")
        s = self.end if start is None else _as_pos(start, self.device)
        pos = s + torch.arange(T, device=self.device)
        slots = pos % self.capacity if self.window is not None else pos
        self.k.index_copy_(0, slots, k.to(self.k.dtype))
        self.v.index_copy_(0, slots, v.to(self.v.dtype))
        self.slot_pos.index_copy_(0, slots, pos)
        self.end.copy_(s + T)
        return self.k, self.v, self.slot_pos

    def visible(self, q_pos: torch.Tensor) -> torch.Tensor:
        """Boolean [T, slots]: which stored keys queries at q_pos [T] attend to."""
        kp = self.slot_pos[None, :]
        qp = q_pos.reshape(-1, 1)
        ok = (kp >= 0) & (kp <= qp)
        if self.window is not None:
            ok &= kp > qp - self.window
        return ok

    def attend(self, q: torch.Tensor, q_pos: torch.Tensor, k_new: torch.Tensor | None = None,
               v_new: torch.Tensor | None = None, tree: torch.Tensor | None = None, scale: float | None = None,
               weight: torch.Tensor | None = None, out: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None) -> torch.Tensor:
        """The attention of queries q [T, heads, dim] at positions q_pos [T]
        over the stored keys that visible(q_pos) names and, for a tree of
        drafted tokens, over their own k_new, v_new [T, self.heads, dim] by
        tree [T, T]; see tree_attention.  Drafts are not stored: append the
        accepted ones.  A whole call can be captured in a HIP graph."""
        return tree_attention(q, self.k, self.v, self.slot_pos, q_pos, k_new, v_new, tree, self.window, scale, weight,
                              out, workspace)

    def truncate(self, length) -> None:
        """Forget positions >= length (the engine's prefix reuse restores a
        shorter length, model.py:119-127); length may be a device tensor."""
        n = _as_pos(length, self.device)
        self.slot_pos.masked_fill_(self.slot_pos >= n, -1)
        self.end.copy_(torch.minimum(self.end, n))


class DeviceBudgetKVBuffer(DeviceKVBuffer):
    """A full-attention buffer of `capacity` slots for more positions than
    that: once it is full, an append takes the slots which received the least
    attention weight so far, the `recent` newest positions (the appended ones
    among them) last.  `weight` [capacity] holds the running sums, which
    attend adds to; a new token starts at 0.  No counterpart in the reference,
    whose softmax layers keep every position.

    GPU only (attend and append are kernels of libsbq.so).  Every tensor keeps
    its address, so append and attend can be captured in a HIP graph."""

    def __init__(self, heads: int, dim: int, capacity: int, recent: int = 0, device: torch.device | str | None = None,
                 dtype: torch.dtype = torch.float32):
        if not 0 <= recent <= capacity:
            raise ValueError("DeviceBudgetKVBuffer: recent must be between 0 and capacity")
        super().__init__(heads, dim, capacity, None, device, dtype)
        self.recent = recent
        self.weight = torch.zeros(capacity, dtype=torch.float32, device=self.k.device)

    def reset(self) -> None:
        super().reset()
        self.weight.zero_()

    def append(self, k: torch.Tensor, v: torch.Tensor, start=None):
        """Store k, v [T, heads, dim] at positions start .. start + T - 1
        (default: after the last append), T <= capacity; start may be an int
        or a device tensor.  Free slots are taken first, then those of least
        weight (equal ones by slot), in ascending slot order.  Going back to an
        earlier start, truncate(start) first: positions from start on that the
        buffer holds would stay beside the new ones (and count as newest)."""
        kv = self.k
        gpu = kv.get_device()
        if k.shape != v.shape or k.dim() != 3 or k.shape[1] != self.heads or k.shape[2] != self.dim:
            raise ValueError(f"DeviceBudgetKVBuffer.append: expected [T, {self.heads}, {self.dim}] keys and values")
        T = k.shape[0]
        if T > self.capacity:
            raise ValueError("DeviceBudgetKVBuffer.append: more tokens than slots")
        if not kv.is_cuda or k.get_device() != gpu or v.get_device() != gpu:
            raise ValueError("DeviceBudgetKVBuffer.append: the buffer, k and v must be on one GPU")
        if T == 0:
            if start is not None:
                self.end.copy_(_as_pos(start, kv.device))
            return kv, self.v, self.slot_pos
        if k.dtype not in _DTYPE_CODE or v.dtype != k.dtype:
            k, v = k.to(kv.dtype), v.to(kv.dtype)
        k, v = _rows_of(k), _rows_of(v)
        if k.stride() != v.stride():
            k, v = k.contiguous(), v.contiguous()
        if T > 1 and (_within(k, kv) or _within(k, self.v) or _within(v, kv) or _within(v, self.v)):
            k, v = k.clone(), v.clone()  # rows of the cache itself would be overwritten as they are read
        s = self.end if start is None else _as_pos(start, kv.device)
        L = _lib.load()
        ws = torch.empty(L.sbq_kv_workspace_bytes(self.capacity, T), dtype=torch.uint8, device=kv.device)
        ks, ns = kv.stride(), k.stride()
        with _on_device(kv.device):
            _lib.check(L.sbq_kv_append(
                self.slot_pos.data_ptr(), self.weight.data_ptr(), self.capacity, self.end.data_ptr(), s.data_ptr(),
                self.recent, kv.data_ptr(), self.v.data_ptr(), _DTYPE_CODE[kv.dtype], self.heads, self.dim, ks[0], ks[1],
                k.data_ptr(), v.data_ptr(), _DTYPE_CODE[k.dtype], T, ns[0], ns[1], ws.data_ptr(), ws.numel(),
                _stream(kv.device)), "sbq_kv_append")
        return kv, self.v, self.slot_pos

    def take(self, source: DeviceKVBuffer, weight: torch.Tensor | None = None):
        """Become what is worth keeping of `source` (after a long prompt): its
        slots in the order of append's rule, the last `capacity` of them kept
        in slot order with their positions and weights.  weight: fp32, one per
        slot of source (default: source.weight); end becomes source.end."""
        kv = self.k
        if weight is None:
            weight = getattr(source, "weight", None)
        if source is self or not kv.is_cuda or source.k.device != kv.device:
            raise ValueError("DeviceBudgetKVBuffer.take: source must be another buffer on this buffer's GPU")
        if source.k.shape[1:] != kv.shape[1:] or source.k.dtype != kv.dtype:
            raise ValueError("DeviceBudgetKVBuffer.take: source must have this buffer's heads, dim and dtype")
        if (weight is None or weight.dtype != torch.float32 or weight.device != kv.device
                or weight.shape != (source.capacity,) or not weight.is_contiguous()):
            raise ValueError(f"DeviceBudgetKVBuffer.take: weight must be a contiguous float32 [{source.capacity}] tensor on "
                             f"{kv.device}")
        if _within(weight, self.weight) or _within(self.weight, weight):
            raise ValueError("DeviceBudgetKVBuffer.take: weight must not be this buffer's own")
        L = _lib.load()
        ws = torch.empty(L.sbq_kv_workspace_bytes(source.capacity, self.capacity), dtype=torch.uint8, device=kv.device)
        ks, ts = source.k.stride(), kv.stride()
        with _on_device(kv.device):
            _lib.check(L.sbq_kv_take(
                source.slot_pos.data_ptr(), weight.data_ptr(), source.capacity, source.end.data_ptr(), source.k.data_ptr(),
                source.v.data_ptr(), _DTYPE_CODE[kv.dtype], self.heads, self.dim, ks[0], ks[1], self.capacity, self.recent,
                self.slot_pos.data_ptr(), self.weight.data_ptr(), self.end.data_ptr(), kv.data_ptr(), self.v.data_ptr(),
                ts[0], ts[1], ws.data_ptr(), ws.numel(), _stream(kv.device)), "sbq_kv_take")
        return kv, self.v, self.slot_pos

    def attend(self, q: torch.Tensor, q_pos: torch.Tensor, k_new: torch.Tensor | None = None,
               v_new: torch.Tensor | None = None, tree: torch.Tensor | None = None, scale: float | None = None,
               weight: torch.Tensor | None = None, out: torch.Tensor | None = None,
               workspace: torch.Tensor | None = None, count: bool = True) -> torch.Tensor:
        """DeviceKVBuffer.attend, which also adds the attention weight that
        every slot received to `weight` (this buffer's own by default; count
        False: nowhere).  All T query rows count, drafts that are rejected
        later among them."""
        if weight is None and count:
            weight = self.weight
        return super().attend(q, q_pos, k_new, v_new, tree, scale, weight, out, workspace)

    def truncate(self, length) -> None:
        super().truncate(length)
        self.weight.masked_fill_(self.slot_pos < 0, 0.0)


_CACHE_CODE = {**_DTYPE_CODE, torch.int8: _lib.SBQ_I8, torch.float8_e4m3fn: _lib.SBQ_E4M3}


@functools.lru_cache(maxsize=256)
def _paged_workspace_bytes(*sizes: int) -> int:
    return _lib.load().sbq_paged_attn_workspace_bytes(*sizes)


class DevicePagedKVBuffer:
    """Keys and values of several sequences in pages of one pool, for a step
    that runs all of them at once.  No counterpart in the reference, whose
    engine holds one sequence.

    dtype: float32, float16 or bfloat16, or int8 or float8_e4m3fn: then a
    token's keys (values) of a head are kept as 8-bit codes and one fp32 scale,
    max |x| / 127 or / 448, as they are written, and multiplied out as they are
    read.  The pool is k, v [pages, heads, page, dim] (rows padded to 16
    columns in memory; k_scale, v_scale [pages, heads, page]).  Sequence b's
    position p stands in page table[b, p // page] (int32 [sequences,
    max_pages], -1: none), row p % page, and length [sequences] (int64) is how
    many positions it holds.

    The host gives pages out: reserve(sequence, length) before an append that
    reaches so far, release(sequence) when it is done.  append, attend, read
    and truncate find everything else on the device and keep every address, so
    a step can be captured in a HIP graph, and replayed for as long as its
    tokens fit what is reserved.  What an append finds no page for is dropped,
    counted in the length all the same up to max_pages * page positions: reserve
    first.  GPU only."""

    def __init__(self, sequences: int, heads: int, dim: int, pages: int, page: int = 64, max_pages: int | None = None,
                 window: int | None = None, device: torch.device | str | None = None, dtype: torch.dtype = torch.float32):
        max_pages = pages if max_pages is None else max_pages
        if dtype not in _CACHE_CODE:
            raise ValueError(f"DevicePagedKVBuffer: unsupported dtype {dtype}; expected float32, float16, bfloat16, int8 or "
                             "float8_e4m3fn")
        if not 1 <= sequences <= 65536 or not 1 <= heads <= 65536 or not 1 <= dim <= 256 or not 1 <= pages <= 1 << 30:
            raise ValueError("DevicePagedKVBuffer: 1 to 65536 sequences and heads, a dim of at most 256, and pages >= 1")
        if page not in (16, 32, 64, 128, 256, 512, 1024) or max_pages < 1 or max_pages * page > 1 << 30:
            raise ValueError("DevicePagedKVBuffer: page must be a power of two from 16 to 1024, and max_pages * page at most 2^30")
        if window is not None and not 1 <= window < 1 << 62:
            raise ValueError("DevicePagedKVBuffer: window must be 1 to 2^62 - 1")
        self.sequences, self.heads, self.dim, self.page, self.window = sequences, heads, dim, page, window
        self._tensors: dict[str, torch.Tensor | None] = {}
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        row, b8 = -(-dim // 16) * 16, dtype in (torch.int8, torch.float8_e4m3fn)
        self.k = torch.zeros(pages, heads, page, row, dtype=dtype, device=dev)[..., :dim]
        self.v = torch.zeros(pages, heads, page, row, dtype=dtype, device=dev)[..., :dim]
        self.k_scale = torch.zeros(pages, heads, page, device=dev) if b8 else None
        self.v_scale = torch.zeros(pages, heads, page, device=dev) if b8 else None
        self.table = torch.full((sequences, max_pages), -1, dtype=torch.int32, device=dev)
        self.length = torch.zeros(sequences, dtype=torch.long, device=dev)
        self._free = list(range(pages - 1, -1, -1))
        self._held: list[dict[int, int]] = [{} for _ in range(sequences)]  # page of the sequence -> page of the pool
        self._first = [0] * sequences  # pages of the sequence before this one were given back

    # The pool's tensors may be replaced (a caller's own memory, its columns from dim on 0 and e4m3 codes
    # finite throughout); they are checked when that happens.
    k = property(lambda self: self._tensors["k"], lambda self, t: self._replace("k", t))
    v = property(lambda self: self._tensors["v"], lambda self, t: self._replace("v", t))
    k_scale = property(lambda self: self._tensors["k_scale"], lambda self, t: self._replace("k_scale", t))
    v_scale = property(lambda self: self._tensors["v_scale"], lambda self, t: self._replace("v_scale", t))
    table = property(lambda self: self._tensors["table"], lambda self, t: self._replace("table", t))
    length = property(lambda self: self._tensors["length"], lambda self, t: self._replace("length", t))

    def _replace(self, name: str, t: torch.Tensor | None) -> None:
        self._tensors[name] = t
        self._sizes = None  # to be checked again

    @property
    def device(self) -> torch.device:
        return self.k.device

    def _row(self, fn: str, sequence: int) -> int:
        if not 0 <= sequence < self.sequences:
            raise ValueError(f"DevicePagedKVBuffer.{fn}: sequence must be 0 .. {self.sequences - 1}")
        return sequence

    def reserve(self, sequence: int, length: int) -> None:
        """Give `sequence` the pages that positions below `length` need and it
        does not have, but for those that release(before) took back.  All or none
        of them: ValueError if the table's row is too short or all of them were
        taken back, RuntimeError if the pool has too few free pages."""
        held = self._held[self._row("reserve", sequence)]
        last = -(-length // self.page)
        if last > self.table.shape[1]:
            raise ValueError(f"DevicePagedKVBuffer.reserve: {length} positions are more than the table's row holds")
        if 0 < last <= self._first[sequence]:
            raise ValueError(f"DevicePagedKVBuffer.reserve: the pages of the first {self._first[sequence] * self.page} positions "
                             "were released")
        want = [i for i in range(self._first[sequence], last) if i not in held]
        if len(want) > len(self._free):
            raise RuntimeError(f"DevicePagedKVBuffer.reserve: {len(want)} pages wanted, {len(self._free)} free")
        if not want:
            return
        for i in want:
            held[i] = self._free.pop()
        # (what is held lies side by side from the first page not given back)
        self.table[sequence, want[0]:want[-1] + 1] = torch.tensor([held[i] for i in range(want[0], want[-1] + 1)],
                                                                  dtype=torch.int32, device=self.device)

    def release(self, sequence: int, before: int | None = None) -> None:
        """Take the sequence's pages back and forget its positions; with
        `before` only the pages that end at or below that position (which a
        window has left behind): nothing is stored there again before the whole
        sequence is released or truncated to 0."""
        held = self._held[self._row("release", sequence)]
        first = self.table.shape[1] if before is None else max(0, before // self.page)
        for i in [i for i in held if i < first]:
            self._free.append(held.pop(i))
        if before is None:
            self._first[sequence] = 0
            self.table[sequence] = -1
            self.length[sequence] = 0
        else:
            self._first[sequence] = max(self._first[sequence], first)
            self.table[sequence, :first] = -1

    def reset(self) -> None:
        for i in range(self.sequences):
            self._held[i].clear()
            self._first[i] = 0
        self._free = list(range(self.k.shape[0] - 1, -1, -1))
        self.table.fill_(-1)
        self.length.zero_()

    def _check(self) -> tuple:
        """(cache type, pages, page, heads, dim, max_pages) of the pool, once its tensors fit each other."""
        k, v, table, length = self.k, self.v, self.table, self.length
        dev, code, n = k.device, _CACHE_CODE.get(k.dtype), self.sequences
        row = -(-self.dim // 16) * 16
        strides = (self.heads * self.page * row, self.page * row, row)
        if not k.is_cuda:
            raise ValueError("DevicePagedKVBuffer: the buffer must be on a GPU")
        if code is None or k.dim() != 4 or any(
                t.shape != k.shape or t.shape[1:] != (self.heads, self.page, self.dim) or t.dtype != k.dtype or t.device != dev
                or t.stride()[:3] != strides or (self.dim > 1 and t.stride(3) != 1) for t in (k, v)):
            raise ValueError(f"DevicePagedKVBuffer: k and v must be [pages, {self.heads}, {self.page}, {self.dim}] of one cache "
                             f"dtype, in rows of {row}, on one GPU")
        if code >= _lib.SBQ_I8:
            for s in (self.k_scale, self.v_scale):
                if s is None or s.dtype != torch.float32 or s.shape != k.shape[:3] or s.device != dev or not s.is_contiguous():
                    raise ValueError("DevicePagedKVBuffer: k_scale and v_scale must be contiguous float32 [pages, heads, page]")
        if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != n or not table.is_contiguous() \
                or table.device != dev or length.dtype != torch.int64 or length.shape != (n,) \
                or not length.is_contiguous() or length.device != dev:
            raise ValueError(f"DevicePagedKVBuffer: table must be int32 [{n}, max_pages] and length int64 [{n}], contiguous")
        self._sizes = (code, k.shape[0], self.page, self.heads, self.dim, table.shape[1])
        self._dev, self._gpu, self._b8 = dev, k.get_device(), code >= _lib.SBQ_I8
        self._bytes = k.shape[0] * strides[0] * k.element_size()
        self._spans = [_span(t) for t in self._tensors.values() if t is not None]
        return self._sizes

    def _cache(self, fn: str, sequence: int | None) -> tuple:
        """The C ABI's description of the cache (of one sequence's row), from k to length."""
        code, pages, page, heads, dim, width = self._sizes or self._check()
        t, at = self._tensors, 0 if sequence is None else self._row(fn, sequence)
        ks, vs = (t["k_scale"].data_ptr(), t["v_scale"].data_ptr()) if self._b8 else (None, None)
        return (t["k"].data_ptr(), t["v"].data_ptr(), ks, vs, code, pages, page, heads, dim,
                t["table"].data_ptr() + 4 * width * at, self.sequences if sequence is None else 1, width,
                t["length"].data_ptr() + 8 * at)

    def _not_released(self, fn: str, position: int, sequence: int | None) -> None:
        """No page from `position` on was released."""
        first = max(self._first) if sequence is None else self._first[sequence]
        if first and position < first * self.page:
            raise ValueError(f"DevicePagedKVBuffer.{fn}: the pages of the first {first * self.page} positions were released")

    def _places(self, fn: str, name: str, t, n: int) -> torch.Tensor:
        """int64 [n] on the device; an int for every sequence."""
        if not isinstance(t, torch.Tensor):
            return torch.full((n,), int(t), dtype=torch.long, device=self.device)
        if t.dtype is not torch.int64 or t.numel() != n or t.get_device() != self._tensors["length"].get_device() \
                or not t.is_contiguous():
            raise ValueError(f"DevicePagedKVBuffer.{fn}: {name} must be a contiguous int64 tensor of {n} on {self.device}")
        return t

    def append(self, k: torch.Tensor, v: torch.Tensor, start=None, counts: torch.Tensor | None = None,
               sequence: int | None = None) -> None:
        """Store k, v [sequences, T, heads, dim] at each sequence's positions
        start .. start + T - 1 (default: after those it holds; an int or int64
        [sequences]), the first counts[b] of them where counts (int64
        [sequences]) is given; length becomes start + counts (0, and nothing is
        stored, for a start below 0).  With `sequence` k, v [T, heads, dim] go
        to that one alone, and start and counts are of one entry."""
        cache = self._cache("append", sequence)
        n, heads, dim, shape = cache[10], self.heads, self.dim, k.shape
        if sequence is None:
            if len(shape) != 4 or shape[0] != n or shape[2] != heads or shape[3] != dim or v.shape != shape:
                raise ValueError(f"DevicePagedKVBuffer.append: expected [{n}, T, {heads}, {dim}] keys and values")
        else:
            if len(shape) != 3 or shape[1] != heads or shape[2] != dim or v.shape != shape:
                raise ValueError(f"DevicePagedKVBuffer.append: expected [T, {heads}, {dim}] keys and values")
            k, v = k[None], v[None]
        gpu = self._gpu
        if k.get_device() != gpu or v.get_device() != gpu:
            raise ValueError(f"DevicePagedKVBuffer.append: keys and values must be on {self.device}")
        code = _DTYPE_CODE.get(k.dtype)
        if code is None or v.dtype != k.dtype:
            k, v, code = k.float(), v.float(), _lib.SBQ_F32
        st = k.stride()
        if (st[3] != 1 and dim > 1) or st != v.stride():
            k, v = k.contiguous(), v.contiguous()
            st = k.stride()
        at_k, at_v = k.data_ptr(), v.data_ptr()
        pool_k, pool_v, room, length = cache[0], cache[1], self._bytes, cache[12]
        if 0 <= at_k - pool_k < room or 0 <= at_k - pool_v < room or 0 <= at_v - pool_k < room or 0 <= at_v - pool_v < room:
            # (rows of the pool itself: they would be overwritten as they are read)
            k, v = k.clone(memory_format=torch.contiguous_format), v.clone(memory_format=torch.contiguous_format)
            at_k, at_v, st = k.data_ptr(), v.data_ptr(), k.stride()
        at = length
        if start is not None:
            if not isinstance(start, torch.Tensor):
                self._not_released("append", start, sequence)
            start = self._places("append", "start", start, n)
            at = start.data_ptr()
            if at != length and abs(at - length) < 8 * n:  # (other sequences' lengths, which this call moves)
                start = start.clone()
                at = start.data_ptr()
        at_counts = None
        if counts is not None:
            counts = self._places("append", "counts", counts, n)
            if abs(counts.data_ptr() - length) < 8 * n:
                counts = counts.clone()
            at_counts = counts.data_ptr()
        dev = self._dev
        with _on_device(dev):
            _lib.check(_lib.load().sbq_paged_append(*cache, at, at_counts, at_k, at_v, code, k.shape[1], st[0], st[1], st[2],
                                                    _stream(dev)), "sbq_paged_append")

    def read(self, start, count: int, dtype: torch.dtype | None = None,
             sequence: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values [sequences, count, heads, dim] of the positions from
        start (an int or int64 [sequences]) on, multiplied out and rounded to
        dtype (default: the pool's, float32 for 8 bits); positions that a
        sequence does not hold are 0.  With `sequence` [count, heads, dim] of
        that one."""
        cache = self._cache("read", sequence)
        n = cache[10]
        if dtype is None:
            dtype = self.k.dtype if self.k.dtype in _DTYPE_CODE else torch.float32
        if dtype not in _DTYPE_CODE or count < 0:
            raise ValueError("DevicePagedKVBuffer.read: dtype must be float32, float16 or bfloat16, and count >= 0")
        start = self._places("read", "start", start, n)
        heads, dim, dev = self.heads, self.dim, self._dev
        shape = (n, count, heads, dim) if sequence is None else (count, heads, dim)
        k = torch.empty(shape, dtype=dtype, device=dev)
        v = torch.empty_like(k)
        with _on_device(dev):
            _lib.check(_lib.load().sbq_paged_read(*cache, start.data_ptr(), count, k.data_ptr(), v.data_ptr(), _DTYPE_CODE[dtype],
                                                  count * heads * dim, heads * dim, dim, _stream(dev)), "sbq_paged_read")
        return k, v

    def _query(self, fn: str, q: torch.Tensor) -> int:
        """The C ABI's type of queries that attend takes."""
        n, kv_heads, shape = self.sequences, self.heads, q.shape
        if len(shape) not in (3, 4) or shape[0] != n or shape[-1] != self.dim or shape[-2] % kv_heads or shape[-2] == 0:
            raise ValueError(f"DevicePagedKVBuffer.{fn}: expected q [{n}, T, heads, {self.dim}], heads a multiple of {kv_heads}")
        if len(shape) == 4 and shape[1] > _lib.SBQ_PAGED_MAX_T:
            raise ValueError(f"DevicePagedKVBuffer.{fn}: at most {_lib.SBQ_PAGED_MAX_T} tokens per call")
        code = _DTYPE_CODE.get(q.dtype)
        if q.get_device() != self._gpu or code is None or not (self._b8 or code in (self._sizes[0], _lib.SBQ_F32)):
            raise ValueError(f"DevicePagedKVBuffer.{fn}: q must be on {self.device}, of the pool's dtype or float32 (8-bit pools: "
                             "float32, float16 or bfloat16)")
        return code

    def attend(self, q: torch.Tensor, start=None, counts: torch.Tensor | None = None, scale: float | None = None,
               out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
        """The attention of q [sequences, T, q heads, dim] (or [sequences, q
        heads, dim], one token each) over each sequence's positions: token t,
        at start + t, sees those held up to its own, with a window only the
        last `window` of them.  start (an int or int64 [sequences]) defaults to
        the tokens appended last: length - counts, counts (int64 [sequences],
        default T) being how many of the T are there; the others' rows are 0,
        as is a row that sees nothing.  Query head h reads key head h // (q
        heads / heads).  q has the pool's dtype or float32 (8-bit pools: any);
        the result has q's.  out and workspace lie apart from everything else."""
        cache = self._cache("attend", None)
        n, gpu, dim, kv_heads, dev, shape = cache[10], self._gpu, self.dim, self.heads, self._dev, q.shape
        code = self._query("attend", q)
        given, room_given = out is not None, workspace is not None
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != shape or out.dtype != q.dtype or out.get_device() != gpu or (dim > 1 and out.stride(-1) != 1):
            raise ValueError("DevicePagedKVBuffer.attend: out must have q's shape, dtype and device, with unit stride in dim")
        T, heads = shape[1] if len(shape) == 4 else 1, shape[-2]
        if T == 0:
            return out
        if dim > 1 and q.stride(-1) != 1:
            q = q.contiguous()
        room, window = 0, self.window or 0
        if workspace is None:
            room = _paged_workspace_bytes(n, T, heads, kv_heads, dim, self.page, cache[11], window, cache[4])
            if room:
                workspace = torch.empty(room, dtype=torch.uint8, device=dev)
        elif workspace.get_device() != gpu or not workspace.is_contiguous():
            raise ValueError(f"DevicePagedKVBuffer.attend: workspace must be a contiguous tensor on {dev}")
        else:
            room = workspace.numel() * workspace.element_size()
        if start is not None:
            start = self._places("attend", "start", start, n)
        if counts is not None:
            counts = self._places("attend", "counts", counts, n)
        if given or room_given:
            self._apart(out if given else None, workspace if room_given else None, q, start, counts)
        qs, os_ = q.stride(), out.stride()
        with _on_device(dev):
            _lib.check(_lib.load().sbq_paged_attention(
                q.data_ptr(), code, T, heads, qs[0], qs[-3], qs[-2], *cache, None if start is None else start.data_ptr(),
                None if counts is None else counts.data_ptr(), window, dim ** -0.5 if scale is None else scale,
                out.data_ptr(), os_[0], os_[-3], os_[-2], workspace.data_ptr() if room else None, room, _stream(dev)),
                "sbq_paged_attention")
        return out

    def _apart(self, out, workspace, q, start, counts) -> None:
        """Refuses an output or a workspace of attend that meets the other, an input or the buffer."""
        for t in (out, workspace):
            if t is not None:
                lo, hi = _span(t)
                if any(lo < b and a < hi for a, b in self._spans):
                    break
        else:
            if (out is None or not (_meet(out, q) or any(t is not None and _meet(out, t) for t in (start, counts)))) \
                    and (workspace is None or not _reached(workspace, (q, out, start, counts))):
                return
        raise ValueError("DevicePagedKVBuffer.attend: out and workspace must lie apart from each other, the inputs and the buffer")

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, inv_freq: torch.Tensor,
             q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
             interleaved: bool = False, counts: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
        """What stands between a softmax layer's projections (model.py:260-270)
        for the next T tokens of every sequence: q [sequences, T, q heads, dim]
        and k, v [sequences, T, heads, dim] as projected; norms and rotation at
        the sequences' next positions (qk_norm_rope), append, attend."""
        if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[0] != self.sequences:
            raise ValueError(f"DevicePagedKVBuffer.step: expected q [{self.sequences}, T, q heads, dim] and k, v "
                             f"[{self.sequences}, T, heads, dim]")
        if v.shape != k.shape or v.get_device() != k.get_device():
            raise ValueError(f"DevicePagedKVBuffer.step: v must have k's shape, and be on {self.device}")
        self._cache("step", None)
        self._query("step", q)  # (refused before anything is stored)
        if scale is not None and scale != scale:
            raise ValueError("DevicePagedKVBuffer.step: scale must be a number")
        qr, kr = qk_norm_rope(q.flatten(0, 1), k.flatten(0, 1), self.length, inv_freq, q_weight, k_weight, eps, interleaved)
        self.append(kr.view(k.shape), v, None, counts)
        return self.attend(qr.view(q.shape), None, counts, scale)

    def truncate(self, length) -> None:
        """Forget positions >= length (an int or int64 [sequences]), for
        instance the drafts that were refused; below 0 as 0.  No further back
        than pages that were released, but for an int of 0, which forgets all
        positions: then those pages can be reserved again."""
        if isinstance(length, torch.Tensor):
            self.length.copy_(torch.minimum(self.length, self._places("truncate", "length", length, self.sequences)).clamp_(min=0))
        else:
            length = max(0, int(length))
            if length:
                self._not_released("truncate", length, None)
            self.length.clamp_(max=length)
            if not length:
                self._first = [0] * self.sequences


@dataclass
class DeviceLayerState:
    """model.py:94-97 LayerState: the layer's key / value buffer and, for a
    hybrid layer, its shared [H, K, V] and partition [P, H, K, V] states."""

    kv: DeviceKVBuffer
    shared: torch.Tensor | None = None
    partitions: torch.Tensor | None = None

    def reset(self) -> None:
        self.kv.reset()
        if self.shared is not None:
            self.shared.zero_()
            self.partitions.zero_()


@dataclass
class DeviceInferenceState:
    """model.py:99-103 InferenceState on the device: ``position`` is the next
    token's position (device long [1]), ``tokens`` the ids fed so far
    (device long [capacity], written at their positions) and ``next_token``
    the id the next decode step embeds (the greedy token of the last one)."""

    layers: list[DeviceLayerState]
    position: torch.Tensor
    tokens: torch.Tensor
    next_token: torch.Tensor = field(default=None)

    def reset(self, token: int | None = None) -> None:
        for layer in self.layers:
            layer.reset()
        self.position.zero_()
        self.tokens.zero_()
        if token is not None:
            self.next_token.fill_(int(token))

    def record(self, token_ids: torch.Tensor) -> None:
        """Write the ids of the tokens about to be fed at the current position."""
        T = token_ids.numel()
        idx = self.position + torch.arange(T, device=self.position.device)
        self.tokens.index_copy_(0, idx.clamp_(max=self.tokens.numel() - 1), token_ids.reshape(-1).long())

    def advance(self, T: int) -> None:
        self.position += T


def new_device_state(hybrid: list[bool], heads: int, head_dim: int, kv_heads: int, partitions: int,
                     window: int, capacity: int, device: torch.device | str | None = None,
                     ring_extra: int = 1, budget: int | None = None, recent: int = 0) -> DeviceInferenceState:
    """model.py:412-424 new_state on the device: per layer a key / value
    buffer (windowed, a ring of window + ring_extra slots, for hybrid layers;
    `capacity` positions for softmax layers) and, for hybrid layers, zeroed
    shared [heads, head_dim, head_dim] and partition [partitions, heads,
    head_dim, head_dim] fp32 states.  ring_extra is the most tokens one call
    appends (1 for decode; the prefill chunk otherwise).  budget: slots of a
    softmax layer's buffer when it is to be smaller than `capacity` positions
    (DeviceBudgetKVBuffer, the `recent` newest positions kept)."""
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    layers = []
    for is_hybrid in hybrid:
        if is_hybrid:
            layers.append(DeviceLayerState(
                kv=DeviceKVBuffer(kv_heads, head_dim, window + ring_extra, window, dev),
                shared=torch.zeros(heads, head_dim, head_dim, device=dev),
                partitions=torch.zeros(partitions, heads, head_dim, head_dim, device=dev)))
        elif budget is not None and budget < capacity:
            layers.append(DeviceLayerState(kv=DeviceBudgetKVBuffer(kv_heads, head_dim, budget, recent, dev)))
        else:
            layers.append(DeviceLayerState(kv=DeviceKVBuffer(kv_heads, head_dim, capacity, None, dev)))
    return DeviceInferenceState(layers=layers, position=torch.zeros((1,), dtype=torch.long, device=dev),
                                tokens=torch.zeros((capacity,), dtype=torch.long, device=dev),
                                next_token=torch.zeros((1,), dtype=torch.long, device=dev))
