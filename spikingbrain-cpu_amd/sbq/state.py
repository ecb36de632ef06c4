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

Capacity: a full-attention buffer holds ``capacity`` positions (slot =
position).  A sliding-window buffer is a ring of ``capacity`` slots (slot =
position mod capacity); it must hold the window plus the tokens appended by
one call, so that no key a query of that call sees is overwritten.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import torch

from . import _lib
from .quant import _DTYPE_CODE, _on_device, _stream


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
