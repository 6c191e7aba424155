"""Device storage of the cache, laid out from what the model's runs declare.

Paged group: every run that owns a cache slot gets K and V tensors
[num_pages, num_kv_heads, page_size, head_dim] in the activation dtype.  A
page id indexes the same page in every run of the group, like the reference's
block ids index every layer's buffer (crates/rllm-cache/src/spec.rs:26-32).
Inside a page the tokens of one kv head are contiguous rows of head_dim, so a
(page, head) tile is one contiguous block (the reference's
[blocks, heads, head_dim, block_size], spec.rs:63-68, strides the hot axis).
State group: every owning run gets float32 [max_seqs, *shape], indexed by a
request's state slot.  In 8 bits (``e4m3``) K and V are float8 e4m3 pages, and beside
each stands a tensor of scales [num_pages, num_kv_heads, page_size], a power of two (e8m0) a row.
A mixer that declared several needs (pages and state,
or two states) owns storage in several groups.  All storage is allocated once, here.

Every paged buffer has one page more than the manager hands out: page
``spare_page(group)`` belongs to no request; every state buffer has one slot
more, ``spare_slot``.  The rows that pad a decode step to a captured batch size
read and write there.
"""
from __future__ import annotations

from typing import Dict, List, Sequence

import torch

from ..parts.base import KVCacheView, StateCacheView
from ..parts.spec import KVPagesNeed, StateNeed


def page_bytes(need: KVPagesNeed, page_size: int, elem_size: int, scale_bytes: int = 0) -> int:
    """Bytes of one page of one run: K and V (one buffer where keys serve as values), a row with ``scale_bytes`` more."""
    row = need.head_dim + (need.value_dim if need.values else 0)
    return need.num_kv_heads * page_size * (row * elem_size + scale_bytes * (2 if need.values else 1))


class CacheStorage:
    def __init__(self, layout, page_size: int, num_pages: Sequence[int], max_seqs: int,
                 dtype: torch.dtype, device: torch.device, e4m3: bool = False):
        self.layout = layout
        self.page_size = page_size
        self.e4m3 = e4m3
        self.scales: Dict[int, tuple] = {}
        self.kv: Dict[int, tuple] = {}
        self.state: Dict[int, torch.Tensor] = {}
        paged = [g for g, n in enumerate(layout.groups) if isinstance(n, KVPagesNeed)]
        pages_of = dict(zip(paged, num_pages))
        self._pages_of = pages_of
        self.spare_slot = max_seqs           # the state slot that no request ever holds
        for g, need in enumerate(layout.groups):
            for run in layout.owners[g]:
                if isinstance(need, KVPagesNeed):
                    shape = (pages_of[g] + 1, need.num_kv_heads, page_size, need.head_dim)
                    vshape = shape[:3] + (need.value_dim,)
                    if e4m3:
                        if not need.values:
                            raise ValueError("pages of one row for keys and values have no 8-bit form")
                        byte = lambda size, dt: torch.zeros(size, dtype=torch.uint8, device=device).view(dt)  # noqa: E731
                        self.kv[run] = (byte(shape, torch.float8_e4m3fn), byte(vshape, torch.float8_e4m3fn))
                        self.scales[run] = (byte(shape[:3], torch.float8_e8m0fnu), byte(shape[:3], torch.float8_e8m0fnu))
                        continue
                    self.kv[run] = (torch.zeros(shape, dtype=dtype, device=device),
                                    torch.zeros(vshape, dtype=dtype, device=device) if need.values else None)
                elif isinstance(need, StateNeed):
                    self.state[run] = torch.zeros((max_seqs + 1,) + tuple(need.shape), dtype=torch.float32,
                                                  device=device)
                else:
                    raise TypeError(f"unknown cache need {need!r}")

    def spare_page(self, group: int) -> int:
        """The id of the page of this paged group that no request ever holds."""
        return self._pages_of[group]

    def view(self, run_index: int):
        """The cache view of a run's mixer; a tuple of views, in the order of its needs, for a mixer that
        declared several (their storage is keyed (owning run, number of the need))."""
        g = self.layout.run_group[run_index]
        if g is None:
            return None
        owner = self.layout.run_owner[run_index]
        writes = owner == run_index
        if isinstance(g, tuple):
            return tuple(self._view((owner, j), gj, writes) for j, gj in enumerate(g))
        return self._view(owner, g, writes)

    def _view(self, key, g: int, writes: bool):
        if key in self.kv:
            k, v = self.kv[key]
            return KVCacheView(k, v, g, writes, *self.scales.get(key, (None, None)))
        return StateCacheView(self.state[key], g, writes)

    def zero_slots(self, slots: List[int]) -> None:
        """Zero the state of newly handed-out slots."""
        if not slots or not self.state:
            return
        idx = torch.tensor(slots, dtype=torch.long, device=next(iter(self.state.values())).device)
        for t in self.state.values():
            t.index_fill_(0, idx, 0.0)

    def copy_for_fork(self, copies, slots) -> None:
        """The device side of ``CacheManager.fork``: every owning run of a group copies the
        page (K and V, one device-to-device copy each, on the current stream) and every
        state buffer copies the slot.  The reference has the copy kernel
        (crates/rllm-kernels/src/cuda/cache_ops.cu:252-279) and never calls it."""
        for g, src, dst in copies:
            for run in self.layout.owners[g]:
                k, v = self.kv[run]
                k[dst].copy_(k[src], non_blocking=True)
                if v is not None:
                    v[dst].copy_(v[src], non_blocking=True)
                for t in self.scales.get(run, ()):
                    t[dst].copy_(t[src], non_blocking=True)
        src, dst = slots
        for t in self.state.values():
            t[dst].copy_(t[src], non_blocking=True)

    def num_bytes(self) -> int:
        n = sum(k.numel() * k.element_size() * (1 if v is None else 2) for k, v in self.kv.values())
        n += sum(t.numel() for pair in self.scales.values() for t in pair)
        return n + sum(t.numel() * 4 for t in self.state.values())

    def read_tokens(self, run_index: int, table: torch.Tensor, positions: torch.Tensor, token_seq: torch.Tensor,
                    dtype: torch.dtype = torch.bfloat16):
        """(keys, values) [T, num_kv_heads, head_dim] of a run's tokens at ``positions`` (int32) of the sequences
        ``token_seq``, whose pages ``table`` (int32 [sequences, blocks]) names, read back from pages kept in 8 bits."""
        from ..kernels import ops
        view = self.view(run_index)
        if not isinstance(view, KVCacheView) or view.k_scale is None:
            raise ValueError(f"run {run_index} has no pages in 8 bits")
        nkv, d = view.k.shape[1], view.k.shape[3]
        k, v = (torch.empty((positions.numel(), nkv * d), dtype=dtype, device=view.k.device) for _ in range(2))
        err = torch.zeros(1, dtype=torch.int32, device=view.k.device)
        ops.kv_read_e4m3(positions, token_seq, table, view.k, view.v, view.k_scale, view.v_scale, k, v, err)
        if int(err.item()):
            raise ValueError("a token lies in a page that its sequence does not hold")
        return k.view(-1, nkv, d), v.view(-1, nkv, d)
