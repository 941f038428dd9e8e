"""Device memory of the cache: page tensors of every group and per-request state.

The reference allocates, per layer, K and V tensors ``[blocks * block_size,
kv_heads, head_dim]`` (inferrs-models/src/kv_cache.rs:249-270).  Here one
tensor per group holds all its caches,

    [caches in group, 2 (keys, values; 1 for a cache of latents), pages, kv_heads, page_size, head_dim]

so that one page of one head is a contiguous ``[page_size, head_dim]`` tile.
Writes are plain stores; a page that is used again needs no clearing because a
request never reads beyond the tokens it has written.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Any, Dict, List, Optional, Sequence, Tuple

import torch

from ..kernels import Kv8Pages
from .manager import GroupLayout


@dataclass(frozen=True)
class KVNeed:
    """What a mixer asks of the paged cache for one schedule entry."""

    n_kv_heads: int
    head_dim: int
    window: Optional[int] = None
    # 2: keys and values each have their pages; 1: one vector per token serves as both (a cache of latents)
    planes: int = 2
    # size of a value head where it differs from a key head's (None: the same; such a group keeps its values in
    # a tensor of their own)
    value_dim: Optional[int] = None
    # how many of a sequence's first tokens stay visible beside the window
    keep_first: int = 0


@dataclass(frozen=True)
class StateNeed:
    """Per-request state of fixed size that a mixer keeps for one schedule entry."""

    shape: Tuple[int, ...]
    dtype: torch.dtype = torch.float32


def bytes_of_vectors(need: KVNeed, dtype: torch.dtype, bits: Optional[int]) -> int:
    """Bytes of one token's keys and values in one cache."""
    if bits == 8:
        return need.n_kv_heads * 2 * (need.head_dim + 4)
    return need.n_kv_heads * (need.head_dim * (need.planes - 1) + (need.value_dim or need.head_dim)) \
        * torch.empty((), dtype=dtype).element_size()


class CacheStorage:
    def __init__(self, kv_needs: Dict[int, KVNeed], state_needs: Dict[int, StateNeed], page_size: int,
                 n_pages: int, max_requests: int, dtype: torch.dtype, device: torch.device,
                 n_pages_per_group: Optional[Sequence[int]] = None,
                 side_state_needs: Optional[Dict[Tuple[int, Any], StateNeed]] = None, bits: Optional[int] = None):
        """``bits`` 8: keys and values in 8 bits (``pages8``; ``pages`` then has nothing to give).
        ``side_state_needs``: per-request states beside a mixer's own, keyed by (cache id, the description that
        owns the state): the inputs that a short convolution in front of a sub-layer or behind a projection keeps."""
        self.page_size = page_size
        self.max_requests = max_requests
        self.dtype = dtype
        self.device = device
        self.bits = bits
        if bits not in (None, 8):
            raise ValueError(f"keys and values are cached in the activations' type or in 8 bits, got {bits} bits")
        if bits == 8 and any(k.planes != 2 or k.value_dim not in (None, k.head_dim) or k.head_dim % 4 for k in kv_needs.values()):
            raise ValueError("a cache in 8 bits holds keys and values of one size, a multiple of four numbers")
        # caches with equal needs form a group, in order of first appearance
        keys: List[KVNeed] = []
        self.group_of: Dict[int, int] = {}
        self.index_in_group: Dict[int, int] = {}
        members: List[List[int]] = []
        for cid in sorted(kv_needs):
            need = kv_needs[cid]
            if need not in keys:
                keys.append(need)
                members.append([])
            g = keys.index(need)
            self.group_of[cid] = g
            self.index_in_group[cid] = len(members[g])
            members[g].append(cid)
        if not keys:
            # a model whose mixers all keep fixed-size state: one group without caches still counts every request's
            # tokens page by page (positions, the longest context), and holds no memory
            keys.append(KVNeed(n_kv_heads=0, head_dim=0))
            members.append([])
        self.needs = keys
        self.members = members
        if any(k.planes not in (1, 2) for k in keys):
            raise ValueError("a cache has one plane (latents) or two (keys and values)")
        self.layouts = [GroupLayout(name=f"group{g}(heads={k.n_kv_heads},dim={k.head_dim},window={k.window})",
                                    window=k.window, keep_first=k.keep_first) for g, k in enumerate(keys)]
        self.n_pages = list(n_pages_per_group) if n_pages_per_group is not None else [n_pages] * len(keys)
        if any(k.value_dim is not None and k.planes != 2 for k in keys):
            raise ValueError("values of a size of their own need a cache of two planes")
        self.kv: List[torch.Tensor] = []
        # in 8 bits: codes in ``kv``, and one float32 scale per vector [caches in group, 2, pages, kv_heads, page_size]
        self.scales: List[torch.Tensor] = []
        self._pages8: Dict[int, Kv8Pages] = {}
        # values whose heads have another size than the keys': [caches in group, pages, kv_heads, page_size, value_dim]
        # (the group's tensor in ``kv`` then holds the keys alone)
        self.values: List[Optional[torch.Tensor]] = []
        for g, k in enumerate(keys):
            if bits == 8:
                shape = (len(members[g]), 2, self.n_pages[g], k.n_kv_heads, page_size, k.head_dim)
                self.kv.append(torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn))
                self.scales.append(torch.zeros(shape[:-1], dtype=torch.float32, device=device))
                self.values.append(None)
                continue
            own_values = k.value_dim is not None and k.value_dim != k.head_dim
            self.kv.append(torch.zeros((len(members[g]), 1 if own_values else k.planes, self.n_pages[g], k.n_kv_heads,
                                        page_size, k.head_dim), dtype=dtype, device=device))
            self.values.append(torch.zeros((len(members[g]), self.n_pages[g], k.n_kv_heads, page_size, k.value_dim),
                                           dtype=dtype, device=device) if own_values else None)
        # one slot more than there are requests: the requests that only pad a replayed step write their state there
        self.states: Dict[int, torch.Tensor] = {
            cid: torch.zeros((max_requests + 1,) + tuple(need.shape), dtype=need.dtype, device=device)
            for cid, need in state_needs.items()}
        self.side_states: Dict[Tuple[int, Any], torch.Tensor] = {
            key: torch.zeros((max_requests + 1,) + tuple(need.shape), dtype=need.dtype, device=device)
            for key, need in (side_state_needs or {}).items()}

    def pages(self, cache_id: int) -> Tuple[torch.Tensor, torch.Tensor, int]:
        """(key pages, value pages, group index) of one cache; pages are [n_pages, kv_heads, page_size, head_dim]
        (value pages end in the group's ``value_dim`` where it has one).
        A cache of one plane gives the same pages twice."""
        if self.bits is not None:
            raise ValueError(f"this cache holds {self.bits} bits a number: ask pages8")
        g = self.group_of[cache_id]
        t = self.kv[g][self.index_in_group[cache_id]]
        if self.values[g] is not None:
            return t[0], self.values[g][self.index_in_group[cache_id]], g
        return t[0], t[t.shape[0] - 1], g

    def pages8(self, cache_id: int) -> Tuple[Kv8Pages, int]:
        """(pages of keys and values in 8 bits, group index) of one cache."""
        g = self.group_of[cache_id]
        if cache_id not in self._pages8:
            i = self.index_in_group[cache_id]
            codes, scales = self.kv[g][i], self.scales[g][i]
            self._pages8[cache_id] = Kv8Pages(codes[0], codes[1], scales[0], scales[1])
        return self._pages8[cache_id], g

    def state(self, cache_id: int) -> torch.Tensor:
        return self.states[cache_id]

    def side_state(self, cache_id: int, owner: Any) -> torch.Tensor:
        """The per-request state [slots, ...] that the description ``owner`` keeps under this cache id."""
        return self.side_states[(cache_id, owner)]

    def clear_slot(self, slot: int):
        """A new request takes the slot: its fixed-size states start at zero."""
        for t in list(self.states.values()) + list(self.side_states.values()):
            t[slot].zero_()

    def snapshot_states(self) -> Dict[Any, torch.Tensor]:
        """Copies of all fixed-size states (for a caller that has to run a step more than once)."""
        saved = {cid: t.clone() for cid, t in self.states.items()}
        saved.update({("side",) + key: t.clone() for key, t in self.side_states.items()})
        return saved

    def restore_states(self, saved: Dict[Any, torch.Tensor]):
        for key, t in saved.items():
            if isinstance(key, tuple) and key and key[0] == "side":
                self.side_states[key[1:]].copy_(t)
            else:
                self.states[key].copy_(t)

    def bytes_per_token(self) -> int:
        """Bytes of keys and values that one token adds, over all groups."""
        return sum(len(self.members[g]) * bytes_of_vectors(k, self.dtype, self.bits) for g, k in enumerate(self.needs))

    def total_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self.kv) + \
            sum(t.numel() * t.element_size() for t in self.values if t is not None) + \
            sum(t.numel() * t.element_size() for t in self.scales) + \
            sum(t.numel() * t.element_size() for t in self.states.values()) + \
            sum(t.numel() * t.element_size() for t in self.side_states.values())
