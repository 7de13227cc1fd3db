"""Device tensors behind the cache manager's page and slot numbers.

For every paged group one tensor `[layers in group, 2 (keys, values), pages + 1, kv heads, page size,
head size]`: the rows of one (page, kv head) lie together, so a kernel reads a page of one head as
one contiguous tile. A group whose values have another head size than its keys has two tensors instead
(`[layers in group, pages + 1, kv heads, page size, head size]` each), and one whose values are the first
values of its key rows has the keys' tensor alone; `keys()` / `values()` give a layer's pages either way. For every state group one tensor `[layers in group, request slots, *shape]`.
Keys are stored after rotation, values as projected (src/model.br:1814-1820).
"""
from __future__ import annotations

from typing import List

import torch

from .manager import CacheManager

_TORCH_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "int32": torch.int32}


class CacheStorage:
    def __init__(self, manager: CacheManager, kv_dtype: torch.dtype, device):
        self.manager = manager
        self.kv_dtype = kv_dtype
        self.device = torch.device(device)
        # One page and one slot more than the manager hands out: rows that only pad a batch to a fixed
        # size (captured CUDA graphs) write there, where no request ever reads.
        self.trash_page = manager.num_pages
        self.trash_slot = manager.max_requests
        self.kv: List[torch.Tensor] = []           # joint tensors (groups with two tensors have None here)
        self.k_pages: List[torch.Tensor] = []      # per group [layers, pages + 1, kv heads, page size, head size]
        self.v_pages: List[torch.Tensor] = []
        for g in manager.paged_groups:
            lead = (manager.num_pages + 1, g.spec.n_kv_heads, manager.page_size)
            if g.spec.values_in_keys:
                if g.spec.value_dim > g.spec.head_dim:
                    raise ValueError(f"values of {g.spec.value_dim} cannot lie inside keys of {g.spec.head_dim}")
                k = torch.zeros((len(g.cache_layers),) + lead + (g.spec.head_dim,), dtype=kv_dtype, device=self.device)
                self.kv.append(None)
                self.k_pages.append(k)
                self.v_pages.append(k[..., :g.spec.value_dim])
            elif g.spec.value_dim == g.spec.head_dim:
                kv = torch.zeros((len(g.cache_layers), 2) + lead + (g.spec.head_dim,), dtype=kv_dtype, device=self.device)
                self.kv.append(kv)
                self.k_pages.append(kv[:, 0])
                self.v_pages.append(kv[:, 1])
            else:
                self.kv.append(None)
                self.k_pages.append(torch.zeros((len(g.cache_layers),) + lead + (g.spec.head_dim,), dtype=kv_dtype, device=self.device))
                self.v_pages.append(torch.zeros((len(g.cache_layers),) + lead + (g.spec.value_dim,), dtype=kv_dtype, device=self.device))
        self.state: List[torch.Tensor] = []
        for sg in manager.state_groups:
            self.state.append(torch.zeros(
                (len(sg.cache_layers), manager.max_requests + 1) + tuple(sg.spec.shape),
                dtype=_TORCH_DTYPES[sg.spec.dtype], device=self.device))
        manager._on_slot_assigned = self.zero_slot

    def poison_freed_pages(self) -> int:
        """Debugging aid: fills every page that was given back since the last call (and, the first time, every page
        that no request holds, the spare page included) with NaN, keys and values in all layers. Freed pages are
        otherwise left as they are, because nothing may read a request's cache past its length; with poison a
        kernel that does read there, even with weight zero, turns its output into NaN. Returns the pages filled."""
        n = 0
        for gi, g in enumerate(self.manager.paged_groups):
            if g.pool.freed_log is None:
                g.pool.freed_log = []
                pages = [p for p in range(g.pool.num_pages) if g.pool.owner_of(p) is None] + [self.trash_page]
            else:
                pages, g.pool.freed_log = [p for p in set(g.pool.freed_log) if g.pool.owner_of(p) is None], []
            if pages and self.kv_dtype.is_floating_point:
                idx = torch.tensor(pages, dtype=torch.long, device=self.device)
                self.k_pages[gi][:, idx] = float("nan")
                self.v_pages[gi][:, idx] = float("nan")
                n += len(pages)
        return n

    def zero_slot(self, slot: int) -> None:
        for t in self.state:
            t[:, slot].zero_()

    def copy_pages(self) -> None:
        """Copies, in all layers, the shared pages that requests are about to write (`CacheManager.take_copies`), on the current stream."""
        if not self.manager.has_copies:
            return
        from ..kernels import ops
        for gi, pairs in enumerate(self.manager.take_copies()):
            # a page that was copied and given back may have become another request's copy meanwhile: such pairs go in their order
            while pairs:
                sources, targets, n = set(), set(), 0
                for s, d in pairs:
                    if d in sources or d in targets or s in targets:
                        break
                    sources.add(s)
                    targets.add(d)
                    n += 1
                own_values = not self.manager.paged_groups[gi].spec.values_in_keys
                ops.copy_blocks([self.k_pages[gi]] + ([self.v_pages[gi]] if own_values else []), pairs[:n])
                pairs = pairs[n:]

    def copy_slot(self, source: int, target: int) -> None:
        """The state of one request slot into another, in all layers."""
        if self.state:
            from ..kernels import ops
            for i in range(0, len(self.state), 8):
                ops.copy_blocks(self.state[i:i + 8], [(source, target)])

    def keys(self, cache_layer: int) -> torch.Tensor:
        kind, gi, li = self.manager.layer_location[cache_layer]
        assert kind == "paged"
        return self.k_pages[gi][li]

    def values(self, cache_layer: int) -> torch.Tensor:
        kind, gi, li = self.manager.layer_location[cache_layer]
        assert kind == "paged"
        return self.v_pages[gi][li]

    def layer_state(self, cache_layer: int) -> torch.Tensor:
        """`[request slots, *shape]` of one cache layer with fixed-size state."""
        kind, gi, li = self.manager.layer_location[cache_layer]
        assert kind == "state"
        return self.state[gi][li]

    def bytes(self) -> int:
        own_values = [v for g, v in zip(self.manager.paged_groups, self.v_pages) if not g.spec.values_in_keys]
        return sum(t.numel() * t.element_size() for t in self.k_pages + own_values + self.state)
