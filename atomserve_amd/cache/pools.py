"""The tensors behind the cache manager's ids.

A paged group has one pool [caches in group, 2 (k, v), num_pages, KV, block_size, D]
in the compute dtype: the block_size keys of one head in one page are contiguous;
the value half of a page is stored transposed, [D, block_size].  It
starts zeroed, so that no slot ever holds a non-finite value
(reference atomserve/kv_cache.py:112-118).  A paged group that asks for 8 bits
has e4m3 numbers (a page's values as blocks of 16 tokens, [block_size / 16, D, 16])
and scales [caches in group, 2, num_pages, KV, block_size / 16] in fp32.  A state group has
[caches in group, max_num_seqs + 1, *shape]: one slot per running request and a last one
(`scrap_slot`) that belongs to nobody, for the rows that only pad a captured step.
"""

import torch

from atomserve_amd.cache.manager import CacheManager

BLOCK = 16  # tokens that share a scale in a cache of 8 bits

class CachePools:
    def __init__(self, manager: CacheManager, dtype: torch.dtype, device):
        self.manager = manager
        self.dtype = dtype
        self.paged = []
        self.scales = []  # per paged group: None, or the scales of a cache in 8 bits
        for g in manager.paged_groups:
            r = g.request
            shape = (len(g.cache_ids), 2, manager.num_blocks, r.num_kv_heads, manager.block_size, r.head_dim)
            if r.bits == 8:
                if manager.block_size % BLOCK:
                    raise ValueError(f"a cache in 8 bits has pages of a multiple of {BLOCK} tokens, not {manager.block_size}")
                self.paged.append(torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn))
                self.scales.append(torch.zeros((*shape[:4], manager.block_size // BLOCK), dtype=torch.float32, device=device))
            elif r.bits == 0:
                self.paged.append(torch.zeros(shape, dtype=dtype, device=device))
                self.scales.append(None)
            else:
                raise ValueError(f"a cache holds the compute dtype or 8 bits, not {r.bits}")
        self.state = []
        self.scrap_slot = manager.max_num_seqs
        for g in manager.state_groups:
            shape = (len(g.cache_ids), manager.max_num_seqs + 1, *g.request.shape)
            self.state.append(torch.zeros(shape, dtype=g.request.dtype, device=device))
        # every cache's views of its pool, made once: every layer of every step asks for its own
        self._views, self._scales = {}, {}
        for cache_id, (kind, gi, li) in manager.group_of_cache.items():
            if kind == "paged":
                nb, kv, bs, d = self.paged[gi].shape[2:]
                scales = self.scales[gi]
                turned = (nb, kv, d, bs) if scales is None else (nb, kv, bs // BLOCK, d, BLOCK)
                self._views[cache_id] = gi, self.paged[gi][li, 0], self.paged[gi][li, 1].view(turned)
                self._scales[cache_id] = (None, None) if scales is None else (scales[li, 0], scales[li, 1])
            elif kind == "state":
                self._views[cache_id] = gi, self.state[gi][li]

    def pages(self, cache_id: int):
        """(group index, k_pages, v_pages) of one cache: k_pages [num_pages, KV, block_size, D];
        v_pages [num_pages, KV, D, block_size], each page of values transposed so that the keys
        of one coordinate are contiguous (what the matrix-core kernels read directly); in 8 bits v_pages
        [num_pages, KV, block_size / 16, D, 16]."""
        if self.manager.group_of_cache[cache_id][0] != "paged":
            raise KeyError(f"cache {cache_id} is not paged")
        return self._views[cache_id]

    def scales_of(self, cache_id: int):
        """(k_scales, v_scales) of one paged cache in 8 bits, [num_pages, KV, block_size / 16] each; (None, None) of another."""
        if self.manager.group_of_cache[cache_id][0] != "paged":
            raise KeyError(f"cache {cache_id} is not paged")
        return self._scales[cache_id]

    def state_of(self, cache_id: int):
        """(group index, state tensor [max_num_seqs + 1, *shape]) of one cache."""
        if self.manager.group_of_cache[cache_id][0] != "state":
            raise KeyError(f"cache {cache_id} holds no fixed-size state")
        return self._views[cache_id]

    @staticmethod
    def bytes_per_block(requests: dict, block_size: int, dtype: torch.dtype) -> int:
        """Memory one page id costs across all paged caches, keys and values, with the scales of those in 8 bits
        (reference atomserve/kv_cache.py:129-135)."""
        from atomserve_amd.parts.base import PagedCacheRequest

        item = torch.empty((), dtype=dtype).element_size()
        return sum(2 * r.num_kv_heads * (r.head_dim * block_size + 4 * (block_size // BLOCK) if r.bits == 8 else r.head_dim * item * block_size)
                   for r in requests.values() if isinstance(r, PagedCacheRequest))  # fmt: skip
