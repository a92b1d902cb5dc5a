"""Paged caches: keys and values head-sharded over the tensor-parallel ranks, one latent row per token and layer, or pages and
recurrent states side by side.

Same interface as the reference's dense cache (``python/triton_dist/models/kv_cache.py:29-66``:
``update_kv_cache``, ``rand_fill_kv_cache``, ``inc_offset``, ``clear``, ``get_kv_len``) but stored as pages
``[layers, num_blocks, page, kv_heads / world, head_dim]`` with a block table, which is the layout the
decode-attention kernel reads. Sequence b owns blocks ``b * blocks_per_seq ...`` so the table is static
and a decode step can be captured in a CUDA graph. ``PagedCache`` owns the pages' bookkeeping (slots, block table,
offsets), the subclasses own what a page holds.
"""
from __future__ import annotations

import dataclasses

import torch

from .. import ops


class PagedCache:

    def __init__(self, num_layers: int, batch_size: int, max_length: int, dtype, page_size: int = 64, device="cuda") -> None:
        self.num_layers, self.batch_size, self.max_length = num_layers, batch_size, max_length
        self.dtype, self.page_size = dtype, page_size
        self.blocks_per_seq = (max_length + page_size - 1) // page_size
        self.num_blocks = batch_size * self.blocks_per_seq
        self.kv_offset = torch.zeros(batch_size, dtype=torch.int32, device=device)
        self.block_table = torch.arange(self.num_blocks, dtype=torch.int32, device=device).view(batch_size, self.blocks_per_seq)

    def slots(self, positions: torch.Tensor) -> torch.Tensor:
        """Flat slot index (block * page + offset) of token position [B, S] of every sequence -> int64 [B*S]."""
        B, S = positions.shape
        base = torch.arange(B, device=positions.device, dtype=torch.int64)[:, None] * (self.blocks_per_seq * self.page_size)
        return (base + positions.to(torch.int64)).reshape(-1)

    def inc_offset(self, n: int = 1) -> None:
        self.kv_offset += n

    def clear(self) -> None:
        self.kv_offset.zero_()

    def save_state(self):
        """What a decode step changes beyond the slots it writes (running a step again would change it again); None here: pages
        are written at their slot, whatever was there."""
        return None

    def restore_state(self, saved) -> None:
        """Back to ``save_state``'s result, in place."""

    def get_kv_len(self) -> torch.Tensor:
        return self.kv_offset


class KV_Cache(PagedCache):

    def __init__(self, num_layers: int = 32, batch_size: int = 1, max_length: int = 32 * 1024, kv_heads: int = 8,
                 head_dim: int = 128, dtype=torch.bfloat16, world_size: int = 8, page_size: int = 64,
                 device="cuda") -> None:
        super().__init__(num_layers, batch_size, max_length, dtype, page_size, device)
        self.kv_heads, self.head_dim, self.world_size = kv_heads, head_dim, world_size
        self.local_kv_heads = max(1, kv_heads // world_size)
        shape = (num_layers, self.num_blocks, page_size, self.local_kv_heads, head_dim)
        self.k_cache = torch.zeros(shape, device=device, dtype=dtype)
        self.v_cache = torch.zeros(shape, device=device, dtype=dtype)

    def layer(self, layer_idx: int):
        """(k pages, v pages) of one layer: [num_blocks, page, kv_heads_local, head_dim]."""
        return self.k_cache[layer_idx], self.v_cache[layer_idx]

    def update_kv_cache(self, new_k: torch.Tensor, new_v: torch.Tensor, layer_idx: int):
        """Append [B, S, kv_heads_local, D] at the current offsets (the fused rope kernel normally does this)."""
        B, S = new_k.shape[:2]
        pos = self.kv_offset[:, None].to(torch.int64) + torch.arange(S, device=new_k.device)[None, :]
        sl = self.slots(pos)
        self.k_cache[layer_idx].view(-1, self.local_kv_heads, self.head_dim)[sl] = new_k.reshape(-1, self.local_kv_heads, self.head_dim)
        self.v_cache[layer_idx].view(-1, self.local_kv_heads, self.head_dim)[sl] = new_v.reshape(-1, self.local_kv_heads, self.head_dim)
        return self.k_cache[layer_idx], self.v_cache[layer_idx], self.kv_offset

    def rand_fill_kv_cache(self, offset: int) -> None:
        self.k_cache.copy_(torch.rand_like(self.k_cache) / 10)
        self.v_cache.copy_(torch.rand_like(self.v_cache) / 10)
        self.kv_offset.fill_(offset)


class LatentCache(PagedCache):
    """Latent attention's cache: layer i keeps one row of ``widths[i]`` elements per token (shared by all heads, so it is
    replicated over tensor-parallel ranks), as pages ``[num_blocks, page, widths[i]]``."""

    def __init__(self, widths: list[int], batch_size: int, max_length: int, dtype=torch.bfloat16, page_size: int = 64,
                 device="cuda") -> None:
        super().__init__(len(widths), batch_size, max_length, dtype, page_size, device)
        self.c_cache = [torch.zeros((self.num_blocks, page_size, w), device=device, dtype=dtype) for w in widths]

    def layer(self, layer_idx: int) -> torch.Tensor:
        """Pages of one layer: [num_blocks, page, width]."""
        return self.c_cache[layer_idx]

    def rows(self, layer_idx: int, count: int) -> torch.Tensor:
        """The first `count` latent rows of every sequence as one matrix [batch * count, width] (a sequence's pages are
        consecutive; a view where the rows of the batch are, else a copy)."""
        c = self.c_cache[layer_idx].view(self.batch_size, self.blocks_per_seq * self.page_size, -1)[:, :count]
        return c.reshape(self.batch_size * count, -1)

    def blank(self, layer_idx: int, start: int, stop: int) -> None:
        """Zero the unused rows [start, stop) of every sequence."""
        if stop > start:
            self.c_cache[layer_idx].view(self.batch_size, self.blocks_per_seq * self.page_size, -1)[:, start:stop].zero_()


class HybridCache(PagedCache):
    """Layers of different kinds: some keep rows per token in pages, some a state of fixed size per sequence, some both.

    ``layers[i]`` maps names to shapes: ``pages`` name -> the shape of a token's row, stored ``[num_blocks, page, *row]`` in the
    cache's type; ``states`` name -> (shape, type), stored ``[batch, *shape]``. States start at zero: ``clear`` zeroes them (pages need
    not be), in place, so that a captured decode step keeps its addresses."""

    @dataclasses.dataclass
    class Layer:
        pages: dict[str, tuple[int, ...]] = dataclasses.field(default_factory=dict)
        states: dict[str, tuple[tuple[int, ...], torch.dtype]] = dataclasses.field(default_factory=dict)

    def __init__(self, layers: list["HybridCache.Layer"], batch_size: int, max_length: int, dtype=torch.bfloat16, page_size: int = 64,
                 device="cuda") -> None:
        super().__init__(len(layers), batch_size, max_length, dtype, page_size, device)
        self._pages = [{n: torch.zeros((self.num_blocks, page_size, *row), device=device, dtype=dtype) for n, row in layer.pages.items()}
                       for layer in layers]
        self._states = [{n: torch.zeros((batch_size, *shape), device=device, dtype=dt) for n, (shape, dt) in layer.states.items()}
                        for layer in layers]

    def pages(self, layer_idx: int, name: str) -> torch.Tensor:
        return self._pages[layer_idx][name]

    def state(self, layer_idx: int, name: str) -> torch.Tensor:
        return self._states[layer_idx][name]

    def _all_states(self) -> list[torch.Tensor]:
        return [t for layer in self._states for t in layer.values()]

    def clear(self) -> None:
        super().clear()
        for t in self._all_states():
            t.zero_()

    def save_state(self):
        return [t.clone() for t in self._all_states()]

    def restore_state(self, saved) -> None:
        for t, old in zip(self._all_states(), saved):
            t.copy_(old)


class PagePool:
    """Keys and values of rows that may hold the same pages: several samples of a prompt, beams, drafts that are taken back.

    Unlike in a ``PagedCache`` no row owns a fixed run of pages: ``block_table`` int32 [batch, max_blocks] (-1: not held), ``kv_lens`` int32 [batch] and
    ``refs`` int32 [num_blocks] (how many rows hold a page) live on the device and are changed in place by kernels, so that a step can be
    captured. A step of S tokens: ``reserve(S)``, keys and values to ``slots(S)``, ``advance(S)``, attention over ``layer(i)``, ``kv_lens`` and
    ``block_table`` (``ops.decode_attention``, ``ops.shared_prefix_attention``); drafts that were refused go with ``trim``. The caches have one page
    more than ``refs`` counts: rows without room of their own write there."""

    def __init__(self, num_layers: int, num_blocks: int, batch_size: int, max_length: int, kv_heads: int, head_dim: int = 128, dtype=torch.bfloat16,
                 page_size: int = 64, device="cuda") -> None:
        self.num_layers, self.num_blocks, self.batch_size, self.max_length = num_layers, num_blocks, batch_size, max_length
        self.kv_heads, self.head_dim, self.dtype, self.page_size = kv_heads, head_dim, dtype, page_size
        shape = (num_layers, num_blocks + 1, page_size, kv_heads, head_dim)
        self.k_cache = torch.zeros(shape, device=device, dtype=dtype)
        self.v_cache = torch.zeros(shape, device=device, dtype=dtype)
        self.block_table = torch.full((batch_size, (max_length + page_size - 1) // page_size), -1, dtype=torch.int32, device=device)
        self.kv_lens = torch.zeros(batch_size, dtype=torch.int32, device=device)
        self.refs = torch.zeros(num_blocks, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)

    def layer(self, layer_idx: int):
        """(k pages, v pages) of one layer: [num_blocks + 1, page, kv_heads, head_dim]."""
        return self.k_cache[layer_idx], self.v_cache[layer_idx]

    def fork(self, src, dst) -> None:
        """Rows `dst[i]` continue what rows `src[i]` hold (``ops.fork_pages``); no data moves."""
        ops.fork_pages(self.block_table, self.kv_lens, self.refs, src, dst, self.page_size)

    def reserve(self, count, check: bool = True) -> None:
        """Room for `count` more tokens (a number, or int32 [batch]) in every row (``ops.reserve_pages``). ``check``: wait for the outcome and
        raise where there are too few pages; without it (inside a capture) ``status`` keeps the worst outcome until the next ``check``."""
        ops.reserve_pages(self.block_table, self.kv_lens, self.refs, count, (self.k_cache, self.v_cache), dim=1, status=self.status, keep=True)
        if check:
            self.check()

    def check(self) -> None:
        """Raise if a ``reserve`` since the last check found too few pages, a row that would outgrow its table or one without a page for its last token (it
        has changed nothing then). Rows that were advanced all the same count tokens that no page holds: ``trim`` or ``free`` them."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise RuntimeError("PagePool: " + {1: "too few free pages", 2: "a row would exceed max_length"}.get(code, "a row has no page for its last token"))

    def slots(self, count: int) -> torch.Tensor:
        """Flat slot (page * page_size + offset) of the next `count` tokens of every row -> int64 [batch * count]. What has no room is sent to the spare
        page: positions without a page, and those in a page that other rows hold too (their tokens may lie there: a row that paused, or whose
        ``reserve`` failed, has got no copy of it). So forks come before the ``reserve`` of a step."""
        pos = self.kv_lens[:, None].to(torch.int64) + torch.arange(count, device=self.kv_lens.device)[None, :]
        at = pos // self.page_size
        blk = self.block_table.gather(1, at.clamp_max(self.block_table.shape[1] - 1)).to(torch.int64)
        alone = self.refs[blk.clamp(0, self.num_blocks - 1)] <= 1
        blk = torch.where((blk >= 0) & (at < self.block_table.shape[1]) & alone, blk, self.num_blocks)
        return (blk * self.page_size + pos % self.page_size).reshape(-1)

    def prefix_table(self, shared: int, tokens: int = 1) -> torch.Tensor:
        """Pages of the first row that attends beyond its first `shared` keys with all its last `tokens` tokens -> int32 [max_blocks], for
        ``ops.shared_prefix_attention``: row 0, its default, may have ended. Of this step: pages change with ``trim``, ``free`` and ``compact``."""
        row = (self.kv_lens - tokens + 1 >= shared).to(torch.int32).argmax()
        return self.block_table.index_select(0, row.view(1))[0]

    def advance(self, count) -> None:
        """The next `count` tokens (a number, or int32 [batch]) of every row have been written."""
        self.kv_lens += count

    def trim(self, lens: torch.Tensor, rows=None) -> None:
        """Rows keep their first `lens` tokens (``ops.trim_pages``)."""
        ops.trim_pages(self.block_table, self.kv_lens, self.refs, self.page_size, lens, rows)

    def free(self, rows) -> None:
        """Rows give back all they hold."""
        ops.trim_pages(self.block_table, self.kv_lens, self.refs, self.page_size, None, rows)

    def compact(self) -> None:
        """The pages in use move to the front of the caches (``ops.compact_pages``)."""
        ops.compact_pages(self.block_table, self.refs, (self.k_cache, self.v_cache), dim=1, out=(self.block_table, self.refs))
