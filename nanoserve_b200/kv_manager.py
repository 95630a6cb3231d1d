"""KV manager: how the scheduler and the engine get KV memory for a request.

`PagedKVManager` keeps the reference's two protocols (nanoserve/kv_manager.py:70-202):
  scheduler side  can_ever_fit / can_admit / admit / try_append / free
  engine side     begin_step / seq_input / decode_meta / forward_kwargs / graph_inputs / commit / usage
and makes the same integer decisions (block ids, slots, prefix hits, watermark).

What is new is `step_records`: instead of building Python lists of slots / tables / lengths and uploading
them as tensors every step, the engine sends one small packed record per scheduled sequence (seat, cached
tokens, new tokens, token offset) plus the block-table entries appended since the last step; a device kernel
expands that into the graph's static buffers. Each admitted request holds a "seat" = one row of the
device-resident block-table mirror.
"""
from __future__ import annotations

import torch

from nanoserve_b200.kv_cache import BlockTable, PagedKVCache, PrefixCachingAllocator
from nanoserve_b200.model import DecodeMeta, ModelConfig, SeqInput


class PagedKVManager:
    kind = "paged"

    def __init__(self, cfg: ModelConfig, budget_tokens: int, block_size: int = 16, device="cuda",
                 dtype=torch.bfloat16, watermark: float = 0.01, attn_backend: str = "native",
                 prefix_caching: bool = False, max_seats: int = 256, kv_dtype=None):
        self.pool = PagedKVCache.from_token_budget(cfg, budget_tokens, block_size, device, dtype, kv_dtype)
        self.block_size = block_size
        self.device = device
        self.attn_backend = attn_backend
        self.prefix_caching = prefix_caching
        self.alloc = PrefixCachingAllocator(self.pool.allocator, block_size) if prefix_caching else self.pool.allocator
        self.prefix_query_tokens = 0
        self.prefix_hit_tokens = 0
        # a few blocks stay free at admission so a fresh request does not force a preemption on its first
        # decode step [kv_manager.py:88-90]
        self.watermark_blocks = int(watermark * self.pool.num_blocks)
        self._slots: list[int] = []
        # seats: rows of the device block-table mirror
        self.max_seats = max_seats
        self._free_seats = list(range(max_seats - 1, -1, -1))
        self._synced = [0] * max_seats            # table entries of each seat already sent to the device

    @property
    def num_free_blocks(self) -> int:
        return self.alloc.num_free

    def reset_stats(self) -> None:
        self.prefix_query_tokens = self.prefix_hit_tokens = 0

    def _blocks_for(self, n_tokens: int) -> int:
        return -(-n_tokens // self.block_size)

    def _hits(self, seq) -> list[int]:
        """Cached blocks of the longest known prefix, leaving at least one token to compute (its logits are
        needed) [kv_manager.py:101-107]."""
        if not self.prefix_caching:
            return []
        toks = seq.prompt_ids + seq.output_ids
        return self.alloc.lookup(toks, max_blocks=(len(toks) - 1) // self.block_size)

    # ---- scheduler side ---------------------------------------------------------------------------------
    def can_ever_fit(self, n_tokens: int) -> bool:
        return self._blocks_for(n_tokens) <= self.pool.num_blocks

    def can_admit(self, seq) -> bool:
        hits = self._hits(seq)
        # hit blocks cost nothing new, but those parked in the LRU list stop being free once pinned
        parked = sum(1 for b in hits if self.alloc.ref.get(b, 0) == 0)
        need = self._blocks_for(seq.step_cost) - len(hits) + parked
        return need <= self.num_free_blocks - self.watermark_blocks

    def admit(self, seq) -> None:
        table = BlockTable(self.block_size)
        if self.prefix_caching:
            hits = self._hits(seq)
            self.prefix_query_tokens += seq.num_tokens
            if hits:
                self.alloc.pin(hits)
                table.blocks = list(hits)
                table.num_hashed = len(hits)
                table.num_tokens = len(hits) * self.block_size
                table.prefix_node = self.alloc.node_of[hits[-1]]
                seq.num_cached = table.num_tokens
                self.prefix_hit_tokens += table.num_tokens
        seq.block_table = table
        table.reserve(seq.step_cost, self.alloc)
        if not self._free_seats:
            raise RuntimeError(f"more than {self.max_seats} requests admitted at once: raise max_seats")
        seq.seat = self._free_seats.pop()
        seq.token_on_device = False
        self._synced[seq.seat] = 0

    def try_append(self, seq) -> bool:
        bt = seq.block_table
        if bt.num_tokens < len(bt.blocks) * bt.block_size:
            return True                      # the next token fits the last block (15 of 16 decode steps): nothing to reserve
        if bt.blocks_needed(1) > self.num_free_blocks:
            return False
        bt.reserve(1, self.alloc)
        return True

    def free(self, seq) -> None:
        if seq.block_table is not None:
            seq.block_table.release(self.alloc)
            seq.block_table = None
        if seq.seat >= 0:
            self._free_seats.append(seq.seat)
            seq.seat = -1
            seq.token_on_device = False

    # ---- engine side: packed records for the device metadata kernel -----------------------------------------
    def step_records(self, scheduled, chunks):
        """For one step: (records, appends, token_ids) as flat int lists.
        records: 4 ints per sequence (seat, cached tokens, new tokens, offset into token_ids or -1 = "the token
        sampled last step, still on the device"); appends: 3 ints per new block-table entry (seat, index, block)."""
        records: list[int] = []
        appends: list[int] = []
        token_ids: list[int] = []
        synced = self._synced
        for seq, n in zip(scheduled, chunks):
            seat, table = seq.seat, seq.block_table
            blocks = table.blocks
            have = synced[seat]
            if have < len(blocks):
                for j in range(have, len(blocks)):
                    appends += (seat, j, blocks[j])
                synced[seat] = len(blocks)
            ctx = seq.num_cached
            if n == 1 and seq.token_on_device and seq.remaining == 1:
                records += (seat, ctx, 1, -1)
            else:
                records += (seat, ctx, n, len(token_ids))
                token_ids += seq.step_tokens(n)[0]
        return records, appends, token_ids

    # ---- engine side: the reference's host-list protocol (kept for inspection and parity tests) ----------
    def begin_step(self) -> None:
        self._slots = []
        self._offset = 0
        self._dec_idx, self._dec_tables, self._dec_lens = [], [], []

    def seq_input(self, seq, n_tokens: int) -> SeqInput:
        table = seq.block_table
        self._slots += table.slots(n_tokens)
        ctx = table.num_tokens
        is_decode = n_tokens == 1 and ctx > 0
        if is_decode:
            self._dec_idx.append(self._offset)
            self._dec_tables.append(table.blocks)
            self._dec_lens.append(ctx + 1)
        self._offset += n_tokens
        return SeqInput(n_tokens, block_table=list(table.blocks), ctx_len=ctx, use_kernel=is_decode)

    def decode_meta(self) -> DecodeMeta | None:
        if not self._dec_idx:
            return None
        width = max(len(t) for t in self._dec_tables)
        rows = [t + [0] * (width - len(t)) for t in self._dec_tables]
        return DecodeMeta(token_idx=torch.tensor(self._dec_idx, device=self.device),
                          block_tables=torch.tensor(rows, dtype=torch.int32, device=self.device),
                          context_lens=torch.tensor(self._dec_lens, dtype=torch.int32, device=self.device))

    def forward_kwargs(self) -> dict:
        kw = {"paged": self.pool, "slot_mapping": torch.tensor(self._slots, device=self.device)}
        meta = self.decode_meta()
        if meta is not None:
            kw["decode_meta"] = meta
        return kw

    def graph_inputs(self) -> tuple[list[int], list[list[int]], list[int]]:
        return self._slots, self._dec_tables, self._dec_lens

    def commit(self, seq, n_tokens: int) -> None:
        table = seq.block_table
        table.commit(n_tokens)
        if self.prefix_caching and table.num_tokens // self.block_size > table.num_hashed:
            self.alloc.register(table, seq.prompt_ids + seq.output_ids)

    def usage(self, running) -> tuple[int, int]:
        used = held = 0
        for s in running:
            if s.block_table:
                used += s.block_table.num_tokens
                held += len(s.block_table.blocks)
        return used, held * self.block_size
