"""Keys and values of a batch of sequences, in blocks, on top of the ``torch.ops.npu.npu_paged_*`` operators.

What stands between the qkv projection and the output projection of a decode step::

    cache = PagedKVCache(batch, max_tokens, kv_heads, head_dim, budget=4096, quantized=True, device="cuda")
    cache.prefill(b, key, value)              # the prompt of sequence b, [tokens, kv_heads, head_dim]
    query, key = cache.rotate(query, key, cos_sin_cache)      # to the positions of the tokens that follow
    cache.append(key, value)                  # one new token per sequence, [batch, kv_heads, head_dim]
    out = cache.attend(query)                 # [batch, heads, head_dim]
    cache.evict()                             # back to the budget

Lengths live on the device, so a step of ``rotate``, ``append``, ``attend`` and ``evict`` can be captured in a graph and replayed.
"""
from __future__ import annotations

import torch

__all__ = ["PagedKVCache"]


class PagedKVCache:
    """``max_tokens``: what a sequence can hold at once.  ``quantized``: codes in place of ``dtype``, of ``bits`` 8 (int8, a float32
    scale per token and head) or 4 (eight in an int32 word, a scale and an offset; head_dim a multiple of 8).  ``budget``: the tokens
    that ``evict`` leaves, each key/value head choosing its own by the attention they got from ``attend``; the newest ``recent``
    (default: a quarter) always stay.  The cache needs room for at least one token beyond it.  Tokens of a prompt have got none before
    the first ``attend``: an ``evict`` before it keeps the recent tokens and the first ones.

    Tensors on ``device``: ``key_cache``, ``value_cache`` [blocks, block_size, kv_heads, head_dim] (4 bits: head_dim / 8) and, with
    codes, ``key_scale`` and ``value_scale``, with 4 bits also ``key_offset`` and ``value_offset``, without the last dimension; all
    stored so that the tokens of one head of a block follow each other; ``block_table`` [batch, blocks per sequence], which an
    allocator of blocks may rewrite; ``context_lens`` [batch]; with a budget ``attn_sums`` and ``positions``
    [batch, kv_heads, capacity] and ``next_position`` [batch].

    A call that would overfill a sequence raises, as far as the host knows the lengths: replays of a captured step pass it by.
    What does not fit then is not written and gets no position, and a length stays at the capacity.  ``append`` takes a token for
    every sequence; one that has ended is cleared, so that it does not fill up.
    """

    def __init__(self, batch: int, max_tokens: int, kv_heads: int, head_dim: int, *, block_size: int = 64, budget: int | None = None,
                 recent: int | None = None, quantized: bool = False, device=None, dtype=torch.bfloat16, bits: int = 8) -> None:
        if min(batch, max_tokens, kv_heads, head_dim, block_size) < 1:
            raise ValueError("batch, max_tokens, kv_heads, head_dim and block_size should be at least 1, but now they are "
                             f"{batch}, {max_tokens}, {kv_heads}, {head_dim}, {block_size}.")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"dtype should be torch.bfloat16 or torch.float16, but now it is {dtype}.")
        if bits not in (4, 8) or (bits == 4 and not quantized):
            raise ValueError(f"bits should be 8, or 4 with quantized=True, but now it is {bits} with quantized={quantized}.")
        if bits == 4 and head_dim % 8:
            raise ValueError(f"head_dim should be a multiple of 8 with 4 bits, but now it is {head_dim}.")
        per_sequence = -(-max_tokens // block_size)
        self.capacity = per_sequence * block_size
        if budget is None and recent is not None:
            raise ValueError("recent needs a budget.")
        if budget is not None and not 0 < budget < self.capacity:
            raise ValueError(f"budget should be at least 1 and below the {self.capacity} tokens that a sequence can hold, but now it is {budget}.")
        self.budget, self.recent = budget, budget // 4 if budget is not None and recent is None else recent
        if budget is not None and not 0 <= self.recent <= budget:
            raise ValueError(f"recent should be between 0 and the budget, but now it is {recent}.")
        self.block_size, self.dtype, self.quantized, self.bits = block_size, dtype, quantized, bits if quantized else 16
        blocks = batch * per_sequence

        def heads_first(*row, dtype):
            return torch.zeros(blocks, kv_heads, block_size, *row, dtype=dtype, device=device).transpose(1, 2)

        for name in ("key", "value"):
            row, kind = {4: (head_dim // 8, torch.int32), 8: (head_dim, torch.int8), 16: (head_dim, dtype)}[self.bits]
            setattr(self, name + "_cache", heads_first(row, dtype=kind))
            setattr(self, name + "_scale", heads_first(dtype=torch.float32) if quantized else None)
            setattr(self, name + "_offset", heads_first(dtype=torch.float32) if self.bits == 4 else None)
        self.block_table = torch.arange(blocks, dtype=torch.int32, device=device).view(batch, per_sequence)
        self.context_lens = torch.zeros(batch, dtype=torch.int32, device=device)
        kept = budget is not None
        shape = (batch, kv_heads, self.capacity)
        self.attn_sums = torch.zeros(shape, dtype=torch.float32, device=device) if kept else None
        self.positions = torch.full(shape, -1, dtype=torch.int32, device=device) if kept else None
        self.next_position = torch.zeros(batch, dtype=torch.int32, device=device) if kept else None
        self._held = [0] * batch                 # tokens of a sequence at most, as far as the host has seen

    def _room(self, sequences, tokens: int) -> None:
        full = [b for b in sequences if self._held[b] + tokens > self.capacity]
        if full:
            raise RuntimeError(f"sequence {full[0]} holds up to {self._held[full[0]]} tokens, {tokens} more do not fit into {self.capacity}")

    def _count(self, sequences, tokens: int) -> None:
        for b in sequences:
            self._held[b] += tokens

    def _params(self) -> dict:
        """Scales and offsets, as the operators take them."""
        scales = {"key_scale": self.key_scale, "value_scale": self.value_scale}
        return scales if self.bits != 4 else {**scales, "key_offset": self.key_offset, "value_offset": self.value_offset}

    def _slots(self, table, place):
        """Slots, in 64 bits, of `place` (int64 [tokens], below the capacity) of the sequences in the rows of `table`."""
        return torch.add(place % self.block_size, table.gather(1, (place // self.block_size)[:, None])[:, 0], alpha=self.block_size)

    def _write(self, key, value, table, place, fits) -> None:
        """key, value of the tokens that go to `place` of the sequence in their row of `table`, if they fit."""
        slots = torch.where(fits, self._slots(table, place), -1)  # (a replayed step does not pass through _room)
        torch.ops.npu.npu_paged_cache_write(key, value, self.key_cache, self.value_cache, slots, **self._params())

    def rotate(self, query: torch.Tensor, key: torch.Tensor, cos_sin_cache: torch.Tensor, *, mrope_section: list[int] | None = None,
               rotary_mode: str = "half", offset: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """query and key of the tokens that ``append`` takes next, turned to their positions by ``npu_mrope``.  A sequence's position is
        the number of tokens that it was given, on every axis of ``mrope_section``; ``offset`` [batch] is added to it (an image takes
        fewer positions than it has tokens)."""
        at = self.context_lens if self.budget is None else self.next_position
        at = at if offset is None else at + offset
        if mrope_section is not None:
            at = at.expand(len(mrope_section), -1)
        return torch.ops.npu.npu_mrope(at, query, key, cos_sin_cache, query.shape[-1], mrope_section=mrope_section, rotary_mode=rotary_mode)

    def append(self, key: torch.Tensor, value: torch.Tensor) -> None:
        """One new token for every sequence."""
        everyone = range(len(self._held))
        self._room(everyone, 1)
        fits = self.context_lens < self.capacity
        place = self.context_lens.clamp(max=self.capacity - 1).long()
        self._write(key, value, self.block_table, place, fits)
        self._count(everyone, 1)                                  # (the operator has taken them)
        if self.budget is not None:
            at = place[:, None, None].expand(-1, self.positions.shape[1], 1)
            # (of a token that does not fit: the last place keeps its position)
            self.positions.scatter_(2, at, torch.where(fits[:, None], self.next_position[:, None], self.positions[:, :, -1])[..., None])
            self.next_position += fits
        self.context_lens += fits

    def prefill(self, sequence: int, key: torch.Tensor, value: torch.Tensor) -> None:
        """Tokens of one sequence behind those that it has."""
        tokens = key.shape[0]
        self._room([sequence], tokens)
        place = self.context_lens[sequence] + torch.arange(tokens, device=self.context_lens.device)
        self._write(key, value, self.block_table[sequence].expand(tokens, -1), place.clamp(max=self.capacity - 1), place < self.capacity)
        self._count([sequence], tokens)
        held = (self.context_lens[sequence] + tokens).clamp(max=self.capacity)
        if self.budget is not None:
            at = place.clamp(max=self.capacity).expand(self.positions.shape[1], -1)
            position = self.next_position[sequence] + torch.arange(tokens, dtype=torch.int32, device=at.device)
            row = torch.nn.functional.pad(self.positions[sequence], (0, 1))       # (what does not fit goes to the place behind)
            self.positions[sequence] = row.scatter_(1, at, position.expand_as(at))[:, :-1]
            self.next_position[sequence] += held - self.context_lens[sequence]
        self.context_lens[sequence] = held

    def attend(self, query: torch.Tensor, *, scale_value: float | None = None, atten_mask: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of one token per sequence over what the sequence holds; with a budget the weights are summed."""
        return torch.ops.npu.npu_paged_decode_attention(query, self.key_cache, self.value_cache, self.block_table, self.context_lens,
                                                        **self._params(), scale_value=scale_value, atten_mask=atten_mask,
                                                        attn_sums=self.attn_sums)[0]

    def evict(self) -> None:
        """Sequences of more than ``budget`` tokens are brought down to it."""
        if self.budget is None:
            raise RuntimeError("the cache has no budget")
        lens, sums, positions = torch.ops.npu.npu_paged_cache_evict(self.key_cache, self.value_cache, self.block_table, self.context_lens,
                                                                    self.attn_sums, self.positions, self.budget, self.recent,
                                                                    **self._params())
        self.context_lens.copy_(lens)
        self.attn_sums.copy_(sums)
        self.positions.copy_(positions)
        capturing = self.context_lens.is_cuda and torch.cuda.is_current_stream_capturing()        # (replays may fill it up to the budget)
        self._held = [self.budget if capturing else min(held, self.budget) for held in self._held]

    def read(self, sequence: int, start: int, stop: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values in places [start, stop) of one sequence, as ``dtype``: what a later chunk of a prompt attends to."""
        if not 0 <= start <= stop <= self.capacity:
            raise IndexError(f"places [{start}, {stop}) of {self.capacity}")
        place = torch.arange(start, stop, device=self.block_table.device)
        slots = self._slots(self.block_table[sequence].expand(stop - start, -1), place)
        return torch.ops.npu.npu_paged_cache_read(self.key_cache, self.value_cache, slots, **self._params(), dtype=self.dtype)

    def clear(self, sequence: int) -> None:
        """Makes room for a new sequence."""
        self.context_lens[sequence] = 0
        self._held[sequence] = 0
        if self.budget is not None:
            self.attn_sums[sequence] = 0
            self.positions[sequence] = -1
            self.next_position[sequence] = 0
