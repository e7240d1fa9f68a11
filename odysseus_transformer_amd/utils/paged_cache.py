"""A key / value cache in pages for decoding many sequences at once.

The reference hands its keys and values to the host's cache (decoder/odysseus.py:215-220), which holds one sequence (or a padded
batch) in a row and copies all of it with every token.  Here sequences own pages of a pool by a table: a sequence grows without
moving, ends without leaving a hole, and lengths differ freely.  The attention module and the decoder layer of decoder/odysseus.py
take it as their `past_key_value(s)`:

    cache = PagedKVCache(layers, pages, page_size=64, max_sequences=8, max_length=4096, n_kv_heads=8, head_dim=128, device="cuda")
    with torch.no_grad():
        cache.begin([300, 17])                    # sequences 0 and 1: so many new tokens each, padded on the left to 300
        y = layer(x, past_key_values=cache)       # x (8, 300, hidden): one row of the batch for each of max_sequences
        cache.begin(1)                            # a token more of every sequence that has some
        y = layer(x1, past_key_values=cache)      # x1 (8, 1, hidden)

`page_table`, `lengths`, `new_tokens` and `position_ids` are device tensors that stay where they are and are rewritten by begin(): a step
that was captured into a graph is replayed after it.  A step that runs again before the next begin() (a rehearsal in front of a capture) writes its tokens'
rows anew.  begin() works on the host, once a step for all layers, on the stream that runs the steps; it
refuses to be captured itself, as free() and truncate() do.
"""
from __future__ import annotations

from typing import List, Sequence, Union

import torch


class PagedKVCache:
    is_compileable = False   # a host model asks

    def __init__(self, num_layers: int, num_pages: int, *, max_sequences: int, max_length: int, n_kv_heads: int, head_dim: int, page_size: int = 64,
                 dtype=torch.bfloat16, device="cuda"):
        for name, value in (("num_layers", num_layers), ("num_pages", num_pages), ("max_sequences", max_sequences), ("max_length", max_length),
                            ("n_kv_heads", n_kv_heads), ("head_dim", head_dim)):
            if value <= 0:
                raise ValueError(f"{name} must be positive, got {value}")
        if page_size < 8 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 8 on, got {page_size}")
        self.num_layers, self.num_pages, self.page_size = num_layers, num_pages, page_size
        self.max_sequences, self.max_length = max_sequences, max_length
        device = torch.device(device)
        # heads outside of rows: what a block reads of a page is one piece (64 sequences of up to 8192 tokens in pages of 64 171 us a layer, 197 with rows of all heads)
        pools = [torch.empty((2, num_pages, n_kv_heads, page_size, head_dim), dtype=dtype, device=device) for _ in range(num_layers)]
        self._layers = [(p[0].transpose(1, 2), p[1].transpose(1, 2)) for p in pools]
        self._columns = (max_length + page_size - 1) // page_size
        self.page_table = torch.full((max_sequences, self._columns), -1, dtype=torch.int32, device=device)
        self._counts = torch.zeros((2, max_sequences), dtype=torch.int32, device=device)
        self.lengths, self.new_tokens = self._counts[0], self._counts[1]
        self.position_ids = None                                   # (max_sequences, n) int64 of the present step, 0 for padding; None: there is none
        self._positions = torch.zeros(max_sequences * max_length, dtype=torch.int64, device=device)
        self._owned: List[List[int]] = [[] for _ in range(max_sequences)]
        self._free = list(range(num_pages - 1, -1, -1))
        self._length = [0] * max_sequences                         # tokens, those of the present step included
        self._new = [0] * max_sequences
        self.fresh = False                                         # the present step's tokens are all that is there, as many of every sequence

    # ------------------------------------------------------------------ steps
    def begin(self, tokens: Union[int, Sequence[int]]) -> int:
        """Makes room for the next step's new tokens: as many of each sequence as `tokens` says -- fewer numbers than max_sequences leave
        the others out -- or, for one number, of every sequence that holds some.  Returns n, the most of them; the step's inputs are
        (max_sequences, n, ...), shorter ones padded on the left.  Nothing changes if there are not enough pages (MemoryError) or a
        sequence would outgrow max_length (ValueError)."""
        self._not_captured()
        if not hasattr(tokens, "__iter__"):
            new = [int(tokens) if length else 0 for length in self._length]
        else:
            new = [int(t) for t in tokens]
            if len(new) > self.max_sequences:
                raise ValueError(f"{len(new)} sequences, the cache is for {self.max_sequences}")
            new += [0] * (self.max_sequences - len(new))
        if min(new) < 0:
            raise ValueError(f"numbers of new tokens must not be negative, got {tokens}")
        n = max(new)
        if n == 0:
            raise ValueError("a step without a new token: give the numbers of new tokens as a list to begin sequences")
        after = [length + t for length, t in zip(self._length, new)]
        if max(after) > self.max_length:
            raise ValueError(f"sequence {after.index(max(after))} would have {max(after)} tokens, the cache is for {self.max_length}")
        wanted = [self._pages_for(a) - len(owned) if t else 0 for a, t, owned in zip(after, new, self._owned)]
        if sum(wanted) > len(self._free):
            raise MemoryError(f"{sum(wanted)} pages wanted, {len(self._free)} of {self.num_pages} are free")
        self.fresh = all(t == n and a == n for a, t in zip(after, new))
        rows, columns, pages = [], [], []
        for s, count in enumerate(wanted):
            for _ in range(count):
                page = self._free.pop()
                rows.append(s), columns.append(len(self._owned[s])), pages.append(page)
                self._owned[s].append(page)
        self._length, self._new = after, new
        device = self.page_table.device
        if pages:
            entries = torch.tensor([rows, columns, pages], dtype=torch.int64).to(device)
            self.page_table[entries[0], entries[1]] = entries[2].to(torch.int32)
        self._write_counts()
        self.position_ids = self._positions[:self.max_sequences * n].view(self.max_sequences, n)
        first = self._counts[0].to(torch.int64)[:, None] - n
        self.position_ids.copy_((first + torch.arange(n, device=device)[None, :]).clamp_(min=0))
        return n

    def free(self, sequence: int) -> None:
        """Ends a sequence: its pages go back to the pool, and its row takes no part until it begins anew."""
        self.truncate(sequence, 0)

    def truncate(self, sequence: int, length: int) -> None:
        """Takes back tokens behind the first `length` of a sequence (proposed ones that were not accepted), after their step, and the pages that they
        leave empty.  The step is over then: begin() comes before the next one."""
        self._not_captured()
        if not 0 <= sequence < self.max_sequences:
            raise ValueError(f"sequence {sequence} of {self.max_sequences}")
        if not 0 <= length <= self._length[sequence]:
            raise ValueError(f"sequence {sequence} has {self._length[sequence]} tokens, {length} of them cannot be kept")
        keep, owned = self._pages_for(length), self._owned[sequence]
        if len(owned) > keep:
            self.page_table[sequence, keep:] = -1
            self._free.extend(reversed(owned[keep:]))
            del owned[keep:]
        if length and self._new[sequence]:
            self.position_ids = None   # modules ask for it; the storage stays
        self._length[sequence], self._new[sequence], self.fresh = length, 0, False
        self._write_counts()

    def _not_captured(self) -> None:
        if self.page_table.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("PagedKVCache: the book-keeping of a step belongs in front of its replay, not into a captured graph")

    def _pages_for(self, length: int) -> int:
        return (length + self.page_size - 1) // self.page_size

    def _write_counts(self) -> None:
        # one copy from pageable memory, which has been read when it returns
        self._counts.copy_(torch.tensor([[a if t else 0 for a, t in zip(self._length, self._new)], self._new], dtype=torch.int32))

    # ------------------------------------------------------------------ what layers and callers ask
    def layer(self, index: int):
        """(k_pages, v_pages) of a layer, (pages, page_size, kv heads, head_dim) each."""
        return self._layers[index]

    def sequence_lengths(self) -> List[int]:
        """Tokens of every sequence, those of the present step included."""
        return list(self._length)

    def free_pages(self) -> int:
        return len(self._free)

    def get_seq_length(self, layer_idx: int = 0) -> int:
        """What a host model takes for the number of earlier tokens: the most of any sequence, without the present step's.  (It counts positions from
        there; the attention module goes by those of the cache.)"""
        return max(a - t for a, t in zip(self._length, self._new))

    def get_query_offset(self, layer_idx: int = 0) -> int:
        return self.get_seq_length(layer_idx)

    def get_mask_sizes(self, query_length, layer_idx: int = 0):
        return self.get_seq_length(layer_idx) + int(query_length), 0
