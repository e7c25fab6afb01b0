"""Generation over a paged cache: many sequences, each at its own length.

``Parrot.prefill`` / ``decode_step`` keep one dense cache per batch and one
position for all of its rows.  Here the layers share pools of pages
(``bridge.PagedKV``), a sequence owns the pages its tokens fill, and
``Parrot.extend`` appends any number of new tokens to any of the sequences in
one pass: prompts, pieces of prompts and single tokens side by side.  The host
keeps the pages and the lengths; the kernels read both from device memory.

    state = model.paged_state(sequences=8, pages=256, kv_dtype=torch.float8_e4m3fn)
    logits = model.extend(torch.cat([prompt_a, prompt_b]), [len(prompt_a), len(prompt_b)], state,
                          sequences=[0, 1])
    ids, logp = model.sample(logits, uniform, temperature=0.8, top_p=0.9)
    logits = model.extend(ids[:, 0], [1, 1], state, sequences=[0, 1])
    state.release(1)                     # its pages may be taken by another sequence
    assert state.read_status()[0] == 0   # nothing was out of range, no wait ran out (synchronises)
"""
from __future__ import annotations

from typing import Sequence

import torch
from torch import Tensor

from . import bridge


class PagedState:
    """The pools of every layer, and which sequence owns which pages."""

    def __init__(self, cfg, sequences: int, pages: int, page_size: int, kv_dtype: torch.dtype,
                 sink_tokens: int, device, is_local: Sequence[bool]):
        if sequences < 1 or pages < 1:
            raise ValueError("sequences and pages must be positive")
        if kv_dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            raise ValueError("kv_dtype must be bfloat16 or float8_e4m3fn")
        if sink_tokens < 0:
            raise ValueError("sink_tokens must be >= 0")
        for name in ("head_dim", "kv_latent_dim"):
            if getattr(cfg, name) not in bridge.PAGED_HEAD_DIMS:
                raise ValueError(f"a paged cache needs {name} in {bridge.PAGED_HEAD_DIMS}")
        if page_size not in bridge.PAGE_SIZES:
            raise ValueError(f"page_size must be one of {bridge.PAGE_SIZES}")
        self.page_size, self.sink_tokens, self.device = page_size, sink_tokens, torch.device(device)
        self.max_positions = cfg.max_seq_len
        width = -(-cfg.max_seq_len // page_size)
        self.layers = [bridge.PagedKV.allocate(
            pages, cfg.n_kv_heads if local else 1, page_size,
            cfg.head_dim if local else cfg.kv_latent_dim, self.device, kv_dtype, latent=not local)
            for local in is_local]
        self.lengths = [0] * sequences
        self._free = list(range(pages - 1, -1, -1))
        self._owned: list[list[int]] = [[] for _ in range(sequences)]
        self._table = torch.full((sequences, width), -1, dtype=torch.int32)
        self.status = torch.zeros(4, dtype=torch.int32, device=self.device)

    @torch.inference_mode()
    def read_status(self, clear: bool = False) -> list[int]:
        """The status word {code, site, info, 0} of the steps so far (synchronises): code 0 is ok,
        1 a wait that ran out, 2 a page, position or length out of range.  The first entry stays
        until it is read with ``clear``."""
        word = self.status.tolist()
        if clear:
            self.status.zero_()
        return word

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _index(self, sequence: int) -> int:
        b = int(sequence)
        if not 0 <= b < len(self.lengths):
            raise ValueError(f"sequences must be in [0, {len(self.lengths)}), got {b}")
        return b

    def _step(self, sequences: Sequence[int], counts: Sequence[int]) -> tuple[list[int], list[int]]:
        """The step's sequences and counts as numbers, checked."""
        seqs, counts = [self._index(b) for b in sequences], [int(n) for n in counts]
        if len(seqs) != len(counts) or not seqs:
            raise ValueError("one count for each sequence, and at least one sequence")
        if len(set(seqs)) != len(seqs):
            raise ValueError("sequences must be different")
        if min(counts) < 0:
            raise ValueError("counts must be >= 0")
        return seqs, counts

    def pages_of(self, sequence: int) -> list[int]:
        return list(self._owned[self._index(sequence)])

    def reserve(self, sequences: Sequence[int], counts: Sequence[int]) -> None:
        """Pages for ``counts[i]`` more tokens of sequence ``sequences[i]``; all or none."""
        sequences, counts = self._step(sequences, counts)
        need = []
        for b, n in zip(sequences, counts):
            if self.lengths[b] + n > self.max_positions:
                raise ValueError(f"sequence {b} would exceed max_seq_len model positions")
            need.append(max(0, -(-(self.lengths[b] + n) // self.page_size) - len(self._owned[b])))
        if sum(need) > len(self._free):
            raise RuntimeError(f"the paged cache has {len(self._free)} free pages, {sum(need)} are needed")
        for b, n in zip(sequences, need):
            for _ in range(n):
                page = self._free.pop()
                self._table[b, len(self._owned[b])] = page
                self._owned[b].append(page)

    def release(self, sequence: int) -> None:
        """Forget a sequence; its pages are free again."""
        sequence = self._index(sequence)
        self._free.extend(reversed(self._owned[sequence]))
        self._owned[sequence] = []
        self._table[sequence] = -1
        self.lengths[sequence] = 0

    def with_tokens(self, sequences: Sequence[int], counts: Sequence[int]) -> tuple[list[int], list[int]]:
        """Of a step's sequences those that have new tokens, with their counts."""
        step = [(b, n) for b, n in zip(*self._step(sequences, counts)) if n]
        return [b for b, _ in step], [n for _, n in step]

    def batch(self, sequences: Sequence[int], counts: Sequence[int]) -> "PagedBatch":
        """Device lists of a step that appends ``counts[i]`` tokens to ``sequences[i]``
        (reserves their pages; the lengths grow when the step is done).  Sequences
        without new tokens may be among them, but count when the attention kernel is
        chosen by the tokens of a sequence: ``with_tokens`` leaves them out."""
        seqs, counts = self._step(sequences, counts)
        if sum(counts) == 0:
            raise ValueError("one of the counts must be positive")
        self.reserve(seqs, counts)
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        lengths = [self.lengths[b] + n for b, n in zip(seqs, counts)]
        # one copy: starts, lengths, then the sequences' rows of the table
        width = max(1, max(-(-n // self.page_size) for n in lengths))
        table = self._table[seqs, :width]
        ints = torch.cat([torch.tensor(starts + lengths, dtype=torch.int32), table.reshape(-1)])
        ints = ints.to(self.device)
        n = len(seqs)
        return PagedBatch(ints[2 * n + 1:].view(n, width), ints[:n + 1], ints[n + 1:2 * n + 1],
                          starts[-1], self.status)

    def advance(self, sequences: Sequence[int], counts: Sequence[int]) -> None:
        """The tokens of a step are in the cache: on the pages that ``reserve`` gave them."""
        sequences, counts = self._step(sequences, counts)
        for b, n in zip(sequences, counts):
            if self.lengths[b] + n > len(self._owned[b]) * self.page_size:
                raise ValueError(f"sequence {b} has no pages for {n} more tokens")
        for b, n in zip(sequences, counts):
            self.lengths[b] += n

    @torch.inference_mode()
    def dense(self, layer: int, sequences: Sequence[int], max_len: int | None = None):
        """A layer's cache of these sequences as dense bf16 (key, value or None),
        [sequences, kv heads, max_len, width], zeros past each length."""
        sequences = [self._index(b) for b in sequences]
        if not sequences:
            raise ValueError("at least one sequence")
        lengths = [self.lengths[b] for b in sequences]
        max_len = max(lengths) if max_len is None else max_len
        width = max(1, max(-(-n // self.page_size) for n in lengths))
        table = self._table[sequences, :width].to(self.device)
        return bridge.b200_paged_gather(self.layers[layer], table, torch.tensor(
            lengths, dtype=torch.int32, device=self.device), max_len, status=self.status)


class PagedBatch:
    """The device lists of one step (``bridge.b200_paged_*``), and where its calls report."""

    __slots__ = ("page_table", "query_start", "context_len", "tokens", "status")

    def __init__(self, page_table: Tensor, query_start: Tensor, context_len: Tensor, tokens: int,
                 status: Tensor | None = None):
        self.page_table, self.query_start, self.context_len = page_table, query_start, context_len
        self.tokens, self.status = tokens, status


def padded_rows(tokens: int) -> int:
    """Rows that a step of ``tokens`` tokens runs with: four sizes an octave from
    16 on, so that the per-size workspaces of the MoE blocks stay few."""
    if tokens <= 16:
        return tokens
    step = 1 << (tokens.bit_length() - 3)
    return -(-tokens // step) * step
