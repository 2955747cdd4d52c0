"""Packed batches: sequences of different lengths served in one step.

The uniform path (:class:`~memopt.kv_cache.PagedKVCache`) takes the same number
of tokens for every sequence and builds its tables in Python lists.  Here the
tokens of a batch lie behind one another (``[num_tokens, heads, head_dim]``)
and everything that depends on the lengths is built on the GPU:

* :class:`DevicePageTable` — block tables, lengths and the ring of free pages
  in device memory.  ``reserve`` appends tokens to rows and returns the
  batch's ``cu_seqlens``, slot mapping, positions and tables; ``truncate``
  gives pages back (a finished sequence, rejected draft tokens).  Pages are
  handed out in the order of the host free-list (:class:`PageTable`).  Nothing
  synchronises, so a step can be captured into a CUDA graph; ``check`` reports
  refused calls.
* :class:`RotaryPositions` — rotary positions with 1 to 4 axes (time, height,
  width), applied to q and k and fused with the write into an fp16 pool.
* :class:`PackedKVCache` — pages of the process-wide pool behind both:
  ``admit`` / ``prompt`` run a batch of whole prompts (causal attention over
  the packed tokens), ``extend`` / ``decode`` the steps after them (paged
  attention).

These operators serve; they carry no gradient and refuse inputs that ask for
one while gradients are recorded (serve under ``torch.no_grad()``).
"""
from __future__ import annotations

import contextlib
import gc
import threading
import weakref
from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple, Union

import torch

__all__ = ["DevicePageTable", "PackedBatch", "PackedKVCache", "RotaryPositions"]

_STATUS = (
    (1, "more new pages than free ones"),
    (2, "a row would exceed its block table"),
    (4, "a row out of range, or twice in a batch"),
    (8, "a negative length, more tokens than max_tokens, or a kept length past the row's"),
    (16, "lengths, ring or table entries out of range"),
)

Ints = Union[torch.Tensor, Sequence[int]]
_WHOLE = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)


def _device(device: Optional[torch.device]) -> torch.device:
    """With its index, as tensors have it; the current CUDA device by default."""
    dev = torch.device("cuda" if device is None else device)
    return torch.device("cuda", torch.cuda.current_device()) if dev.type == "cuda" and dev.index is None else dev


@dataclass
class PackedBatch:
    """What ``reserve`` built for a batch of rows (device tensors, int32)."""

    rows: torch.Tensor          # [B] table rows
    cu_seqlens: torch.Tensor    # [B + 1] first packed token of each sequence
    slot_mapping: torch.Tensor  # [max_tokens] slot of each new token, -1 past the last
    positions: torch.Tensor     # [max_tokens] position of each new token in its sequence, evicted tokens counted
    block_tables: torch.Tensor  # [B, max_blocks_per_seq]
    context_lens: torch.Tensor  # [B] lengths with the new tokens
    whole: bool = False         # the new tokens are the whole sequences
    attend_lens: Optional[torch.Tensor] = None  # [B] context_lens, 0 if the batch was refused


class DevicePageTable:
    """Block tables and free pages in device memory, one sequence per row of
    up to ``max_seq_len`` tokens (rounded up to whole pages).  ``pages``: those of the pool's ``num_blocks`` pages that the table may
    hand out, in this order (all of them by default)."""

    def __init__(self, num_blocks: int, block_size: int, max_seqs: int, max_seq_len: int,
                 device: Optional[torch.device] = None, pages: Optional[Sequence[int]] = None) -> None:
        if min(num_blocks, block_size, max_seqs, max_seq_len) <= 0:
            raise ValueError("DevicePageTable: num_blocks, block_size, max_seqs and max_seq_len must be > 0")
        ring = list(range(num_blocks)) if pages is None else list(pages)
        if len(set(ring)) != len(ring) or any(not 0 <= p < num_blocks for p in ring):
            raise ValueError("DevicePageTable: pages must be distinct pages of the pool")
        import memopt_C

        self._C = memopt_C
        self.num_blocks, self.block_size, self.max_seqs = num_blocks, block_size, max_seqs
        self.max_seq_len = max_seq_len
        self.device = _device(device)
        width = (max_seq_len + block_size - 1) // block_size

        def int32(value, *shape):
            return torch.full(shape, value, dtype=torch.int32, device=self.device)

        self.block_tables = int32(-1, max_seqs, width)
        self.context_lens = int32(0, max_seqs)
        self.position_offsets = int32(0, max_seqs)  # tokens that evictions took out of a row
        self.free_pages = torch.tensor(ring + [-1] * (num_blocks - len(ring)), dtype=torch.int32, device=self.device)
        self.pool_state = torch.tensor([0, len(ring), 0, 0], dtype=torch.int32, device=self.device)

    def ints(self, values: Ints) -> torch.Tensor:
        """Whole numbers as an int32 tensor on the table's device; what passes
        32 bits stays out of any range and is refused there.  Those of
        the host are copied from pinned memory, so the call does not wait for
        the stream; a graph would replay the copy of what is no longer there,
        so they are refused during a capture."""
        given = isinstance(values, torch.Tensor)
        if given and values.dtype == torch.int32 and values.device == self.device:
            return values
        pin = self.device.type == "cuda" and not (given and values.is_cuda)
        if pin and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("DevicePageTable: a captured call takes its rows and lengths as tensors of the GPU")
        if not given:
            values = torch.tensor(list(values), dtype=torch.int32, pin_memory=pin)
        elif values.dtype not in _WHOLE:
            raise TypeError(f"DevicePageTable: rows and lengths are whole numbers, not {values.dtype}")
        elif values.dtype == torch.int64:
            values = values.clamp(-(1 << 31), (1 << 31) - 1)
        if given and pin:
            values = values.to(torch.int32)
            # pin_memory gives pinned memory back as it is, and the caller may write there after the call
            values = (values.clone() if values.is_pinned() else values).pin_memory()
        return values.to(device=self.device, dtype=torch.int32, non_blocking=True)

    def reserve(self, rows: Ints, new_lens: Ints, max_tokens: Optional[int] = None) -> PackedBatch:
        """Appends ``new_lens[b]`` tokens to row ``rows[b]``.  ``max_tokens``
        sizes the per-token outputs (default: the sum of ``new_lens``, which
        must then be a Python sequence); the sum may be smaller, a larger one
        is refused.  A refused batch changes nothing (see :meth:`check`): its
        ``cu_seqlens`` are zero and its slots -1."""
        return self._reserve(rows, new_lens, max_tokens, False)

    def replace(self, rows: Ints, new_lens: Ints, max_tokens: Optional[int] = None) -> PackedBatch:
        """:meth:`reserve` for sequences that begin: what the rows held is
        given back first, unless the batch is refused."""
        return self._reserve(rows, new_lens, max_tokens, True)

    def _reserve(self, rows: Ints, new_lens: Ints, max_tokens: Optional[int], replace: bool) -> PackedBatch:
        if max_tokens is None:
            if isinstance(new_lens, torch.Tensor):
                raise ValueError("reserve: max_tokens is needed when new_lens is a tensor")
            max_tokens = sum(new_lens)
        r = self.ints(rows)
        cu, slots, pos, tables, lens, attend = self._C.reserve_rows(
            self.block_tables, self.context_lens, self.position_offsets, self.free_pages, self.pool_state, r,
            self.ints(new_lens), self.block_size, max_tokens, replace)
        return PackedBatch(r, cu, slots, pos, tables, lens, attend_lens=attend)

    def truncate(self, rows: Ints, keep_lens: Optional[Ints] = None) -> None:
        """Cuts each row to its first ``keep_lens`` tokens (None: to nothing)
        and gives the pages behind them back.  Positions go on from there:
        those of the tokens cut off are given out again."""
        keep = None if keep_lens is None else self.ints(keep_lens)
        self._C.truncate_rows(self.block_tables, self.context_lens, self.free_pages, self.pool_state,
                              self.ints(rows), keep, self.block_size)

    def release_pages(self, pages: torch.Tensor, counts: torch.Tensor) -> None:
        """Gives back the first ``counts[i]`` pages of each row of ``pages``
        (the ``freed_pages`` and ``freed_count`` of an exact eviction; both
        are cleared)."""
        n = torch.arange(min(pages.shape[0], 8192), dtype=torch.int32, device=self.device)
        for at in range(0, pages.shape[0], 8192):  # the most rows of a call
            some = slice(at, at + 8192)
            part = counts[some]
            self._C.truncate_rows(pages[some], part, self.free_pages, self.pool_state, n[:part.shape[0]], None, 1)

    def free_count(self) -> int:
        """Number of free pages (synchronises)."""
        return int(self.pool_state[1].item())

    def check(self) -> None:
        """Raises if a call since the last check was refused (synchronises)."""
        bits = int(self.pool_state[2].item())
        if bits == 0:
            return
        self.pool_state[2] = 0
        why = "; ".join(text for bit, text in _STATUS if bits & bit)
        if bits == 1:
            raise MemoryError(f"DevicePageTable: a call was refused: {why}")
        raise RuntimeError(f"DevicePageTable: a call was refused: {why}")


class RotaryPositions:
    """Rotary positions of the heads: ``rotary_dim`` leading dims turn (all of
    ``head_dim`` by default), pair i by ``base ** (-2i / rotary_dim)`` per
    position of its axis (or by ``inv_freq[i]``); ``sections`` share the pairs
    out among the axes, one axis by default."""

    def __init__(self, head_dim: int, base: float = 10000.0, rotary_dim: Optional[int] = None,
                 sections: Optional[Sequence[int]] = None, interleaved: bool = False,
                 inv_freq: Optional[torch.Tensor] = None, device: Optional[torch.device] = None) -> None:
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        pairs = rotary_dim // 2
        if rotary_dim <= 0 or rotary_dim > head_dim or rotary_dim % 16 != 0:
            raise ValueError("RotaryPositions: rotary_dim must be a multiple of 16, at most head_dim")
        self.sections: List[int] = [pairs] if sections is None else [int(s) for s in sections]
        if min(self.sections, default=-1) < 0 or sum(self.sections) != pairs or len(self.sections) > 4:
            raise ValueError(f"RotaryPositions: sections must be 1 to 4 counts that sum to {pairs}")
        if inv_freq is None:
            inv_freq = float(base) ** (-torch.arange(pairs, dtype=torch.float64) / pairs)
        if inv_freq.shape != (pairs,):
            raise ValueError(f"RotaryPositions: inv_freq must hold {pairs} values")
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, rotary_dim, interleaved
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.inv_freq = inv_freq.to(device=self.device, dtype=torch.float64)

    def apply(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """q [T, H, D] and k [T, KVH, D] turned by ``positions`` int32 [axes, T]
        (or [T] for one axis)."""
        import memopt_C

        q2, k2 = memopt_C.apply_rotary(q, k, positions, self.inv_freq, self.sections, self.interleaved)
        return q2, k2

    def write(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
              slot_mapping: torch.Tensor, key_cache: torch.Tensor,
              value_cache: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """:meth:`apply`, and the turned keys and the values written to the
        fp16 pool at ``slot_mapping`` in the same pass."""
        import memopt_C

        q2, k2 = memopt_C.rotary_write_cache(q, k, v, positions, self.inv_freq, self.sections, slot_mapping,
                                             key_cache, value_cache, self.interleaved)
        return q2, k2


_caches: "weakref.WeakSet[PackedKVCache]" = weakref.WeakSet()
_taking = threading.Lock()


def _pool_kind(C) -> Optional[tuple]:
    """(block_size, heads, head_dim, format, device) and the number of pages of
    the process-wide pool, None where there is none."""
    try:
        fmt = C.pool_format()
    except RuntimeError:
        return None
    k = C.get_pool_tensors()[0]
    if fmt == "int4":  # codes [NB, H, BS, D / 2]
        return (k.shape[2], k.shape[1], 2 * k.shape[3], fmt, k.device), k.shape[0]
    return (k.shape[1], k.shape[2], k.shape[3], fmt, k.device), k.shape[0]


def _take_pages(C, num_blocks: int, kind: tuple) -> Tuple[List[int], int]:
    """``num_blocks`` pages off the free-list of a pool of this kind, and the
    pool's number of pages.  A pool that has them free is used as it is;
    otherwise the pool is initialised, unless a cache still lives in it."""
    pool = _pool_kind(C)
    if pool is None or pool[0] != kind or C.free_blocks_count() < num_blocks:
        if any(c._owns() for c in _caches):
            gc.collect()  # one that only a reference cycle keeps does not count
        if any(c._owns() for c in _caches):
            raise RuntimeError("PackedKVCache: the process-wide pool belongs to another PackedKVCache and has not "
                               f"{num_blocks} free pages of this kind; call memopt_C.init_pool with the pages of all "
                               "caches before the first one is made, or close the other one")
        C.init_pool(num_blocks, *kind[:3], kv_format=kind[3])
    pages: List[int] = []
    while len(pages) < num_blocks and (page := C.allocate_block()) >= 0:
        pages.append(page)
    if len(pages) < num_blocks:
        _give_back(C, C.pool_generation(), pages)
        raise RuntimeError(f"PackedKVCache: the pool has {len(pages)} free pages, {num_blocks} are asked for; the others "
                           "are held through allocate_block")
    return pages, _pool_kind(C)[1]


def _give_back(C, generation: int, pages: List[int]) -> None:
    if C.pool_generation() == generation:
        for page in pages:
            C.free_block(page)


class PackedKVCache:
    """Packed-batch KV cache of one attention layer.

    It takes ``num_blocks`` pages from the free-list of the process-wide pool,
    as :class:`PagedKVCache` does page by page, and gives them back when it is
    closed or dropped.  A pool of its kind (block size, heads, head_dim,
    format) that has so many free pages is used as it is, otherwise it is
    initialised with ``num_blocks`` pages: for several caches, one per layer,
    call ``memopt_C.init_pool`` with the pages of all of them first.  While a
    cache lives in the pool another one does not replace it.  The pool holds
    fp16 or INT4 whatever the inputs' type: bf16 keys and values past 65504
    are infinite there."""

    def __init__(self, num_blocks: int, num_heads: int, head_dim: int, block_size: int = 16, max_seqs: int = 256,
                 max_seq_len: int = 32768, kv_format: str = "fp16", rotary: Optional[RotaryPositions] = None,
                 device: Optional[torch.device] = None) -> None:
        import memopt_C

        self._C = memopt_C
        if rotary is not None and rotary.head_dim != head_dim:
            raise ValueError("PackedKVCache: rotary.head_dim differs from head_dim")
        if num_blocks <= 0:
            raise ValueError("PackedKVCache: num_blocks must be > 0")
        self.num_heads, self.head_dim, self.block_size, self.rotary = num_heads, head_dim, block_size, rotary
        dev = _device(device)
        with torch.cuda.device(dev) if dev.type == "cuda" else contextlib.nullcontext():
            with _taking:
                pages, total = _take_pages(memopt_C, num_blocks, (block_size, num_heads, head_dim, kv_format, dev))
                self._generation = memopt_C.pool_generation()
                self._pages = weakref.finalize(self, _give_back, memopt_C, self._generation, pages)
                self._pages.atexit = False
                _caches.add(self)
        self.table = DevicePageTable(total, block_size, max_seqs, max_seq_len, dev, pages)

    def close(self) -> None:
        """Gives the cache's pages back to the pool; the cache is then empty
        and refuses further use."""
        self._pages()

    def _owns(self) -> bool:
        return self._pages.alive and self._C.pool_generation() == self._generation

    def _need_pool(self) -> None:
        if not self._pages.alive:
            raise RuntimeError("PackedKVCache: the cache was closed")
        if self._C.pool_generation() != self._generation:
            raise RuntimeError("PackedKVCache: the process-wide pool was initialised anew, the cache's pages are gone")

    @property
    def kv_format(self) -> str:
        return self._C.pool_format()

    # ---- tables --------------------------------------------------------------
    def admit(self, rows: Ints, prompt_lens: Ints, max_tokens: Optional[int] = None) -> PackedBatch:
        """Starts a sequence in each row (what the row held is given back) and
        reserves its prompt; a refused batch changes nothing."""
        self._need_pool()
        batch = self.table.replace(rows, prompt_lens, max_tokens)
        batch.whole = True
        return batch

    def extend(self, rows: Ints, tokens_per_row: int = 1) -> PackedBatch:
        """Reserves the next ``tokens_per_row`` tokens of each row."""
        self._need_pool()
        r = self.table.ints(rows)
        n = torch.full_like(r, tokens_per_row)
        return self.table.reserve(r, n, int(r.numel()) * tokens_per_row)

    def finish(self, rows: Ints) -> None:
        """Gives the pages of finished rows back."""
        self._need_pool()
        self.table.truncate(rows)

    # ---- data path -------------------------------------------------------------
    @staticmethod
    def _no_grad(*tensors: torch.Tensor) -> None:
        """Before anything is written: paged attention and the cache write
        would drop the gradient in silence."""
        if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
            raise RuntimeError("PackedKVCache: the operators have no gradient; detach their inputs or call them under "
                               "torch.no_grad()")

    def _store(self, q, k, v, batch: PackedBatch, positions):
        if self.rotary is not None:
            pos = batch.positions if positions is None else positions
            if positions is None and len(self.rotary.sections) > 1:
                pos = batch.positions.expand(len(self.rotary.sections), -1)
            if self.kv_format == "fp16":
                kc, vc = self._C.get_pool_tensors()
                return self.rotary.write(q, k, v, pos, batch.slot_mapping, kc, vc)
            q, k = self.rotary.apply(q, k, pos)
        elif positions is not None:
            raise ValueError("PackedKVCache: positions without rotary")
        self._C.write_cache(k.to(torch.float16).contiguous(), v.to(torch.float16).contiguous(), batch.block_tables,
                            batch.slot_mapping)
        return q, k

    def prompt(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, batch: PackedBatch, max_seqlen: int,
               window_size: int = -1, causal: bool = True, positions: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Whole prompts (a batch of :meth:`admit`): rotary positions (the
        tokens' own, or ``positions`` [axes, T]), the cache write, and
        attention inside each prompt.  q [T, H, D], k and v [T, KVH, D]; rows
        past the batch's last token, and all rows of a refused batch, are 0.
        A window is the last ``window_size`` tokens up to the row's own
        (causal), or of the whole prompt for every row (not causal: what a
        decode step sees, not a band around the row)."""
        if not batch.whole:
            raise ValueError("PackedKVCache.prompt: the batch must come from admit (whole sequences)")
        self._no_grad(q, k, v)
        self._need_pool()
        q, k = self._store(q, k, v, batch, positions)
        return self._C.packed_attention(q, k, v, batch.cu_seqlens, max_seqlen, window_size, causal, zero_rest=True)

    def decode(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, batch: PackedBatch, window_size: int = -1,
               positions: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The next tokens of each row (a batch of :meth:`extend`, the same
        number n of tokens per row): causal paged attention over the cached
        context.  q [B * n, H, D]; the result has q's shape, in fp16 (the
        pool's type; 0 for a refused batch).  A window counts cached tokens."""
        if batch.whole:
            raise ValueError("PackedKVCache.decode: the batch must come from extend")
        B = batch.rows.numel()
        if B == 0 or q.shape[0] % B != 0:
            raise ValueError(f"PackedKVCache.decode: {q.shape[0]} tokens for {B} rows")
        self._no_grad(q, k, v)
        self._need_pool()
        q, _ = self._store(q, k, v, batch, positions)
        q4 = q.to(torch.float16).contiguous().reshape(B, q.shape[0] // B, q.shape[1], q.shape[2])
        reach = batch.block_tables.shape[1] * self.block_size
        window = reach if window_size <= 0 else window_size
        lens = batch.context_lens if batch.attend_lens is None else batch.attend_lens
        if self.kv_format == "int4":
            out = self._C.dynamic_sparse_attention_int4(q4, self._C.get_int4_pages(), batch.block_tables, lens,
                                                        reach, window, True)
        else:
            kc, vc = self._C.get_pool_tensors()
            out = self._C.dynamic_sparse_attention(q4, kc, vc, batch.block_tables, lens, reach, window, True)
        return out.reshape(q.shape)

    def evict(self, scores: torch.Tensor, retain_ratio: float, num_sink_tokens: int = 4):
        """``evict_topk_compact`` over every row of the table (scores fp32
        [max_seqs, heads, L], L at least the longest row): kept tokens move to
        the front, lengths shrink, emptied pages return to the ring.  Positions
        go on from the sequence's own length: kept keys stay turned by those
        that they were written with.  Returns (kept_idx, kept_count)."""
        self._need_pool()
        t = self.table
        before = t.context_lens.clone()
        try:
            kept, count, freed, freed_count = self._C.evict_topk_compact(scores, t.block_tables, t.context_lens,
                                                                         float(retain_ratio), int(num_sink_tokens))
        finally:  # a failed one may have shrunk the lengths too
            t.position_offsets += before - t.context_lens
        t.release_pages(freed, freed_count)
        return kept, count
