"""PagedKVCache: a compressed KV cache in pages, with page-sparse attention and eviction by attention weight.

Where ``RawKVCache`` keeps one growing buffer per layer, this keeps a fixed
pool of pages and hands them to the sequences of a batch as they grow, so
ragged batches share the memory and a finished sequence gives its pages back.
On top of the pool:

* ``attention(layer, q)`` attends to every cached token (``pkv_paged_attn``);
* ``attention(layer, q, top_pages=n)`` attends to the n pages per KV head whose
  summaries promise the highest scores (``pkv_pages_select``);
* with ``track_weights`` every call adds each token's attention weights, and
  ``evict(layer, keep)`` keeps the first, the latest and the most attended
  tokens of every sequence (``pkv_tokens_select``, ``pkv_tokens_gather``).

The reference has no paged cache; its RawKVCache (cache/raw_cache.py:57-292) is
the nearest relative.  Tensors and pages belong to one CUDA stream at a time:
a page is reused as soon as it is free, in stream order.  Threads that share
the stream may share the cache.
"""

from __future__ import annotations

import threading
from dataclasses import dataclass, field
from typing import Dict, List, Optional, Sequence, Union

import torch

from ..quantizer.stacked_plane import _cuda_device
from .backend import CacheBackend


@dataclass
class _PagedLayer:
    k: torch.Tensor                    # (num_pages, kv_heads, page_size, m)
    v: torch.Tensor
    table: torch.Tensor                # (batch, max_pages) int32
    lens: torch.Tensor                 # (batch,) int32
    rows: List[List[int]]              # the pages of each sequence, on the host
    lengths: List[int]
    free: List[int] = field(default_factory=list)
    summaries: Optional[torch.Tensor] = None
    weights: Optional[torch.Tensor] = None


def _capturing(dev: torch.device) -> bool:
    """Whether the device's current stream records a CUDA graph, to be replayed when the sequences are longer."""
    if dev.type != "cuda":
        return False
    if torch.cuda.current_device() == dev.index:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(dev):
        return torch.cuda.is_current_stream_capturing()


class PagedKVCache:
    """backend: one CacheBackend for every layer, or a dict keyed by layer index; batch sequences of kv_heads
    heads share num_pages pages (per layer) of page_size tokens.  max_tokens: the longest sequence (default: all
    pages in one).  page_summaries: keep what ``top_pages`` needs; track_weights: keep what ``evict`` needs.

    Attention weights are a buffer of (batch, kv_heads, slots) floats.  With ``max_tokens``, and wherever slots for
    the whole pool take at most a quarter of what the codes take, it is made once; otherwise it is replaced by a wider
    one when the longest sequence outgrows it, and attention cannot be captured into a CUDA graph."""

    def __init__(self, backend: Union[CacheBackend, Dict[int, CacheBackend]], batch: int, kv_heads: int, num_pages: int,
                 page_size: int = 16, max_tokens: Optional[int] = None, page_summaries: bool = False,
                 track_weights: bool = False, device: Optional[torch.device] = None) -> None:
        if batch < 1 or kv_heads < 1 or num_pages < 1:
            raise ValueError(f"batch, kv_heads and num_pages must be positive, got {batch}, {kv_heads}, {num_pages}")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        self._backends = dict(backend) if isinstance(backend, dict) else {}
        self._default_backend = None if isinstance(backend, dict) else backend
        self.batch, self.kv_heads, self.num_pages, self.page_size = batch, kv_heads, num_pages, page_size
        self.max_pages = num_pages if max_tokens is None else min(num_pages, -(-int(max_tokens) // page_size))
        if self.max_pages < 1:
            raise ValueError(f"max_tokens must be positive, got {max_tokens}")
        self.page_summaries, self.track_weights = page_summaries, track_weights
        self._whole = max_tokens is not None                  # weights for the longest possible sequence at once
        self._device = device
        self._layers: Dict[int, _PagedLayer] = {}
        self._lock = threading.Lock()

    # ------------------------------------------------------------------
    def _backend(self, layer_idx: int) -> CacheBackend:
        b = self._backends.get(layer_idx, self._default_backend)
        if b is None:
            raise KeyError(f"No backend for layer {layer_idx}.")
        return b

    def _layer(self, layer_idx: int) -> _PagedLayer:
        if layer_idx not in self._layers:
            raise KeyError(f"Layer {layer_idx} has no cached data.")
        return self._layers[layer_idx]

    def _new_layer(self, backend: CacheBackend, dev: torch.device) -> _PagedLayer:
        codec = backend.codec(dev)
        k, v = (codec.empty_pages(self.num_pages, self.kv_heads, self.page_size, backend.quantizer.code_dtype)
                for _ in range(2))
        st = _PagedLayer(k, v, torch.full((self.batch, self.max_pages), -1, dtype=torch.int32, device=dev),
                         torch.zeros(self.batch, dtype=torch.int32, device=dev), [[] for _ in range(self.batch)],
                         [0] * self.batch, list(range(self.num_pages - 1, -1, -1)))
        if self.page_summaries:
            st.summaries = codec.empty_summaries(self.num_pages, self.kv_heads)
        if self.track_weights:
            slots = self.max_pages * self.page_size
            codes = 2 * self.num_pages * self.page_size * k.stride(2) * k.element_size()
            whole = self._whole or 4 * (4 * self.batch * slots) <= codes
            st.weights = torch.zeros((self.batch, self.kv_heads, slots if whole else 0), device=dev)
        return st

    def _wide_enough(self, st: _PagedLayer, pages: int) -> Optional[torch.Tensor]:
        """The layer's weights, in a wider buffer where sequences of so many pages need it."""
        w, ps = st.weights, self.page_size
        if w is None or w.shape[2] >= pages * ps:
            return w
        wide = w.new_zeros((self.batch, self.kv_heads, min(self.max_pages, max(pages, w.shape[2] // ps * 3 // 2)) * ps))
        wide[..., :w.shape[2]] = w
        return wide

    def _ints(self, values: Sequence[int], dev: torch.device) -> torch.Tensor:
        return torch.tensor(list(values), dtype=torch.int32, device=dev)

    def _table_of(self, rows: List[List[int]]) -> torch.Tensor:
        """The page table of these rows, on the host."""
        return torch.tensor([r + [-1] * (self.max_pages - len(r)) for r in rows], dtype=torch.int32)

    # ------------------------------------------------------------------
    # A change is made on copies, or behind a sequence's end where nothing reads, and becomes the layer's state after
    # its last launch: a call that raises leaves the layer as it was.
    def append(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor, lengths: Optional[Sequence[int]] = None) -> List[int]:
        """Compress and append (batch, kv_heads, s, head_dim) tokens; ``lengths`` (host integers) takes only the
        first lengths[b] of a padded row.  Returns the sequences' new lengths."""
        backend = self._backend(layer_idx)
        B, H, ps = self.batch, self.kv_heads, self.page_size
        if k.dim() != 4 or k.shape[:2] != (B, H) or k.shape[3] != backend.head_dim or v.shape != k.shape:
            raise ValueError(f"expected K and V of ({B}, {H}, s, {backend.head_dim}), got {tuple(k.shape)}, {tuple(v.shape)}")
        s = k.shape[2]
        counts = [s] * B if lengths is None else [int(n) for n in lengths]
        if len(counts) != B or any(n < 0 or n > s for n in counts):
            raise ValueError(f"lengths must be {B} numbers from 0 to {s}, got {counts}")
        st = self._layers.get(layer_idx)
        dev = st.lens.device if st is not None else self._device if self._device is not None else _cuda_device(k)
        codec = backend.codec(dev)
        codes = [codec.encode(backend.aligner.pad(x.to(dev).reshape(B * H * s, x.shape[3]))).view(B, H, s, codec.m)
                 for x in (k, v)]
        with self._lock:
            st = self._layers.get(layer_idx)
            if st is None:
                st = self._new_layer(backend, dev)
            new = [n + c for n, c in zip(st.lengths, counts)]
            need = [-(-n // ps) - len(r) for n, r in zip(new, st.rows)]
            if any(-(-n // ps) > self.max_pages for n in new):
                raise ValueError(f"sequences of {new} tokens exceed {self.max_pages} pages of {ps}")
            if sum(need) > len(st.free):
                raise RuntimeError(f"layer {layer_idx}: {sum(need)} pages needed, {len(st.free)} free")
            total = sum(need)
            rows, weights = st.rows, st.weights
            if total:
                fresh = iter(st.free[len(st.free) - total:][::-1])
                rows = [r + [next(fresh) for _ in range(n)] for r, n in zip(rows, need)]
                weights = self._wide_enough(st, max(map(len, rows)))
                st.table.copy_(self._table_of(rows))
            start = st.lens.clone()
            cnt = None if lengths is None else self._ints(counts, st.lens.device)
            more = s if cnt is None else cnt
            codec.store_pages(codes[0], st.k, st.table, start, cnt)
            codec.store_pages(codes[1], st.v, st.table, start, cnt)
            if st.summaries is not None:
                codec.summarize_pages(st.k, st.table, start + more, st.summaries, start=start)
            st.lens += more
            st.rows, st.lengths, st.weights = rows, new, weights
            del st.free[len(st.free) - total:]
            self._layers[layer_idx] = st
            return list(new)

    def attention(self, layer_idx: int, q: torch.Tensor, scale: Optional[float] = None, top_pages: Optional[int] = None,
                  sinks: int = 1, recent: int = 1, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """Decode attention of q (batch, q_heads, head_dim) -> the same shape.

        ``top_pages``: attend to that many pages per KV head at most, the first
        ``sinks`` and last ``recent`` among them.  Captured into a CUDA graph,
        the call follows the cache's later changes when it is replayed.
        """
        backend = self._backend(layer_idx)
        if q.dim() != 3 or q.shape[2] != backend.head_dim:
            raise ValueError(f"q must be ({self.batch}, q_heads, {backend.head_dim}), got {tuple(q.shape)}")
        if scale is None:
            scale = backend.head_dim ** -0.5
        with self._lock:
            st = self._layer(layer_idx)
            codec = backend.codec(st.lens.device)
            qp = backend.aligner.pad(q.to(st.lens.device))
            longest, capturing = max(map(len, st.rows)), _capturing(st.lens.device)
            # Scratch and grids go by the width of the table and the weights: where that is more than twice the longest
            # sequence, only the first columns are passed. A graph will be replayed over longer sequences.
            width = self.max_pages if capturing or 2 * longest > self.max_pages else max(longest, 1)
            table, weights = st.table, st.weights
            if weights is not None:
                slots = weights.shape[2]
                if slots < width * self.page_size:
                    if capturing:
                        raise RuntimeError("attention captured into a graph needs weights that are not replaced as "
                                           "sequences grow: make the cache with max_tokens")
                    width = max(1, slots // self.page_size)
                elif slots > width * self.page_size:
                    weights = weights[..., :width * self.page_size]
            if width < self.max_pages:
                table = table[:, :width]
            pages = None
            if top_pages is not None:
                if not self.page_summaries:
                    raise RuntimeError("top_pages needs a cache made with page_summaries=True")
                if top_pages < 1 or sinks < 0 or recent < 0 or sinks + recent > top_pages:
                    raise ValueError("need 0 <= sinks + recent <= top_pages and top_pages >= 1, "
                                     f"got {sinks}, {recent}, {top_pages}")
                if (self.max_pages if capturing else longest) > top_pages:
                    pages = codec.select_pages(qp, st.summaries, table, st.lens, self.page_size, top_pages, sinks=sinks,
                                               recent=recent)
            out = codec.paged_attention(qp, st.k, st.v, table, st.lens, scale=scale, pages=pages, weights=weights,
                                        out_dtype=out_dtype)
        return backend.aligner.unpad(out)

    def evict(self, layer_idx: int, keep: int, sinks: int = 4, recent: int = 32) -> List[int]:
        """Cut every sequence of more than ``keep`` tokens to ``keep``: its first ``sinks``, its last ``recent`` and
        the most attended others of each KV head, in their order.  Returns the new lengths.  The kept tokens move to
        free pages and the old ones come free, as many sequences at a time as the free pages take
        (ceil(keep / page_size) each); one that finds no room moves through a buffer of that size into its own first
        pages, so a full pool can be cut too.  A call that raises leaves sequences as they were or cut."""
        backend = self._backend(layer_idx)
        if not self.track_weights:
            raise RuntimeError("evict needs a cache made with track_weights=True")
        if keep < 1 or sinks < 0 or recent < 0 or sinks + recent > keep:
            raise ValueError(f"need 0 <= sinks + recent <= keep and keep >= 1, got {sinks}, {recent}, {keep}")
        with self._lock:
            st = self._layer(layer_idx)
            dev = st.lens.device
            codec = backend.codec(dev)
            cut = [b for b in range(self.batch) if st.lengths[b] > keep]
            if not cut:
                return list(st.lengths)
            per = -(-keep // self.page_size)
            lens = self._ints([n if n > keep else 0 for n in st.lengths], dev)
            longest = max(map(len, st.rows)) * self.page_size
            kept, kw = codec.select_tokens(st.weights[..., :longest], lens, keep, sinks=sinks, recent=recent)
            at = 0
            while at < len(cut):
                n = max(1, min(len(cut) - at, len(st.free) // per))
                self._move(st, codec, cut[at:at + n], kept, kw, n < len(cut))
                at += n
            return list(st.lengths)

    def _move(self, st: _PagedLayer, codec, group: List[int], kept: torch.Tensor, kw: torch.Tensor, some: bool) -> None:
        """Cut the group's sequences to their kept slots: into free pages or, one without room, its own first ones.
        some: kept has slots of other sequences too."""
        dev, keep = st.lens.device, kept.shape[2]
        per = -(-keep // self.page_size)
        room = per * len(group) <= len(st.free)
        taken = per * len(group) if room else 0
        fresh = iter(st.free[len(st.free) - taken:][::-1])
        to = {b: [next(fresh) for _ in range(per)] if room else st.rows[b][:per] for b in group}
        table2 = torch.tensor([to.get(b, [-1] * per) for b in range(self.batch)], dtype=torch.int32, device=dev)
        picks = kept.masked_fill(table2[:, :1, None] < 0, -1) if some else kept
        rows = [to.get(b, r) for b, r in enumerate(st.rows)]
        lengths = [keep if b in to else n for b, n in enumerate(st.lengths)]
        table, lens = self._table_of(rows).to(dev), self._ints(lengths, dev)
        if room:
            codec.gather_tokens(st.k, st.v, st.table, picks, st.k, st.v, table2)
            if st.summaries is not None:
                start = self._ints([0 if b in to else n for b, n in enumerate(lengths)], dev)
                codec.summarize_pages(st.k, table, lens, st.summaries, start=start)
        else:                                             # all that can fail comes before the pages are written over
            k, v = (codec.empty_pages(per, self.kv_heads, self.page_size, st.k.dtype) for _ in range(2))
            side = torch.tensor([list(range(per)) if b in to else [-1] * per for b in range(self.batch)], dtype=torch.int32,
                                device=dev)
            order = torch.arange(keep, dtype=torch.int32, device=dev).expand(kept.shape).masked_fill(picks < 0, -1)
            codec.gather_tokens(st.k, st.v, st.table, picks, k, v, side)
            if st.summaries is not None:
                sums = codec.summarize_pages(k, side, lens.masked_fill(table2[:, 0] < 0, 0),
                                             codec.empty_summaries(per, self.kv_heads))
            codec.gather_tokens(k, v, side, order, st.k, st.v, table2)
            if st.summaries is not None:
                st.summaries[table2[group[0]].long()] = sums
        for b in group:
            st.weights[b] = 0
            st.weights[b, :, :keep] = kw[b]
        st.table.copy_(table)
        st.lens.copy_(lens)
        old, st.rows, st.lengths = st.rows, rows, lengths
        del st.free[len(st.free) - taken:]
        for b in group:
            st.free.extend(reversed(old[b] if room else old[b][per:]))

    # ------------------------------------------------------------------
    def release(self, layer_idx: int, sequence: int) -> None:
        """Forget one sequence of a layer; its pages come free."""
        if not 0 <= sequence < self.batch:
            raise IndexError(f"sequence {sequence} outside a batch of {self.batch}")
        with self._lock:
            st = self._layer(layer_idx)
            st.table.copy_(self._table_of([[] if b == sequence else r for b, r in enumerate(st.rows)]))
            st.lens[sequence] = 0
            if st.weights is not None:
                st.weights[sequence] = 0
            st.free.extend(reversed(st.rows[sequence]))
            st.rows[sequence], st.lengths[sequence] = [], 0

    def clear(self, layer_idx: Optional[int] = None) -> None:
        with self._lock:
            if layer_idx is None:
                self._layers.clear()
            else:
                self._layers.pop(layer_idx, None)

    def get_seq_lengths(self, layer_idx: int = 0) -> List[int]:
        with self._lock:
            st = self._layers.get(layer_idx)
            return [0] * self.batch if st is None else list(st.lengths)

    def free_pages(self, layer_idx: int = 0) -> int:
        with self._lock:
            st = self._layers.get(layer_idx)
            return self.num_pages if st is None else len(st.free)

    def get_weights(self, layer_idx: int) -> Optional[torch.Tensor]:
        """(batch, kv_heads, slots) accumulated attention weights, slots for the longest sequence at least; a
        sequence's tokens come first."""
        with self._lock:
            return self._layer(layer_idx).weights

    def get_pages(self, layer_idx: int):
        """The device buffers: K and V pools, page table and lengths."""
        with self._lock:
            st = self._layer(layer_idx)
            return st.k, st.v, st.table, st.lens

    @property
    def cached_layers(self) -> list:
        with self._lock:
            return sorted(self._layers)

    def memory_footprint(self) -> dict:
        """codes_bytes (K + V codes of cached tokens), fp16_bytes (the same in FP16), compression, pool_bytes, n_layers."""
        codes = fp16 = pool = 0
        with self._lock:
            for layer_idx, st in self._layers.items():
                n = sum(st.lengths) * self.kv_heads
                codes += 2 * n * st.k.shape[3] * st.k.element_size()
                fp16 += 4 * n * self._backend(layer_idx).head_dim
                pool += 2 * st.k.shape[0] * self.kv_heads * self.page_size * st.k.stride(2) * st.k.element_size()
            layers = len(self._layers)
        return {"codes_bytes": codes, "fp16_bytes": fp16, "compression": fp16 / codes if codes else float("nan"),
                "pool_bytes": pool, "n_layers": layers}

    def __repr__(self) -> str:
        return (f"PagedKVCache(batch={self.batch}, kv_heads={self.kv_heads}, pages={self.num_pages}x{self.page_size}, "
                f"n_layers={len(self._layers)})")
