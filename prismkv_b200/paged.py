"""Calls over a paged cache of packed codes: the paged half of ``DeviceCodec``.

A pool of pages holds K and V codes as (num_pages, kv_heads, page_size, m)
tensors (``empty_pages`` makes one); row b of an int32 ``page_table``
(batch, max_pages) names sequence b's pages in order and int32 ``seq_lens``
(batch) its tokens, both on the codec's device.  Token t of sequence b sits in
slot ``t % page_size`` of page ``page_table[b, t // page_size]``; entries past
the last token are never read.  ``page_size`` is a power of two, 16 to 1024.
Any strides serve whose rows start on 16-byte boundaries with unit code stride,
so (num_pages, page_size, kv_heads, m) pools pass as transposed views.

Nothing here synchronises, keeps state between calls or allocates beyond its
outputs and a workspace from torch's allocator, so every call can be captured
into a CUDA graph.  A page id outside the pool, a token past the table or a
page list out of order is skipped on the device and shows in
``_lib.device_error()`` as 6.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import numpy as np
import torch

from . import _lib

PAGE_CODE_DTYPES = {torch.uint8: 1, torch.int16: 2, torch.uint16: 2}
ROW_BYTES = 16          # code rows start on multiples of this


def _summary_grid(dec_z: np.ndarray, dec_xy: np.ndarray, total_codes: int) -> Tuple[np.ndarray, np.ndarray]:
    """Decoded values on the summaries' grid in 1/128 steps, the largest magnitude at 127 steps (int16)."""
    z, xy = dec_z.astype(np.float64).reshape(-1), dec_xy.astype(np.float64).reshape(-1, 2)
    top = max(np.abs(z).max(), np.abs(xy).max())
    f = 127.0 * 128.0 / top if top > 0 else 0.0
    xy = np.tile(xy, (total_codes // xy.shape[0], 1))
    return np.rint(z * f).astype(np.int16), np.rint(xy * f).astype(np.int16)


class PagedOps:
    """Mixed into DeviceCodec: needs its struct, host, device, dim, m, bits_total and stream."""

    # ------------------------------------------------------------------
    def empty_pages(self, num_pages: int, kv_heads: int, page_size: int,
                    code_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """Uninitialised (num_pages, kv_heads, page_size, m) codes with rows on 16-byte boundaries."""
        if code_dtype is None:
            code_dtype = torch.uint8 if self.bits_total <= 8 else torch.int16
        if code_dtype not in PAGE_CODE_DTYPES:
            raise ValueError("codes must be stored as uint8 or 16-bit integers")
        per = ROW_BYTES // PAGE_CODE_DTYPES[code_dtype]
        pitch = -(-self.m // per) * per
        return torch.empty((num_pages, kv_heads, page_size, pitch), dtype=code_dtype, device=self.device)[..., :self.m]

    @property
    def summary_pitch(self) -> int:
        """Bytes per summary row: dim rounded up to 16."""
        return -(-self.dim // 16) * 16

    def empty_summaries(self, num_pages: int, kv_heads: int) -> torch.Tensor:
        """Uninitialised (num_pages, kv_heads, 2, summary_pitch) int8 page summaries."""
        return torch.empty((num_pages, kv_heads, 2, self.summary_pitch), dtype=torch.int8, device=self.device)

    # ------------------------------------------------------------------
    # The checks run on every call of a decode step, so they read each property of a tensor once.
    def _index(self) -> int:
        """The codec's CUDA device index."""
        i = self.device.index
        return torch.cuda.current_device() if i is None else i

    def _on_device(self, t: torch.Tensor, name: str) -> None:
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor")
        if t.get_device() != self._index():
            raise ValueError(f"{name} is on {t.device}, the codec on {self.device}")

    def _check_ints(self, t: torch.Tensor, name: str, shape) -> torch.Tensor:
        self._on_device(t, name)
        if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor of shape {tuple(shape)}, "
                             f"got {t.dtype} {tuple(t.shape)}")
        return t

    def _check_table(self, page_table: torch.Tensor):
        """(data pointer, row stride, batch, max_pages) of a page table."""
        self._on_device(page_table, "page_table")
        if page_table.dtype != torch.int32 or page_table.dim() != 2:
            raise ValueError("page_table must be an int32 (batch, max_pages) tensor with unit inner stride")
        B, n = page_table.shape
        stride, inner = page_table.stride()
        if n > 1 and inner != 1:
            raise ValueError("page_table must be an int32 (batch, max_pages) tensor with unit inner stride")
        return page_table.data_ptr(), stride if B > 1 else n, B, n

    def _pages(self, k: torch.Tensor, v: Optional[torch.Tensor], page_table: torch.Tensor,
               name: str = "k_pages") -> _lib.PkvPages:
        self._on_device(k, name)
        if k.dim() != 4 or k.shape[3] != self.m or k.shape[1] < 1:
            raise ValueError(f"{name} must be (num_pages, kv_heads, page_size, {self.m}), got {tuple(k.shape)}")
        P, H, ps, _ = shape = k.shape
        code_bytes = PAGE_CODE_DTYPES.get(k.dtype)
        if code_bytes is None:
            raise ValueError("codes must be stored as uint8 or 16-bit integers")
        strides = k.stride()
        if v is not None:
            self._on_device(v, "v_pages")
            if v.shape != shape or v.dtype != k.dtype or v.stride() != strides:
                raise ValueError("k_pages and v_pages must have the same shape, dtype and strides")
        if strides[3] != 1:
            raise ValueError("codes need unit stride within a row")
        if ps < 16 or ps > 1024 or ps & (ps - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {ps}")
        table, table_stride, B, max_pages = self._check_table(page_table)
        # (a dimension of one element has no stride of its own)
        return _lib.PkvPages(k.data_ptr(), v.data_ptr() if v is not None else None, code_bytes, P, H, ps,
                             strides[0] if P > 1 else 0, strides[1] if H > 1 else 0, strides[2], table, table_stride, B,
                             max_pages)

    def _query(self, q: torch.Tensor, kv_heads: int, batch: int) -> torch.Tensor:
        self._on_device(q, "q")
        if q.dim() == 4:
            if q.shape[2] != 1:
                raise ValueError("paged attention takes one query token (Sq == 1)")
            q = q[:, :, 0, :]
        if q.dim() != 3 or q.shape[0] != batch or q.shape[2] != self.dim:
            raise ValueError(f"q must be ({batch}, q_heads, {self.dim}), got {tuple(q.shape)}")
        if q.shape[1] < 1 or q.shape[1] % kv_heads:
            raise ValueError(f"{q.shape[1]} query heads do not divide among {kv_heads} KV heads")
        if q.dtype not in _lib.DTYPE_CODES:
            q = q.float()
        return q if q.stride(2) == 1 else q.contiguous()

    def _call(self, fn, what: str, *args) -> None:
        """fn(*args, stream) with the codec's device current; a non-zero status raises."""
        i = self._index()
        if torch.cuda.current_device() == i:
            rc = fn(*args, _lib.raw_stream(i))
        else:
            with torch.cuda.device(i):
                rc = fn(*args, _lib.raw_stream(i))
        if rc:
            _lib.check(rc, what)

    # ------------------------------------------------------------------
    def paged_attention(self, q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                        page_table: torch.Tensor, seq_lens: torch.Tensor, scale: Optional[float] = None,
                        pages: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None,
                        weights_out: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                        out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """Decode attention over a paged cache: q (B, Hq, dim) [or (B, Hq, 1, dim)] -> (B, Hq, dim) of out_dtype.

        ``pages`` (B, Hkv, n) int32 restricts each KV head to the listed logical
        pages (``select_pages`` makes such lists): strictly ascending, -1 behind
        the last.  ``weights`` (B, Hkv, slots) fp32: every attended token's
        softmax weights, summed over the KV head's query heads, are added --
        in place, or into ``weights_out`` of the same shape, whose other entries
        are not touched; slots must cover every token.  A sequence without
        tokens gives zeros.
        """
        g = self._pages(k_pages, v_pages, page_table)
        q = self._query(q, g.kv_heads, g.batch)
        B, Hq, _ = q.shape
        self._check_ints(seq_lens, "seq_lens", (B,))
        if out is None:
            if out_dtype not in _lib.DTYPE_CODES:
                raise ValueError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
            out = torch.empty((B, Hq, self.dim), dtype=out_dtype, device=q.device)
        else:
            self._on_device(out, "out")
            if out.shape != (B, Hq, self.dim) or out.dtype not in _lib.DTYPE_CODES or out.stride(2) != 1:
                raise ValueError(f"out must be a ({B}, {Hq}, {self.dim}) float tensor with unit inner stride")
        selected = n_selected = 0
        if pages is not None:
            if pages.dim() != 3:
                raise ValueError(f"pages must be ({B}, {g.kv_heads}, n), got {tuple(pages.shape)}")
            n_selected = pages.shape[2]
            self._check_ints(pages, "pages", (B, g.kv_heads, n_selected))
            if n_selected == 0:
                raise ValueError("pages lists no page; leave it out to attend to every token")
            selected = pages.data_ptr()
        w_in = w_out = slots = 0
        if weights_out is not None and weights is None:
            raise ValueError("weights_out needs weights")
        if weights is not None:
            to = weights if weights_out is None else weights_out
            for t, n in ((weights, "weights"), (to, "weights_out")):
                self._on_device(t, n)
                if t.dtype != torch.float32 or t.dim() != 3 or t.shape[:2] != (B, g.kv_heads) or not t.is_contiguous():
                    raise ValueError(f"{n} must be a contiguous float32 ({B}, {g.kv_heads}, slots) tensor")
            if to.shape != weights.shape:
                raise ValueError("weights and weights_out must have the same shape")
            w_in, w_out, slots = weights.data_ptr(), to.data_ptr(), weights.shape[2]
        qs, os = q.stride(), out.stride()
        a = _lib.PkvPagedAttnArgs(g, Hq, _lib.DTYPE_CODES[q.dtype], q.data_ptr(), qs[0], qs[1], seq_lens.data_ptr(),
                                  selected or None, n_selected, self.dim ** -0.5 if scale is None else float(scale),
                                  out.data_ptr(), _lib.DTYPE_CODES[out.dtype], os[0], os[1], w_in or None, w_out or None,
                                  slots, slots)
        args = ctypes.byref(a)
        lib = _lib.load()
        # the workspace's size follows from the shapes alone
        key = (B, Hq, g.kv_heads, g.page_size, g.max_pages, n_selected, w_in != 0)
        sizes = self.__dict__.setdefault("_paged_sizes", {})
        need = sizes.get(key)
        if need is None:
            with torch.cuda.device(self._index()):
                need = max(int(lib.pkv_paged_attn_workspace_size(self._struct_ref(), args)), 256)
            if len(sizes) > 256:
                sizes.clear()
            sizes[key] = need
        ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        self._call(lib.pkv_paged_attn, "pkv_paged_attn", self._struct_ref(), args, ws.data_ptr(), need)
        return out

    def _struct_ref(self):
        return ctypes.byref(self.struct)

    # ------------------------------------------------------------------
    def store_pages(self, codes: torch.Tensor, pages: torch.Tensor, page_table: torch.Tensor, start: torch.Tensor,
                    counts: Optional[torch.Tensor] = None) -> None:
        """Copy codes (B, Hkv, n, m) into slots start[b] .. of one pool; counts[b] < n leaves padded rows out."""
        g = self._pages(pages, None, page_table, "pages")
        self._on_device(codes, "codes")
        if codes.dim() != 4 or codes.dtype != pages.dtype or (codes.shape[0], codes.shape[1], codes.shape[3]) != (
                g.batch, g.kv_heads, self.m):
            raise ValueError(f"codes must be ({g.batch}, {g.kv_heads}, n, {self.m}) of the pool's dtype")
        codes = codes.contiguous()
        self._check_ints(start, "start", (g.batch,))
        if counts is not None:
            self._check_ints(counts, "counts", (g.batch,))
        self._call(_lib.load().pkv_pages_store, "pkv_pages_store", ctypes.byref(g), self.m, pages.data_ptr(),
                   codes.data_ptr(), codes.shape[2], start.data_ptr(), counts.data_ptr() if counts is not None else None)

    def _grid(self):
        """Device tables of the summaries' grid, built on first use."""
        if getattr(self, "_grid_z", None) is None:
            z, xy = _summary_grid(np.asarray(self.host.dec_z), np.asarray(self.host.dec_xy), 1 << self.bits_total)
            if (np.diff(z.astype(np.int64)) < 0).any():
                raise ValueError("page summaries need decoded z values that rise with the bin")
            self._grid_xy = torch.from_numpy(np.ascontiguousarray(xy)).to(self.device)
            self._grid_z = torch.from_numpy(z).to(self.device)
        return self._grid_z, self._grid_xy

    def _check_summaries(self, t: torch.Tensor, g: _lib.PkvPages) -> None:
        self._on_device(t, "summaries")
        want = (g.kv_heads, 2, self.summary_pitch)
        if t.dtype != torch.int8 or t.dim() != 4 or tuple(t.shape[1:]) != want or not t.is_contiguous():
            raise ValueError(f"summaries must be a contiguous int8 (num_pages, {', '.join(map(str, want))}) tensor")

    def summarize_pages(self, k_pages: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                        summaries: torch.Tensor, start: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Least and greatest decoded key per page, KV head and rotated channel, rounded outwards to int8.

        Writes the summaries of the pages that hold a token >= start[b] of
        sequence b (of every page without ``start``) into ``summaries``
        (num_pages, Hkv, 2, summary_pitch) and returns it.  One step is 1/127 of
        the codec's largest decoded magnitude; values within 1/256 of a step of
        a whole number count as it.
        """
        g = self._pages(k_pages, None, page_table)
        self._check_ints(seq_lens, "seq_lens", (g.batch,))
        self._check_summaries(summaries, g)
        if summaries.shape[0] != g.num_pages:
            raise ValueError(f"summaries hold {summaries.shape[0]} pages, the pool {g.num_pages}")
        if start is not None:
            self._check_ints(start, "start", (g.batch,))
        gz, gxy = self._grid()
        self._call(_lib.load().pkv_pages_summarize, "pkv_pages_summarize", self._struct_ref(), ctypes.byref(g),
                   seq_lens.data_ptr(), start.data_ptr() if start is not None else None, gz.data_ptr(), gxy.data_ptr(),
                   summaries.data_ptr())
        return summaries

    def select_pages(self, q: torch.Tensor, summaries: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                     page_size: int, top: int, sinks: int = 1, recent: int = 1,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The pages worth attending to: (B, Hkv, top) int32 logical pages, ascending, -1 behind the last.

        The first ``sinks`` and last ``recent`` pages of a sequence are always
        taken, the others by an upper bound of their tokens' scores: the KV
        head's queries, rotated and rounded to int8 on a common scale, against
        the summaries' greatest (positive) and least (negative) values; the
        largest over the heads counts, ties go to the lower page.
        """
        if summaries.dim() != 4:
            raise ValueError("summaries must be (num_pages, kv_heads, 2, summary_pitch)")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        if top < 1 or sinks < 0 or recent < 0 or sinks + recent > top:
            raise ValueError(f"need 0 <= sinks + recent <= top and top >= 1, got {sinks}, {recent}, {top}")
        table, table_stride, B, max_pages = self._check_table(page_table)
        g = _lib.PkvPages(None, None, 1, summaries.shape[0], summaries.shape[1], page_size, 0, 0,
                          -(-self.m // ROW_BYTES) * ROW_BYTES, table, table_stride, B, max_pages)
        self._check_summaries(summaries, g)
        q = self._query(q, g.kv_heads, g.batch)
        self._check_ints(seq_lens, "seq_lens", (g.batch,))
        if out is None:
            out = torch.empty((g.batch, g.kv_heads, top), dtype=torch.int32, device=q.device)
        self._check_ints(out, "out", (g.batch, g.kv_heads, top))
        qs = q.stride()
        self._call(_lib.load().pkv_pages_select, "pkv_pages_select", self._struct_ref(), ctypes.byref(g), q.data_ptr(),
                   _lib.DTYPE_CODES[q.dtype], q.shape[1], qs[0], qs[1], seq_lens.data_ptr(), summaries.data_ptr(), top,
                   sinks, recent, out.data_ptr())
        return out

    # ------------------------------------------------------------------
    def select_tokens(self, weights: torch.Tensor, seq_lens: torch.Tensor, keep: int, sinks: int = 0,
                      recent: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
        """Slots to keep per (sequence, KV head) by accumulated weight, and their weights: both (B, Hkv, keep).

        Of the first seq_lens[b] entries of weights (B, Hkv, slots): the first
        ``sinks``, the last ``recent``, then the largest (ties: the lower slot;
        NaN last), ascending; -1 and 0 behind the last.
        """
        self._on_device(weights, "weights")
        if weights.dim() != 3 or weights.dtype != torch.float32 or not weights.is_contiguous():
            raise ValueError("weights must be a contiguous float32 (batch, kv_heads, slots) tensor")
        if keep < 1 or sinks < 0 or recent < 0 or sinks + recent > keep:
            raise ValueError(f"need 0 <= sinks + recent <= keep and keep >= 1, got {sinks}, {recent}, {keep}")
        B, H, T = weights.shape
        self._check_ints(seq_lens, "seq_lens", (B,))
        kept = torch.empty((B, H, keep), dtype=torch.int32, device=weights.device)
        kw = torch.empty((B, H, keep), dtype=torch.float32, device=weights.device)
        self._call(_lib.load().pkv_tokens_select, "pkv_tokens_select", weights.data_ptr(), B, H, T, T, seq_lens.data_ptr(),
                   keep, sinks, recent, kept.data_ptr(), kw.data_ptr())
        return kept, kw

    def gather_tokens(self, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, kept: torch.Tensor,
                      k_out: torch.Tensor, v_out: torch.Tensor, out_table: torch.Tensor) -> None:
        """Copy the codes of slots kept[b, hk, i] (negative: none) into slots i of out_table's pages.

        The destination pages may lie in the same pool but must not be among the
        pages that are read.
        """
        src = self._pages(k_pages, v_pages, page_table)
        dst = self._pages(k_out, v_out, out_table, "k_out")
        if k_out.dtype != k_pages.dtype or dst.batch != src.batch or dst.kv_heads != src.kv_heads:
            raise ValueError("source and destination must agree in dtype, batch and KV heads")
        if kept.dim() != 3:
            raise ValueError(f"kept must be ({src.batch}, {src.kv_heads}, keep), got {tuple(kept.shape)}")
        keep = kept.shape[2]
        self._check_ints(kept, "kept", (src.batch, src.kv_heads, keep))
        if keep > dst.max_pages * dst.page_size:
            raise ValueError(f"{keep} tokens do not fit {dst.max_pages} pages of {dst.page_size}")
        self._call(_lib.load().pkv_tokens_gather, "pkv_tokens_gather", ctypes.byref(src), self.m, kept.data_ptr(), keep,
                   ctypes.byref(dst), k_out.data_ptr(), v_out.data_ptr())
