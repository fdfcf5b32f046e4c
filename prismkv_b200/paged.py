"""Calls over a paged cache of packed codes: the paged half of ``DeviceCodec``.

A pool of pages holds K and V codes as (num_pages, kv_heads, page_size, m)
tensors (``empty_pages`` makes one); row b of an int32 ``page_table``
(batch, max_pages) names sequence b's pages in order and int32 ``seq_lens``
(batch) its tokens, both on the codec's device.  Token t of sequence b sits in
slot ``t % page_size`` of page ``page_table[b, t // page_size]``; entries past
the last token are never read.  ``page_size`` is a power of two, 16 to 1024.
Any strides serve whose rows start on 16-byte boundaries with unit code stride,
so (num_pages, page_size, kv_heads, m) pools pass as transposed views.

Nothing here synchronises, keeps results between calls or allocates beyond its
outputs and a workspace from torch's allocator, so every call can be captured
into a CUDA graph (``empty_summaries`` or a first ``summarize_pages`` uploads the
summaries' grid: make one of them before a capture).  A page id outside the
pool, a token past the table or a listed page not above the one before it is
skipped on the device and shows in ``_lib.device_error()`` as 6.
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
        self._grid()                                      # uploaded here, so that a capture need not
        return torch.empty((num_pages, kv_heads, 2, self.summary_pitch), dtype=torch.int8, device=self.device)

    # ------------------------------------------------------------------
    # The checks run on every call of a decode step, where the GPU may need less than 20 us: each property of a
    # tensor is read once, and the device is compared as an index (-1 for CPU tensors).
    def _index(self) -> int:
        """The codec's CUDA device index."""
        return self.device.index

    def _elsewhere(self, t: torch.Tensor, name: str) -> Exception:
        if not t.is_cuda:
            return RuntimeError(f"{name} must be a CUDA tensor")
        return ValueError(f"{name} is on {t.device}, the codec on {self.device}")

    def _check_ints(self, t: torch.Tensor, name: str, shape, dev: int) -> int:
        """Data pointer of a contiguous int32 tensor of that shape."""
        if t.get_device() != dev:
            raise self._elsewhere(t, name)
        if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor of shape {tuple(shape)}, "
                             f"got {t.dtype} {tuple(t.shape)}")
        return t.data_ptr()

    def _check_table(self, page_table: torch.Tensor, dev: int):
        """(data pointer, row stride, batch, max_pages) of a page table."""
        if page_table.get_device() != dev:
            raise self._elsewhere(page_table, "page_table")
        shape = page_table.shape
        if page_table.dtype is torch.int32 and len(shape) == 2:
            B, n = shape
            stride, inner = page_table.stride()
            if n <= 1 or inner == 1:
                return page_table.data_ptr(), stride if B > 1 else n, B, n
        raise ValueError("page_table must be an int32 (batch, max_pages) tensor with unit inner stride")

    def _pages(self, k: torch.Tensor, v: Optional[torch.Tensor], page_table: torch.Tensor, dev: int,
               name: str = "k_pages") -> _lib.PkvPages:
        if k.get_device() != dev:
            raise self._elsewhere(k, name)
        shape = k.shape
        if len(shape) != 4 or shape[3] != self.m or shape[1] < 1:
            raise ValueError(f"{name} must be (num_pages, kv_heads, page_size, {self.m}), got {tuple(shape)}")
        P, H, ps, _ = shape
        dtype = k.dtype
        code_bytes = PAGE_CODE_DTYPES.get(dtype)
        if code_bytes is None:
            raise ValueError("codes must be stored as uint8 or 16-bit integers")
        strides = k.stride()
        vp = None
        if v is not None:
            if v.get_device() != dev:
                raise self._elsewhere(v, "v_pages")
            # (a dimension of one element has no stride of its own)
            if v.shape != shape or v.dtype is not dtype or (v.stride() != strides and any(
                    n > 1 and a != b for n, a, b in zip(shape, strides, v.stride()))):
                raise ValueError("k_pages and v_pages must have the same shape, dtype and strides")
            vp = v.data_ptr()
        if strides[3] != 1:
            raise ValueError("codes need unit stride within a row")
        if ps < 16 or ps > 1024 or ps & (ps - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {ps}")
        table, table_stride, B, max_pages = self._check_table(page_table, dev)
        return _lib.PkvPages(k.data_ptr(), vp, code_bytes, P, H, ps, strides[0] if P > 1 else 0,
                             strides[1] if H > 1 else 0, strides[2], table, table_stride, B, max_pages)

    def _query(self, q: torch.Tensor, kv_heads: int, batch: int, dev: int):
        """(q, its shape, strides and dtype code) with unit inner stride, in a type the kernels read."""
        if q.get_device() != dev:
            raise self._elsewhere(q, "q")
        if q.dim() == 4:
            if q.shape[2] != 1:
                raise ValueError("paged attention takes one query token (Sq == 1)")
            q = q[:, :, 0, :]
        shape = q.shape
        if len(shape) != 3 or shape[0] != batch or shape[2] != self.dim:
            raise ValueError(f"q must be ({batch}, q_heads, {self.dim}), got {tuple(shape)}")
        if shape[1] < 1 or shape[1] % kv_heads:
            raise ValueError(f"{shape[1]} query heads do not divide among {kv_heads} KV heads")
        code = _lib.DTYPE_CODES.get(q.dtype)
        if code is None:
            q, code = q.float(), _lib.PKV_F32
        strides = q.stride()
        if strides[2] != 1:
            q = q.contiguous()
            strides = q.stride()
        return q, shape, strides, code

    def _weight_rows(self, t: torch.Tensor, name: str, B: int, H: int, dev: int) -> int:
        """Floats from one (sequence, KV head) row of weights to the next."""
        if t.get_device() != dev:
            raise self._elsewhere(t, name)
        if t.dtype is torch.float32 and t.dim() == 3 and t.shape[:2] == (B, H):
            n = t.shape[2]
            if t.is_contiguous():
                return n
            s0, s1, s2 = t.stride()
            row = s1 if H > 1 else s0 if B > 1 else n
            if (n <= 1 or s2 == 1) and (B <= 1 or H <= 1 or s0 == H * s1) and row >= n:
                return row
        raise ValueError(f"{name} must be a float32 ({B}, {H}, slots) tensor, contiguous or the first slots of one")

    def _call(self, fn, what: str, dev: int, *args) -> None:
        """fn(*args, stream) with CUDA device ``dev`` current; a non-zero status raises."""
        if torch.cuda.current_device() == dev:
            rc = fn(*args, _lib.raw_stream(dev))
        else:
            with torch.cuda.device(dev):
                rc = fn(*args, _lib.raw_stream(dev))
        if rc:
            _lib.check(rc, what)

    # ------------------------------------------------------------------
    def paged_attention(self, q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                        page_table: torch.Tensor, seq_lens: torch.Tensor, scale: Optional[float] = None,
                        pages: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None,
                        weights_out: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                        out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """Decode attention over a paged cache: q (B, Hq, dim) [or (B, Hq, 1, dim)] -> (B, Hq, dim) of out_dtype.

        The workspace holds a float per query head and slot of the page table
        when there are ``weights``: pass the table's first columns, as far as
        the longest sequence goes, and the weights' first slots.
        ``pages`` (B, Hkv, n) int32 restricts each KV head to the listed logical
        pages (``select_pages`` makes such lists): strictly ascending, -1 behind
        the last.  ``weights`` (B, Hkv, slots) fp32: every attended token's
        softmax weights, summed over the KV head's query heads, are added --
        in place, or into ``weights_out`` of the same shape, whose other entries
        are not touched; slots must cover every token.  A sequence without
        tokens gives zeros.  Operands are fp16 (hi, lo) pairs, so a codec with
        ``fp32_attention`` set is refused.
        """
        dev = self._index()
        g = self._pages(k_pages, v_pages, page_table, dev)
        B, kv_heads = g.batch, g.kv_heads
        q, shape, qs, q_code = self._query(q, kv_heads, B, dev)
        Hq = shape[1]
        lens = self._check_ints(seq_lens, "seq_lens", (B,), dev)
        if out is None:
            out_code = _lib.DTYPE_CODES.get(out_dtype)
            if out_code is None:
                raise ValueError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
            out = q.new_empty(shape, dtype=out_dtype)
        else:
            if out.get_device() != dev:
                raise self._elsewhere(out, "out")
            out_code = _lib.DTYPE_CODES.get(out.dtype)
            if out.shape != shape or out_code is None or out.stride(2) != 1:
                raise ValueError(f"out must be a ({B}, {Hq}, {self.dim}) float tensor with unit inner stride")
        os = out.stride()
        selected, n_selected = None, 0
        if pages is not None:
            if pages.dim() != 3:
                raise ValueError(f"pages must be ({B}, {kv_heads}, n), got {tuple(pages.shape)}")
            n_selected = pages.shape[2]
            selected = self._check_ints(pages, "pages", (B, kv_heads, n_selected), dev)
            if n_selected == 0:
                raise ValueError("pages lists no page; leave it out to attend to every token")
        w_in = w_out = None
        slots = row = 0
        if weights_out is not None and weights is None:
            raise ValueError("weights_out needs weights")
        if weights is not None:
            to = weights if weights_out is None else weights_out
            row = self._weight_rows(weights, "weights", B, kv_heads, dev)
            if to is not weights:
                if self._weight_rows(to, "weights_out", B, kv_heads, dev) != row or to.shape != weights.shape:
                    raise ValueError("weights and weights_out must have the same shape and strides")
            w_in, w_out, slots = weights.data_ptr(), to.data_ptr(), weights.shape[2]
        args = ctypes.byref(_lib.PkvPagedAttnArgs(
            g, Hq, q_code, q.data_ptr(), qs[0], qs[1], lens, selected, n_selected,
            self.dim ** -0.5 if scale is None else float(scale), out.data_ptr(), out_code, os[0], os[1], w_in, w_out, row,
            slots))
        lib = _lib.load()
        # the workspace's size follows from the shapes alone
        key = (B, Hq, kv_heads, g.page_size, g.max_pages, n_selected, not w_in)    # (no slots: a null pointer)
        sizes = self.__dict__.setdefault("_paged_sizes", {})
        need = sizes.get(key)
        if need is None:
            with torch.cuda.device(dev):
                need = int(lib.pkv_paged_attn_workspace_size(self._struct_ref(), args))
            if need:                                      # 0: nothing to do, or arguments that the call refuses
                if len(sizes) > 256:
                    sizes.clear()
                sizes[key] = need
        ws = q.new_empty(need, dtype=torch.uint8)
        self._call(lib.pkv_paged_attn, "pkv_paged_attn", dev, self._struct_ref(), args, ws.data_ptr(), need)
        return out

    def _struct_ref(self):
        return ctypes.byref(self.struct)

    # ------------------------------------------------------------------
    def store_pages(self, codes: torch.Tensor, pages: torch.Tensor, page_table: torch.Tensor, start: torch.Tensor,
                    counts: Optional[torch.Tensor] = None) -> None:
        """Copy codes (B, Hkv, n, m) into slots start[b] .. of one pool; counts[b] < n leaves padded rows out."""
        dev = self._index()
        g = self._pages(pages, None, page_table, dev, "pages")
        if codes.get_device() != dev:
            raise self._elsewhere(codes, "codes")
        if codes.dim() != 4 or codes.dtype != pages.dtype or (codes.shape[0], codes.shape[1], codes.shape[3]) != (
                g.batch, g.kv_heads, self.m):
            raise ValueError(f"codes must be ({g.batch}, {g.kv_heads}, n, {self.m}) of the pool's dtype")
        codes = codes.contiguous()
        first = self._check_ints(start, "start", (g.batch,), dev)
        taken = None if counts is None else self._check_ints(counts, "counts", (g.batch,), dev)
        self._call(_lib.load().pkv_pages_store, "pkv_pages_store", dev, ctypes.byref(g), self.m, pages.data_ptr(),
                   codes.data_ptr(), codes.shape[2], first, taken)

    def _grid(self):
        """Device tables of the summaries' grid, built on first use."""
        if getattr(self, "_grid_z", None) is None:
            z, xy = _summary_grid(np.asarray(self.host.dec_z), np.asarray(self.host.dec_xy), 1 << self.bits_total)
            if (np.diff(z.astype(np.int64)) < 0).any():
                raise ValueError("page summaries need decoded z values that rise with the bin")
            self._grid_xy = torch.from_numpy(np.ascontiguousarray(xy)).to(self.device)
            self._grid_z = torch.from_numpy(z).to(self.device)
        return self._grid_z, self._grid_xy

    def _check_summaries(self, t: torch.Tensor, g: _lib.PkvPages, dev: int) -> int:
        """Data pointer of the pool's summaries."""
        if t.get_device() != dev:
            raise self._elsewhere(t, "summaries")
        want = (g.num_pages, g.kv_heads, 2, self.summary_pitch)
        if t.dtype is not torch.int8 or t.shape != want or not t.is_contiguous():
            raise ValueError(f"summaries must be a contiguous int8 {want} tensor, got {t.dtype} {tuple(t.shape)}")
        return t.data_ptr()

    def summarize_pages(self, k_pages: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                        summaries: torch.Tensor, start: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Least and greatest decoded key per page, KV head and rotated channel, rounded outwards to int8.

        Writes the summaries of the pages that hold a token >= start[b] of
        sequence b (of every page without ``start``) into ``summaries``
        (num_pages, Hkv, 2, summary_pitch) and returns it.  One step is 1/127 of
        the codec's largest decoded magnitude; values within 1/256 of a step of
        a whole number count as it.
        """
        dev = self._index()
        g = self._pages(k_pages, None, page_table, dev)
        lens = self._check_ints(seq_lens, "seq_lens", (g.batch,), dev)
        to = self._check_summaries(summaries, g, dev)
        first = None if start is None else self._check_ints(start, "start", (g.batch,), dev)
        gz, gxy = self._grid()
        self._call(_lib.load().pkv_pages_summarize, "pkv_pages_summarize", dev, self._struct_ref(), ctypes.byref(g), lens,
                   first, gz.data_ptr(), gxy.data_ptr(), to)
        return summaries

    def select_pages(self, q: torch.Tensor, summaries: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                     page_size: int, top: int, sinks: int = 1, recent: int = 1,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The pages worth attending to: (B, Hkv, top) int32 logical pages, ascending, -1 behind the last.

        The first ``sinks`` and last ``recent`` pages of a sequence are always
        taken, the others by the greatest score that a token within the page's
        bounds could have: the KV head's queries, rotated and rounded to int8
        on a common scale, against the summaries' greatest (positive) and least
        (negative) values (an upper bound for the rounded queries, not for the
        queries themselves); the largest over the heads counts, ties go to the
        lower page.  A page table
        of more than about 300000 columns is refused (``pkv_pages_select`` gives
        the limit): pass the columns that the sequences use.
        """
        if summaries.dim() != 4:
            raise ValueError("summaries must be (num_pages, kv_heads, 2, summary_pitch)")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        if top < 1 or sinks < 0 or recent < 0 or sinks + recent > top:
            raise ValueError(f"need 0 <= sinks + recent <= top and top >= 1, got {sinks}, {recent}, {top}")
        dev = self._index()
        table, table_stride, B, max_pages = self._check_table(page_table, dev)
        g = _lib.PkvPages(None, None, 1, summaries.shape[0], summaries.shape[1], page_size, 0, 0,
                          -(-self.m // ROW_BYTES) * ROW_BYTES, table, table_stride, B, max_pages)
        sums = self._check_summaries(summaries, g, dev)
        q, shape, qs, q_code = self._query(q, g.kv_heads, B, dev)
        lens = self._check_ints(seq_lens, "seq_lens", (B,), dev)
        if out is None:
            out = q.new_empty((B, g.kv_heads, top), dtype=torch.int32)
            to = out.data_ptr()
        else:
            to = self._check_ints(out, "out", (B, g.kv_heads, top), dev)
        self._call(_lib.load().pkv_pages_select, "pkv_pages_select", dev, self._struct_ref(), ctypes.byref(g), q.data_ptr(),
                   q_code, shape[1], qs[0], qs[1], lens, sums, top, sinks, recent, to)
        return out

    # ------------------------------------------------------------------
    def select_tokens(self, weights: torch.Tensor, seq_lens: torch.Tensor, keep: int, sinks: int = 0,
                      recent: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
        """Slots to keep per (sequence, KV head) by accumulated weight, and their weights: both (B, Hkv, keep).

        Of the first seq_lens[b] entries of weights (B, Hkv, slots): the first
        ``sinks``, the last ``recent``, then the largest (ties: the lower slot;
        NaN last), ascending; -1 and 0 behind the last.
        """
        dev = self._index()
        if weights.dim() != 3:
            raise ValueError("weights must be a float32 (batch, kv_heads, slots) tensor")
        row = self._weight_rows(weights, "weights", weights.shape[0], weights.shape[1], dev)
        if keep < 1 or sinks < 0 or recent < 0 or sinks + recent > keep:
            raise ValueError(f"need 0 <= sinks + recent <= keep and keep >= 1, got {sinks}, {recent}, {keep}")
        B, H, T = weights.shape
        lens = self._check_ints(seq_lens, "seq_lens", (B,), dev)
        kept = weights.new_empty((B, H, keep), dtype=torch.int32)
        kw = weights.new_empty((B, H, keep))
        self._call(_lib.load().pkv_tokens_select, "pkv_tokens_select", dev, weights.data_ptr(), B, H, T, row, lens, keep,
                   sinks, recent, kept.data_ptr(), kw.data_ptr())
        return kept, kw

    def gather_tokens(self, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, kept: torch.Tensor,
                      k_out: torch.Tensor, v_out: torch.Tensor, out_table: torch.Tensor) -> None:
        """Copy the codes of slots kept[b, hk, i] (negative: none) into slots i of out_table's pages.

        The destination pages may lie in the same pool but must not be among the
        pages that are read.
        """
        dev = self._index()
        src = self._pages(k_pages, v_pages, page_table, dev)
        dst = self._pages(k_out, v_out, out_table, dev, "k_out")
        if k_out.dtype is not k_pages.dtype or dst.batch != src.batch or dst.kv_heads != src.kv_heads:
            raise ValueError("source and destination must agree in dtype, batch and KV heads")
        if kept.dim() != 3:
            raise ValueError(f"kept must be ({src.batch}, {src.kv_heads}, keep), got {tuple(kept.shape)}")
        keep = kept.shape[2]
        slots = self._check_ints(kept, "kept", (src.batch, src.kv_heads, keep), dev)
        if keep > dst.max_pages * dst.page_size:
            raise ValueError(f"{keep} tokens do not fit {dst.max_pages} pages of {dst.page_size}")
        self._call(_lib.load().pkv_tokens_gather, "pkv_tokens_gather", dev, ctypes.byref(src), self.m, slots, keep,
                   ctypes.byref(dst), dst.k, dst.v)
