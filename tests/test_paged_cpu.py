"""The paged entry points refuse malformed arguments before any CUDA call, and the summaries' grid is
what its definition says (no GPU needed)."""

import ctypes

import numpy as np
import pytest
import torch

from prismkv_b200 import _lib
from prismkv_b200.paged import _summary_grid

INVALID, UNSUPPORTED, ALIGNMENT, WORKSPACE = 1, 2, 3, 4


def _codec(dim=96, bits=(4, 4, 4)):
    c = _lib.PkvCodec()
    c.dim = dim
    c.bits_z, c.bits_r, c.bits_theta = bits
    c.R = c.dec_z = c.dec_xy = 16
    return c


def _pages(**kw):
    g = _lib.PkvPages()
    g.k = g.v = g.table = 256
    g.code_bytes, g.num_pages, g.kv_heads, g.page_size = 2, 8, 4, 16
    g.token_stride, g.head_stride, g.page_stride = 32, 512, 2048
    g.batch, g.max_pages, g.table_stride = 2, 4, 4
    for k, v in kw.items():
        setattr(g, k, v)
    return g


def _args(pages=None, **kw):
    a = _lib.PkvPagedAttnArgs()
    a.pages = pages or _pages()
    a.q_heads, a.q_dtype, a.out_dtype, a.scale = 8, 0, 0, 0.1
    a.q = a.out = a.seq_lens = 256
    for k, v in kw.items():
        setattr(a, k, v)
    return a


PAGE_FAULTS = [
    (dict(page_size=8), INVALID), (dict(page_size=48), INVALID), (dict(page_size=2048), INVALID),
    (dict(kv_heads=0), INVALID), (dict(num_pages=-1), INVALID), (dict(batch=-1), INVALID),
    (dict(code_bytes=4), INVALID), (dict(token_stride=31), INVALID), (dict(table=None), INVALID),
    (dict(table_stride=3), INVALID), (dict(token_stride=36), ALIGNMENT), (dict(head_stride=516), ALIGNMENT),
    (dict(page_stride=2049), ALIGNMENT), (dict(k=264), ALIGNMENT), (dict(k=None), INVALID),
    (dict(max_pages=1 << 27, table_stride=1 << 27, page_size=16), UNSUPPORTED),
]


@pytest.mark.parametrize("kw,code", PAGE_FAULTS)
def test_attention_refuses_bad_pages(kw, code):
    lib = _lib.load()
    assert lib.pkv_paged_attn(ctypes.byref(_codec()), ctypes.byref(_args(_pages(**kw))), 256, 1 << 30, None) == code
    assert lib.pkv_paged_attn_workspace_size(ctypes.byref(_codec()), ctypes.byref(_args(_pages(**kw)))) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(q_heads=6), INVALID), (dict(q_heads=0), INVALID), (dict(q_heads=68), UNSUPPORTED), (dict(q_dtype=3), INVALID),
    (dict(out_dtype=-1), INVALID), (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
    (dict(n_selected=-1), INVALID), (dict(n_selected=4), INVALID), (dict(weights=256), INVALID),
    (dict(weights_out=256), INVALID), (dict(weights=256, weights_out=256, weights_slots=64, weights_row_stride=63), INVALID),
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(seq_lens=None), INVALID)])
def test_attention_refuses_bad_arguments(kw, code):
    lib = _lib.load()
    assert lib.pkv_paged_attn(ctypes.byref(_codec()), ctypes.byref(_args(**kw)), 256, 1 << 30, None) == code


@pytest.mark.parametrize("kw,code", [(dict(dim=95), INVALID), (dict(dim=195), UNSUPPORTED), (dict(bits=(0, 4, 4)), INVALID),
                                     (dict(bits=(5, 4, 4)), UNSUPPORTED)])
def test_attention_refuses_bad_codec(kw, code):
    lib = _lib.load()
    assert lib.pkv_paged_attn(ctypes.byref(_codec(**kw)), ctypes.byref(_args()), 256, 1 << 30, None) == code


def test_one_byte_codes_hold_eight_bits():
    lib = _lib.load()
    g = _pages(code_bytes=1)
    assert lib.pkv_paged_attn(ctypes.byref(_codec()), ctypes.byref(_args(g)), 256, 1 << 30, None) == INVALID
    assert lib.pkv_pages_summarize(ctypes.byref(_codec()), ctypes.byref(g), 256, None, 256, 256, 256, None) == INVALID


def test_empty_batch_launches_nothing():
    lib = _lib.load()
    g = _pages(batch=0)
    c = _codec()
    assert lib.pkv_paged_attn(ctypes.byref(c), ctypes.byref(_args(g)), None, 0, None) == 0
    assert lib.pkv_pages_store(ctypes.byref(g), 32, 256, 256, 3, 256, None, None) == 0
    assert lib.pkv_pages_store(ctypes.byref(_pages()), 32, 256, 256, 0, 256, None, None) == 0
    assert lib.pkv_pages_summarize(ctypes.byref(c), ctypes.byref(g), 256, None, 256, 256, 256, None) == 0
    assert lib.pkv_pages_select(ctypes.byref(c), ctypes.byref(g), 256, 0, 8, 96, 96, 256, 256, 4, 1, 1, 256, None) == 0
    assert lib.pkv_tokens_select(256, 0, 4, 16, 16, 256, 4, 0, 0, 256, 256, None) == 0
    assert lib.pkv_tokens_gather(ctypes.byref(g), 32, 256, 4, ctypes.byref(g), 256, 256, None) == 0


def test_other_calls_refuse_bad_arguments():
    lib = _lib.load()
    c, g = _codec(), _pages()
    sel = lambda **k: lib.pkv_pages_select(  # noqa: E731
        ctypes.byref(c), ctypes.byref(k.get("g", g)), k.get("q", 256), k.get("dt", 0), k.get("hq", 8), 768, 96,
        k.get("lens", 256), k.get("sums", 256), k.get("top", 4), k.get("sinks", 1), k.get("recent", 1), k.get("out", 256), None)
    assert sel(top=0) == INVALID and sel(sinks=-1) == INVALID and sel(sinks=3, recent=2) == INVALID
    assert sel(hq=7) == INVALID and sel(hq=68) == UNSUPPORTED and sel(dt=5) == INVALID
    assert sel(q=None) == INVALID and sel(out=None) == INVALID and sel(sums=None) == INVALID and sel(sums=8) == ALIGNMENT
    assert sel(g=_pages(page_size=24)) == INVALID
    # pages past what the cluster's shared memory holds
    keep = lambda **k: lib.pkv_tokens_select(  # noqa: E731
        k.get("w", 256), k.get("B", 1), k.get("H", 4), k.get("T", 64), k.get("rs", 64), k.get("lens", 256), k.get("keep", 8),
        k.get("sinks", 1), k.get("recent", 1), k.get("kept", 256), k.get("kw", 256), None)
    assert keep(keep=0) == INVALID and keep(sinks=5, recent=4) == INVALID and keep(recent=-1) == INVALID
    assert keep(rs=63) == INVALID and keep(H=0) == INVALID and keep(B=-1) == INVALID and keep(w=None) == INVALID
    assert keep(kept=None) == INVALID and keep(kw=None) == INVALID and keep(lens=None) == INVALID
    gather = lambda d, keep=8, kept=256, dk=256: lib.pkv_tokens_gather(  # noqa: E731
        ctypes.byref(g), 32, kept, keep, ctypes.byref(d), dk, 256, None)
    assert gather(_pages(kv_heads=2)) == INVALID and gather(_pages(batch=1)) == INVALID
    assert gather(_pages(code_bytes=1)) == INVALID and gather(_pages(), keep=65) == INVALID
    assert gather(_pages(), kept=None) == INVALID and gather(_pages(), dk=None) == INVALID
    assert gather(_pages(), dk=264) == ALIGNMENT and gather(_pages(), keep=-1) == INVALID
    store = lambda n=1, dst=256, start=256: lib.pkv_pages_store(  # noqa: E731
        ctypes.byref(g), 32, dst, 256, n, start, None, None)
    assert store(n=-1) == INVALID and store(dst=None) == INVALID and store(start=None) == INVALID and store(dst=8) == ALIGNMENT
    assert lib.pkv_pages_summarize(ctypes.byref(c), ctypes.byref(g), 256, None, 256, 256, 264, None) == ALIGNMENT
    assert lib.pkv_pages_summarize(ctypes.byref(c), ctypes.byref(g), None, None, 256, 256, 256, None) == INVALID


def test_workspace_is_checked():
    lib = _lib.load()
    if not torch.cuda.is_available():
        pytest.skip("the size depends on the device")
    a = _args()
    need = lib.pkv_paged_attn_workspace_size(ctypes.byref(_codec()), ctypes.byref(a))
    assert need > 0
    assert lib.pkv_paged_attn(ctypes.byref(_codec()), ctypes.byref(a), None, 0, None) == WORKSPACE
    assert lib.pkv_paged_attn(ctypes.byref(_codec()), ctypes.byref(a), 256, need - 1, None) == WORKSPACE


def test_cpu_tensors_are_refused():
    from prismkv_b200.paged import PagedOps

    class Stub(PagedOps):
        dim, m, bits_total, device = 96, 32, 12, torch.device("cuda", 0)

    k = torch.zeros(2, 1, 16, 32, dtype=torch.int16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        Stub().paged_attention(torch.zeros(1, 1, 96), k, k, table, lens)
    with pytest.raises(RuntimeError, match="CUDA"):
        Stub().select_tokens(torch.zeros(1, 1, 4), lens, 2)


def test_summary_grid():
    z = np.linspace(-3, 3, 16).astype(np.float32)
    xy = np.stack([np.linspace(-6, 6, 256), np.zeros(256)], -1).astype(np.float32)
    gz, gxy = _summary_grid(z, xy, 4096)
    assert gz.dtype == np.int16 and gxy.shape == (4096, 2)
    assert gxy[255, 0] == 127 * 128 and gxy[0, 0] == -127 * 128 and (gxy[:, 1] == 0).all()
    assert np.array_equal(gxy[:256], gxy[256:512])
    assert np.abs(gz / 128.0 * (6 / 127) - z).max() <= 6 / 127 / 256 + 1e-7
    gz, gxy = _summary_grid(np.zeros(2, np.float32), np.zeros((4, 2), np.float32), 8)     # a table of zeros
    assert not gz.any() and not gxy.any()


def test_indexes_that_pass_32_bits_are_refused():
    lib = _lib.load()
    c, big = _codec(), 0x7fffffff
    keep = lambda slots, keep: lib.pkv_tokens_select(256, 1, 1, slots, big, 256, keep, 0, 0, 256, 256, None)  # noqa: E731
    assert keep(big, 8) == UNSUPPORTED and keep(0x7fff0001, 8) == UNSUPPORTED and keep(64, big) == UNSUPPORTED
    assert lib.pkv_pages_select(ctypes.byref(c), ctypes.byref(_pages()), 256, 0, 8, 96, 96, 256, 256, big, 1, 1, 256,
                                None) == UNSUPPORTED
    wide = _pages(max_pages=0x7ffffff, table_stride=0x7ffffff)           # 2^31 - 16 tokens
    assert lib.pkv_paged_attn(ctypes.byref(c), ctypes.byref(_args(wide)), 256, 1 << 30, None) == UNSUPPORTED
    assert lib.pkv_tokens_gather(ctypes.byref(_pages()), 32, 256, 8, ctypes.byref(wide), 256, 256, None) == UNSUPPORTED
    assert lib.pkv_paged_attn(ctypes.byref(c), ctypes.byref(_args(selected=256, n_selected=0x7ffffff)), 256, 1 << 30,
                              None) == UNSUPPORTED
