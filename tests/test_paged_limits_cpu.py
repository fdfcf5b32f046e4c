"""Limits of the paged entry points, refused before any CUDA call (no GPU needed)."""

import ctypes

import pytest

from prismkv_b200 import _lib
from test_paged_cpu import UNSUPPORTED, _args, _codec, _pages


@pytest.mark.parametrize("flags", [_lib.PKV_CODEC_FP32_ATTN, _lib.PKV_CODEC_FP32_ATTN | _lib.PKV_CODEC_Z_UNIFORM])
def test_attention_refuses_a_codec_that_asks_for_fp32_throughout(flags):
    lib, c = _lib.load(), _codec()
    c.flags = flags
    assert lib.pkv_paged_attn(ctypes.byref(c), ctypes.byref(_args()), 256, 1 << 30, None) == UNSUPPORTED
    assert lib.pkv_paged_attn_workspace_size(ctypes.byref(c), ctypes.byref(_args())) == 0


@pytest.mark.parametrize("dim,group,most", [(192, 16, 303104), (96, 1, 386432), (96, 4, 378368), (129, 8, 359744)])
def test_page_selection_refuses_tables_past_its_shared_memory(dim, group, most):
    lib, c = _lib.load(), _codec(dim)
    per = 64                                                             # codes to a row: 128 bytes, whatever the head size
    for pages in (most + 1, 0x7ffefff):
        g = _pages(kv_heads=1, token_stride=per, head_stride=per * 16, page_stride=per * 16, max_pages=pages, table_stride=pages)
        assert lib.pkv_pages_select(ctypes.byref(c), ctypes.byref(g), 256, 0, group, dim * group, dim, 256, 256, 4, 1, 1, 256,
                                    None) == UNSUPPORTED
