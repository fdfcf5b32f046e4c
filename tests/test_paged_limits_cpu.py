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
