"""What the 8-bit caches' calls refuse by sizes and by where tensors lie, on the CPU: before anything is launched."""

import ctypes

import pytest
import torch

from whisper_trt_b200 import _lib, kv8


def test_append_is_refused_before_the_attention():
    """More appended tokens than the append counts: the call does nothing, not its first half."""
    lib = _lib.load()
    buf = (ctypes.c_char * 1088)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    st = lib.wt_kv8_self_attn(0, p, p, p, p, p, p, p, p, 1 << 13, 1 << 18, 1, 4, 64, 1, None)
    assert st == _lib.WT_ERR_ARG and b"too many new tokens" in lib.wt_last_error()
