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


def _cache(r, h, c, blocks):
    kv = [torch.zeros(r, h, c, 64, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)]
    return kv8.Cache8(*kv, *(torch.ones(r, h, blocks) for _ in range(2)))


def test_results_over_the_inputs_are_refused():
    """Other rows' new tokens are read, and appended, while a row's result is written."""
    base = torch.zeros(2 * 4 * 3 * 192, dtype=torch.float16)
    qkv, cache = base.view(2, 4, 576), _cache(2, 3, 100, 100)
    off, src = torch.zeros(2, dtype=torch.int64), torch.zeros(2, 100, dtype=torch.int32)
    for at in (0, 512, base.numel() - 8 * 192):
        with pytest.raises(ValueError, match="overlap"):
            kv8.self_attn(qkv, cache, off, src, out=base[at:at + 8 * 192].view(2, 4, 192))
    with pytest.raises(ValueError, match="CUDA"):  # (apart: refused for the device alone)
        kv8.self_attn(qkv, cache, off, src, out=torch.zeros(2, 4, 192, dtype=torch.float16))
    q, cross = base[:1536].view(2, 4, 192), _cache(2, 3, 100, 2)
    with pytest.raises(ValueError, match="overlap"):
        kv8.cross_attn(q, cross, out=base[192:1728].view(2, 4, 192))
    with pytest.raises(ValueError, match="CUDA"):  # (in place)
        kv8.cross_attn(q, cross, out=q)
