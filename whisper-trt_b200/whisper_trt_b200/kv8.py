"""The decoder's attention over caches held in 8 bits: half the memory and half the traffic of the 16-bit caches of
:mod:`whisper_trt_b200.attn_plugin`, beside whose calls these stand (``wt_kv8_*`` of the C ABI).

A :class:`Cache8` holds e4m3 values and float32 scales, powers of two: a value is ``stored * scale``. The scale is the
smallest power of two, at least 2^-120, with which the largest finite magnitude of its block is at most 448; a block is

* 64 frames of one head of a window in a cross-attention cache (:func:`empty_cross`): k, v [W, H, T, 64], scales
  [W, H, ceil(T / 64)];
* one slot of one head of a row in a self-attention cache (:func:`empty_self`), whose slots are appended one by one and
  gathered one by one through the slot table: k, v [N, H, C, 64], scales [N, H, C].

Values that are not finite are stored as NaN and leave the scale to the others. A cache keeps its type whatever the
activations' (float16 or bfloat16).

:func:`quantize_cross` fills a cross cache from the encoder's keys and values, :func:`cross_attn` reads it;
:func:`self_attn` attends one or many new tokens per row and appends them. Every call launches on torch's current
stream, allocates nothing but its result, keeps nothing between calls, and can be captured into a CUDA graph (after one call,
which makes the error word of the device's waits). CUDA tensors only, contiguous; there is no CPU path.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .attn_plugin import NAMESPACE, _cuda, _dtype_code, _on, _stream, _workspace

HEAD_DIM = 64
FRAME_BLOCK = 64  # frames of a cross-attention cache that share a scale


class Cache8(NamedTuple):
    """One layer's keys and values in 8 bits: k, v float8_e4m3fn [R, H, C, 64], their scales float32 [R, H, blocks]."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def _empty(rows: int, heads: int, capacity: int, blocks: int, device) -> Cache8:
    kv = [torch.zeros(rows, heads, capacity, HEAD_DIM, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
          for _ in range(2)]
    return Cache8(*kv, *(torch.ones(rows, heads, blocks, dtype=torch.float32, device=device) for _ in range(2)))


def empty_cross(windows: int, heads: int, frames: int, device="cuda") -> Cache8:
    """A cross-attention cache of zeros."""
    return _empty(windows, heads, frames, -(-frames // FRAME_BLOCK), device)


def empty_self(rows: int, heads: int, capacity: int, device="cuda") -> Cache8:
    """A self-attention cache of zeros."""
    return _empty(rows, heads, capacity, capacity, device)


def _check_cache(what: str, cache: Cache8, frames_per_scale: int) -> tuple[int, int, int]:
    k, v, ks, vs = cache
    shape = k.shape
    if len(shape) != 4 or v.shape != shape or shape[3] != HEAD_DIM:
        raise ValueError(f"{what}: the cache's k and v must be [R, H, C, {HEAD_DIM}] of the same shape (got "
                         f"{tuple(shape)}, {tuple(v.shape)})")
    if k.dtype != torch.float8_e4m3fn or v.dtype != torch.float8_e4m3fn:
        raise TypeError(f"{what}: the cache's k and v must be float8_e4m3fn (got {k.dtype}, {v.dtype})")
    r, h, c, _ = shape
    want = (r, h, -(-c // frames_per_scale))
    if ks.shape != want or vs.shape != want:
        raise ValueError(f"{what}: the cache's scales must be {list(want)} (got {tuple(ks.shape)}, {tuple(vs.shape)})")
    if ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise TypeError(f"{what}: the cache's scales must be float32")
    return r, h, c


def _check_apart(what: str, out: torch.Tensor, x: torch.Tensor) -> None:
    a, b = out.data_ptr(), x.data_ptr()
    if a < b + x.nbytes and b < a + out.nbytes:
        raise ValueError(f"{what}: out must not overlap the input")


def _check_lengths(what: str, lengths: torch.Tensor | None, windows: int) -> tuple:
    if lengths is None:
        return ()
    if lengths.shape != (windows,) or lengths.dtype != torch.int64:
        raise ValueError(f"{what}: lengths must be [W] int64")
    return (lengths,)


def quantize_cross(k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor | None = None,
                   out: Cache8 | None = None) -> Cache8:
    """The encoder's keys and values of one layer, k, v [W, H, T, 64], as an 8-bit cache (``out``, or a new one of
    zeros). ``lengths`` [W] int64: a window's first ``lengths[w]`` frames (clamped to [0, T]) are taken, and a block's scale
    is theirs alone; later frames, and the scales of blocks that hold none of them, stay as they are in ``out``."""
    what = "kv8.quantize_cross"
    if k.dim() != 4 or v.shape != k.shape or k.shape[3] != HEAD_DIM:
        raise ValueError(f"{what}: k and v must be [W, H, T, {HEAD_DIM}] of the same shape (got {tuple(k.shape)}, "
                         f"{tuple(v.shape)})")
    w, h, t, _ = k.shape
    code = _dtype_code(k, what)
    if v.dtype != k.dtype:
        raise TypeError(f"{what}: k and v must have one dtype")
    more = _check_lengths(what, lengths, w)
    cache = empty_cross(w, h, t, k.device) if out is None else out
    if _check_cache(what, cache, FRAME_BLOCK) != (w, h, t):
        raise ValueError(f"{what}: out {tuple(cache.k.shape)} does not match k {tuple(k.shape)}")
    dev = _cuda(what, k, v, *cache, *more)
    if 0 in k.shape:
        return cache
    with _on(dev):
        st = _lib.load().wt_kv8_quantize_cross(code, k.data_ptr(), v.data_ptr(),
                                               lengths.data_ptr() if more else None,
                                               cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(),
                                               cache.v_scale.data_ptr(), w, h, t, HEAD_DIM, _stream(dev))
    _lib.check(st, what)
    return cache


def cross_attn(q: torch.Tensor, cache: Cache8, lengths: torch.Tensor | None = None, *,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q [W, S, H*64] to the 8-bit cross cache of T frames -> [W, S, H*64] in q's dtype: the attention of
    :func:`attn_plugin.cross_attn_triton` to the values the cache stands for. ``lengths`` [W] int64: a window attends to
    its first ``lengths[w]`` frames (clamped to [0, T]); what lies behind them is not read, and a window without
    frames gives zeros (a query whose scores are all -inf gives NaN, as its softmax does). ``out`` may be q itself."""
    what = "kv8.cross_attn"
    w, h, t = _check_cache(what, cache, FRAME_BLOCK)
    shape = q.shape
    if len(shape) != 3 or shape[0] != w or shape[2] != h * HEAD_DIM:
        raise ValueError(f"{what}: q {tuple(q.shape)} does not match the cache {tuple(cache.k.shape)}: it must be "
                         "[W, S, H*64]")
    s = shape[1]
    code = _dtype_code(q, what)
    more = _check_lengths(what, lengths, w)
    if out is None:
        dev = _cuda(what, q, *cache, *more)
        y = torch.empty_like(q)
    else:
        y = out
        if y.shape != shape or y.dtype != q.dtype:
            raise ValueError(f"{what}: out must be shaped and typed like q")
        if y.data_ptr() != q.data_ptr():
            _check_apart(what, y, q)
        dev = _cuda(what, q, y, *cache, *more)
    if w * s * h == 0:
        return y
    if t == 0:
        return y.zero_()
    err = _workspace(dev, "logits", (), 256)
    with _on(dev):
        st = _lib.load().wt_kv8_cross_attn(code, q.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(),
                                           cache.k_scale.data_ptr(), cache.v_scale.data_ptr(),
                                           lengths.data_ptr() if more else None, y.data_ptr(), w, s, h, t, HEAD_DIM,
                                           err.data_ptr(), _stream(dev))
    _lib.check(st, what)
    return y


def self_attn(qkv: torch.Tensor, cache: Cache8, offset: torch.Tensor, src: torch.Tensor, write_cache: bool = False, *,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """Self-attention of S >= 1 new tokens per row (qkv [N, S, 3*H*64]) over the row's cache slots below offset [N]
    int64 (clamped to [0, C]), slot j read from the row ``src[r, j]`` names (src [N, C] int32, clamped to [0, N-1]),
    and causally over the new tokens up to itself, these at their own 16 bits -> [N, S, H*64] in qkv's dtype: the
    attention of :func:`attn_plugin.self_attn_triton` and :func:`attn_plugin.self_attn_step_triton`. What a later token
    holds, values that are not finite included, does not reach a query.

    ``write_cache``: afterwards the new keys and values go, in 8 bits, into the row's own slots offset, offset + 1, ...
    (those below C) in place. The attention sees the cache as it was before the call, whatever the slot table names.
    ``out`` must not overlap qkv: other rows' tokens are read, and appended, while it is written."""
    what = "kv8.self_attn"
    n, h, c = _check_cache(what, cache, 1)
    shape = qkv.shape
    if len(shape) != 3 or shape[0] != n or shape[2] != 3 * h * HEAD_DIM:
        raise ValueError(f"{what}: qkv {tuple(qkv.shape)} does not match the cache {tuple(cache.k.shape)}: it must be "
                         "[N, S, 3*H*64]")
    s = shape[1]
    if offset.shape != (n,) or offset.dtype != torch.int64:
        raise ValueError(f"{what}: offset must be [N] int64")
    if src.shape != (n, c) or src.dtype != torch.int32:
        raise ValueError(f"{what}: src must be [N, C] int32")
    code = _dtype_code(qkv, what)
    if out is None:
        dev = _cuda(what, qkv, *cache, offset, src)
        y = torch.empty(n, s, h * HEAD_DIM, dtype=qkv.dtype, device=dev)
    else:
        y = out
        if y.shape != (n, s, h * HEAD_DIM) or y.dtype != qkv.dtype:
            raise ValueError(f"{what}: out must be [N, S, H*64] of qkv's dtype")
        _check_apart(what, y, qkv)
        dev = _cuda(what, qkv, y, *cache, offset, src)
    if n * s * h == 0:
        return y
    if c == 0:
        raise ValueError(f"{what}: the cache has no slots")
    with _on(dev):
        st = _lib.load().wt_kv8_self_attn(code, qkv.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(),
                                          cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), offset.data_ptr(),
                                          src.data_ptr(), y.data_ptr(), n, s, h, c, HEAD_DIM, int(bool(write_cache)),
                                          _stream(dev))
    _lib.check(st, what)
    return y


# --- torch custom ops (for tracing: fake kernels, and what a call writes declared) --------------------------
@torch.library.custom_op(f"{NAMESPACE}::kv8_quantize_cross", mutates_args=())
def quantize_cross_op(k: torch.Tensor, v: torch.Tensor, lengths: Optional[torch.Tensor]
                      ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """:func:`quantize_cross` into a new cache, whose four tensors it returns."""
    return tuple(quantize_cross(k, v, lengths))


@quantize_cross_op.register_fake
def _(k, v, lengths):
    w, h, t, _ = k.shape
    blocks = (t + FRAME_BLOCK - 1) // FRAME_BLOCK
    return (*(k.new_empty(k.shape, dtype=torch.float8_e4m3fn) for _ in range(2)),
            *(k.new_empty(w, h, blocks, dtype=torch.float32) for _ in range(2)))


@torch.library.custom_op(f"{NAMESPACE}::kv8_quantize_cross_into", mutates_args=("k8", "v8", "k_scale", "v_scale"))
def quantize_cross_into_op(k: torch.Tensor, v: torch.Tensor, lengths: Optional[torch.Tensor], k8: torch.Tensor,
                           v8: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
    """:func:`quantize_cross` into the cache of the last four."""
    quantize_cross(k, v, lengths, out=Cache8(k8, v8, k_scale, v_scale))


@quantize_cross_into_op.register_fake
def _(k, v, lengths, k8, v8, k_scale, v_scale):
    return None


@torch.library.custom_op(f"{NAMESPACE}::kv8_cross_attn", mutates_args=())
def cross_attn_op(q: torch.Tensor, k8: torch.Tensor, v8: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                  lengths: Optional[torch.Tensor]) -> torch.Tensor:
    """:func:`cross_attn`."""
    return cross_attn(q, Cache8(k8, v8, k_scale, v_scale), lengths)


@cross_attn_op.register_fake
def _(q, k8, v8, k_scale, v_scale, lengths):
    return torch.empty_like(q)


@torch.library.custom_op(f"{NAMESPACE}::kv8_self_attn", mutates_args=())
def self_attn_op(qkv: torch.Tensor, k8: torch.Tensor, v8: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                 offset: torch.Tensor, src: torch.Tensor) -> torch.Tensor:
    """:func:`self_attn` without the append."""
    return self_attn(qkv, Cache8(k8, v8, k_scale, v_scale), offset, src)


@torch.library.custom_op(f"{NAMESPACE}::kv8_self_attn_append", mutates_args=("k8", "v8", "k_scale", "v_scale"))
def self_attn_append_op(qkv: torch.Tensor, k8: torch.Tensor, v8: torch.Tensor, k_scale: torch.Tensor,
                        v_scale: torch.Tensor, offset: torch.Tensor, src: torch.Tensor) -> torch.Tensor:
    """:func:`self_attn` that appends the new keys and values at ``offset``."""
    return self_attn(qkv, Cache8(k8, v8, k_scale, v_scale), offset, src, write_cache=True)


@self_attn_op.register_fake
@self_attn_append_op.register_fake
def _(qkv, k8, v8, k_scale, v_scale, offset, src):
    return qkv.new_empty(qkv.shape[0], qkv.shape[1], k8.shape[1] * HEAD_DIM)
