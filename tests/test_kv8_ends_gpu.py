"""The 8-bit caches' attention at the ends of its range, against the definition in 64 bits: weights that nearly cancel, zero
queries over zero keys, scores past 2^24, scores of minus infinity, value scales far apart."""

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

from test_kv8_gpu import DTYPES, _attend, _check, _check_cross, _cross_reference, _gen, _randn, _self_case, _values  # noqa: E402
from whisper_trt_b200 import kv8  # noqa: E402


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("s,t", [(5, 2), (8, 6), (16, 2), (24, 6), (32, 2), (40, 2), (70, 6), (130, 2)])
def test_cross_weights_in_two_parts(dtype, s, t):
    """Frames in pairs of opposite values and nearly equal weights: what is left of a pair shows the weights' own bits. Scores
    of about 2^-6, so that their fp32 sums are no part of the error; weights in two parts of 11 bits err by 2^-22."""
    g = _gen(s + t)
    k, v = _randn(g, 30, 4, t, 64, dtype=dtype), _randn(g, 30, 4, t, 64, dtype=dtype)
    v[:, :, 1::2] = -v[:, :, ::2]
    cache = kv8.quantize_cross(k, v)
    q = _randn(g, 30, s, 256, std=2.0**-7, dtype=dtype)
    _check(kv8.cross_attn(q, cache), *_cross_reference(q, cache, None), 2.0**-22)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("s", [5, 40, 130])
@pytest.mark.parametrize("w,t", [(20, 100), (1, 100), (1, 1500)])
def test_cross_zero_queries_over_zero_keys(dtype, s, w, t):
    """Zero rows and a last, partly filled block of zero keys (a padded transcript over a padded window): their scores are 0,
    whatever the product of the two scales is in fp32. Tiny ones alike."""
    g = _gen(s + t)
    k, v = _randn(g, w, 2, t, 64, dtype=dtype), _randn(g, w, 2, t, 64, dtype=dtype)
    k[:, :, t // 64 * 64:] = 0
    q = _randn(g, w, s, 128, dtype=dtype)
    q[:, ::3] = 0
    q[:, 1::3] *= 2.0**-100 if dtype == torch.bfloat16 else 2.0**-20
    y = _check_cross(q, kv8.quantize_cross(k, v))
    assert torch.isfinite(y).all()
    zero = kv8.quantize_cross(torch.zeros_like(k), v)
    _check_cross(torch.zeros_like(q), zero)
    _check_cross(torch.zeros_like(q), zero, torch.full((w,), t - 1, device="cuda"))
