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


# A score of 8 a b (natural units) at the frames that count, all of them equal, and far below it at the others.
_LARGE = [(torch.float16, 2000.0, 1024.0), (torch.float16, 2000.0, 2048.0), (torch.float16, 60000.0, 28672.0),
          (torch.float16, 2000.0, -1024.0), (torch.float16, 60000.0, -14336.0), (torch.bfloat16, 1024.0, 2048.0),
          (torch.bfloat16, 2.0**20, 2.0**23), (torch.bfloat16, 2.0**40, -2.0**60), (torch.bfloat16, 1920.0, -2048.0)]


def _others(b):
    return -b if b > 0 else 2 * b


@pytest.mark.parametrize("dtype,a,b", _LARGE)
@pytest.mark.parametrize("w,s,t", [(20, 5, 150), (1, 16, 300), (20, 32, 150), (20, 40, 150), (1, 70, 700)])
def test_cross_scores_past_2_24(dtype, a, b, w, s, t):
    """Scores whose unit in the last place is 1 or more: the softmax subtracts its maximum, and equal scores stay equal, so
    the output is the mean over the frames that have it (no error of scores enters)."""
    g = _gen(s + t)
    k = torch.full((w, 1, t, 64), b, device="cuda")
    k[:, :, torch.rand(t, generator=g, device="cuda") < 0.6] = _others(b)
    k[:, :, [3, -1]] = b
    cache = kv8.quantize_cross(k.to(dtype), _randn(g, w, 1, t, 64, dtype=dtype))
    q = torch.full((w, s, 64), a, dtype=dtype, device="cuda")
    ref, mass, _, sv = _cross_reference(q, cache, None)
    _check(kv8.cross_attn(q, cache), ref, mass, 0.0, sv, 2.0**-20)


@pytest.mark.parametrize("dtype,a,b", _LARGE)
@pytest.mark.parametrize("n,s,c", [(3, 1, 150), (200, 1, 70), (3, 20, 150), (2, 100, 100)])
def test_self_scores_past_2_24(dtype, a, b, n, s, c):
    """The same over cached slots, the new tokens below them, and at the new tokens alone (rows without slots)."""
    h = 20 if n == 200 else 1
    g = _gen(s + c)
    qkv, cache, src = _self_case(g, n, s, h, c, 1, dtype)
    low = torch.rand(c, generator=g, device="cuda") < 0.6
    low[3] = low[40] = False
    k = torch.where(low[:, None], _others(b), b).expand(n, h, c, 64).contiguous().to(dtype)
    scale = torch.exp2(torch.ceil(torch.log2(k.float().abs().amax(-1) / 448)))
    cache.k.copy_((k.float() / scale[..., None]).to(torch.float8_e4m3fn))
    cache.k_scale.copy_(scale)
    offset = torch.full((n,), c, device="cuda")
    offset[0] = 0
    q3 = qkv.unflatten(-1, (3, h, 64))
    q3[:, :, 0] = a
    q3[1:, :, 1] = _others(b)
    q3[0, :, 1] = b
    y = kv8.self_attn(qkv, cache, offset, src).unflatten(-1, (h, 64))
    v = _values(cache, 1)[1]
    q64 = qkv.double().unflatten(-1, (3, h, 64))
    for r in (0, 1, n - 1):
        m = int(offset[r])
        for i in (0, s // 2, s - 1):
            seen = v[r, :, :m][:, ~low[:m]] if m else q64[r, :i + 1, 2].transpose(0, 1)
            _check(y[r, i], seen.mean(1), seen.abs().mean(1), 0.0, seen.abs().sum(1), 2.0**-16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("s,t", [(5, 100), (20, 1500), (40, 100), (40, 1500)])
def test_cross_scores_of_minus_infinity(dtype, s, t):
    """A query all of whose scores are minus infinity has no softmax (NaN); the others, and windows without frames, have."""
    g = _gen(s)
    k, v = _randn(g, 3, 2, t, 64, dtype=dtype), _randn(g, 3, 2, t, 64, dtype=dtype)
    k[..., 0] = k[..., 0].abs() + 1
    q = _randn(g, 3, s, 128, dtype=dtype)
    q[:, 1, 0] = -torch.inf
    lengths = torch.tensor([t, 0, 70], device="cuda")
    y = kv8.cross_attn(q, kv8.quantize_cross(k, v), lengths)
    assert torch.isnan(y[[0, 2], 1, :64]).all() and (y[1] == 0).all()
    y[:, 1, :64] = 0
    assert torch.isfinite(y).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("s", [1, 40])
def test_self_scores_of_minus_infinity(dtype, s):
    n, h, c = 3, 2, 90
    qkv, cache, src = _self_case(_gen(s), n, s, h, c, 1, dtype)
    cache.k.view(torch.uint8)[..., 0] &= 0x7F  # (keys at least 0 there: minus infinity, or NaN where they are 0)
    q3 = qkv.unflatten(-1, (3, h, 64))
    q3[..., 1, :, 0] = q3[..., 1, :, 0].abs() + 1
    q3[1, s - 1, 0, 1, 0] = -torch.inf
    y = kv8.self_attn(qkv, cache, torch.tensor([5, 60, 90], device="cuda"), src).unflatten(-1, (h, 64))
    assert torch.isnan(y[1, s - 1, 1]).all()
    y[1, s - 1, 1] = 0
    assert torch.isfinite(y).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("far", [30, 90])
@pytest.mark.parametrize("w,s,t", [(20, 5, 300), (20, 40, 300), (1, 70, 700), (1, 130, 1500)])
def test_cross_value_scales_far_apart(dtype, far, w, s, t):
    """Blocks of values 2^`far` times the others', at frames that next to no weight falls on: what the weight does fall on keeps
    its bits (errors are relative to a row's own sum of p |v|). Every third block, all but those, the first, the last."""
    g = _gen(s + t + far)
    q = _randn(g, w, s, 64, dtype=dtype)
    q[..., 0] = 16
    last = (t - 1) // 64
    for big in ([b for b in range(last) if b % 3 == 1], [b for b in range(last) if b % 3 != 1], [0], [last]):
        k = _randn(g, w, 1, t, 64, dtype=dtype)
        k[..., 0] = 0
        for b in big:
            k[:, :, 64 * b:64 * b + 64, 0] = -0.4 * far - 16  # (weights of about 2^-(1.15 far + 46))
        cache = kv8.quantize_cross(k, _randn(g, w, 1, t, 64, dtype=dtype))
        cache.v_scale[:, :, big] *= 2.0**far
        _check(kv8.cross_attn(q, cache), *_cross_reference(q, cache, None), 2.0**-20, least=0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("far", [30, 90])
@pytest.mark.parametrize("n,s", [(3, 1), (200, 1), (3, 20)])
def test_self_value_scales_far_apart(dtype, far, n, s):
    """The same of slots next to one another."""
    h, c = (20, 70) if n == 200 else (1, 150)
    qkv, cache, src = _self_case(_gen(s + far), n, s, h, c, 1, dtype)
    big = torch.arange(2, c, 5, device="cuda")
    cache.v_scale[:, :, big] *= 2.0**far
    cache.k_scale[:, :, big] = 2.0**-3
    cache.k.view(torch.uint8)[..., 0] = 0
    cache.k.view(torch.uint8)[:, :, big, 0] = 0xFE  # (-448: -56 with the scale)
    q3 = qkv.unflatten(-1, (3, h, 64))
    q3[:, :, 0, :, 0] = 0.0625 * far + 8  # (weights of 2^-100 and 2^-137)
    q3[:, :, 1, :, 0] = 0
    y = kv8.self_attn(qkv, cache, torch.full((n,), c, device="cuda"), src).unflatten(-1, (h, 64))
    k, v = _values(cache, 1)
    q64 = qkv.double().unflatten(-1, (3, h, 64))
    for r in (0, n - 1):
        for j in (0, h - 1):
            for i in (0, s - 1):
                kr, vr = (torch.cat((x[r, j], q64[r, :i + 1, 1 + e, j])) for e, x in enumerate((k, v)))
                _check(y[r, i:i + 1, j], *_attend(q64[r, i:i + 1, 0, j], kr[None], vr[None]), 2.0**-16, least=0.0)


@pytest.mark.parametrize("s", [2097121, 4000000])
def test_cross_queries_past_2_21(s):
    """One window and head, more queries than a grid has rows of 32 for."""
    g = _gen(s)
    cache = kv8.quantize_cross(_randn(g, 1, 1, 70, 64, dtype=torch.float16), _randn(g, 1, 1, 70, 64, dtype=torch.float16))
    q = torch.randn(1, s, 64, generator=g, device="cuda", dtype=torch.float16)
    y = kv8.cross_attn(q, cache)
    pick = torch.tensor([0, 1, s // 2, s - 129, s - 2, s - 1], device="cuda")
    _check(y[:, pick], *_cross_reference(q[:, pick], cache, None), 2.0**-20)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("w,s,t", [(3, 5, 100), (1, 5, 1500), (1, 20, 1500), (3, 130, 300), (1, 223, 1500)])
def test_cross_in_place(dtype, w, s, t):
    """The result over the queries: every query is read before its result is written, by clusters too."""
    g = _gen(s)
    cache = kv8.quantize_cross(_randn(g, w, 4, t, 64, dtype=dtype), _randn(g, w, 4, t, 64, dtype=dtype))
    q = _randn(g, w, s, 256, dtype=dtype)
    want = kv8.cross_attn(q, cache)
    for _ in range(5):
        y = q.clone()
        assert kv8.cross_attn(y, cache, out=y) is y and torch.equal(y, want)
