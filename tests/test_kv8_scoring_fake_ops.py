"""The 8-bit caches' and the scoring's torch custom ops: their fake kernels on meta tensors, without a GPU; on one, a decode step
of them traced as one graph, against the calls themselves."""

import pytest
import torch

from whisper_trt_b200 import kv8, scoring

OPS = torch.ops.whisper_trt_b200
M = {"device": "meta"}
E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_kv8_fakes(dtype):
    k = torch.empty(3, 20, 1500, 64, dtype=dtype, **M)
    lengths = torch.empty(3, dtype=torch.int64, **M)
    cross = OPS.kv8_quantize_cross(k, k, lengths)
    want = kv8.empty_cross(3, 20, 1500, "meta")
    assert [(x.shape, x.dtype) for x in cross] == [(x.shape, x.dtype) for x in want]
    assert OPS.kv8_quantize_cross_into(k, k, None, *want) is None
    for s in (5, 223):
        q = torch.empty(3, s, 1280, dtype=dtype, **M)
        y = OPS.kv8_cross_attn(q, *cross, None)
        assert y.shape == q.shape and y.dtype == dtype
    cache = kv8.empty_self(10, 20, 448, "meta")
    off, src = torch.empty(10, dtype=torch.int64, **M), torch.empty(10, 448, dtype=torch.int32, **M)
    for s in (1, 17):
        qkv = torch.empty(10, s, 3840, dtype=dtype, **M)
        for op in (OPS.kv8_self_attn, OPS.kv8_self_attn_append):
            y = op(qkv, *cache, off, src)
            assert y.shape == (10, s, 1280) and y.dtype == dtype


def test_scoring_fakes():
    tokens = torch.empty(4, 7, dtype=torch.int64, **M)
    for top in (0, 5):
        for out in (OPS.token_logprobs(torch.empty(4, 7, 51866, **M), tokens, top, None),
                    OPS.score_tokens(torch.empty(4, 7, 1280, dtype=torch.float16, **M),
                                     torch.empty(51866, 1280, dtype=torch.float16, **M), tokens, top,
                                     torch.empty(51866, dtype=torch.bool, **M))):
            assert [x.shape for x in out] == [(4, 7), (4, 7), (4, 7, top), (4, 7, top)]
            assert [x.dtype for x in out] == [torch.float32] * 3 + [torch.int64]


def test_ops_declare_what_they_write():
    for op, names in ((OPS.kv8_self_attn_append, {"k8", "v8", "k_scale", "v_scale"}),
                      (OPS.kv8_quantize_cross_into, {"k8", "v8", "k_scale", "v_scale"}), (OPS.kv8_self_attn, set()),
                      (OPS.kv8_cross_attn, set()), (OPS.kv8_quantize_cross, set()), (OPS.token_logprobs, set()),
                      (OPS.score_tokens, set())):
        args = op.default._schema.arguments
        assert {a.name for a in args if a.alias_info is not None and a.alias_info.is_write} == names


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")
def test_a_traced_decode_step():
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").half()
    n, h, c, t, v = 6, 4, 40, 150, 1000
    k, val = rand(2, h, t, 64), rand(2, h, t, 64)
    lengths = torch.tensor([150, 70], device="cuda")
    src = torch.arange(n, device="cuda", dtype=torch.int32).unsqueeze(1).repeat(1, c)
    tokens, w = torch.randint(0, v, (n,), generator=g, device="cuda"), rand(v, h * 64)
    cache, plain = kv8.empty_self(n, h, c), kv8.empty_self(n, h, c)
    cross = kv8.quantize_cross(k, val, lengths)

    def step(qkv, offset, k8, v8, ks, vs, k, val, lengths, src, w, tokens):
        cross = OPS.kv8_quantize_cross(k, val, lengths)
        y = OPS.kv8_self_attn_append(qkv, k8, v8, ks, vs, offset, src)
        y = OPS.kv8_cross_attn(y.view(2, 3, -1), *cross, lengths).view(y.shape[0], -1)
        return y, *OPS.score_tokens(y, w, tokens, 3, None), *OPS.token_logprobs((y @ w.t()).float(), tokens, 2, None)

    traced = torch.compile(step, backend="aot_eager", fullgraph=True)
    for at in range(3):
        qkv, offset = rand(n, 1, 3 * h * 64), torch.full((n,), at, device="cuda")
        got = traced(qkv, offset, *cache, k, val, lengths, src, w, tokens)
        y = kv8.self_attn(qkv, plain, offset, src, write_cache=True)
        y = kv8.cross_attn(y.view(2, 3, -1), cross, lengths).view(n, -1)
        want = (y, *scoring.score_tokens(y, w, tokens, 3), *scoring.token_logprobs((y @ w.t()).float(), tokens, 2))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, plain))
