"""Scores of given tokens at the ends of what the calls accept: rows past 2^30, vocabularies near 2^20, rows enough to be taken in
parts, contiguous logits of one token."""

import math

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA GPU")]

from test_scoring_gpu import DTYPES, _case, _check, _gen, _states  # noqa: E402,F401
from whisper_trt_b200 import attn_plugin, scoring  # noqa: E402,F401


@pytest.mark.parametrize("suppress", [False, True])
def test_logprobs_rows_past_2_30(suppress):
    n = 2**30 + 5
    if torch.cuda.mem_get_info()[0] < 32 << 30:
        pytest.skip("needs 32 GB of device memory")
    logits = torch.zeros(n, 2, dtype=torch.bfloat16, device="cuda")
    logits[-2] = torch.tensor([3.0, 1.0])
    tokens = torch.zeros(n, dtype=torch.int64, device="cuda")
    tokens[-1] = 1
    sup = torch.tensor([False, True], device="cuda") if suppress else None
    got = scoring.token_logprobs(logits, tokens, 0, sup).logprob
    if suppress:
        assert (got[:-1] == 0).all() and got[-1] == -torch.inf
        return
    assert (got[:-2] == got[0]).all() and abs(got[0].item() + math.log(2)) < 1e-6
    assert abs(got[-2].item() + math.log1p(math.exp(-2))) < 1e-6 and got[-1] == got[0]


@pytest.mark.parametrize("n", [4100, 6000])
def test_score_rows_in_passes_over_one_scratch(n):
    """Rows and alternatives enough to pass the scratch's bound; every row right, and the same bits every time, captured too."""
    x, w, tokens, sup = _states(n, 51866, 64, torch.float16, n, True)
    tokens[5] = -100
    got = scoring.score_tokens(x, w, tokens, 16, sup)
    for a in range(0, n, 1500):
        part = slice(a, a + 1500)
        _check(scoring.TokenScores(*(y[part] for y in got)), x[part].double() @ w.double().t(), tokens[part], 16, sup)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = scoring.score_tokens(x, w, tokens, 16, sup)
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(u, z) for u, z in zip(again, got))
    assert attn_plugin.workspace_errors() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_logprobs_of_one_token_at_any_stride(dtype):
    """[N, 1]: contiguous whatever the stride of the dimension of one."""
    logits, tokens, _ = _case(9, 1, dtype, 3, False)
    tokens[4] = 1
    row = logits.flatten().as_strided((9, 1), (1, 9))
    assert row.is_contiguous() and row.stride(1) != 1
    _check(scoring.token_logprobs(row, tokens, 2), logits, tokens, 2, None)
    wide = torch.full((9, 7), torch.nan, device="cuda").to(dtype)
    wide[:, 3:4] = logits
    _check(scoring.token_logprobs(wide[:, 3:4], tokens, 2), logits, tokens, 2, None)
    with pytest.raises(ValueError, match="rows apart"):
        scoring.token_logprobs(logits[:1].expand(9, 1), tokens)


@pytest.mark.parametrize("suppress", [False, True])
@pytest.mark.parametrize("n,v", [(3, 2**20), (5, 2**20 - 7), (300, 2**20 - 1)])
def test_vocabularies_near_2_20(n, v, suppress):
    """The largest masks, and more records a row than a CTA of the merge takes at once."""
    logits, tokens, sup = _case(n, v, torch.bfloat16, n, suppress)
    tokens[0] = v - 1
    _check(scoring.token_logprobs(logits, tokens, 16, sup), logits, tokens, 16, sup)
    x, w, tokens, sup = _states(n, v, 64, torch.float16, n, suppress)
    tokens[0] = v - 1
    got = scoring.score_tokens(x, w, tokens, 16, sup)
    for a in range(0, n, 50):
        part = slice(a, a + 50)
        _check(scoring.TokenScores(*(y[part] for y in got)), x[part].double() @ w.double().t(), tokens[part], 16, sup)
    assert attn_plugin.workspace_errors() == 0


def test_vocabularies_past_2_20_are_refused():
    with pytest.raises(ValueError):
        scoring.token_logprobs(torch.zeros(1, 2**20 + 1, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="too large"):
        scoring.score_tokens(torch.zeros(1, 8, device="cuda").half(), torch.zeros(2**20 + 1, 8, device="cuda").half(),
                             torch.zeros(1, dtype=torch.int64, device="cuda"))
