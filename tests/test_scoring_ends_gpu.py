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
