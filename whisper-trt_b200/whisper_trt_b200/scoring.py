"""How likely a given text is: per row the log-probability of one token, the entropy of the distribution it was drawn
from, and the most likely alternatives -- what word confidences, a segment's average log-probability and the comparison of two
builds of a model on one transcript are made of (``wt_token_logprobs``, ``wt_score_tokens`` of the C ABI).

:func:`token_logprobs` takes the logits a decode step has in hand (:func:`attn_plugin.logits32_triton`'s, or 16-bit
ones), :func:`score_tokens` the hidden states before the vocabulary projection: it computes the logits as
:func:`attn_plugin.logits32_triton` does, on the tensor cores with fp32 sums, and reduces them on the way, so that a batch of
forced transcripts does not write and read its [N, V] logits. Both launch on torch's current stream, keep nothing
between calls and can be captured into a CUDA graph (after one call, which makes the error word of the device's waits).
CUDA tensors only; there is no CPU path.

Definitions, for a row's logits x with the suppressed tokens at -inf: p = softmax(x); ``logprob`` = ln p[token],
-inf for a suppressed token, 0 for a row whose token is outside [0, V) (padding: it then adds nothing to a sum);
``entropy`` = -sum p ln p; ``top_logprob`` / ``top_token``: the ``top`` largest logits, equal ones in the order of their
tokens, as ln p and token; places that no token with a logit above -inf is left for hold (-inf, -1). A row without any
such token has entropy 0 and log-probability -inf. A NaN or +inf logit makes a row's log-probabilities and entropy NaN.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .attn_plugin import NAMESPACE, _cuda, _dtype_code, _on, _stream, _workspace

MAX_TOP = 16


class TokenScores(NamedTuple):
    """logprob [...], entropy [...], top_logprob [..., top] float32; top_token [..., top] int64."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: torch.Tensor
    top_token: torch.Tensor


def _prepare(what: str, lead: torch.Size, vocab: int, tokens: torch.Tensor, top: int, suppress: torch.Tensor | None,
             dev: torch.device) -> TokenScores:
    if tokens.shape != lead or tokens.dtype != torch.int64:
        raise ValueError(f"{what}: tokens must be {list(lead)} int64 (got {list(tokens.shape)} {tokens.dtype})")
    if max(tokens.numel(), vocab) >= 2**31:
        raise ValueError(f"{what}: too large ({tokens.numel()} rows, {vocab} tokens)")
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"{what}: top must be 0 to {MAX_TOP} (got {top})")
    if suppress is not None and (suppress.shape != (vocab,) or suppress.dtype != torch.bool):
        raise ValueError(f"{what}: suppress must be [V] = [{vocab}] bool")
    f32 = torch.float32
    return TokenScores(torch.empty_like(tokens, dtype=f32), torch.empty_like(tokens, dtype=f32),
                       torch.empty(*lead, top, dtype=f32, device=dev),
                       torch.empty(*lead, top, dtype=torch.int64, device=dev))


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0,
                   suppress: torch.Tensor | None = None) -> TokenScores:
    """The scores of ``tokens`` [N] int64 under ``logits`` [N, V] (float32, float16 or bfloat16), or tokens [...] under
    logits [..., V]. The rows of 2-D logits may lie any distance apart (a slice of a padded vocabulary). ``suppress``
    [V] bool: tokens that are left out."""
    what = "token_logprobs"
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError(f"{what}: logits must be [..., V] with V > 0 (got {tuple(logits.shape)})")
    vocab = logits.shape[-1]
    code = _lib.WT_F32 if logits.dtype == torch.float32 else _dtype_code(logits, what)
    more = () if suppress is None else (suppress,)
    dev = _cuda(what, tokens, *more)
    if logits.device != dev:
        raise ValueError(f"{what}: tensors on different devices ({logits.device}, {dev})")
    if logits.dim() == 2 and logits.shape[0] > 1:
        if (logits.stride(1) != 1 and vocab > 1) or logits.stride(0) < vocab:
            raise ValueError(f"{what}: the tokens of a row of logits must be adjacent, its rows apart (strides "
                             f"{logits.stride()})")
        stride = logits.stride(0)
    else:
        _cuda(what, logits)
        stride = vocab
    out = _prepare(what, logits.shape[:-1], vocab, tokens, top, suppress, dev)
    n = tokens.numel()
    if n == 0:
        return out
    with _on(dev):
        st = _lib.load().wt_token_logprobs(code, logits.data_ptr(), stride, tokens.data_ptr(),
                                           suppress.data_ptr() if more else None, out.logprob.data_ptr(),
                                           out.entropy.data_ptr(), out.top_logprob.data_ptr() if top else None,
                                           out.top_token.data_ptr() if top else None, n, vocab, top, _stream(dev))
    _lib.check(st, what)
    return out


def score_tokens(x: torch.Tensor, w: torch.Tensor, tokens: torch.Tensor, top: int = 0,
                 suppress: torch.Tensor | None = None) -> TokenScores:
    """The scores of ``tokens`` [...] int64 under the logits x . w^T of hidden states ``x`` [..., d] and a vocabulary
    projection ``w`` [V, d] (both float16 or both bfloat16, d a multiple of 8), logits in fp32. The call takes scratch from
    torch's allocator, 2 * slices of the vocabulary * (16 + 4 * (2 + 32) * top) bytes a row (at 51866 tokens some 9 kB a row
    with one alternative, 41 kB with five), at most 320 MiB: further rows go in passes over the same scratch."""
    what = "score_tokens"
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1] or 0 in w.shape:
        raise ValueError(f"{what}: x must be [..., d] and w [V, d] (got {tuple(x.shape)}, {tuple(w.shape)})")
    vocab, d = w.shape
    code = _dtype_code(x, what)
    if w.dtype != x.dtype:
        raise TypeError(f"{what}: x and w must have the same dtype")
    more = () if suppress is None else (suppress,)
    dev = _cuda(what, x, w, tokens, *more)
    out = _prepare(what, x.shape[:-1], vocab, tokens, top, suppress, dev)
    n = tokens.numel()
    if n == 0:
        return out
    err = _workspace(dev, "logits", (), 256)
    lib = _lib.load()
    with _on(dev):
        nbytes = int(lib.wt_score_tokens_workspace(n, vocab, d, top))
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        st = lib.wt_score_tokens(code, x.data_ptr(), w.data_ptr(), tokens.data_ptr(),
                                 suppress.data_ptr() if more else None, out.logprob.data_ptr(),
                                 out.entropy.data_ptr(), out.top_logprob.data_ptr() if top else None,
                                 out.top_token.data_ptr() if top else None, n, vocab, d, top, err.data_ptr(),
                                 scratch.data_ptr(), nbytes, _stream(dev))
    _lib.check(st, what)
    return out


# --- torch custom ops (for tracing) -------------------------------------------------------------------------
def _fake(tokens: torch.Tensor, top: int):
    lead = tokens.shape
    f32 = torch.float32
    return (tokens.new_empty(lead, dtype=f32), tokens.new_empty(lead, dtype=f32),
            tokens.new_empty((*lead, top), dtype=f32), tokens.new_empty((*lead, top)))


@torch.library.custom_op(f"{NAMESPACE}::token_logprobs", mutates_args=())
def token_logprobs_op(logits: torch.Tensor, tokens: torch.Tensor, top: int, suppress: Optional[torch.Tensor]
                      ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """:func:`token_logprobs`: logprob, entropy, top_logprob, top_token."""
    return tuple(token_logprobs(logits, tokens, top, suppress))


@token_logprobs_op.register_fake
def _(logits, tokens, top, suppress):
    return _fake(tokens, top)


@torch.library.custom_op(f"{NAMESPACE}::score_tokens", mutates_args=())
def score_tokens_op(x: torch.Tensor, w: torch.Tensor, tokens: torch.Tensor, top: int, suppress: Optional[torch.Tensor]
                    ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """:func:`score_tokens`, likewise."""
    return tuple(score_tokens(x, w, tokens, top, suppress))


@score_tokens_op.register_fake
def _(x, w, tokens, top, suppress):
    return _fake(tokens, top)
