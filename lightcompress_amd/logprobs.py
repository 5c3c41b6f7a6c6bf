"""Log probabilities of given tokens, with entropy and best alternatives, from a model's logits in one pass: what the
reference's perplexity (llmc/eval/eval_ppl.py) and token-consistency evaluations
take from a whole log-softmax and an argmax.  Forward only: nothing here records a gradient."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib as L
from .w8a8 import _code, _here

MOST_TOP = 64


class TokenLogprobs(NamedTuple):
    logprobs: Optional[torch.Tensor]          # fp32, like tokens
    entropy: torch.Tensor                     # fp32 [...], in nats
    top_logprobs: torch.Tensor                # fp32 [..., top], largest first
    top_tokens: torch.Tensor                  # int64 [..., top]


def _sequences(x):
    """Logits [..., V] as B sequences of S rows -> (x or a contiguous copy, B, S, distance between sequences, between rows).
    Dimensions that one stride covers are one; a copy is made only where more than two are left, or a row is not in one piece."""
    V = x.shape[-1]
    if x.is_contiguous():
        return x, 1, x.numel() // V, 0, V
    dims = []
    for n, stride in zip(x.shape[:-1], x.stride()[:-1]):
        if n == 1:
            continue
        if dims and dims[-1][1] == n * stride:
            n *= dims.pop()[0]
        dims.append((n, stride))
    if len(dims) > 2 or (x.stride(-1) != 1 and V > 1):
        return _sequences(x.contiguous())
    (B, lds), (S, ldx) = [(1, 0)] * (2 - len(dims)) + dims
    return x, B, S, lds, ldx


def token_logprobs(logits, tokens=None, top=0, ignore_index=-100):
    """logits [..., V] (fp32, bf16, fp16); tokens int64 [...] or [..., m], the ids whose log probability is asked for.

    A token equal to `ignore_index` gives 0, any other id outside the vocabulary NaN.  Masked logits (-inf) have
    probability 0 and log probability -inf; a row that is masked everywhere, or holds a NaN or +inf, gives NaN, as
    log_softmax does.  The `top` (at most 64) alternatives come largest first, equal logits by the lowest id, a NaN first."""
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError(f'logits need a vocabulary, got shape {tuple(logits.shape)}')
    shape = logits.shape
    V, lead = shape[-1], (shape[0],) if len(shape) == 2 else tuple(shape[:-1])
    code = _code(logits.dtype)
    if not 0 <= top <= min(MOST_TOP, V):
        raise ValueError(f'top {top}: between 0 and {min(MOST_TOP, V)}')
    m = 0
    if tokens is not None:
        if tokens.dtype != torch.int64:
            raise L.LcqError(f'tokens are int64, got {tokens.dtype}')
        if tokens.shape == lead:
            m = 1
        elif tokens.dim() == logits.dim() and tokens.shape[:-1] == lead:
            m = tokens.shape[-1]
        else:
            raise ValueError(f'tokens {tuple(tokens.shape)} next to logits {tuple(logits.shape)}')
    if not _here(logits, tokens):
        with torch.cuda.device(logits.device):
            return token_logprobs(logits, tokens, top, ignore_index)
    ids = None if tokens is None else tokens.contiguous()
    logprobs = None if ids is None else torch.empty_like(ids, dtype=torch.float32)
    entropy = logits.new_empty(lead, dtype=torch.float32)
    top_logprobs = logits.new_empty((*lead, top), dtype=torch.float32)
    top_tokens = logits.new_empty((*lead, top), dtype=torch.int64)
    if logits.numel():
        x, B, S, lds, ldx = _sequences(logits)
        L.check(L.lib().lcq_token_logprobs_of(x.data_ptr(), code, B, S, V, lds, ldx, ids.data_ptr() if m else None, m, ignore_index,
                                              logprobs.data_ptr() if m else None, entropy.data_ptr(), top,
                                              top_logprobs.data_ptr() if top else None, top_tokens.data_ptr() if top else None,
                                              L.stream()), 'lcq_token_logprobs_of')
    return TokenLogprobs(logprobs, entropy, top_logprobs, top_tokens)
