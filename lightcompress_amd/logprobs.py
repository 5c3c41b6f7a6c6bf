"""Log probabilities of given tokens, with entropy and best alternatives, from a model's logits in one pass: what the
reference's perplexity (llmc/eval/eval_ppl.py) and token-consistency evaluations
take from a whole log-softmax and an argmax.  Forward only: nothing here records a gradient."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib as L
from .w8a8 import _code, _here, _rows

MOST_TOP = 64


class TokenLogprobs(NamedTuple):
    logprobs: Optional[torch.Tensor]          # fp32, like tokens
    entropy: torch.Tensor                     # fp32 [...], in nats
    top_logprobs: torch.Tensor                # fp32 [..., top], largest first
    top_tokens: torch.Tensor                  # int64 [..., top]


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

    def run(x, at):
        """The logits x, whose rows are the rows from `at` on of all of them."""
        if apart and x.dim() > 2:                   # logits[:, :-1]: a call per sequence, and no copy
            rows = x[0].numel() // V
            for i in range(x.shape[0]):
                run(x[i], at + i * rows)
            return
        rows, T, ld = _rows(x, V)
        if T:
            L.check(L.lib().lcq_token_logprobs(rows.data_ptr(), code, T, V, ld, ids.data_ptr() + 8 * m * at if m else None, m, ignore_index,
                                               logprobs.data_ptr() + 4 * m * at if m else None, entropy.data_ptr() + 4 * at, top,
                                               top_logprobs.data_ptr() + 4 * top * at if top else None,
                                               top_tokens.data_ptr() + 8 * top * at if top else None, L.stream()), 'lcq_token_logprobs')

    if logits.numel():
        apart = logits.dim() > 2 and logits.stride(-1) == 1 and not logits.is_contiguous()
        if apart:                                   # many short sequences (a transposed batch): one copy is faster than their calls
            each = V * lead[-1]
            apart = logits.numel() // each <= 64 or each * logits.element_size() >= 1 << 25
        run(logits, 0)
    return TokenLogprobs(logprobs, entropy, top_logprobs, top_tokens)
