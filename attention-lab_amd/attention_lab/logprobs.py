"""Log probabilities of given tokens, with the entropy and the most likely alternatives, on gfx950.

What a program does with a runner's logits: score a prompt token by token, compare a sparse read's distribution with the full
one's, follow the likeliest continuations. Each logit is read once, whatever is asked for. No counterpart in the reference's
package, whose scripts take log_softmax of the logits on the host.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native as nat

MAX_TOP = 64
MAX_VOCAB = (1 << 20) - 16
_DTYPES = {torch.bfloat16: nat.DT_BF16, torch.float16: nat.DT_F16, torch.float32: nat.DT_F32}


class TokenLogprobs(NamedTuple):
    logprobs: Optional[torch.Tensor]       # float32 [...], of the given tokens; None without tokens
    entropy: Optional[torch.Tensor]        # float32 [...], in nats; None if not asked for
    top_logprobs: torch.Tensor             # float32 [..., top], largest first
    top_tokens: torch.Tensor               # int64 [..., top]


def token_logprobs(logits, tokens=None, *, top: int = 0, entropy: bool = False) -> TokenLogprobs:
    """logits [..., V] (bfloat16, float16 or float32, V up to 2^20 - 16); tokens [...] (int64 or int32) -> TokenLogprobs.

    logprobs = logits[token] - log sum exp(logits); a token below 0 is padding and gives 0, one of V or more NaN. top (up to
    64): the most likely tokens, equal logits by the lower token (-0 equals +0, NaN last). A row with a NaN or +inf, or of
    nothing but -inf, has no distribution: its values are NaN. Sums are float32. Rows may have any stride; logits whose last
    dimension has another stride than 1 are copied. There is no gradient: logits that ask for one are refused."""
    code = _DTYPES.get(logits.dtype)
    if code is None or logits.dim() < 1 or not logits.is_cuda:
        raise ValueError("logits must be a bfloat16, float16 or float32 [..., V] tensor on a HIP device")
    *lead, V = logits.shape
    if not 1 <= V <= MAX_VOCAB:
        raise ValueError(f"V={V} must be in [1, {MAX_VOCAB}]")
    top = int(top)
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top={top} must be in [0, {min(MAX_TOP, V)}]")
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("token_logprobs has no gradient: give it logits that need none (detach them, or use torch.no_grad)")
    device = logits.device
    if tokens is not None:
        if tokens.dtype not in (torch.int64, torch.int32) or list(tokens.shape) != lead or tokens.device != device:
            raise ValueError(f"tokens must be an int64 or int32 {lead} tensor on the logits' device")
        tokens = tokens.contiguous()
    if logits.stride(-1) != 1 and V > 1:
        logits = logits.contiguous()
    rows = logits if len(lead) == 1 else logits.reshape(-1, V)
    N = rows.shape[0]
    stride = rows.stride(0) if N > 1 else V
    made = lambda *n, dtype=torch.float32: torch.empty((*lead, *n), dtype=dtype, device=device)  # noqa: E731
    found = made() if tokens is not None else None
    spread = made() if entropy else None
    best, at = made(top), made(top, dtype=torch.int64)
    if N == 0:
        return TokenLogprobs(found, spread, best, at)
    nbytes = nat.lib().attnlab_logprob_part_bytes(N, V, code, top)
    part = torch.empty(nbytes, dtype=torch.uint8, device=device)
    nat.call_on(device, "attnlab_token_logprobs", rows.data_ptr(), code, stride, N, V, nat.ptr(tokens),
                tokens is not None and tokens.dtype == torch.int64, top, nat.ptr(found), nat.ptr(spread), best.data_ptr(),
                at.data_ptr(), part.data_ptr(), nbytes, nat.stream_of(device))
    return TokenLogprobs(found, spread, best, at)
