"""Log probabilities of given tokens, with the entropy and the most likely alternatives, on gfx950.

What a program does with a runner's logits: score a prompt token by token, compare a sparse read's distribution with the full
one's, follow the likeliest continuations. Each logit is read once, whatever is asked for. Few rows take one launch, in which the
last workgroup of a row merges it, counted by counters of the stream's; a captured call takes two, and shares nothing. No
counterpart in the reference's package, whose scripts take log_softmax of the logits on the host.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch

from . import _native as nat
from .hip_range import capturing, stream_counters

MAX_TOP = 64
MAX_VOCAB = (1 << 20) - 16
# Up to as many rows are merged in the segments' launch: V = 151936, float32, top 20, merged and in two launches: 64 rows 16.4 and
# 16.9 us, 128 rows 23.3 and 22.5, 512 rows 61.7 and 53.7 (bfloat16, top 5: 64 rows 14.5 and 15.7, 256 rows 23.1 and 22.1).
MERGED_ROWS = 64
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
    dimension has another stride than 1 are copied. There is no gradient: logits that ask for one, or carry a tangent, are
    refused."""
    shape = logits.shape
    code = _DTYPES.get(logits.dtype)
    if code is None or not shape or not logits.is_cuda:
        raise ValueError("logits must be a bfloat16, float16 or float32 [..., V] tensor on a HIP device")
    lead, V, device = shape[:-1], shape[-1], logits.device
    if not 1 <= V <= MAX_VOCAB:
        raise ValueError(f"V={V} must be in [1, {MAX_VOCAB}]")
    top = int(top)
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top={top} must be in [0, {min(MAX_TOP, V)}]")
    nat.refuse_gradients("token_logprobs", logits)
    if tokens is not None:
        wide = tokens.dtype is torch.int64
        if not (wide or tokens.dtype is torch.int32) or tokens.shape != lead or tokens.device != device:
            raise ValueError(f"tokens must be an int64 or int32 {list(lead)} tensor on the logits' device")
        tokens = tokens.contiguous()
    *strides, last = logits.stride()
    if last != 1 and V > 1:
        logits = logits.contiguous()
        *strides, last = logits.stride()
    if len(lead) != 1:
        logits = logits.reshape(-1, V)
        strides = logits.stride()
    N = logits.shape[0]
    # an empty_like is half the time of an empty with its arguments, and the host's part is most of a small call's time
    like = torch.empty(lead, dtype=torch.float32, device=device)
    found = like if tokens is not None else None
    spread = None if not entropy else torch.empty_like(like) if found is like else like
    best = torch.empty((*lead, top), dtype=torch.float32, device=device)
    at = torch.empty_like(best, dtype=torch.int64)
    if N == 0:
        return TokenLogprobs(found, spread, best, at)
    nbytes = _part_bytes(N, V, code, top)
    part = torch.empty(nbytes, dtype=torch.uint8, device=device)
    stream = nat.stream_of(device)
    held, arrive = (None, None) if N > MERGED_ROWS or capturing(device) else stream_counters(device, stream)
    nat.call_on(device, "attnlab_token_logprobs", logits.data_ptr(), code, strides[0] if N > 1 else V, N, V,
                None if tokens is None else tokens.data_ptr(), tokens is not None and wide, top,
                None if found is None else found.data_ptr(), None if spread is None else spread.data_ptr(), best.data_ptr(),
                at.data_ptr(), part.data_ptr(), nbytes, arrive, stream)
    return TokenLogprobs(found, spread, best, at)


@functools.lru_cache(maxsize=256)
def _part_bytes(N: int, V: int, code: int, top: int) -> int:
    return nat.lib().attnlab_logprob_part_bytes(N, V, code, top)
