"""Token log probabilities without a GPU: what the C entry and its Python caller refuse before any launch."""
from __future__ import annotations

import pytest
import torch

import attention_lab
from attention_lab import _native, token_logprobs

ARGS = dict(logits=16, dtype=0, stride=1000, N=3, V=1000, tokens=16, tokens64=1, top=5, logprobs=16, entropy=None, top_logprobs=16,
            top_tokens=16, part=16, part_bytes=1 << 20, arrive=None, stream=None)


@pytest.mark.parametrize("change,match", [
    (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(V=0), "V=0"), (dict(V=1 << 20), "V="), (dict(N=-1), "negative"),
    (dict(top=65), "top"), (dict(top=-1), "top"), (dict(V=4), "top"), (dict(tokens=None), "together"), (dict(logprobs=None), "together"),
    (dict(top_tokens=None), "top_tokens"), (dict(logits=None), "logits"), (dict(logits=17), "aligned"),
    (dict(dtype=2, logits=18), "aligned"), (dict(part=None), "part"), (dict(part=8), "part"), (dict(part_bytes=64), "part"),
    (dict(N=1 << 40), "too many"),
])
def test_refused_before_any_launch(native_lib, change, match):
    assert len(ARGS) == len(_native.SIGNATURES["attnlab_token_logprobs"][1])
    with pytest.raises(ValueError, match=match):
        _native.call("attnlab_token_logprobs", *dict(ARGS, **change).values())


def test_nothing_to_do_is_no_launch(native_lib):
    _native.call("attnlab_token_logprobs", *dict(ARGS, N=0, logits=None, part=None).values())


def test_part_bytes(native_lib):
    size = native_lib.attnlab_logprob_part_bytes
    assert size(1, 1000, 0, 5) == 16 + 40                    # one segment
    assert size(0, 1000, 0, 5) == 0
    assert size(4096, 151936, 0, 5) == 4096 * 10 * (16 + 40)  # 16384 logits a segment
    assert size(1, (1 << 20) - 16, 2, 64) == 64 * (16 + 512)
    for bad in ((-1, 10, 0, 0), (1, 0, 0, 0), (1, 1 << 20, 0, 0), (1, 10, 5, 0), (1, 10, 0, 65)):
        assert size(*bad) == -1


class OnDevice(torch.Tensor):
    """A CPU tensor that says it is on a HIP device: for the checks, which look no further."""
    is_cuda = True


def test_python_refuses():
    x = torch.zeros(3, 10).as_subclass(OnDevice)
    for call, match in (
        (lambda: token_logprobs(torch.zeros(3, 10)), "HIP device"), (lambda: token_logprobs(x.double()), "float32"),
        (lambda: token_logprobs(x[0, 0]), "V"), (lambda: token_logprobs(x[:, :0]), "V=0"),
        (lambda: token_logprobs(x, top=11), "top"), (lambda: token_logprobs(x, top=-1), "top"),
        (lambda: token_logprobs(x, torch.zeros(3)), "tokens"), (lambda: token_logprobs(x, torch.zeros(2, dtype=torch.int64)), "tokens"),
        (lambda: token_logprobs(x, torch.zeros(3, 1, dtype=torch.int64)), "tokens"),
        (lambda: token_logprobs(torch.zeros(3, 10, requires_grad=True).as_subclass(OnDevice)), "gradient"),
    ):
        with pytest.raises(ValueError, match=match):
            call()
    assert "token_logprobs" in attention_lab.__all__ and "TokenLogprobs" in attention_lab.__all__
