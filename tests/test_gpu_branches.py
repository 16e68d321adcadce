"""The paged cache, the shared read and the log probabilities together, as a beam search and a prompt's scoring use them."""
from __future__ import annotations

import copy

import pytest
import torch

from attention_lab import (PagedCache, page_append, page_compact, page_fork, page_reserve, page_truncate,
                           shared_prefix_attention, token_logprobs)

pytestmark = pytest.mark.gpu
V, G, H, D, LAYERS = 61, 2, 2, 128, 2


class Toy:
    """A language model without an MLP: a token's query, key and value come from tables, layer by layer, and the logits from the
    layers' attention outputs."""

    def __init__(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.q = torch.randn(LAYERS, V, G, H, D, generator=g).to(torch.bfloat16)
        self.k, self.v = (torch.randn(LAYERS, V, G, D, generator=g).to(torch.bfloat16) for _ in "kv")
        self.w = torch.randn(LAYERS, G * H * D, V, generator=g) * 0.15

    def to(self, gpu):
        new = copy.copy(self)
        new.q, new.k, new.v, new.w = (t.to(gpu) for t in (self.q, self.k, self.v, self.w))
        return new

    def logits(self, outs):
        """outs: [n, G, H, D] of each layer -> [n, V]."""
        return sum(o.flatten(1).to(self.w.dtype) @ w for o, w in zip(outs, self.w))

    def exact(self, tokens):
        """float64 log probabilities behind the last of `tokens`, and how far bf16 outputs may move one: with A = sum w |v|, an
        output is off by 2^-8 of itself and 2^-8 A and fp32 sums (2^-12 A), times |w|; a log probability by twice the most."""
        t = torch.tensor(tokens)
        total, off = torch.zeros(V, dtype=torch.float64), torch.zeros(V, dtype=torch.float64)
        for layer in range(LAYERS):
            q, k, v, w = (x[layer].double() for x in (self.q, self.k, self.v, self.w))
            p = torch.softmax(q[t[-1]] @ k[t].permute(1, 2, 0) / D ** 0.5, dim=-1)
            o, size = p @ v[t].transpose(0, 1), p @ v[t].transpose(0, 1).abs()
            total += o.flatten() @ w
            off += (2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -12) * size).flatten() @ w.abs()
        return torch.log_softmax(total, dim=0), 2 * off.max() + 1e-5


def test_beam_search(gpu):
    """Two prompts, four beams each: every beam's score is the sum of its tokens' float64 log probabilities along its own
    history, whatever pages it shares; the pool is compacted midway and gives the same reads."""
    host = Toy(1)
    m = host.to(gpu)
    prompts = [torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (37, 50)]
    beams, slots, page, T = 4, 8, 8, 50
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    cache = PagedCache.empty(LAYERS, slots, G, 80, page, 10, device=gpu)

    # the prompts, in slots 0 and 4: rows from the front, queries at the last positions
    tokens = ints([37, 0, 0, 0, 50, 0, 0, 0])
    front, back = (torch.zeros(slots, T, dtype=torch.int64, device=gpu) for _ in range(2))
    for i, p in enumerate(prompts):
        front[4 * i, :len(p)] = torch.tensor(p, device=gpu)
        back[4 * i, T - len(p):] = torch.tensor(p, device=gpu)
    page_reserve(cache, tokens)
    outs = []
    for layer in range(LAYERS):
        page_append(cache, layer, m.k[layer][front].transpose(1, 2), m.v[layer][front].transpose(1, 2), tokens)
        q = m.q[layer][back].permute(0, 2, 3, 1, 4)
        outs.append(shared_prefix_attention(q, cache.k[layer], cache.v[layer], cache.table, cache.lengths)[:, :, :, -1])
    first = token_logprobs(m.logits(outs)[::4], top=beams)
    scores = first.top_logprobs.clone()                          # [2, beams]
    last = first.top_tokens.reshape(-1)
    page_fork(cache, ints([0] * 4 + [4] * 4))
    held = [list(prompts[i // 4]) for i in range(slots)]
    runs, prefix = ints([0, 4, 8]), ints([37, 50])
    exact = [sum(host.exact(prompts[i // 4])[0][int(last[i])].tolist() for _ in [0]) for i in range(slots)]
    off = [host.exact(prompts[i // 4])[1] for i in range(slots)]

    for step in range(9):
        for i in range(slots):
            held[i] = held[i] + [int(last[i])]
        page_reserve(cache, 1)
        outs = []
        for layer in range(LAYERS):
            page_append(cache, layer, m.k[layer][last][:, :, None], m.v[layer][last][:, :, None])
            q = m.q[layer][last][:, :, :, None]
            args = q, cache.k[layer], cache.v[layer], cache.table, cache.lengths, prefix
            outs.append(shared_prefix_attention(*args, runs=runs)[:, :, :, 0])
            alone = shared_prefix_attention(*args, runs=runs, partitions=(0, 1))[:, :, :, 0]
            assert (outs[-1].float() - alone.float()).abs().max() <= 2.0 ** -5   # two ways to round weights and outputs of ~1
        assert cache.lengths.tolist() == [len(h) for h in held]
        r = token_logprobs(m.logits(outs), top=beams, entropy=True)
        both = (scores.view(slots, 1) + r.top_logprobs).view(2, -1)
        scores, pick = both.topk(beams, dim=1)
        parents = (pick // beams + beams * torch.arange(2, device=gpu)[:, None]).reshape(-1)
        last = r.top_tokens.reshape(2, -1).gather(1, pick).reshape(-1)
        new_exact, new_off = [], []
        for i, p in enumerate(parents.tolist()):
            lp, tol = host.exact(held[p])
            new_exact.append(exact[p] + float(lp[int(last[i])]))
            new_off.append(off[p] + tol)
            assert abs(float(r.entropy[p]) + float((lp.exp() * lp).sum())) <= 12 * tol
        exact, off, held = new_exact, new_off, [list(held[p]) for p in parents.tolist()]
        for got, want, tol in zip(scores.reshape(-1).tolist(), exact, off):
            assert abs(got - want) <= tol, (step, got, want, float(tol))
        page_fork(cache, parents.to(torch.int32))
        if step == 4:
            page_compact(cache)
            used = int((cache.refs > 0).sum())
            assert int(cache.table.max()) < used and int(cache.missing) == 0
    # the beams share their prompts to the end, and leave nothing behind
    assert cache.refs[cache.table[0, :4].long()].tolist() == [4] * 4
    page_truncate(cache)
    assert int(cache.refs.abs().sum()) == 0 and int((cache.table >= 0).sum()) == 0


def test_scores_of_a_prompt(gpu):
    """LabRunner.score: the log probabilities of a prefill's own logits, chunk by chunk, in every format and mode."""
    transformers = pytest.importorskip("transformers")  # noqa: F841
    from attention_lab.qwen_wrap import LabRunner, make_state, tiny_qwen3, wrap_model
    m = tiny_qwen3(seed=0, layers=2, hidden=256, heads=4, groups=2, head_dim=128, intermediate=256, vocab=256,
                   dtype=torch.bfloat16).to(gpu)
    ids = torch.randint(0, 256, (2, 75), generator=torch.Generator().manual_seed(3)).to(gpu)
    holder = wrap_model(m)
    with torch.inference_mode():
        for kw in (dict(mode="full"), dict(mode="full", kv_format="e4m3"), dict(mode="window", window=40, sinks=4)):
            for chunk in (75, 74, 32, 25):
                run = LabRunner(m, holder, make_state(m, 100, batch=2, **kw))
                r = run.score(ids, chunk, top=6, entropy=True)
                assert run.cache.valid_length == 75
                other = LabRunner(m, holder, make_state(m, 100, batch=2, **kw))
                y = torch.log_softmax(other.prefill(ids, chunk, keep_logits=True).double(), dim=-1)[:, :-1]
                want = y.gather(-1, ids[:, 1:, None]).squeeze(-1)
                assert r.logprobs.shape == (2, 74) and r.top_tokens.shape == (2, 74, 6)
                # fp32 sums over 256 logits of a few nats: 2^-18 and the result's rounding
                assert (r.logprobs.double() - want).abs().max() <= 2.0 ** -16
                assert (r.top_logprobs.double() - y.gather(-1, r.top_tokens)).abs().max() <= 2.0 ** -16
                assert (r.entropy.double() + (y.exp() * y).sum(-1)).abs().max() <= 2.0 ** -14
    with torch.no_grad():
        plain = LabRunner(m, holder, make_state(m, 100, "full"))
        for p in m.parameters():
            p.requires_grad_(True)
        r = plain.score(ids[:1], 40)
        assert r.logprobs.shape == (1, 74) and r.entropy is None and r.top_tokens.shape == (1, 74, 0)
        with pytest.raises(ValueError, match="two tokens"):
            plain.score(ids[:1, :1], 40)
