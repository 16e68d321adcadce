"""Operators for several answers to one prompt: the work whose speed is measured.

The kinds:

  branch    one decode step's bookkeeping and writes over a cache of shared pages: the sequences that go on are chosen
            (`page_fork`), room is made for their next tokens, which takes a page apart that two of them would write
            (`page_reserve`), and every layer's new rows are written (`page_append`). Without a fork: a prompt chunk.
  compact   the pages of a cache moved to the pool's low end, after sequences have ended (`page_compact`).
  shared    attention of sequences that share long prompts, a prompt's keys read once for all that share it
            (`shared_prefix_attention`): one query each, or a chunk each.
  logprob   log probabilities of given tokens, the entropy and the most likely alternatives (`token_logprobs`).

Shapes: 8 KV groups, head_dim 128, 1 to 8 query heads per KV group and the vocabulary of 151936, as in the Qwen3 shapes
of bench.py; contexts from some hundred positions to 32K. Synthetic data: K, V and queries ~ N(0, 1), logits ~ N(0, 2.5) with
a few likely tokens.

`own` False: every operator in elementary torch operations. True: the framework's calls.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
G, D = 8, 128
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # a small beam search: four beams of a short question
        dict(name="branch_beams4", kind="branch", prompts=1, branches=4, history=300, tokens=1, page=16, layers=2, pool=64,
             fork=True),
        # sampling: eight prompts of up to 2K with eight answers each, where some have ended and others go on twice
        dict(name="branch_8x8", kind="branch", prompts=8, branches=8, history=2048, tokens=1, page=64, layers=8, pool=512,
             fork=True),
        # a draft of odd length checked for many beams, long prompts in large pages
        dict(name="branch_4x31_draft", kind="branch", prompts=4, branches=31, history=12345, tokens=5, page=128, layers=4,
             pool=768, fork=True),
        # an odd prompt chunk of three requests, begun inside a page
        dict(name="append_chunk_odd", kind="branch", prompts=3, branches=1, history=517, tokens=1003, page=32, layers=4,
             pool=256, fork=False),
        # a pool after half of the sequences have ended
        dict(name="compact_half", kind="compact", pool=2048, sequences=48, live=0.5, page=64, layers=4),
        # a small pool of small pages that is nearly full
        dict(name="compact_small", kind="compact", pool=501, sequences=7, live=0.9, page=16, layers=2),
        # four answers to a short question: latency
        dict(name="shared_1x4_512", kind="shared", prompts=1, branches=4, heads=2, tokens=1, prefix=512, suffix=40, page=16),
        # sixteen answers to one 8K prompt
        dict(name="shared_1x16_8k", kind="shared", prompts=1, branches=16, heads=4, tokens=1, prefix=8192, suffix=300, page=64),
        # four prompts of odd lengths with unequal numbers of answers, many query heads to a KV head
        dict(name="shared_4x13_odd", kind="shared", prompts=4, branches=13, heads=8, tokens=1, prefix=9001, suffix=1021,
             page=32),
        # sixteen questions of 211 tokens about one 16K document
        dict(name="shared_questions", kind="shared", prompts=1, branches=16, heads=2, tokens=211, prefix=16384, suffix=211,
             page=64),
        # the next token of 64 sequences, out of a float32 head
        dict(name="logprob_step", kind="logprob", rows=64, vocab=151936, type="f32", top=20),
        # a prompt scored token by token
        dict(name="logprob_prompt", kind="logprob", rows=4096, vocab=151936, type="bf16", top=5),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["branch", "branch", "compact", "shared", "shared", "shared", "logprob", "logprob"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "branch":
        prompts, history = _log(rng, 1, 8), _log(rng, 20, 12000)
        fork = rng.random() < 0.7
        branches = _log(rng, 2, 32) if fork else 1
        tokens = _log(rng, 1, 6) if fork else _log(rng, 1, 1500)
        need = prompts * (history // page + 1) + 2 * prompts * branches * (tokens // page + 2)
        return dict(kind=kind, prompts=prompts, branches=branches, history=history, tokens=tokens, page=page,
                    layers=rng.choice([1, 2, 4]) if page * need > 65536 else rng.choice([1, 2, 4, 8]),
                    pool=need + _log(rng, 1, 200), fork=fork)
    if kind == "compact":
        return dict(kind=kind, pool=_log(rng, 100, 131072 // page), sequences=_log(rng, 1, 64),
                    live=round(rng.uniform(0.2, 0.95), 2), page=page, layers=rng.choice([1, 2, 4]))
    if kind == "shared":
        heads, prompts = rng.choice([1, 2, 3, 4, 6, 8]), _log(rng, 1, 6)
        if rng.random() < 0.65:    # one query of every sequence
            prefix = _log(rng, 200, 32768 // prompts)
            return dict(kind=kind, prompts=prompts, branches=_log(rng, 2, max(2, min(48, 700000 // (prompts * prefix)))), heads=heads,
                        tokens=1, prefix=prefix, suffix=_log(rng, 1, 1500), page=page)
        tokens, prefix = _log(rng, 2, 300), _log(rng, 200, 12000 // prompts)
        most = 2 * 16 * 211 * 16000 // (heads * tokens * prompts * (prefix + tokens))
        return dict(kind=kind, prompts=prompts, branches=_log(rng, 2, max(2, min(16, most))), heads=heads, tokens=tokens,
                    prefix=prefix, suffix=tokens + rng.choice([0, _log(rng, 1, 200)]), page=page)
    vocab = rng.choice([151936, _log(rng, 1000, 200000)])
    kind_of = rng.choice(["bf16", "bf16", "f16", "f32"])
    rows = _log(rng, 1, min(4096, (2 if kind_of == "f32" else 4) * 151936000 // vocab))
    return dict(kind=kind, rows=rows, vocab=vocab, type=kind_of, top=rng.choice([0, 1, 5, 8, 20, 32]))


# ---------------------------------------------------------------------------------------------------------------------
# inputs: made on the GPU from the seed alone
# ---------------------------------------------------------------------------------------------------------------------
def _randn(gen, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=dtype)


def _between(gen, lo, hi, n):
    """n whole numbers of [lo, hi]."""
    return torch.randint(lo, hi + 1, (n,), generator=gen, device=DEV)


def _book(s, table, lengths, refs):
    """A cache's table, lengths and reference counts as parts of one tensor, and how they stand before a step: a pass
    begins by putting them back."""
    parts = [t.to(torch.int32).reshape(-1) for t in (table, lengths, refs)]
    s["book"] = torch.cat(parts)
    s["before"] = s["book"].clone()
    a, b, c = s["book"].split([p.numel() for p in parts])
    s["table"], s["lengths"], s["refs"] = a.view(table.shape), b, c


def _shared_tables(gen, prefix, run_of, lengths, page, pool, width):
    """Tables [B, width] and reference counts of sequences whose whole pages below prefix[run] are their run's, in pages
    placed at random."""
    entry = torch.arange(width, device=DEV)
    common = (prefix // page)[run_of].unsqueeze(1)
    mine = (entry >= common) & (entry < ((lengths + page - 1) // page).unsqueeze(1))
    first = torch.cumsum(prefix // page, 0) - prefix // page
    place = torch.randperm(pool, generator=gen, device=DEV)
    own_at = (prefix // page).sum() + torch.cumsum(mine.reshape(-1), 0).view(mine.shape) - 1
    at = torch.where(mine, own_at, first[run_of].unsqueeze(1) + entry)
    used = mine | (entry < common)
    table = torch.where(used, place[at.clamp(0, pool - 1)], -1)
    refs = torch.zeros(pool + 1, dtype=torch.int64, device=DEV)
    refs.scatter_add_(0, torch.where(used, table, pool).reshape(-1), torch.ones_like(table).reshape(-1))
    return table, refs[:pool]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind = case["kind"]
    s = dict(kind=kind)
    if kind == "logprob":
        N, V = case["rows"], case["vocab"]
        x = _randn(gen, N, V, dtype=TYPES[case["type"]]).mul_(2.5)
        likely = torch.randint(0, V, (N, 4), generator=gen, device=DEV)
        x.scatter_add_(1, likely, 6.0 * torch.rand(N, 4, generator=gen, device=DEV).to(x.dtype))
        s["logits"], s["top"] = x, case["top"]
        s["tokens"] = torch.where(torch.rand(N, generator=gen, device=DEV) < 0.7, likely[:, 0],
                                  torch.randint(0, V, (N,), generator=gen, device=DEV))
        return s
    page = case["page"]
    s["page"] = page
    if kind == "compact":
        pool, S = case["pool"], case["sequences"]
        live = max(1, round(pool * case["live"]))
        each = torch.bincount(torch.randint(0, S, (live,), generator=gen, device=DEV), minlength=S)   # pages of a sequence
        width = live
        entry = torch.arange(width, device=DEV)
        used = entry < each.unsqueeze(1)
        place = torch.randperm(pool, generator=gen, device=DEV)
        at = (torch.cumsum(each, 0) - each).unsqueeze(1) + entry
        table = torch.where(used, place[at.clamp(max=pool - 1)], -1)
        refs = torch.zeros(pool, dtype=torch.int64, device=DEV)
        refs[place[:live]] = 1
        lengths = (each * page - torch.randint(0, page, (S,), generator=gen, device=DEV)).clamp(min=0)
        _book(s, table, lengths, refs)
        s["k"], s["v"] = (_randn(gen, case["layers"], pool, G, page, D) for _ in "kv")
        return s
    P, n = case["prompts"], case["branches"]
    B = P * n
    if kind == "branch":
        T = case["tokens"]
        run_of = torch.arange(B, device=DEV) // n
        prefix = _between(gen, max(1, case["history"] // 2), case["history"], P)
        lengths = prefix[run_of]
        table, refs = _shared_tables(gen, prefix, run_of, lengths, page, case["pool"], (case["history"] + T) // page + 2)
        _book(s, table, lengths, refs)
        s["k"], s["v"] = (_randn(gen, case["layers"], case["pool"], G, page, D) for _ in "kv")
        s["parents"] = torch.arange(B, device=DEV, dtype=torch.int32)
        if case["fork"]:    # within its prompt a sequence may go on several times, and one slot of eight or so ends
            pick = run_of * n + torch.randint(0, n, (B,), generator=gen, device=DEV)
            ends = (torch.rand(B, generator=gen, device=DEV) < 0.12) & (torch.arange(B, device=DEV) % n > 0)
            s["parents"] = torch.where(ends, -1, pick).to(torch.int32)
        s["tokens"] = torch.where(s["parents"] >= 0, T, 0).to(torch.int32)
        s["new_k"], s["new_v"] = (_randn(gen, case["layers"], B, T, G, D).transpose(2, 3) for _ in "kv")
        s["fork"] = case["fork"]
        return s
    T, h = case["tokens"], case["heads"]
    prefix = _between(gen, max(1, case["prefix"] * 3 // 4), case["prefix"], P) if P > 1 else \
        torch.full((1,), case["prefix"], device=DEV)
    cut = torch.sort(torch.randint(1, B, (P - 1,), generator=gen, device=DEV)).values if P > 1 else prefix[:0]
    runs = torch.cat([cut.new_zeros(1), cut, cut.new_full((1,), B)])
    run_of = torch.searchsorted(cut, torch.arange(B, device=DEV), right=True)
    lengths = prefix[run_of] + _between(gen, max(T, case["suffix"] // 4), case["suffix"], B)
    width = (case["prefix"] + case["suffix"]) // page + 1
    pool = P * (case["prefix"] // page) + B * (case["suffix"] // page + 2) + 7
    s["table"], _ = _shared_tables(gen, prefix, run_of, lengths, page, pool, width)
    s["table"], s["lengths"] = s["table"].to(torch.int32), lengths.to(torch.int32)
    s["runs"], s["prefix"] = runs.to(torch.int32), prefix.to(torch.int32)
    s["k"], s["v"] = (_randn(gen, pool, G, page, D) for _ in "kv")
    s["q"] = _randn(gen, B, G, h, T, D)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "logprob":
        return _plain_logprobs(s)
    if s["kind"] == "shared":
        return _plain_shared(s)
    s["book"].copy_(s["before"])
    if s["kind"] == "compact":
        _plain_compact(s)
    else:
        if s["fork"]:
            _plain_fork(s)
        _plain_reserve(s)
        _plain_append(s)
    return _held(s)


def _run_own(s):
    al = _package()
    if s["kind"] == "logprob":
        r = al.token_logprobs(s["logits"], s["tokens"], top=s["top"], entropy=True)
        return {"logprobs": r.logprobs, "entropy": r.entropy, "top_logprobs": r.top_logprobs, "top_tokens": r.top_tokens}
    if s["kind"] == "shared":
        return al.shared_prefix_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["prefix"], runs=s["runs"])
    s["book"].copy_(s["before"])
    cache = al.PagedCache(s["k"], s["v"], s["table"], s["lengths"], s["refs"])
    if s["kind"] == "compact":
        al.page_compact(cache)
    else:
        if s["fork"]:
            al.page_fork(cache, s["parents"])
        al.page_reserve(cache, s["tokens"])
        [al.page_append(cache, i, s["new_k"][i], s["new_v"][i], s["tokens"]) for i in range(s["k"].shape[0])]
    return _held(s)


def _held(s):
    return {"k": s["k"], "v": s["v"], "table": s["table"], "lengths": s["lengths"], "refs": s["refs"]}


def _package():
    if "attention_lab" not in sys.modules:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "attention-lab_amd"))
    import attention_lab
    return attention_lab


def _plain_count(s):
    """Reference counts: how many table entries name each page."""
    pool = s["refs"].numel()
    at = torch.where(s["table"] >= 0, s["table"], pool).reshape(-1).long()
    n = torch.zeros(pool + 1, dtype=torch.int32, device=DEV).scatter_add_(0, at, torch.ones_like(at, dtype=torch.int32))
    s["refs"].copy_(n[:pool])


def _plain_fork(s):
    """Slot i becomes a branch of what slot parents[i] held, or empty."""
    goes = s["parents"] >= 0
    at = s["parents"].clamp(min=0).long()
    s["table"].copy_(torch.where(goes.unsqueeze(1), s["table"][at], -1))
    s["lengths"].copy_(torch.where(goes, s["lengths"][at], 0))
    _plain_count(s)


def _plain_reserve(s):
    """Room for tokens[i] more positions: a shared last page that is not full is copied for all of its holders but the
    last (where all of them go on), and new pages are taken; pages in the order of slots and entries, lowest first."""
    page, table, refs, n = s["page"], s["table"], s["refs"], s["lengths"]
    end = n + s["tokens"]
    last, rows = n // page, n % page
    held = table.gather(1, last.long().unsqueeze(1)).squeeze(1).long()
    writes = (s["tokens"] > 0) & (rows > 0) & (held >= 0)
    same = (held.unsqueeze(1) == held) & writes.unsqueeze(1) & writes
    keeps = (same.sum(1) == refs[held.clamp(min=0)]) & ~same.triu(1).any(1)
    copies = writes & (refs[held.clamp(min=0)] > 1) & ~keeps
    entry = torch.arange(table.shape[1], device=DEV)
    want = (entry >= ((n + page - 1) // page).unsqueeze(1)) & (entry < ((end + page - 1) // page).unsqueeze(1))
    want = want | ((entry == last.unsqueeze(1)) & copies.unsqueeze(1))
    rank = torch.cumsum(want.reshape(-1), 0).view(want.shape) - 1
    free = torch.argsort((refs > 0).to(torch.uint8), stable=True)
    fresh = torch.where(rank < (refs == 0).sum(), free[rank.clamp(0, refs.numel() - 1)], -1)
    table.copy_(torch.where(want, fresh, table))
    s["lengths"].copy_(end)
    _plain_count(s)
    which = copies.nonzero().squeeze(1)
    src, dst = held[which], table[which, last[which].long()].long()
    valid = (torch.arange(page, device=DEV) < rows[which].unsqueeze(1)).view(1, -1, 1, page, 1)
    s["k"][:, dst] = torch.where(valid, s["k"][:, src], s["k"][:, dst])
    s["v"][:, dst] = torch.where(valid, s["v"][:, src], s["v"][:, dst])


def _plain_append(s):
    """Every layer's new rows at the last tokens[i] positions of slot i."""
    page, T = s["page"], s["new_k"].shape[3]
    t = torch.arange(T, device=DEV)
    slot, t = (t < s["tokens"].unsqueeze(1)).nonzero(as_tuple=True)
    pos = (s["lengths"] - s["tokens"])[slot] + t
    at, row = s["table"][slot, (pos // page).long()].long(), (pos % page).long()
    s["k"].transpose(2, 3)[:, at, row] = s["new_k"].transpose(2, 3)[:, slot, t]
    s["v"].transpose(2, 3)[:, at, row] = s["new_v"].transpose(2, 3)[:, slot, t]


def _plain_compact(s):
    """The i-th page in use past the first n (n in use) moves to the i-th free page among them."""
    table, refs = s["table"], s["refs"]
    used = refs > 0
    n = int(used.sum())
    src, dst = used[n:].nonzero().squeeze(1) + n, (~used[:n]).nonzero().squeeze(1)
    s["k"][:, dst], s["v"][:, dst] = s["k"][:, src], s["v"][:, src]
    to = torch.arange(refs.numel(), device=DEV, dtype=torch.int32)
    to[src] = dst.to(torch.int32)
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    refs[dst] = refs[src]
    refs[src] = 0


def _plain_shared(s):
    """Softmax attention of every sequence over its own pages, in 32 bits."""
    q, page = s["q"], s["page"]
    B, _, h, T, _ = q.shape
    C = s["table"].shape[1] * page
    at = s["table"].clamp(min=0).long()
    p = (s["lengths"].view(B, 1) - T + torch.arange(T, device=DEV)).view(B, 1, 1, T, 1)
    seen = torch.arange(C, device=DEV) <= p
    x = q.float().view(B, G, h * T, D) @ s["k"][at].permute(0, 2, 4, 1, 3).float().reshape(B, G, D, C)
    x = torch.where(seen, x.view(B, G, h, T, C) * D ** -0.5, float("-inf"))
    x = torch.exp(x - x.amax(dim=-1, keepdim=True))
    out = x.view(B, G, h * T, C) @ s["v"][at].transpose(1, 2).float().reshape(B, G, C, D)
    return (out.view(B, G, h, T, D) / x.sum(dim=-1, keepdim=True)).to(q.dtype)


def _plain_logprobs(s):
    x = s["logits"].float()
    V = x.shape[1]
    top = x.amax(dim=1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(dim=1, keepdim=True)
    lse = top + torch.log(total)
    entropy = torch.log(total) - (e * (x - top)).sum(dim=1, keepdim=True) / total
    # the largest logits, ties to the lowest token: keys of the value's order and the token counted from the last
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() * (1 << 32) + (V - 1 - torch.arange(V, device=DEV))
    best = order.topk(s["top"], dim=1).indices
    return {"logprobs": (x.gather(1, s["tokens"].unsqueeze(1)) - lse).squeeze(1), "entropy": entropy.squeeze(1),
            "top_logprobs": x.gather(1, best) - lse, "top_tokens": best}


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "logprob":
        N, V = case["rows"], case["vocab"]
        return dict(bytes=N * V * TYPES[case["type"]].itemsize + N * (16 + 12 * case["top"]), flops=5 * N * V)
    page = case["page"]
    row = 2 * G * D * 2             # bytes of a position's K and V
    if kind == "compact":
        pool, f = case["pool"], case["live"]
        live = max(1, round(pool * f))
        return dict(bytes=2 * pool * f * (1 - f) * page * row * case["layers"] + 8 * pool + 8 * live, flops=0)
    P, n = case["prompts"], case["branches"]
    B = P * n
    if kind == "branch":
        T = case["tokens"]
        copies, going = 0.0, B
        if case["fork"]:            # those that go on, but one for every sequence that any of them goes on from
            going = P * (1 + (n - 1) * 0.88)
            copies = going - B * (1 - (1 - going / B / n) ** n)
        entries = B * (case["history"] * 3 // 4) // page
        return dict(bytes=case["layers"] * row * 2 * (copies * page / 2 + going * T) + 8 * entries + 4 * case["pool"], flops=0)
    T, h = case["tokens"], case["heads"]
    prefix = case["prefix"] if P == 1 else case["prefix"] * 7 // 8
    suffix = (max(T, case["suffix"] // 4) + case["suffix"]) / 2
    pairs = B * T * (prefix + suffix - (T - 1) / 2)
    return dict(bytes=(P * prefix + B * suffix) * row + B * G * h * T * D * 4, flops=G * h * pairs * 4 * D)


# ---------------------------------------------------------------------------------------------------------------------
# the same from the definition: step by step, in 64 bits where values are computed
# ---------------------------------------------------------------------------------------------------------------------
def _exact_pages(s):
    page, pool = s["page"], s["refs"].numel()
    table, lengths = s["table"].tolist(), s["lengths"].tolist()
    holders = {}

    def hold(p, by):
        if p >= 0:
            holders[p] = holders.get(p, 0) + by
            if holders[p] == 0:
                del holders[p]

    for row in table:
        for p in row:
            hold(p, 1)

    def take():
        p = next((p for p in range(pool) if p not in holders), -1)
        hold(p, 1)
        return p

    if s["kind"] == "compact":
        n, hole = len(holders), 0
        for p in sorted(x for x in holders if x >= n):
            while hole in holders:
                hole += 1
            for x in "kv":
                s[x][:, hole] = s[x][:, p]
            table = [[hole if e == p else e for e in row] for row in table]
            holders[hole] = holders.pop(p)
    else:
        if s["fork"]:
            parents = s["parents"].tolist()
            table = [list(table[p]) if p >= 0 else [-1] * len(table[0]) for p in parents]
            lengths = [lengths[p] if p >= 0 else 0 for p in parents]
            holders.clear()
            for row in table:
                for p in row:
                    hold(p, 1)
        tokens = s["tokens"].tolist()
        # who keeps a shared page: the last slot of those that write it, where nobody else holds it
        writers = {}
        for i, t in enumerate(tokens):
            if t > 0 and lengths[i] % page:
                writers.setdefault(table[i][lengths[i] // page], []).append(i)
        leaves = [i for p, w in writers.items() for i in (w if holders[p] > len(w) else w[:-1])]
        let_go = []
        for i, t in enumerate(tokens):
            n = lengths[i]
            if i in leaves:
                old, e = table[i][n // page], n // page
                table[i][e] = take()
                let_go.append(old)
                for x in "kv":
                    s[x][:, table[i][e], :, :n % page] = s[x][:, old, :, :n % page]
            for e in range(-(-n // page), -(-(n + t) // page)):
                table[i][e] = take()
            lengths[i] = n + t
        for p in let_go:
            hold(p, -1)
        for i, t in enumerate(tokens):
            for u in range(t):
                pos = lengths[i] - t + u
                for x in "kv":
                    s[x][:, table[i][pos // page], :, pos % page] = s["new_" + x][:, i, :, u]
    refs = [holders.get(p, 0) for p in range(pool)]
    as_ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    return {"k": s["k"], "v": s["v"], "table": as_ints(table), "lengths": as_ints(lengths), "refs": as_ints(refs)}


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] in ("branch", "compact"):
        return _exact_pages(s)
    if s["kind"] == "logprob":
        out = {name: [] for name in ("logprobs", "entropy", "top_logprobs", "top_tokens")}
        for a in range(0, s["logits"].shape[0], 256):
            x = s["logits"][a:a + 256].double()
            y = torch.log_softmax(x, dim=1)
            out["logprobs"].append(y.gather(1, s["tokens"][a:a + 256].unsqueeze(1)).squeeze(1))
            out["entropy"].append(-(y.exp() * y).sum(dim=1))
            best = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :s["top"]]
            out["top_logprobs"].append(y.gather(1, best))
            out["top_tokens"].append(best)
        return {name: torch.cat(v) for name, v in out.items()}
    q, page = s["q"], s["page"]
    B, _, h, T, _ = q.shape
    out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
    for b, L in enumerate(s["lengths"].tolist()):
        pos = torch.arange(L, device=DEV)
        at, row = s["table"][b].long()[pos // page], pos % page
        gone = pos > torch.arange(L - T, L, device=DEV).unsqueeze(1)
        for g in range(G):
            x = q[b, g].double() @ s["k"][at, g, row].double().t().contiguous() / math.sqrt(D)
            out[b, g] = torch.softmax(x.masked_fill(gone, float("-inf")), dim=-1) @ s["v"][at, g, row].double()
    return out
