"""Writes and rollbacks of an 8-bit LabCache against a cache that only ever saw the rows that are left: shared by the host
test (the launches replaced by the oracle) and the GPU one."""
from __future__ import annotations

import random

import numpy as np
import torch

from oracle import quant as oq

L, B, G, D = 2, 2, 2, 128


def rows(seed, length, loud):
    """[L, B, G, length, D] rows of which the share `loud` is up to 2^14 louder than the others, and a few not finite."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(L, B, G, length, D, generator=g)
    x *= torch.exp2(torch.where(torch.rand(L, B, G, length, 1, generator=g) < loud,
                                14 * torch.rand(L, B, G, length, 1, generator=g), torch.zeros(1)))
    x[..., 0, :, :][torch.rand(L, B, length, D, generator=g) < 1e-4] = float("inf")
    return x.to(torch.bfloat16)


class Expected:
    """The oracle's codes and scale bytes of a list of writes."""

    def __init__(self, slots, block):
        self.slots, self.block, self.writes = slots, block, []

    def write(self, start, k, v):
        self.writes.append((start, k, v))

    def rollback(self, length):
        self.writes = [(s, k[:, :, :, :length - s], v[:, :, :, :length - s]) for s, k, v in self.writes if s < length]

    def state(self):
        nb = -(-self.slots // self.block)
        out = {n: np.zeros((L * B, G, self.slots, D), np.uint8) for n in "kv"}
        out |= {n + "_exp": np.full((L * B, G, nb), oq.MIN_EXP, np.uint8) for n in "kv"}
        for start, *kv in self.writes:
            for n, x in zip("kv", kv):
                oq.append(out[n], out[n + "_exp"], x.reshape(L * B, G, -1, D).double().numpy(), start, self.block)
        return out

    def check(self, cache, what):
        n, want = cache.valid_length, self.state()
        blocks = -(-n // self.block)
        for x in "kv":
            codes = cache._store[x].view(torch.uint8).cpu().numpy().reshape(L * B, G, -1, D)[:, :, :n]
            exps = cache._store[x + "_exp"].cpu().numpy().reshape(L * B, G, -1)[:, :, :blocks]
            np.testing.assert_array_equal(exps, want[x + "_exp"][:, :, :blocks], err_msg=f"{what}: scales of {x}")
            nan = (want[x][:, :, :n] & 127) == 127          # a NaN's sign is not defined
            assert ((codes[nan] & 127) == 127).all(), what
            np.testing.assert_array_equal(np.where(nan, 0, codes), np.where(nan, 0, want[x][:, :, :n]),
                                          err_msg=f"{what}: codes of {x}")


def append(cache, expected, x, y):
    start, T = cache.valid_length, x.shape[3]
    for l in range(L):
        cache.append(l, x[l].to(cache.device), y[l].to(cache.device))
    cache.advance(T)
    expected.write(start, x, y)


def walk(cache, seed, steps, loud=0.1):
    """Random writes and rollbacks; after each, the codes and scale bytes of every legal row are those of a cache that saw
    only the writes that are left. Returns how many rollbacks were taken and how many refused."""
    rng, expected, taken, refused = random.Random(seed), Expected(cache.slots, cache.kv_block), 0, 0
    pinned, near = (0, 0), 0      # near: three blocks before the furthest position written
    for n in range(steps):
        room, valid = cache.capacity - cache.valid_length, cache.valid_length
        if room and (rng.random() < 0.6 or not valid):
            T = min(room, rng.choice([1, 1, 1, 1, 2, 5, rng.randint(1, 40), rng.randint(1, 150)]))
            append(cache, expected, rows(1000 * seed + 2 * n, T, loud), rows(1000 * seed + 2 * n + 1, T, loud))
            near = max(near, valid + T - 3 * cache.kv_block)
            if T > 1:
                pinned = ((valid + T) // cache.kv_block * cache.kv_block, valid + T)
        else:
            to = rng.choice([valid - min(valid, rng.randint(1, 12)), rng.randint(0, valid), pinned[1] if pinned[1] <= valid
                             else valid, valid // cache.kv_block * cache.kv_block])
            before = cache._store["k"].view(torch.uint8).clone(), cache._store["v_exp"].clone()
            try:
                cache.rollback(to)
                taken += 1
                expected.rollback(to)
                pinned = (pinned[0], min(pinned[1], to)) if pinned[0] < to else (0, 0)
                near = min(near, to)
            except ValueError:
                refused += 1
                # only where the documentation says so: no multiple, not near the end, not in the pinned block
                assert to % cache.kv_block and to < near and not pinned[0] < to <= pinned[1], (to, valid)
                assert cache.valid_length == valid
                assert torch.equal(before[0], cache._store["k"].view(torch.uint8))
                assert torch.equal(before[1], cache._store["v_exp"])
        if n % 4 == 3 or n == steps - 1:
            expected.check(cache, f"step {n}")
    return taken, refused
