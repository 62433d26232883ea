"""Seeded inputs and checks shared by the tests of the operators for a further turn over cached rows."""
from __future__ import annotations

import numpy as np
import torch

from oracle import turn
from prompt_cases import F32, U, assert_within, attention_tolerance

LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half a step of the subnormals


def angles(positions, rot, base=10000.0):
    """cos_sin [positions, rot] as a model keeps it: computed in 64 bits, stored in 32."""
    rate = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(positions, dtype=torch.float64)[:, None] * rate
    return torch.cat([a.cos(), a.sin()], 1).float()


def rope_tolerance(want, size, dtype):
    """Half a step of the type, and 32-bit arithmetic on the terms that make an element up.  The sum
    of squares (16 roundings of positive terms at most) is half as far off under the root, the
    root's reciprocal is good to 2^-23; with the two products of the norm and the two of the rotation
    that is less than 16 roundings of 2^-24, taken as 32."""
    return U[dtype] * np.abs(want) + LEAST[dtype] + (1 + U[dtype]) * 32 * F32 * size


def i32(x, device="cpu"):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device=device)


class Cache:
    """Rows of `lens` tokens in random pages of pools a quarter larger, every slot that holds no
    token filled with `stale`; the newest `new` tokens of each are the call's."""

    def __init__(self, lens, new, hq, hkv, page, dtype, seed, spare_columns=2, lead=0, trail=0, stale=float("nan")):
        gen = torch.Generator().manual_seed(seed)
        self.lens, self.new, self.hq, self.hkv, self.page, self.dtype = list(lens), list(new), hq, hkv, page, dtype
        counts = [-(-n // page) for n in lens]
        self.pages = max(int(1.25 * sum(counts)) + 1, 2)
        order = torch.randperm(self.pages, generator=gen).tolist()
        columns = max(counts + [1]) + spare_columns
        self.table = np.full((len(lens), columns), -1, dtype=np.int64)
        self.k = torch.full((self.pages, hkv, page, 128), stale).to(dtype)
        self.v = self.k.clone()
        for b, (n, c) in enumerate(zip(lens, counts)):
            self.table[b, :c] = [order.pop() for _ in range(c)]
            pos = torch.arange(n)
            ids = torch.as_tensor(self.table[b])[pos // page]
            for pool in (self.k, self.v):
                pool[ids, :, pos % page] = torch.randn(n, hkv, 128, generator=gen).to(dtype)
        tokens = lead + sum(new) + trail
        self.q = torch.randn(tokens, hq, 128, generator=gen).to(dtype)
        self.offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int64) + lead

    def place(self, row, position):
        """(page, offset) of a token."""
        return int(self.table[row, position // self.page]), position % self.page

    def on(self, device):
        return (self.q.to(device), self.k.to(device), self.v.to(device), i32(self.table, device), i32(self.lens, device),
                i32(self.offsets, device))

    def want(self):
        clean = lambda pool: np.nan_to_num(pool.double().numpy(), nan=0.0, posinf=0.0, neginf=0.0)
        return turn.paged_prefill(self.q.double().numpy(), clean(self.k), clean(self.v), self.table, self.lens, self.offsets)

    def bound(self, want, weight, vmax, score):
        longest = max(list(self.lens) + [1])
        tiny = longest * 2.0 ** -25 * vmax if self.dtype == torch.float16 else 0.0
        return attention_tolerance(np.nan_to_num(want), weight, score, longest, self.dtype, U[self.dtype], tiny)


def run_chunk(ext, cache, device, fill=7.0, workspace=None):
    q, k, v, table, lens, offsets = cache.on(device)
    out = torch.full(q.shape, fill, dtype=cache.dtype, device=device)
    if workspace is None:
        floats = ext.paged_prefill_workspace_floats(len(cache.lens), q.shape[0], cache.hq, cache.hkv)
        workspace = torch.full((floats,), float("nan"), device=device)
    ext.paged_prefill_attention(q, k, v, table, lens, offsets, out, workspace, cache.page)
    return out


def check_chunk(ext, cache, device, what=""):
    out = run_chunk(ext, cache, device)
    want, *rest = cache.want()
    inside = np.zeros(len(want), dtype=bool)
    for s, e in zip(cache.offsets, cache.offsets[1:]):
        inside[s:e] = True
    assert (out[~torch.from_numpy(inside)].float() == 7.0).all()  # left as they were
    bound = cache.bound(want, *rest)
    assert_within(out.cpu()[torch.from_numpy(inside)], want[inside], bound[inside], what)
    return out
