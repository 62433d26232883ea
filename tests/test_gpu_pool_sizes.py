"""Compactions and frees of pools around 2^18 pages, where the one-launch form's LDS passes 64 KB."""
import numpy as np
import pytest
import torch

import test_gpu_pages
from oracle import turn
from turn_cases import i32

pytestmark = pytest.mark.gpu
check = test_gpu_pages.test_large_pools


@pytest.mark.parametrize("pages", [261887, 261888, 261889, 262144, 262145, 524287])
def test_pools_around_64_kilobytes_of_lds(ext, gpu, pages):
    check(ext, gpu, pages)


@pytest.mark.parametrize("pages", [1000, 262144, 600000])
def test_captured_compactions(ext, gpu, pages):
    """In one launch, in one with more than 64 KB of LDS, and pass by pass: replays follow their inputs."""
    rng = np.random.default_rng(pages)
    ins = [i32(np.zeros(n), gpu) for n in (pages, pages, 1)]
    table = i32(np.zeros((3, 50)), gpu)
    outs = [i32(np.zeros(n), gpu) for n in (pages, pages, pages, 1, pages // 2, pages // 2)]
    table_out, space = torch.zeros_like(table), torch.empty(ext.page_workspace_ints(pages), dtype=torch.int32, device=gpu)

    def step():
        ext.compact_pages(table, *ins, outs[0], table_out, outs[1], outs[2], outs[3], outs[4], outs[5], space)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for used in (pages // 2, pages, 0, pages // 3):
        order = rng.permutation(pages)
        shares = np.zeros(pages, dtype=np.int64)
        shares[order[:used]] = rng.integers(0, 4, used)
        free = np.concatenate([order[used:], order[:used]])
        ids = rng.integers(-2, pages + 2, (3, 50))
        for x, y in zip((table, *ins, outs[2]), (ids, shares, free, [pages - used], free)):
            x.copy_(i32(y, gpu))
        graph.replay()
        torch.cuda.synchronize()
        want = turn.compact_pages(ids, shares, free, pages - used, pages // 2)
        for got, w in zip((outs[0], table_out, *outs[1:]), want):
            test_gpu_pages._equal(got, w)
