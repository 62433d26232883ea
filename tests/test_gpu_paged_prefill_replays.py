"""paged_prefill_attention of more than 64 rows, whose plan is a launch of its own: captured calls whose
lengths change between replays, and calls on two streams."""
import pytest
import torch

from turn_cases import Cache, check_chunk

pytestmark = pytest.mark.gpu


def _caches(dtype):
    rows = 80
    shapes = [([40 + 17 * i for i in range(rows)], [1] * rows), ([9] * 40 + [900] * 40, [9, 1] * 20 + [1, 90] * 20),
              ([0, 3000] + [5] * 78, [0, 700] + [0] * 78)]
    tokens = max(sum(n) for _, n in shapes)
    return [Cache(lens, new, 8, 2, 16, dtype, seed=i, trail=tokens - sum(new)) for i, (lens, new) in enumerate(shapes)], rows, tokens


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_plans_of_their_own(ext, gpu, dtype):
    caches, rows, tokens = _caches(dtype)
    refs = [check_chunk(ext, c, gpu) for c in caches]  # tokens behind every row are 7
    columns, pages = max(c.table.shape[1] for c in caches), max(c.pages for c in caches)
    ins = []
    for c in caches:
        q, k, v, table, lens, offsets = c.on(gpu)
        wide = torch.full((rows, columns), -1, dtype=torch.int32, device=gpu)
        wide[:, :table.shape[1]] = table
        pools = [torch.zeros(pages, 2, 16, 128, dtype=dtype, device=gpu) for _ in range(2)]
        for pool, x in zip(pools, (k, v)):
            pool[:c.pages] = x
        ins.append([q, *pools, wide, lens, offsets])
    floats = ext.paged_prefill_workspace_floats(rows, tokens, 8, 2)
    spaces = [torch.empty(floats, device=gpu) for _ in range(2)]
    held, out = [x.clone() for x in ins[0]], torch.zeros_like(refs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ext.paged_prefill_attention(*held, out, spaces[0], 16)
    stream = torch.cuda.Stream()
    for i in (0, 1, 2, 1, 0, 2):
        for dst, src in zip(held, ins[i]):
            dst.copy_(src)
        out.fill_(7.0)
        other = torch.full_like(out, 7.0)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(stream):  # another call beside it, with a workspace of its own
            ext.paged_prefill_attention(*ins[(i + 1) % 3], other, spaces[1], 16)
        torch.cuda.synchronize()
        assert torch.equal(out, refs[i]) and torch.equal(other, refs[(i + 1) % 3]), i
