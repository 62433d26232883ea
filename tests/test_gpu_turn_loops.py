"""The loops around the page operators over the kernels; a captured fork that is taken or not on the GPU."""
import pytest
import torch

from turn_cases import i32
from turn_loops import pages_back_beside_forked_rows, refused_fork_and_retry, rows_that_get_shorter

pytestmark = pytest.mark.gpu


@pytest.fixture
def ops(ext, gpu):
    def fork(parents, children, lens, table, shares, free, num_free, page):
        t, s, left, src, dst = i32(table, gpu), i32(shares, gpu), i32([99], gpu), i32([9] * len(parents), gpu), i32([9] * len(parents), gpu)
        ext.fork_rows(i32(parents, gpu), i32(children, gpu), i32(lens, gpu), t, s, i32(free, gpu), i32([num_free], gpu), left, src, dst, page)
        return t.tolist(), s.tolist(), left.item(), src.tolist(), dst.tolist()

    def release(rows, lens, table, shares, free, num_free, page):
        s, f, left = i32(shares, gpu), i32(free, gpu), i32([99], gpu)
        space = torch.empty(ext.page_workspace_ints(len(shares)), dtype=torch.int32, device=gpu)
        ext.free_rows(i32(rows, gpu), i32(lens, gpu), i32(table, gpu), s, f, i32([num_free], gpu), left, space, page)
        return s.tolist(), f.tolist(), left.item()

    return fork, release


def test_a_refused_fork_is_not_taken(ops):
    refused_fork_and_retry(*ops)


def test_pages_that_other_rows_hold_stay_off_the_list(ops):
    pages_back_beside_forked_rows(*ops)


def test_rows_that_get_shorter_give_their_pages_back(ops):
    rows_that_get_shorter(*ops)


def test_a_captured_step_of_rows_that_get_shorter(ext, gpu):
    """Lengths, the table of what lies behind them and the list all on the GPU, as one graph."""
    page, pages, columns = 16, 40, 5
    table = torch.full((3, columns), -1, dtype=torch.int32, device=gpu)
    lens, kept, num, left = (i32(x, gpu) for x in ([0] * 3, [0] * 3, [0], [0]))
    shares, free, rows = i32([0] * pages, gpu), i32([0] * pages, gpu), i32([0, 1, 2], gpu)
    space = torch.empty(ext.page_workspace_ints(pages), dtype=torch.int32, device=gpu)
    cols = torch.arange(columns, device=gpu)

    def step():
        first = (kept + page - 1) // page
        more = (lens + page - 1) // page - first
        behind = table.gather(1, (first[:, None] + cols).clamp(max=columns - 1))
        ext.free_rows(rows, more * page, behind, shares, free, num, left, space, page)
        num.copy_(left)
        lens.copy_(kept)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for n, keep, shared in (([80, 33, 5], [49, 32, 5], 0), ([80, 80, 80], [0, 16, 80], 0), ([40, 40, 7], [16, 17, 1], 1), ([64, 1, 2], [64, 1, 2], 0)):
        held = [-(-x // page) for x in n]
        ids = torch.randperm(pages).tolist()
        t = [[ids.pop() for _ in range(h)] + [-1] * (columns - h) for h in held]
        count = [0] * pages
        if shared:  # the second row holds the first's leading pages
            ids += t[1][:2]
            t[1][:2] = t[0][:2]
            for p in t[0][:2]:
                count[p] = 1
        for x, y in zip((table, lens, kept, num, shares, free), (t, n, keep, [len(ids)], count, ids + [0] * (pages - len(ids)))):
            x.copy_(i32(y, gpu))
        graph.replay()
        torch.cuda.synchronize()
        behind = [p for row, h, k in zip(t, held, keep) for p in row[-(-k // page):h]]
        gone = sorted(p for p in set(behind) if behind.count(p) > count[p])
        assert num.item() == len(ids) + len(gone) and lens.tolist() == keep
        assert free.tolist()[:num.item()] == ids + gone
        assert shares.tolist() == [max(count[p] - behind.count(p), 0) for p in range(pages)]


def test_a_captured_fork_takes_its_count_on_the_gpu(ext, gpu):
    """The count and the children's lengths by torch.where on the GPU: replays with too few pages
    leave the state as it was, those with enough go through."""
    page, pages = 16, 12
    table = i32([[0, 1, 2], [3, 4, 5], [-1] * 3, [-1] * 3], gpu)
    lens, shares, free = i32([40, 33, 0, 0], gpu), i32([0] * pages, gpu), i32(list(range(11, -1, -1)), gpu)
    num, left, src, dst = i32([1], gpu), i32([0], gpu), i32([0, 0], gpu), i32([0, 0], gpu)
    parents, children = i32([0, 1], gpu), i32([2, 3], gpu)
    pools = [torch.randn(pages, 1, page, 128, device=gpu).half() for _ in range(2)]

    def step():
        ext.fork_rows(parents, children, lens, table, shares, free, num, left, src, dst, page)
        ext.copy_pages(src, dst, *pools)
        fits = left >= 0
        num.copy_(torch.where(fits, left, num))
        lens[children.long()] = torch.where(fits, lens[parents.long()], lens[children.long()])

    held = [x.clone() for x in (table, lens, shares, num, *pools)]

    def restore(free_pages):
        for x, y in zip((table, lens, shares, num, *pools), held):
            x.copy_(y)
        num.fill_(free_pages)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for have in (1, 2, 0, 6, 1):
        restore(have)
        graph.replay()
        torch.cuda.synchronize()
        if have < 2:
            assert num.item() == have and lens.tolist() == [40, 33, 0, 0] and torch.equal(table, held[0]) and not shares.any()
            assert all(torch.equal(x, y) for x, y in zip(pools, held[4:]))
            continue
        taken = free.tolist()[have - 2:have][::-1]
        assert num.item() == have - 2 and lens.tolist() == [40, 33, 40, 33]
        assert table.tolist()[2:] == [[0, 1, taken[0]], [3, 4, taken[1]]] and shares.tolist() == [1, 1, 0, 1, 1] + [0] * 7
        for x, y in zip(pools, held[4:]):
            assert torch.equal(x[taken], y[[2, 5]])
