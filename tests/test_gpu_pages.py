"""fork_rows, free_rows, compact_pages and copy_pages against plain loops: whole numbers and copies,
so every entry must be equal."""
import numpy as np
import pytest
import torch

from oracle import turn
from turn_cases import i32

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def _equal(got, want):
    got = got.cpu().long().reshape(-1)
    want = torch.as_tensor(np.asarray(want)).long().reshape(-1)
    assert torch.equal(got, want), (got[got != want][:8], want[got != want][:8])


def _state(rng, rows, hi, page, columns, spare=3, shared=0):
    """A table of `rows` rows, whose first `shared` pages are the same, page_shares and the list."""
    lens = rng.integers(0, min(hi, columns * page) + 1, rows)
    counts = -(-lens // page)
    pages = int(counts.sum()) + columns * spare + 1
    order = list(rng.permutation(pages))
    prefix = [order.pop() for _ in range(shared)]
    table, shares = rng.integers(-3, pages + 5, (rows, columns)), np.zeros(pages, dtype=np.int64)
    holders = np.zeros(pages, dtype=np.int64)
    for b, n in enumerate(counts):
        for c in range(n):
            table[b, c] = prefix[c] if c < shared and (c + 1) * page <= lens[b] else order.pop()
            holders[table[b, c]] += 1
    shares = np.maximum(holders - 1, 0)
    free = order + [p for p in prefix if holders[p] == 0]
    num_free = len(free)
    return lens, table, shares, np.array(free + [77] * (pages - num_free)), num_free


def _fork(ext, gpu, parents, children, lens, table, shares, free, num_free, page):
    t, s = i32(table, gpu), i32(shares, gpu)
    given = [i32(parents, gpu), i32(children, gpu), i32(lens, gpu), i32(free, gpu), i32([num_free], gpu)]
    before = [x.clone() for x in given]
    left, src, dst = (i32([99] * n, gpu) for n in (1, len(parents), len(parents)))
    ext.fork_rows(*given[:3], t, s, *given[3:], left, src, dst, page)
    want = turn.fork_rows(parents, children, lens, table, shares, free, num_free, page)
    for got, w in zip((t, s, left, src, dst), want):
        _equal(got, w)
    assert all(torch.equal(a, b) for a, b in zip(given, before))
    return t, s, left, src, dst


@pytest.mark.parametrize("rows,ways,hi,page,columns", [(1, 1, 40, 16, 7), (4, 16, 500, 16, 40), (8, 1, 100, 24, 300), (3, 5, 900, 1, 900),
                                                       (60, 2, 64, 16, 6), (300, 4, 90, 8, 12), (1, 1500, 200, 64, 5), (2, 3, 0, 16, 4)])
def test_forks(ext, gpu, rows, ways, hi, page, columns):
    rng = np.random.default_rng(rows * 31 + hi)
    lens, table, shares, free, num_free = _state(rng, rows, hi, page, columns)
    children = rows * ways
    table = np.concatenate([table, rng.integers(-5, 3, (children, columns))])
    lens = np.concatenate([lens, rng.integers(-2, 99, children)])
    parents, kids = [i // ways for i in range(children)], list(rng.permutation(np.arange(rows, rows + children)))
    free = np.concatenate([free, rng.integers(0, 9, children)])
    _fork(ext, gpu, parents, kids, lens, table, shares, free, num_free, page)
    _fork(ext, gpu, parents, kids, lens, table, shares, free, len(free), page)


def test_forks_that_find_no_page_change_nothing(ext, gpu):
    lens, table = [40, 0, 33, 0], [[5, 6, 7, -1], [-1] * 4, [2, 3, 4, -1], [-1] * 4]
    shares, free = [0] * 12, [8, 9]
    t, s, left, src, dst = _fork(ext, gpu, [0, 2, 0], [1, 3, 3], lens, table, shares, free, 2, 16)
    assert left.item() == -1 and src.tolist() == dst.tolist() == [-1] * 3 and t.tolist() == table
    t, s, left, src, dst = _fork(ext, gpu, [0, 2], [1, 3], lens, table, shares, free, 2, 16)
    assert left.item() == 0 and src.tolist() == [7, 4] and dst.tolist() == [9, 8]
    assert t.tolist()[1] == [5, 6, 9, -1] and s.tolist()[2:8] == [1, 1, 0, 1, 1, 0]


def test_forks_of_no_rows_whole_pages_and_odd_pairs(ext, gpu):
    lens, table, shares, free = [32, 5, -4, 10 ** 6], [[1, 2, -1], [3, -1, -1], [-1] * 3, [4, -7, 99]], [0] * 9, [8, 7, 6, 5]
    _fork(ext, gpu, [], [], lens, table, shares, free, 4, 16)
    _fork(ext, gpu, [], [], lens, table, shares, free, -3, 16)
    _fork(ext, gpu, [0], [2], lens, table, shares, free, 0, 16)       # whole pages only: none is needed
    _fork(ext, gpu, [2], [1], lens, table, shares, free, 4, 16)       # a negative length
    _fork(ext, gpu, [3], [2], lens, table, shares, free, 4, 16)       # past its table, with ids that are none
    _fork(ext, gpu, [0, 9, -1, 1, 1], [9, 1, 2, 1, 2], lens, table, shares, free, 4, 16)  # rows outside, a row to itself


def _free(ext, gpu, rows, lens, table, shares, free, num_free, page):
    s, f = i32(shares, gpu), i32(free, gpu)
    given = [i32(rows, gpu), i32(lens, gpu), i32(table, gpu), i32([num_free], gpu)]
    before = [x.clone() for x in given]
    left = i32([99], gpu)
    ws = torch.full((ext.page_workspace_ints(len(shares)),), -12345, dtype=torch.int32, device=gpu)
    ext.free_rows(given[0], given[1], given[2], s, f, given[3], left, ws, page)
    for got, w in zip((s, f, left), turn.free_rows(rows, lens, table, shares, free, num_free, page)):
        _equal(got, w)
    assert all(torch.equal(a, b) for a, b in zip(given, before))
    return s, f, left


@pytest.mark.parametrize("rows,hi,page,columns,shared", [(1, 40, 16, 7, 0), (64, 700, 16, 60, 5), (5, 3000, 2, 1600, 300), (200, 90, 24, 4, 1),
                                                         (3, 0, 16, 3, 0), (900, 60, 1, 60, 7)])
def test_frees(ext, gpu, rows, hi, page, columns, shared):
    rng = np.random.default_rng(rows + hi)
    lens, table, shares, free, num_free = _state(rng, rows, hi, page, columns, shared=shared)
    for gone in ([], [0], list(rng.permutation(rows)[:rows // 2]), list(rng.permutation(rows))):
        _free(ext, gpu, gone, lens, table, shares, free, num_free, page)


def test_rows_listed_twice_or_outside(ext, gpu):
    rng = np.random.default_rng(3)
    lens, table, shares, free, num_free = _state(rng, 40, 300, 16, 20, shared=6)
    gone = list(rng.integers(-3, 45, 700))
    _free(ext, gpu, gone, lens, table, shares, free, num_free, 16)
    lens[:5] = [-4, 10 ** 6, 320, 321, 0]
    _free(ext, gpu, [0, 1, 2, 3, 4, 1], lens, table, shares, free, num_free, 16)


def test_frees_with_a_full_list_stay_inside(ext, gpu):
    """Counts that contradict the table: the list takes no more than its places."""
    _free(ext, gpu, [0], [64], [[0, 1, 2, 3]], [0] * 5, [4, 4, 4, 9, 9], 3, 16)
    _free(ext, gpu, [0], [64], [[0, 1, 2, 3]], [0] * 5, [4, 4, 4, 9, 9], 77, 16)
    _free(ext, gpu, [0], [64], [[0, 0, 0, 9]], [1] * 5, [4, 4, 4, 9, 9], -1, 16)


def _compact(ext, gpu, table, shares, free, num_free, extra=0, in_place=False):
    pages = len(shares)
    copies = pages // 2 + extra
    ins = [i32(x, gpu) for x in (table, shares, free, [num_free])]
    before = [x.clone() for x in ins]
    page_map, shares_out, left = (i32([99] * n, gpu) for n in (pages, pages, 1))
    src, dst = i32([99] * copies, gpu), i32([99] * copies, gpu)
    table_out, free_out = ins[0] if in_place else torch.full_like(ins[0], 99), ins[2].clone()
    ws = torch.full((ext.page_workspace_ints(pages),), -12345, dtype=torch.int32, device=gpu)
    ext.compact_pages(*ins, page_map, table_out, shares_out, free_out, left, src, dst, ws)
    want = turn.compact_pages(table, shares, free, num_free, copies)
    for got, w in zip((page_map, table_out, shares_out, free_out, left, src, dst), want):
        _equal(got, w)
    assert all(torch.equal(a, b) for a, b in list(zip(ins, before))[in_place:])


@pytest.mark.parametrize("rows,hi,page,columns,spare", [(1, 40, 16, 7, 1), (10, 700, 16, 60, 3), (64, 300, 16, 40, 30), (2, 900, 1, 900, 2), (200, 500, 8, 64, 1), (3, 0, 16, 3, 1)])
def test_compactions(ext, gpu, rows, hi, page, columns, spare):
    rng = np.random.default_rng(rows + hi)
    lens, table, shares, free, num_free = _state(rng, rows, hi, page, columns, spare=spare, shared=min(2, columns))
    _compact(ext, gpu, table, shares, free, num_free, extra=5)
    _compact(ext, gpu, table, shares, free, num_free, in_place=True)
    some = num_free // 2  # pages that neither a row nor the list names stay in use
    _compact(ext, gpu, table, shares, free, some)


def test_compactions_of_full_empty_and_single_pools(ext, gpu):
    n = 2500
    shares = list(range(n))
    for free in ([], list(range(n)), list(range(n))[::-1], [5], [n - 1], list(range(0, n, 2)), list(range(n // 2)), list(range(n // 2, n)),
                 [3, 3, 3, -1, n, n + 7]):
        _compact(ext, gpu, [[0, n - 1, -1, n, 7]], shares, free + [0] * (n - len(free)), len(free))
    _compact(ext, gpu, [[0]], [4], [0], 0)
    _compact(ext, gpu, [[0]], [4], [0], 1, extra=2)
    _compact(ext, gpu, np.zeros((0, 3), dtype=np.int64), [0, 0], [1, 0], 1)


@pytest.mark.parametrize("pages", [65535, 65536, 65537, 300001, 524288, 524289, 1100000])
def test_large_pools(ext, gpu, pages):
    """On both sides of the sizes where the counting moves to launches of its own."""
    rng = np.random.default_rng(pages)
    order = rng.permutation(pages)
    used = pages * 2 // 5
    shares = np.zeros(pages, dtype=np.int64)
    shares[order[:used]] = rng.integers(0, 3, used)
    free = np.concatenate([order[used:], np.zeros(used, dtype=np.int64)])
    columns = used // 7
    table = order[:7 * columns].reshape(7, columns)
    # numpy forms of the loops
    in_use = np.ones(pages, dtype=bool)
    in_use[free[:pages - used]] = False
    holes, movers = np.nonzero(~in_use[:used])[0], used + np.nonzero(in_use[used:])[0][::-1]
    page_map = np.where(in_use, np.arange(pages), -1)
    page_map[movers] = holes
    moved = np.zeros(pages, dtype=np.int64)
    moved[page_map[in_use]] = shares[in_use]
    list_out = free.copy()
    list_out[:pages - used] = np.arange(pages - 1, used - 1, -1)
    pad = np.full(pages // 2 - len(holes), -1)
    ins = [i32(x, gpu) for x in (table, shares, free, [pages - used])]
    outs = [i32(np.zeros(n), gpu) for n in (pages, pages, 1, pages // 2, pages // 2)]
    table_out, free_out = torch.zeros_like(ins[0]), ins[2].clone()
    ws = torch.empty(ext.page_workspace_ints(pages), dtype=torch.int32, device=gpu)
    ext.compact_pages(*ins, outs[0], table_out, outs[1], free_out, outs[2], outs[3], outs[4], ws)
    for got, w in zip((outs[0], table_out, outs[1], free_out, outs[2], outs[3], outs[4]),
                      (page_map, page_map[table], moved, list_out, [pages - used], np.concatenate([movers, pad]), np.concatenate([holes, pad]))):
        _equal(got, w)
    # and all rows but two freed
    left = shares.copy()
    np.subtract.at(left, table[:5].reshape(-1), 1)
    gone = np.nonzero(left < 0)[0]
    want = free.copy()
    want[pages - used:pages - used + len(gone)] = gone
    s, n = ins[1].clone(), i32([0], gpu)
    ext.free_rows(i32([4, 2, 0, 1, 3], gpu), i32([columns * 16] * 7, gpu), ins[0], s, ins[2], ins[3], n, ws, 16)
    _equal(s, np.maximum(left, 0))
    _equal(ins[2], want)
    assert n.item() == pages - used + len(gone)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, F8])
@pytest.mark.parametrize("pages,hkv,page,pairs", [(9, 1, 1, 3), (40, 2, 16, 1), (40, 2, 16, 15), (300, 8, 16, 140), (30, 5, 24, 14), (12, 8, 128, 6), (5, 3, 1000, 2)])
def test_copies(ext, gpu, dtype, pages, hkv, page, pairs):
    gen = torch.Generator().manual_seed(pages + page)
    bits = lambda x: x.view(torch.uint8) if x.element_size() == 1 else x.view(torch.int16)
    pools = [torch.randint(0, 255, (pages, hkv, page, 128 * (1 if dtype == F8 else 2)), generator=gen, dtype=torch.uint8).view(dtype).to(gpu) for _ in range(2)]
    scales = torch.randn(pages, hkv, 2, generator=gen).to(gpu)
    order = torch.randperm(pages, generator=gen)
    src, dst = order[:pairs].clone(), order[pairs:2 * pairs].clone()
    src = torch.cat([src, torch.tensor([-1, 0, pages, 2, -1])])
    dst = torch.cat([dst, torch.tensor([0, -1, 0, pages, -1])])  # skipped
    src, dst = torch.cat([src, order[2 * pairs:2 * pairs + 1]]), torch.cat([dst, order[2 * pairs:2 * pairs + 1]])  # to itself
    for with_scales in (False, True):
        a, b, s = pools[0].clone(), pools[1].clone(), scales.clone()
        ext.copy_pages(i32(src, gpu), i32(dst, gpu), a, b, s if with_scales else None)
        to, come = dst[:pairs].to(gpu), src[:pairs].to(gpu)
        for got, was in ((a, pools[0]), (b, pools[1])):
            want = bits(was).clone()
            want[to] = want[come]
            assert torch.equal(bits(got), want)
        want = scales.clone()
        if with_scales:
            want[to] = want[come]
        assert torch.equal(s, want)


def test_copies_past_four_gigabytes(ext, gpu):
    pages = 2 ** 32 // (8 * 16 * 256) + 40
    pools = [torch.zeros(pages, 8, 16, 128, dtype=torch.float16, device=gpu) for _ in range(2)]
    pools[0][pages - 3], pools[1][1] = 2.0, 3.0
    ext.copy_pages(i32([pages - 3, 1], gpu), i32([pages - 20, pages - 1], gpu), *pools)
    assert (pools[0][pages - 20] == 2).all() and (pools[1][pages - 1] == 3).all()
    assert torch.count_nonzero(pools[0]).item() == torch.count_nonzero(pools[1]).item() == 2 * 8 * 16 * 128


def test_captured_calls_follow_their_inputs(ext, gpu):
    rng = np.random.default_rng(9)
    cases = []
    for _ in range(3):
        lens, table, shares, free, num_free = _state(rng, 12, 200, 16, 13, shared=3)
        cases.append((lens, table, shares, free, num_free))
    pages = max(len(c[2]) for c in cases)
    pad = lambda x: np.concatenate([x, np.zeros(pages - len(x), dtype=np.int64)])
    # pages past a case's own are on its list
    cases = [(l, t, pad(s), np.concatenate([f[:n], np.arange(len(s), pages), f[n:]]), n + pages - len(s)) for l, t, s, f, n in cases]
    held = [i32(x, gpu) for x in (*cases[0][:4], [cases[0][4]], [1, 3, 5], [8, 9, 10], [2, 7, 2])]
    lens, table, shares, free, num, parents, children, gone = held
    left, src, dst, s2, f2, l2 = i32([0], gpu), i32([0] * 3, gpu), i32([0] * 3, gpu), shares.clone(), free.clone(), i32([0], gpu)
    t1, s1 = table.clone(), shares.clone()
    out = [i32(np.zeros(x.shape), gpu) for x in (shares, table, shares, free, num)] + [i32([0] * (pages // 2), gpu) for _ in range(2)]
    ws = [torch.empty(ext.page_workspace_ints(pages), dtype=torch.int32, device=gpu) for _ in range(2)]

    def calls():
        t1.copy_(table), s1.copy_(shares), s2.copy_(shares), f2.copy_(free), out[3].copy_(free)
        ext.fork_rows(parents, children, lens, t1, s1, free, num, left, src, dst, 16)
        ext.free_rows(gone, lens, table, s2, f2, num, l2, ws[0], 16)
        ext.compact_pages(table, shares, free, num, *out, ws[1])

    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for i in (0, 1, 2, 0, 2):
        l, t, s, f, n = cases[i]
        for x, y in zip((lens, table, shares, free, num), (l, t, s, f, [n])):
            x.copy_(i32(y, gpu))
        graph.replay()
        torch.cuda.synchronize()
        for got, w in zip((t1, s1, left, src, dst), turn.fork_rows([1, 3, 5], [8, 9, 10], l, t, s, f, n, 16)):
            _equal(got, w)
        for got, w in zip((s2, f2, l2), turn.free_rows([2, 7, 2], l, t, s, f, n, 16)):
            _equal(got, w)
        for got, w in zip(out, turn.compact_pages(t, s, f, n, pages // 2)):
            _equal(got, w)
