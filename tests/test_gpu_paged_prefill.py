"""paged_prefill_attention against attention in 64 bits over the rows' pages, element by element
(tolerances as those of prefill_attention: products and weights are the same; joining a row's parts
adds roundings that the tolerance's exponent and sum terms hold)."""
import numpy as np
import pytest
import torch

from oracle import turn
from prompt_cases import U, assert_within
from turn_cases import Cache, check_chunk, i32, run_chunk

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16

ROWS = [  # lens, new
    ([1], [1]), ([2], [1]), ([33], [33]), ([64], [2]), ([500], [5]), ([1000], [1000]), ([40, 300, 1], [40, 7, 1]),
    ([0, 5, 0], [0, 5, 0]), ([700, 64, 65, 31], [1, 1, 1, 1]), ([90, 1500], [0, 130]), ([3000], [1]), ([129] * 70, [1] * 70),
    ([0, 1, 2, 3] * 30 + [400], [0, 1, 1, 2] * 30 + [90]),
]


@pytest.mark.parametrize("lens,new", ROWS, ids=lambda x: "-".join(map(str, x[:6])))
@pytest.mark.parametrize("hq,hkv,page,dtype", [(8, 2, 16, F16), (8, 2, 24, BF16), (3, 3, 16, BF16), (16, 1, 64, F16)])
def test_rows(ext, gpu, lens, new, hq, hkv, page, dtype):
    check_chunk(ext, Cache(lens, new, hq, hkv, page, dtype, seed=sum(lens) + page), gpu, f"{lens[:6]} {new[:6]}")


@pytest.mark.parametrize("hq,hkv", [(1, 1), (2, 1), (3, 1), (5, 1), (10, 2), (31, 1), (32, 1), (12, 4), (9, 9)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_head_layouts(ext, gpu, hq, hkv, dtype):
    check_chunk(ext, Cache([200, 77, 450], [61, 1, 300], hq, hkv, 16, dtype, seed=hq * 40 + hkv), gpu, f"Hq {hq} Hkv {hkv}")


@pytest.mark.parametrize("page", [1, 2, 3, 7, 8, 16, 31, 32, 33, 48, 128, 1000, 4096])
def test_page_sizes(ext, gpu, page):
    check_chunk(ext, Cache([1100, 37], [100, 37], 4, 2, page, F16, seed=page), gpu, f"pages of {page}")


@pytest.mark.parametrize("page,lens,new", [(1, [2100], [1000]), (2, [1700, 600], [900, 600]), (3, [4000], [700])])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_parts_longer_than_a_window_of_page_ids(ext, gpu, page, lens, new, dtype):
    """Blocks enough that a part of a row is more tiles than 512 pages hold."""
    check_chunk(ext, Cache(lens, new, 32, 4, page, dtype, seed=page + 5), gpu, f"pages of {page}")


@pytest.mark.parametrize("lens,new,hq,hkv", [([300] * 12, [150] * 12, 32, 8), ([600, 40], [600, 40], 32, 16),
                                             ([2000] + [50] * 40, [3] + [50] * 40, 16, 16), ([200] * 100, [64] * 100, 8, 2)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_blocks_for_every_cu(ext, gpu, lens, new, hq, hkv, dtype):
    """Calls of many blocks, whose waves do not share their tiles out; with rows cut and not."""
    check_chunk(ext, Cache(lens, new, hq, hkv, 16, dtype, seed=len(lens)), gpu, f"{lens[:3]} {new[:3]}")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_tokens_that_see_nothing(ext, gpu, dtype):
    """More new tokens than the row has: the first ones give 0; a row without tokens only zeros."""
    cache = Cache([20, 0, 150], [20, 0, 150], 4, 2, 16, dtype, seed=2)
    cache.offsets = np.array([0, 50, 57, 170])
    cache.q = torch.randn(170, 4, 128, generator=torch.Generator().manual_seed(1)).to(dtype)
    out = check_chunk(ext, cache, gpu, "rows shorter than their tokens")
    assert (out[:30] == 0).all() and (out[50:57] == 0).all() and (out[30:50] != 0).any()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_tokens_outside_every_row(ext, gpu, dtype):
    cache = Cache([70, 3, 300], [9, 3, 129], 8, 2, 16, dtype, seed=3, lead=300, trail=90)
    cache.q[:300] = float("nan")
    cache.q[300 + 141:] = float("nan")
    check_chunk(ext, cache, gpu)


def test_lengths_past_the_table_and_bad_pages_stay_inside(ext, gpu):
    """A row longer than its table sees what the table holds; ids outside the pool count as its ends."""
    cache = Cache([100, 64], [10, 64], 4, 2, 16, F16, seed=4, spare_columns=0, stale=0.5)
    cache.lens[0] = 130  # the table holds 112
    cache.table[1, 1], cache.table[1, 3] = -5, 10 ** 6
    check_chunk(ext, cache, gpu)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,more", [(8, 2, 0), (2, 2, 0), (16, 1, 0), (8, 2, 90), (16, 16, 40)])
def test_nonfinite_values_reach_the_tokens_that_see_them(ext, gpu, dtype, hq, hkv, more):
    cache = Cache([400, 150, 64] + [1] * more, [300, 150, 1] + [1] * more, hq, hkv, 16, dtype, seed=5)
    inf, nan = float("inf"), float("nan")
    spots = [(0, 170, 0, 3, inf), (0, 190, 0, 3, -inf), (0, 140, 0, 127, nan), (0, 399, hkv - 1, 0, nan), (1, 149, 0, 64, nan),
             (1, 0, 0, 17, inf), (2, 63, 0, 5, inf)]
    clean = turn.paged_prefill
    k, v = (np.nan_to_num(x.double().numpy(), nan=0.0) for x in (cache.k, cache.v))
    for row, pos, head, dim, x in spots:
        page, off = cache.place(row, pos)
        cache.v[page, head, off, dim] = x
        v[page, head, off, dim] = x
    page, off = cache.place(1, 130)
    cache.k[page, 0, off, 5] = nan  # every score of the tokens from 130 on
    k[page, 0, off, 5] = nan
    want, *rest = clean(cache.q.double().numpy(), k, v, cache.table, cache.lens, cache.offsets)
    out = run_chunk(ext, cache, gpu)
    finite = np.isfinite(want)
    bound = cache.bound(np.where(finite, want, 0.0), *rest)
    assert_within(out, want, np.where(np.isfinite(bound), bound, 0.0), "nonfinite")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_growing_falling_and_peaked_scores(ext, gpu, dtype):
    cache = Cache([900], [200], 4, 1, 16, dtype, seed=6)
    cache.q[:] = 1.0
    pos = torch.arange(900)
    ids, off = torch.as_tensor(cache.table[0])[pos // 16], pos % 16
    ramp = torch.linspace(0.0, 6.0, 900)[:, None]
    for name, keys in (("ramp", ramp), ("falling", -ramp), ("peak", 40.0 * (pos == 399)[:, None])):
        cache.k[ids, 0, off] = keys.to(dtype).expand(-1, 128)
        check_chunk(ext, cache, gpu, name)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hidden", [1, 32, 130, 256, 700])
def test_keys_of_minus_infinity(ext, gpu, dtype, hidden):
    """Whole parts of a row without weight; a token that sees none but such keys is NaN."""
    cache = Cache([900], [300], 4, 2, 16, dtype, seed=hidden)
    cache.q[..., 0] = 1.0
    pos = torch.arange(hidden)
    cache.k[torch.as_tensor(cache.table[0])[pos // 16], :, pos % 16, 0] = -float("inf")
    k, v = (np.nan_to_num(x.double().numpy(), nan=0.0, neginf=-np.inf) for x in (cache.k, cache.v))
    want, weight, vmax, score = turn.paged_prefill(cache.q.double().numpy(), k, v, cache.table, cache.lens, cache.offsets)
    rest = cache.want()[1:]  # without the infinities, in magnitudes
    out = run_chunk(ext, cache, gpu)
    seen = 900 - 300 + np.arange(300) >= hidden
    assert torch.isnan(out[torch.from_numpy(~seen)]).all()
    assert_within(out[torch.from_numpy(seen)], want[seen], cache.bound(want, weight, vmax, rest[2] + 20.0)[seen], f"{hidden} hidden")


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_large_scores(ext, gpu, dtype, sign):
    """Scores about 2^32 (fp16) and 2^100 (bf16): the keys of the largest share all the weight, over
    all parts of the row."""
    cache = Cache([600], [130], 2, 1, 16, dtype, seed=13)
    pos = torch.arange(600)
    ids, off, steps = torch.as_tensor(cache.table[0])[pos // 16], pos % 16, pos % 3
    cache.q[:] = 0.0
    key = torch.zeros(600, 128)
    if dtype == F16:
        cache.q[..., :4] = 16.0 * 2047
        key[:, :4] = (sign * 16.0 * ((2039 if sign > 0 else 2037) - sign * steps))[:, None]
    else:
        cache.q[..., 0] = 255.0 * 2.0 ** 42
        key[:, 0] = sign * 2.0 ** 42 * (249 - sign * steps)
    cache.k[ids, 0, off] = key.to(dtype)
    out = run_chunk(ext, cache, gpu).cpu().double()
    v = cache.v[ids, 0, off].double()
    for i in range(130):
        seen = torch.arange(600) <= 470 + i
        tied = seen & (steps == 0)
        want, most = v[tied].mean(0), v[tied].abs().max()
        bound = U[dtype] * want.abs() + 700 * 2.0 ** -24 * most + 2.0 ** -25
        assert ((out[i] - want).abs() <= bound).all(), i


def test_pools_past_four_gigabytes(ext, gpu):
    """Pages whose bytes lie past 2^32 in the pools."""
    cache = Cache([700, 90], [40, 90], 8, 8, 16, F16, seed=8)
    want = check_chunk(ext, cache, gpu)
    pages = 2 ** 32 // (8 * 16 * 256) + 300
    q, k, v, table, lens, offsets = cache.on(gpu)
    pools = [torch.zeros(pages, 8, 16, 128, dtype=F16, device=gpu) for _ in range(2)]
    for pool, x in zip(pools, (k, v)):
        pool[-cache.pages:] = x
    out = torch.zeros_like(q)
    ws = torch.empty(ext.paged_prefill_workspace_floats(2, q.shape[0], 8, 8), device=gpu)
    ext.paged_prefill_attention(q, *pools, torch.where(table >= 0, table + pages - cache.pages, table), lens, offsets, out, ws, 16)
    assert torch.equal(out, want)


def test_strided_q_and_in_place(ext, gpu):
    cache = Cache([250, 33], [150, 33], 8, 2, 16, F16, seed=9)
    want = check_chunk(ext, cache, gpu)
    q, k, v, table, lens, offsets = cache.on(gpu)
    ws = torch.empty(ext.paged_prefill_workspace_floats(2, 183, 8, 2), device=gpu)
    fused = torch.zeros(183, 12, 128, dtype=F16, device=gpu)
    fused[:, :8] = q
    out = torch.zeros_like(q)
    ext.paged_prefill_attention(fused[:, :8], k, v, table, lens, offsets, out, ws, 16)
    assert torch.equal(out, want)
    ext.paged_prefill_attention(q, k, v, table, lens, offsets, q, ws, 16)
    assert torch.equal(q, want)


def test_bad_offsets_stay_inside(ext, gpu):
    cache = Cache([300, 280], [60, 140], 4, 2, 16, F16, seed=10)
    want = run_chunk(ext, cache, gpu)
    cache.offsets = np.array([-5, 60, 900])
    assert torch.equal(run_chunk(ext, cache, gpu), want)


def test_streams_and_graph_replays(ext, gpu):
    caches = [Cache(*x, 8, 2, 16, F16, seed=s) for s, x in ((1, ([300, 900], [100, 7])), (2, ([1200, 70], [50, 57])))]
    refs = [check_chunk(ext, c, gpu) for c in caches]
    columns, pages = max(c.table.shape[1] for c in caches), max(c.pages for c in caches)
    ins = []
    for c in caches:
        q, k, v, table, lens, offsets = c.on(gpu)
        wide = torch.full((2, columns), -1, dtype=torch.int32, device=gpu)
        wide[:, :table.shape[1]] = table
        pools = [torch.zeros(pages, 2, 16, 128, dtype=F16, device=gpu) for _ in range(2)]
        for pool, x in zip(pools, (k, v)):
            pool[:c.pages] = x
        ins.append([q, *pools, wide, lens, offsets])
    ws = [torch.empty(ext.paged_prefill_workspace_floats(2, 107, 8, 2), device=gpu) for _ in range(2)]
    outs = [torch.zeros_like(r) for r in refs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for st, x, out, w in zip(streams, ins, outs, ws):
            with torch.cuda.stream(st):
                ext.paged_prefill_attention(*x, out, w, 16)
    torch.cuda.synchronize()
    assert all(torch.equal(o, r) for o, r in zip(outs, refs))
    held = [x.clone() for x in ins[0]]
    out = torch.zeros_like(refs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ext.paged_prefill_attention(*held, out, ws[0], 16)
    for i in (0, 1, 0, 1):  # the captured call follows its inputs, the lengths among them
        for dst, src in zip(held, ins[i]):
            dst.copy_(src)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, refs[i])


def test_one_token_a_row_is_the_decode_op(ext, gpu):
    """Within the two operators' roundings of the weights and outputs."""
    cache = Cache([900, 40, 2000, 1], [1] * 4, 8, 2, 16, F16, seed=12, stale=0.0)
    out = check_chunk(ext, cache, gpu)
    q, k, v, table, lens, offsets = cache.on(gpu)
    ref = torch.zeros_like(out)
    ws = torch.empty(ext.workspace_floats(4, 8, 4), device=gpu)
    ext.paged_attention_masked(q, k, v, table, lens, ref, ws, 2000, 16, 4)
    assert (out.float() - ref.float()).abs().max() <= 2e-3
