"""paged_attention_fp8_block against decode attention in 64 bits, element by element.

fp16: weights reach the product with V rounded to half a step (2^-11), and one below 2^-14 of
the running maximum's is subnormal, off by up to 2^-25.  The maximum is of weight times V's
scale, so what all of those lose is at most tokens * 2^-25 * 448 * max_j p_j vs_j.  bf16: the
weight is split into two terms, off by half a step of the second (2^-8 * 2^-8).
"""
import numpy as np
import pytest
import torch

from oracle import prompt
from prompt_cases import assert_within, attention_tolerance

pytestmark = pytest.mark.gpu
F16, BF16, F8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
P_STEP = {F16: 2.0 ** -11, BF16: 2.0 ** -16}


def _case(lengths, hq, hkv, page_size, dtype, seed, low=-9, high=-4, columns=None):
    gen = torch.Generator().manual_seed(seed)
    counts = [-(-max(n, 0) // page_size) for n in lengths]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=gen).tolist()
    columns = columns or max(counts + [1])
    table, at = [], 0
    for c in counts:
        mine = order[at:at + c]
        at += c
        table.append((mine + [pages + 7] * columns)[:columns])  # unused entries point nowhere
    k8, v8 = ((torch.randn(pages, hkv, page_size, 128, generator=gen) * 90).clamp(-448, 448).to(F8) for _ in range(2))
    scales = torch.exp2(torch.randint(low, high + 1, (pages, hkv, 2), generator=gen).float())
    q = torch.randn(len(lengths), hq, 128, generator=gen).to(dtype)
    return q, k8, v8, scales, torch.tensor(table, dtype=torch.int32), torch.tensor(lengths, dtype=torch.int32)


def _run(ext, gpu, case, out=None, ws=None):
    q, k8, v8, scales, table, lens = (x.to(gpu) for x in case)
    hq, hkv = q.shape[1], k8.shape[1]
    out = torch.full_like(q, float("nan")) if out is None else out
    if ws is None:
        ws = torch.full((ext.fp8_block_workspace_floats(len(lens), hq, hkv),), float("nan"), device=gpu)
    ext.paged_attention_fp8_block(q, k8, v8, scales, table, lens, out, ws, k8.shape[2])
    torch.cuda.synchronize()
    return out


def _check(ext, gpu, case, what=""):
    out = _run(ext, gpu, case)
    q, k8, v8, scales, table, lens = case
    want, weight, score, lead = prompt.fp8_block_decode(q.double(), k8.double(), v8.double(), scales.double(), table.numpy(), lens.tolist())
    n = max(lens.tolist() + [1])
    tiny = n * 2.0 ** -25 * 448 * lead[..., None] if q.dtype == F16 else 0.0
    bound = attention_tolerance(want, weight, score, n, q.dtype, P_STEP[q.dtype], tiny)
    assert_within(out, want, bound, what)
    return out


@pytest.mark.parametrize("lengths", [[1], [15, 16, 17], [31, 32, 33, 0, 1], [500], [0, 0], [2000, 3, 64, 65, 130], [1] * 90], ids=str)
@pytest.mark.parametrize("page_size,dtype", [(16, F16), (16, BF16), (32, F16), (48, BF16), (128, F16)])
def test_lengths(ext, gpu, lengths, page_size, dtype):
    _check(ext, gpu, _case(lengths, 8, 2, page_size, dtype, seed=sum(lengths)), f"{lengths[:5]} pages of {page_size}")


@pytest.mark.parametrize("lengths", [[1], [15, 16, 17], [31, 32, 33, 0, 1], [500], [0, 0], [512, 3, 64, 65, 130], [33] * 90], ids=str)
@pytest.mark.parametrize("columns", [32, 33, 400])
@pytest.mark.parametrize("hq,hkv,dtype", [(8, 2, F16), (16, 1, BF16), (17, 1, F16), (3, 3, BF16)])
def test_lengths_under_short_and_wide_tables(ext, gpu, lengths, columns, hq, hkv, dtype):
    """Tables of 512 tokens, a page more, and many: each way to share the work out."""
    _check(ext, gpu, _case(lengths, hq, hkv, 16, dtype, seed=columns + len(lengths), columns=columns), f"{lengths[:5]} of {16 * columns}")


@pytest.mark.parametrize("rows,columns,longest", [(512, 16, 300), (513, 16, 300), (255, 32, 200), (256, 32, 1024), (300, 33, 200)])
def test_rows_of_short_tables(ext, gpu, rows, columns, longest):
    """About a row and two rows a CU, between which a table of up to 1024 tokens is short too."""
    rng = np.random.default_rng(rows)
    lengths = rng.integers(0, 60, rows)
    lengths[::9] = rng.integers(0, longest + 1, len(lengths[::9]))
    _check(ext, gpu, _case(lengths.tolist(), 2, 1, 32, BF16, seed=rows, columns=columns), f"{rows} rows")


def test_scales_far_apart_in_a_wide_table(ext, gpu):
    """Pages whose V is 2^40 larger than others', through the cut over all CUs."""
    case = _case([200, 65, 400], 4, 2, 16, F16, seed=3, columns=64)
    scales = case[3]
    scales[:, :, 0] = 2.0 ** -8
    scales[::2, :, 1] = 2.0 ** -40
    _check(ext, gpu, case, "2^40 apart")


def test_short_tables_in_place_and_replayed(ext, gpu):
    cases = [_case([300, 33, 0, 512], 8, 2, 16, F16, seed=s, columns=32) for s in (31, 32)]
    refs = [_check(ext, gpu, c) for c in cases]
    dev = [[x.to(gpu) for x in c] for c in cases]
    q = dev[0][0].clone()
    ws = torch.empty(ext.fp8_block_workspace_floats(4, 8, 2), device=gpu)
    ext.paged_attention_fp8_block(q, *dev[0][1:], q, ws, 16)  # output over q
    assert torch.equal(q, refs[0])
    ins, out = [x.clone() for x in dev[0]], torch.zeros_like(refs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ext.paged_attention_fp8_block(*ins, out, ws, 16)
    for i in (0, 1, 0, 1):
        for x, y in zip(ins, dev[i]):
            x.view(torch.uint8).copy_(y.view(torch.uint8))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, refs[i])


@pytest.mark.parametrize("hq,hkv", [(1, 1), (2, 1), (3, 1), (5, 1), (8, 1), (10, 2), (16, 1), (17, 1), (31, 1), (32, 1), (40, 2), (12, 12)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_head_layouts(ext, gpu, hq, hkv, dtype):
    _check(ext, gpu, _case([77, 0, 300, 1], hq, hkv, 16, dtype, seed=hq + 50 * hkv), f"Hq {hq} Hkv {hkv}")


@pytest.mark.parametrize("rows", [257, 600])
def test_many_rows(ext, gpu, rows):
    rng = np.random.default_rng(rows)
    _check(ext, gpu, _case(rng.integers(0, 40, rows).tolist(), 2, 1, 16, F16, seed=rows), f"{rows} rows")


def test_one_long_row(ext, gpu):
    _check(ext, gpu, _case([20000], 4, 1, 64, F16, seed=1), "20000 tokens")
    _check(ext, gpu, _case([20000, 1], 4, 1, 64, BF16, seed=2), "20000 and 1 tokens")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_scales_far_apart(ext, gpu, dtype):
    """Pages whose V is 2^40 larger than others', next to pages of zeros under the least scale;
    K's scales keep the scores small."""
    case = _case([200, 65, 400], 4, 2, 16, dtype, seed=3)
    q, k8, v8, scales, table, lens = case
    scales[:, :, 0] = 2.0 ** -8
    scales[::2, :, 1] = 2.0 ** -40
    scales[1::3, :, 1] = 2.0 ** -60
    v8 = v8.float()
    v8[1::3] = 0.0
    _check(ext, gpu, (q, k8, v8.to(F8), scales, table, lens), "2^40 apart")
    # the page with large V has next to no weight: the others' values must survive
    k8 = k8.float()
    k8[:] = 0.0
    big = table[0, 3].item()
    k8[big] = -8.0
    scales[:, :, 1] = 2.0 ** -12
    scales[big, :, 1] = 2.0 ** 7
    scales[:, :, 0] = 2.0 ** -2
    q = torch.ones_like(q)
    _check(ext, gpu, (q, k8.to(F8), v8.to(F8), scales, table, lens), "large V without weight")


@pytest.mark.parametrize("tokens,columns", [(400, 32), (400, 64), (4112, 257)])
def test_scales_at_both_ends(ext, gpu, tokens, columns):
    """bf16: one page whose V is 2^120 larger than the others', and whose tokens weigh 2^7.1 times as
    much each.  Next to weight times V's scale the others' are below fp32's range, but they are
    0.15 to 0.65 of the sum that divides."""
    q, k8, v8, scales, table, lens = _case([tokens], 4, 2, 16, BF16, seed=10, columns=columns)
    q[:] = 1.0
    k8, big = torch.zeros_like(k8.float()), table[0, 3].item()
    k8[big, :, :, 0] = 56.0
    scales[:, :, 0], scales[:, :, 1] = 1.0, 2.0 ** -60
    scales[big, :, 1] = 2.0 ** 60
    _check(ext, gpu, (q, k8.to(F8), v8, scales, table, lens), f"{tokens} tokens")


def test_scales_that_are_no_powers_of_two(ext, gpu):
    case = _case([300, 20], 8, 2, 16, F16, seed=4)
    scales = case[3] * (1 + torch.rand(case[3].shape, generator=torch.Generator().manual_seed(5)))
    _check(ext, gpu, (*case[:3], scales, *case[4:]), "odd scales")
    bad = scales.clone()  # outside the range: clamped, NaN and what is not positive to the least
    bad[::4, :, 1] = 0.0
    bad[1::4, :, 1] = float("nan")
    bad[2::5, :, 0] = -1.0
    _check(ext, gpu, (*case[:3], bad, *case[4:]), "scales out of range")


def test_nothing_behind_a_row_is_read(ext, gpu):
    """NaN codes behind each row's last token, and in pages of no row."""
    case = list(_case([17, 100, 1], 8, 2, 32, F16, seed=6))
    used = torch.zeros(case[1].shape[0], 32, dtype=torch.bool)
    for b, n in enumerate(case[5].tolist()):
        for t in range(n):
            used[case[4][b, t // 32], t % 32] = True
    for i in (1, 2):
        x = case[i].float()
        x[~used[:, None, :, None].expand_as(x)] = float("nan")
        case[i] = x.to(F8)
    _check(ext, gpu, tuple(case), "NaN behind the rows")


def test_lengths_and_pages_out_of_range(ext, gpu):
    """Lengths past the table count as its capacity, page ids as clamped into the pool."""
    q, k8, v8, scales, table, lens = _case([64, 40], 4, 1, 16, F16, seed=7)
    table[1, 0], table[0, 1] = -5, 10 ** 6
    _check(ext, gpu, (q, k8, v8, scales, table, torch.tensor([1000, -3], dtype=torch.int32)))


def test_in_place_streams_and_graph_replays(ext, gpu):
    cases = [_case([900, 33, 400], 8, 2, 16, F16, seed=s) for s in (8, 9)]
    refs = [_check(ext, gpu, c) for c in cases]
    dev = [[x.to(gpu) for x in c] for c in cases]
    floats = ext.fp8_block_workspace_floats(3, 8, 2)
    q = dev[0][0].clone()
    ext.paged_attention_fp8_block(q, *dev[0][1:], q, torch.empty(floats, device=gpu), 16)  # output over q
    assert torch.equal(q, refs[0])
    outs = [torch.zeros_like(r) for r in refs]
    wss = [torch.empty(floats, device=gpu) for _ in refs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for st, d, out, ws in zip(streams, dev, outs, wss):
            with torch.cuda.stream(st):
                ext.paged_attention_fp8_block(*d, out, ws, 16)
    torch.cuda.synchronize()
    assert all(torch.equal(o, r) for o, r in zip(outs, refs))
    held = [x.clone() for x in dev[0]]
    out, graph = torch.zeros_like(refs[0]), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ext.paged_attention_fp8_block(*held, out, wss[0], 16)
    for i, lens in ((0, [900, 33, 400]), (1, [900, 33, 400]), (0, [5, 0, 1]), (0, [900, 33, 400])):
        for h, d in zip(held, dev[i]):
            h.copy_(d)
        held[5].copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.empty_like(out)
        ext.paged_attention_fp8_block(*held, eager, wss[1], 16)
        assert torch.equal(out, eager)
