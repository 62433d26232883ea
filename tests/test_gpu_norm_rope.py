"""norm_rope and norm_rope_write_kv against the formulas in 64 bits, element by element."""
import numpy as np
import pytest
import torch

from oracle import turn
from prompt_cases import assert_within
from turn_cases import angles, i32, rope_tolerance

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
EPS = 1e-6


def _inputs(tokens, hq, hkv, dtype, seed, positions=3000, rot=128, weights="one"):
    gen = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(tokens, hq + 2 * hkv, 128, generator=gen) * torch.exp2(2 * torch.randn(1, hq + 2 * hkv, 1, generator=gen))).to(dtype)
    pos = torch.randint(0, positions, (tokens,), generator=gen, dtype=torch.int32)
    shape = {"one": (128,), "each": (-1, 128), "none": (0,)}[weights]
    w = [(1 + 0.3 * torch.randn(h, 128, generator=gen))[:1 if weights == "one" else h].reshape(-1)[:0 if weights == "none" else None]
         for h in (hq, hkv)]
    return qkv, pos, [x.reshape(shape) for x in w], angles(positions, rot)


def _want(x, weight, table, pos, pairs, eps=EPS):
    return turn.norm_rope(x.double().numpy(), weight.double().numpy() if weight.numel() else None, table.double().numpy(),
                          pos.tolist(), eps, pairs)


def _check(ext, gpu, qkv, pos, w, table, hq, hkv, pairs, eps=EPS, what=""):
    dtype, tokens = qkv.dtype, qkv.shape[0]
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    on = qkv.to(gpu)
    args = [x.to(gpu) for x in w] + [table.to(gpu), pos.to(gpu)]
    outs = [torch.full(x.shape, 7.0, dtype=dtype, device=gpu) for x in (q, k)]
    ext.norm_rope(on[:, :hq], on[:, hq:hq + hkv], *args, *outs, eps, pairs)
    for name, got, x, weight in zip("qk", outs, (q, k), w):
        want, size = _want(x, weight, table, pos, pairs, eps)
        assert_within(got, want, rope_tolerance(np.nan_to_num(want), np.nan_to_num(size), dtype), f"{what} {name}")
    # Straight into the pools: the same bits at the slots, and nothing elsewhere.
    page = 8
    pages = tokens // page + 3
    gen = torch.Generator().manual_seed(tokens)
    slots = torch.randperm(pages * page, generator=gen)[:tokens].to(torch.int32)
    slots[::7] = torch.where(torch.arange(tokens)[::7] % 2 == 0, -1, pages * page)  # skipped
    pools = [torch.full((pages, hkv, page, 128), 3.0, dtype=dtype, device=gpu) for _ in range(2)]
    q2 = torch.full_like(outs[0], 7.0)
    ext.norm_rope_write_kv(on[:, :hq], on[:, hq:hq + hkv], on[:, hq + hkv:], *args, q2, *pools, slots.to(gpu), eps, pairs)
    ref = [torch.full_like(p, 3.0) for p in pools]
    fine = (slots >= 0) & (slots < pages * page)
    at = slots[fine].long().to(gpu)
    ref[0][at // page, :, at % page] = outs[1][fine.to(gpu)]
    ref[1][at // page, :, at % page] = on[:, hq + hkv:][fine.to(gpu)]
    bits = lambda x: x.view(torch.int16)
    assert torch.equal(bits(q2), bits(outs[0])) and all(torch.equal(bits(a), bits(b)) for a, b in zip(pools, ref))
    return outs


@pytest.mark.parametrize("tokens", [1, 2, 3, 5, 64, 333])
@pytest.mark.parametrize("hq,hkv,dtype", [(8, 2, F16), (8, 2, BF16), (3, 3, F16), (1, 1, BF16), (40, 5, BF16), (17, 1, F16)])
def test_sizes(ext, gpu, tokens, hq, hkv, dtype):
    qkv, pos, w, table = _inputs(tokens, hq, hkv, dtype, tokens * 50 + hq)
    _check(ext, gpu, qkv, pos, w, table, hq, hkv, False, what=f"{tokens} tokens")


@pytest.mark.parametrize("hq,hkv,dtype,weights", [(8, 2, F16, "one"), (7, 7, BF16, "each"), (5, 1, F16, "none")])
def test_hundreds_of_thousands_of_heads(ext, gpu, hq, hkv, dtype, weights):
    """Four heads a wave, the last ones of a part of fewer: as the same tokens in calls of few."""
    tokens = (1 << 20) // (hq + hkv) + 37
    gen = torch.Generator(device=gpu).manual_seed(hq)
    qkv = torch.randn(tokens, hq + hkv, 128, generator=gen, device=gpu).to(dtype)
    _, pos, w, table = _inputs(tokens, hq, hkv, dtype, 3, weights=weights)
    args = [x.to(gpu) for x in w] + [table.to(gpu)]
    q, k = qkv[:, :hq], qkv[:, hq:]
    outs = [torch.zeros(tokens, h, 128, dtype=dtype, device=gpu) for h in (hq, hkv)]
    pos = pos.to(gpu)
    ext.norm_rope(q, k, *args, pos, *outs, EPS, False)
    for first, n in ((0, 200), (tokens // 2 - 7, 3), (tokens - 4000, 4000)):
        few = [torch.zeros(n, h, 128, dtype=dtype, device=gpu) for h in (hq, hkv)]
        at = slice(first, first + n)
        ext.norm_rope(q[at], k[at], *args, pos[at], *few, EPS, False)
        assert all(torch.equal(a[at], b) for a, b in zip(outs, few))


@pytest.mark.parametrize("rot", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("weights,tokens", [("one", 20), ("each", 400), ("none", 400), ("each", 3)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rotations_and_weights(ext, gpu, rot, pairs, weights, tokens, dtype):
    qkv, pos, w, table = _inputs(tokens, 10, 2, dtype, rot + pairs, rot=rot, weights=weights)
    _check(ext, gpu, qkv, pos, w, table, 10, 2, pairs, what=f"rot {rot}")


def test_a_norm_of_one_of_the_two(ext, gpu):
    qkv, pos, w, table = _inputs(50, 8, 2, BF16, 4)
    _check(ext, gpu, qkv, pos, [w[0], w[1][:0]], table, 8, 2, False)
    _check(ext, gpu, qkv, pos, [w[0][:0], w[1]], table, 8, 2, False)


def test_far_positions_and_ones_outside_the_table(ext, gpu):
    qkv, _, w, _ = _inputs(40, 4, 2, BF16, 5)
    table = angles(1 << 20, 128, base=500000.0)
    pos = torch.randint((1 << 20) - 5000, 1 << 20, (40,), dtype=torch.int32)
    pos[3], pos[4], pos[5] = -1, 1 << 20, 2 ** 31 - 1  # the table's ends
    _check(ext, gpu, qkv, pos, w, table, 4, 2, False)


@pytest.mark.parametrize("tokens", [3, 300])
def test_large_small_and_nonfinite_heads(ext, gpu, tokens):
    """Squares past 2^128 (bf16 values of 2^127) and below 2^-126; heads of zeros; infinities and
    NaN stay in their head."""
    qkv, pos, w, table = _inputs(tokens, 8, 2, BF16, 6)
    qkv[0, 0] = torch.where(qkv[0, 0] > 0, 2.0 ** 127, -(2.0 ** 126)).to(BF16)
    qkv[0, 1] *= 2.0 ** 64
    qkv[0, 2] *= 2.0 ** -90
    qkv[0, 3] = 0.0
    qkv[1, 0, 5], qkv[1, 1, 7], qkv[1, 9, 0] = float("inf"), float("nan"), -float("inf")
    want = [_want(x, y, table, pos, False) for x, y in ((qkv[:, :8], w[0]), (qkv[:, 8:10], w[1]))]
    outs = [torch.zeros(tokens, h, 128, dtype=BF16, device=gpu) for h in (8, 2)]
    on = qkv.to(gpu)
    ext.norm_rope(on[:, :8], on[:, 8:10], *(x.to(gpu) for x in w), table.to(gpu), pos.to(gpu), *outs, EPS, False)
    for got, (ref, size) in zip(outs, want):
        assert_within(got, ref, rope_tolerance(np.nan_to_num(ref), np.nan_to_num(size), BF16), "extremes")


@pytest.mark.parametrize("eps", [2.0 ** -100, 1e-12, 0.1, 2.0 ** 100])
def test_eps(ext, gpu, eps):
    qkv, pos, w, table = _inputs(30, 4, 2, BF16, 7)
    qkv *= 2.0 ** -20
    eps = float(np.float32(eps))
    _check(ext, gpu, qkv, pos, w, table, 4, 2, False, eps=eps)


@pytest.mark.parametrize("tokens", [1, 5, 700])
@pytest.mark.parametrize("pairs,rot", [(False, 128), (False, 96), (True, 64)])
def test_in_place_and_between_the_inputs(ext, gpu, tokens, pairs, rot):
    qkv, pos, w, table = _inputs(tokens, 8, 2, F16, 8, rot=rot)
    want = _check(ext, gpu, qkv, pos, w, table, 8, 2, pairs)
    args = [x.to(gpu) for x in w] + [table.to(gpu), pos.to(gpu)]
    fused = qkv.to(gpu)
    q, k = fused[:, :8], fused[:, 8:10]
    ext.norm_rope(q, k, *args, q, k, EPS, pairs)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(fused[:, 10:].cpu(), qkv[:, 10:])
    # outputs in columns of the inputs' own buffer, beside them
    wide = torch.zeros(tokens, 30, 128, dtype=F16, device=gpu)
    wide[:, :12] = qkv.to(gpu)
    ext.norm_rope(wide[:, :8], wide[:, 8:10], *args, wide[:, 12:20], wide[:, 20:22], EPS, pairs)
    assert torch.equal(wide[:, 12:20], want[0]) and torch.equal(wide[:, 20:22], want[1])
    assert torch.equal(wide[:, :12].cpu(), qkv) and (wide[:, 22:] == 0).all()


def test_overlapping_outputs_are_refused(ext, gpu):
    qkv, pos, w, table = _inputs(30, 8, 2, F16, 9)
    fused = torch.zeros(30, 14, 128, dtype=F16, device=gpu)
    args = [x.to(gpu) for x in w] + [table.to(gpu), pos.to(gpu)]
    q, k, out, kout = fused[:, :8], fused[:, 8:10], torch.zeros(30, 8, 128, dtype=F16, device=gpu), torch.zeros(30, 2, 128, dtype=F16, device=gpu)
    for bad in ((fused[:, 1:9], kout), (fused[:, 2:10], kout), (out, fused[:, 7:9]), (out, out[:, 6:]), (fused.view(-1)[:30 * 1024].view(30, 8, 128), kout)):
        with pytest.raises(RuntimeError, match="overlap"):
            ext.norm_rope(q, k, *args, *bad, EPS, False)
    assert (fused == 0).all()


def test_slots_past_two_gigabytes(ext, gpu):
    tokens, pages = 20, (2 ** 32) // (8 * 16 * 256) + 64
    qkv, pos, w, table = _inputs(tokens, 8, 8, F16, 10)
    on = qkv.to(gpu)
    args = [x.to(gpu) for x in w] + [table.to(gpu), pos.to(gpu)]
    pools = [torch.zeros(pages, 8, 16, 128, dtype=F16, device=gpu) for _ in range(2)]
    slots = (torch.arange(tokens, device=gpu, dtype=torch.int32) * 3 + (pages - 60) * 16).to(torch.int32)
    outs = [torch.zeros(tokens, 8, 128, dtype=F16, device=gpu) for _ in range(2)]
    ext.norm_rope(on[:, :8], on[:, 8:16], *args, *outs, EPS, False)
    ext.norm_rope_write_kv(on[:, :8], on[:, 8:16], on[:, 16:], *args, torch.empty_like(outs[0]), *pools, slots, EPS, False)
    at = slots.long()
    assert torch.equal(pools[0][at // 16, :, at % 16], outs[1]) and torch.equal(pools[1][at // 16, :, at % 16], on[:, 16:])
    for pool, x in zip(pools, (outs[1], on[:, 16:])):
        assert pool.float().square().sum() == 0 or torch.count_nonzero(pool) == torch.count_nonzero(x)


def test_streams_and_graph_replays(ext, gpu):
    cases = [_inputs(70, 8, 2, BF16, s) for s in (11, 12)]
    want = [_check(ext, gpu, *c, 8, 2, False) for c in cases]
    ins = [[c[0].to(gpu), c[1].to(gpu), c[2][0].to(gpu), c[2][1].to(gpu), c[3].to(gpu)] for c in cases]
    outs = [[torch.zeros_like(x) for x in w] for w in want]
    call = lambda x, o: ext.norm_rope(x[0][:, :8], x[0][:, 8:10], x[2], x[3], x[4], x[1], *o, EPS, False)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st, x, o in zip(streams, ins, outs):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            call(x, o)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o, w in zip(outs, want) for a, b in zip(o, w))
    held, out = [x.clone() for x in ins[0]], [torch.zeros_like(x) for x in want[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(held, out)
    for i in (0, 1, 0, 1):
        for dst, src in zip(held, ins[i]):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
