"""prefill_attention against causal attention in 64 bits, element by element.

Weights reach the product with V in the activation type (half a step: fp16 2^-11, bf16 2^-8),
and in fp16 a weight below 2^-14 of the running maximum's is subnormal, off by up to 2^-25;
the sum of weights is at least 1 in those units (the largest weight is).
"""
import numpy as np
import pytest
import torch

from oracle import prompt
from prompt_cases import U, assert_within, attention_tolerance, packed_inputs, split_qkv

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _check(ext, gpu, qkv, offsets, hq, hkv, what=""):
    dtype = qkv.dtype
    q, k, v = split_qkv(qkv, hq, hkv)
    out = torch.full(q.shape, 7.0, dtype=dtype, device=gpu)
    ext.prefill_attention(*split_qkv(qkv.to(gpu), hq, hkv), offsets.to(gpu), out)
    torch.cuda.synchronize()
    off = offsets.tolist()
    want, weight, vmax, score = prompt.prefill(q.double(), k.double(), v.double(), off)
    inside = np.zeros(len(want), dtype=bool)
    for s, e in zip(off, off[1:]):
        inside[s:e] = True
    assert (out[~torch.from_numpy(inside)].float() == 7.0).all()  # left as they were
    longest = max([e - s for s, e in zip(off, off[1:])] + [1])
    tiny = longest * 2.0 ** -25 * vmax if dtype == F16 else 0.0
    bound = attention_tolerance(want, weight, score, longest, dtype, U[dtype], tiny)
    sel = torch.from_numpy(inside)
    assert_within(out.cpu()[sel], want[inside], bound[inside], what)
    return out


LENGTHS = [[1], [2], [31], [64], [65], [500], [63, 1, 64, 2, 65, 0, 3], [0, 0], [1] * 70, [130, 257, 5], [1000, 17]]


@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda x: "-".join(map(str, x[:8])))
@pytest.mark.parametrize("hq,hkv,dtype", [(8, 2, F16), (8, 2, BF16), (3, 3, F16)])
def test_lengths(ext, gpu, lengths, hq, hkv, dtype):
    qkv, off = packed_inputs(lengths, hq, hkv, dtype, seed=sum(lengths))
    _check(ext, gpu, qkv, off, hq, hkv, f"{lengths[:8]}")


@pytest.mark.parametrize("hq,hkv", [(1, 1), (2, 1), (3, 1), (5, 1), (8, 1), (10, 2), (16, 1), (31, 1), (32, 1), (12, 4), (9, 9)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_head_layouts(ext, gpu, hq, hkv, dtype):
    lengths = [77, 1, 300]
    qkv, off = packed_inputs(lengths, hq, hkv, dtype, seed=hq * 40 + hkv)
    _check(ext, gpu, qkv, off, hq, hkv, f"Hq {hq} Hkv {hkv}")


@pytest.mark.parametrize("lengths", [[1], [64, 33], [500], [130, 257, 5], [1000, 17]], ids=str)
@pytest.mark.parametrize("hq,hkv,empty,dtype", [(8, 2, 150, F16), (3, 3, 60, BF16), (16, 16, 12, F16), (32, 16, 20, BF16)])
def test_blocks_for_every_cu(ext, gpu, lengths, hq, hkv, empty, dtype):
    """Sequences without tokens count as blocks, so that the launch has more blocks of 128 rows
    than half the CUs and its waves do not share rows' tiles out; with up to 64 sequences and
    with more."""
    qkv, off = packed_inputs([0] * (empty // 2) + lengths + [0] * (empty - empty // 2), hq, hkv, dtype, seed=sum(lengths) + empty)
    _check(ext, gpu, qkv, off, hq, hkv, f"{lengths} and {empty} empty")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_tokens_outside_every_sequence(ext, gpu, dtype):
    """Tokens before the first and behind the last sequence hold NaN: nothing reads them, and
    their output rows stay."""
    qkv, off = packed_inputs([70, 3, 129], 8, 2, dtype, seed=3, lead=300, trail=90)
    qkv[:300] = float("nan")
    qkv[300 + 202:] = float("nan")
    _check(ext, gpu, qkv, off, 8, 2)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hq,hkv,empty", [(8, 2, 0), (2, 2, 0), (16, 1, 0), (8, 2, 90), (2, 2, 90), (16, 1, 190)])
def test_nonfinite_values_reach_later_tokens_only(ext, gpu, dtype, hq, hkv, empty):
    qkv, off = packed_inputs([100, 150, 64] + [0] * empty, hq, hkv, dtype, seed=4)
    k, v = qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    inf, nan = float("inf"), float("nan")
    v[70, 0, 3], v[90, 0, 3], v[40, 0, 127], v[99, hkv - 1, 0] = inf, -inf, nan, nan
    v[100 + 149, 0, 64], v[100, 0, 17] = nan, inf
    k[100 + 130, 0, 5] = nan     # every score of the tokens from 130 on
    v[250 + 63, 0, :] = nan
    _check(ext, gpu, qkv, off, hq, hkv)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_growing_and_peaked_scores(ext, gpu, dtype):
    """Scores that grow along the prompt (the running maximum moves in every tile) and ones so
    far apart that a single token takes all the weight."""
    qkv, off = packed_inputs([400], 4, 1, dtype, seed=6)
    ramp = torch.linspace(0.0, 6.0, 400)[:, None]
    qkv[:, :4] = 1.0
    qkv[:, 4] = ramp.to(dtype)
    _check(ext, gpu, qkv, off, 4, 1, "ramp")
    qkv[:, 4] = -ramp.to(dtype)
    _check(ext, gpu, qkv, off, 4, 1, "falling ramp")
    qkv[:, 4] = 0.0
    qkv[199, 4] = 40.0
    _check(ext, gpu, qkv, off, 4, 1, "one peak")


@pytest.mark.parametrize("empty", [0, 90])
def test_scores_at_the_ends_of_the_range(ext, gpu, empty):
    """bf16 scores around -1e36 in every token (their differences decide), and rows of -inf."""
    qkv, off = packed_inputs([90, 40] + [0] * empty, 2, 1, BF16, seed=11)
    qkv[:, :2] = 0.0
    qkv[:, 2] = 0.0
    qkv[:90, :2, 0] = 2.0 ** 60
    steps = torch.arange(90) % 3
    qkv[:90, 2, 0] = (-(2.0 ** 60) * (1 + steps / 4)).to(BF16)
    out = torch.zeros(130, 2, 128, dtype=BF16, device=gpu)
    ext.prefill_attention(*split_qkv(qkv.to(gpu), 2, 1), off.to(gpu), out)
    v = qkv[:90, 3].double()
    for i in range(90):  # the tokens with the largest score share all the weight
        want = v[:i + 1][steps[:i + 1] == 0].mean(0)
        assert (out[i].cpu().double() - want).abs().max() <= 2.0 ** -7 * want.abs().max() + 1e-4
    qkv[90:, :2, 0] = float("inf")
    qkv[90:, 2, 0] = -1.0
    ext.prefill_attention(*split_qkv(qkv.to(gpu), 2, 1), off.to(gpu), out)
    assert torch.isnan(out[90:]).all() and torch.isfinite(out[:90]).all()


@pytest.mark.parametrize("empty", [0, 90])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_large_scores(ext, gpu, dtype, sign, empty):
    """Scores that are exact in 32 bits, about 2^32 (fp16) and 2^100 (bf16), and no powers of two:
    their scaled value is rounded by tens of units and more, and the weights must not show it.
    The tokens with the largest score share all the weight, 1 each, so that only the mean's own
    arithmetic and the output's rounding are left."""
    qkv, off = packed_inputs([90, 40] + [0] * empty, 2, 1, dtype, seed=13)
    qkv[:, :3] = 0.0
    steps = torch.arange(130) % 3
    if dtype == F16:  # four products of 22 bits
        qkv[:, :2, :4] = 16.0 * 2047
        qkv[:, 2, :4] = (sign * 16.0 * ((2039 if sign > 0 else 2037) - sign * steps))[:, None].to(dtype)
    else:
        qkv[:, :2, 0] = 255.0 * 2.0 ** 42
        qkv[:, 2, 0] = (sign * 2.0 ** 42 * (249 - sign * steps)).to(dtype)
    out = torch.zeros(130, 2, 128, dtype=dtype, device=gpu)
    ext.prefill_attention(*split_qkv(qkv.to(gpu), 2, 1), off.to(gpu), out)
    for first, last in ((0, 90), (90, 130)):
        v, s = qkv[first:last, 3].double(), steps[first:last]
        for i in range(last - first):
            tied = s[:i + 1] == s[:i + 1].min()
            want, most = v[:i + 1][tied].mean(0), v[:i + 1][tied].abs().max()
            bound = U[dtype] * want.abs() + 200 * 2.0 ** -24 * most + 2.0 ** -25
            assert ((out[first + i].cpu().double() - want).abs() <= bound).all(), (first, i)


@pytest.mark.parametrize("empty", [0, 90])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hidden", [31, 32, 40, 64, 70])
def test_keys_of_minus_infinity(ext, gpu, dtype, hidden, empty):
    """Keys whose scores are -inf have no weight: a row that sees none but such is NaN, and the
    later ones are as if the sequence began behind them, whole tiles of them or not."""
    qkv, off = packed_inputs([200] + [0] * empty, 4, 2, dtype, seed=hidden)
    qkv[:, :4, 0] = 1.0
    qkv[:hidden, 4:6, 0] = -float("inf")
    out = torch.zeros(200, 4, 128, dtype=dtype, device=gpu)
    ext.prefill_attention(*split_qkv(qkv.to(gpu), 4, 2), off.to(gpu), out)
    assert torch.isnan(out[:hidden]).all()
    q, k, v = (x[hidden:].double() for x in split_qkv(qkv, 4, 2))
    want, weight, vmax, score = prompt.prefill(q, k, v, [0, 200 - hidden])
    tiny = 200 * 2.0 ** -25 * vmax if dtype == F16 else 0.0
    assert_within(out[hidden:], want, attention_tolerance(want, weight, score, 200, dtype, U[dtype], tiny), f"behind {hidden}")


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 3)])
@pytest.mark.parametrize("nats", [10.0, 10.4, 11.0])
def test_many_weights_below_the_normal_range(ext, gpu, hq, hkv, nats):
    """One key ahead of 4999 equal ones by so much that their fp16 weights, 2^-14.4 to 2^-15.9, are
    subnormal, and 0.08 to 0.23 of the sum together; V of one sign.  With rows' tiles shared out
    over two pairs of waves (one KV head) and not."""
    qkv, off = packed_inputs([5000], hq, hkv, F16, seed=14)
    qkv[:, :hq] = 1.0
    qkv[:, hq:hq + hkv] = 0.0
    qkv[0, hq:hq + hkv] = nats * 128 ** 0.5 / 128
    qkv[:, hq + hkv:] = 1.0 + qkv[:, hq + hkv:].abs()
    _check(ext, gpu, qkv, off, hq, hkv, f"{nats} nats ahead")


def test_token_strides_at_their_limit(ext, gpu):
    """2^23 elements between the tokens of K: 300 of them pass 2^32 bytes."""
    qkv, off = packed_inputs([10, 290], 4, 2, F16, seed=12)
    q, k, v = (x.contiguous().to(gpu) for x in split_qkv(qkv, 4, 2))
    far = torch.empty(299 * 2 ** 23 + 256, dtype=F16, device=gpu).as_strided((300, 2, 128), (2 ** 23, 128, 1))
    far.copy_(k)
    a, b = torch.empty_like(q), torch.empty_like(q)
    ext.prefill_attention(q, k, v, off.to(gpu), a)
    ext.prefill_attention(q, far, v, off.to(gpu), b)
    assert torch.equal(a, b)
    far.copy_(v)
    ext.prefill_attention(q, k, far, off.to(gpu), b)
    assert torch.equal(a, b)


def test_contiguous_and_offset_inputs(ext, gpu):
    qkv, off = packed_inputs([150, 33], 8, 2, F16, seed=8)
    ref = _check(ext, gpu, qkv, off, 8, 2)
    q, k, v = (x.contiguous().to(gpu) for x in split_qkv(qkv, 8, 2))
    out = torch.empty_like(q)
    ext.prefill_attention(q, k, v, off.to(gpu), out)
    assert torch.equal(out, ref)
    ext.prefill_attention(q, k, v, off.to(gpu), q)  # in place: a row is read before it is written
    assert torch.equal(q, ref)


def test_outputs_over_and_beside_the_inputs(ext, gpu):
    """A fused projection whose rows lie apart may not be written over, but for one token; memory
    that ends where an input begins, and lies between an input's rows, may be."""
    qkv, off = packed_inputs([40, 25], 8, 2, F16, seed=15)
    ref = _check(ext, gpu, qkv, off, 8, 2)
    fused = qkv.to(gpu)
    parts = split_qkv(fused, 8, 2)
    over = fused.view(-1)[:65 * 8 * 128].view(65, 8, 128)
    for out, message in ((over, "must not be k or v"), (fused.view(-1)[128:65 * 8 * 128 + 128].view(65, 8, 128), "must not be k or v")):
        with pytest.raises(RuntimeError, match=message):
            ext.prefill_attention(*parts, off.to(gpu), out)
    with pytest.raises(RuntimeError, match="not overlap q"):
        ext.prefill_attention(parts[0], *(x.contiguous() for x in parts[1:]), off.to(gpu), over)
    assert torch.equal(fused.cpu(), qkv)
    one, one_off = packed_inputs([1], 8, 2, F16, seed=16)
    want = _check(ext, gpu, one, one_off, 8, 2)
    fused = one.to(gpu)
    q, k, v = split_qkv(fused, 8, 2)
    ext.prefill_attention(q, k, v, one_off.to(gpu), q)
    assert torch.equal(fused[:, :8], want) and torch.equal(fused[:, 8:].cpu(), one[:, 8:])
    wide = torch.zeros(2 * 65 * 12 * 128, dtype=F16, device=gpu)  # the inputs, and the output right behind them
    wide[:65 * 12 * 128].view(65, 12, 128).copy_(qkv)
    out = wide[65 * 12 * 128:][:65 * 8 * 128].view(65, 8, 128)
    ext.prefill_attention(*split_qkv(wide[:65 * 12 * 128].view(65, 12, 128), 8, 2), off.to(gpu), out)
    assert torch.equal(out, ref)
    apart = torch.zeros(65, 12 + 65 * 8, 128, dtype=F16, device=gpu)  # and between the first two rows
    apart[:, :12].copy_(qkv)
    out = apart[0, 12:]
    ext.prefill_attention(*split_qkv(apart[:, :12], 8, 2), off.to(gpu), out.view(65, 8, 128))
    assert torch.equal(out.view(65, 8, 128), ref)


def test_thousands_of_sequences(ext, gpu):
    """More sequences than two rounds of the search for a block's tell apart (63^2)."""
    lengths = [(7 * i) % 3 for i in range(4100)] + [200, 1]
    qkv, off = packed_inputs(lengths, 4, 2, F16, seed=21)
    _check(ext, gpu, qkv, off, 4, 2)


def test_bad_offsets_stay_inside(ext, gpu):
    """Offsets past the tokens, or negative, count as clamped."""
    qkv, _ = packed_inputs([200], 4, 2, F16, seed=9)
    a = torch.full((200, 4, 128), 7.0, dtype=F16, device=gpu)
    b = a.clone()
    parts = split_qkv(qkv.to(gpu), 4, 2)
    ext.prefill_attention(*parts, torch.tensor([-5, 60, 900], dtype=torch.int32, device=gpu), a)
    ext.prefill_attention(*parts, torch.tensor([0, 60, 200], dtype=torch.int32, device=gpu), b)
    assert torch.equal(a, b)


def test_streams_and_graph_replays(ext, gpu):
    cases = [packed_inputs(l, 8, 2, F16, seed=s) for s, l in ((1, [300, 41]), (2, [129, 212]))]
    refs = [_check(ext, gpu, *c, 8, 2) for c in cases]
    outs = [torch.zeros_like(r) for r in refs]
    ins = [(c[0].to(gpu), c[1].to(gpu)) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for st, (qkv, off), out in zip(streams, ins, outs):
            with torch.cuda.stream(st):
                ext.prefill_attention(*split_qkv(qkv, 8, 2), off, out)
    torch.cuda.synchronize()
    assert all(torch.equal(o, r) for o, r in zip(outs, refs))
    qkv, off = ins[0][0].clone(), ins[0][1].clone()
    out = torch.zeros_like(refs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ext.prefill_attention(*split_qkv(qkv, 8, 2), off, out)
    for i in (0, 1, 0, 1):  # the captured call follows its inputs, the lengths among them
        qkv.copy_(ins[i][0])
        off.copy_(ins[i][1])
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, refs[i])
