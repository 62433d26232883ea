"""paged_prefill_attention where a part would be longer than 192 tiles and large rows are cut finer: against
64 bits, the states that the kernels write against those of the plan, and nothing behind the workspace."""
import math

import numpy as np
import pytest
import torch

from chunk_plan import cut, parts, plan_floats, states, states_at_most, written_states
from prompt_cases import F32, U, assert_within, attention_tolerance
from turn_cases import Cache, run_chunk

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _exact(cache, device):
    """turn.paged_prefill on the GPU, in 64 bits: output, and per element the sizes that the tolerance needs."""
    group = cache.hq // cache.hkv
    q = cache.q.to(device).double()
    out, weight, vmax, spread = (torch.zeros_like(q) for _ in range(4))
    score, most = (torch.zeros(q.shape[:2], dtype=torch.float64, device=device) for _ in range(2))
    for b, (size, n) in enumerate(zip(cache.lens, cache.new)):
        if not n:
            continue
        start = int(cache.offsets[b])
        ids = torch.as_tensor(cache.table[b][:-(-size // cache.page)])
        last = torch.arange(size - n, size, device=device).repeat_interleave(group)
        for h in range(cache.hkv):
            k, v = (pool[ids, h].reshape(-1, 128)[:size].to(device).double() for pool in (cache.k, cache.v))
            kt, kabs = k.T.contiguous(), k.abs().T.contiguous()
            heads = slice(h * group, (h + 1) * group)
            rows = q[start:start + n, heads].reshape(-1, 128)
            got = [[], [], [], [], []]
            for at in range(0, rows.shape[0], 4096):
                x = rows[at:at + 4096]
                hidden = torch.arange(size, device=device) > last[at:at + 4096, None]
                p = torch.softmax((torch.mm(x, kt) / math.sqrt(128)).masked_fill_(hidden, -math.inf), -1)
                p[last[at:at + 4096] < 0] = 0.0  # a token that sees nothing
                got[0].append(torch.mm(p, v))
                got[1].append(torch.mm(p, v.abs()))
                got[3].append(torch.mm(p * p, v * v).sqrt_())
                got[4].append(p.amax(1))
                got[2].append(torch.mm(x.abs(), kabs).masked_fill_(hidden, 0.0).amax(1) / math.sqrt(128))
            at = (slice(start, start + n), heads)
            out[at], weight[at], spread[at] = (torch.cat(got[i]).reshape(n, group, 128) for i in (0, 1, 3))
            vmax[at] = v.abs().max()
            score[at], most[at] = (torch.cat(got[i]).reshape(n, group) for i in (2, 4))
    return [x.cpu().numpy() for x in (out, weight, vmax, score, spread, most)]


def _likely(exact, weight, vmax, score, spread, most, longest, dtype):
    """attention_tolerance with roundings as independent errors of mean 0, whose sum passes 8 times the
    root of the sum of their squared bounds with a probability of less than 2 exp(-32) = 3e-14
    (Hoeffding's inequality): the weights', e_j p_j |v_j| with |e_j| <= u, in the numerator and, where
    sqrt(sum p_j^2) is at most 1, in the denominator; and those of at most longest + 16 additions in 32
    bits, each of a partial sum of at most sum p_j |v_j|.  What fp16 weights below its normal range
    lose, 2^-25 each, counts beside a sum of weights of at least 1 / max p_j, since the largest is 1 or
    more."""
    tiny = longest * 2.0 ** -25 * vmax * most[..., None] if dtype == F16 else 0.0
    rest = attention_tolerance(exact, weight, score, 0, dtype, 0.0, tiny)
    return rest + 8 * U[dtype] * (spread + np.abs(exact)) + 16 * math.sqrt(longest + 16) * F32 * weight


LONG = [([26000], [1000]), ([44800], [1200]), ([30000, 9000, 900], [500, 700, 900]), ([17000] * 4, [300] * 4),
        ([40000, 12000] + [37 * i for i in range(1, 31)], [700, 600] + [1] * 30), ([33] * 40 + [26000, 14000] + [300 + i for i in range(38)], [1] * 40 + [900, 500] + [1, 2] * 19)]


@pytest.mark.parametrize("lens,new", LONG, ids=lambda x: f"{len(x)}x{max(x)}")
@pytest.mark.parametrize("hq,hkv,dtype", [(32, 1, BF16), (32, 1, F16), (48, 3, BF16)])
def test_long_parts(ext, gpu, lens, new, hq, hkv, dtype):
    if hkv > 1:  # as many blocks for fewer heads a group
        new = [n * 2 if n > 2 else n for n in new]
    group, tokens, batch = hq // hkv, sum(new), len(lens)
    units = torch.cuda.get_device_properties(gpu).multi_processor_count
    assert cut(lens, new, group, hkv, units)[0] >= 192 and max(c for c, _ in parts(lens, new, group, hkv, units)) > 1
    cache = Cache(lens, new, hq, hkv, 16, dtype, seed=sum(lens))
    floats = ext.paged_prefill_workspace_floats(batch, tokens, hq, hkv)
    most = states_at_most(tokens, group, units)
    assert floats == plan_floats(batch) + 130 * most
    space = torch.full((floats + 4096,), 7.0, device=gpu)
    space[:floats] = float("nan")
    out = run_chunk(ext, cache, gpu, workspace=space[:floats])
    assert (space[floats:] == 7.0).all()
    # the plan's states, and no other
    want = torch.from_numpy(written_states(lens, new, group, hkv, units)).to(gpu)
    assert len(want) == states(lens, new, group, hkv, units)[0] and len(want) * hkv <= most
    first = plan_floats(batch)
    sums = space[first:first + 128 * most].view(most, 128)
    tops = space[first + 128 * most:floats].view(most, 2)
    for x in (sums, tops):
        written = ~torch.isnan(x)
        assert (written.all(1) == written.any(1)).all()
        assert torch.equal(written[:len(want) * hkv, 0].view(-1, hkv), want[:, None].expand(-1, hkv))
        assert not written[len(want) * hkv:].any()
    assert torch.equal(run_chunk(ext, cache, gpu, workspace=space[:floats]).view(torch.int16), out.view(torch.int16))
    exact, *rest = _exact(cache, gpu)
    assert_within(out, exact, cache.bound(exact, *rest[:3]), f"{batch} rows up to {max(lens)}, {tokens} tokens, {hq} / {hkv}")
    assert_within(out, exact, _likely(exact, *rest, max(lens), dtype), "with independent roundings")


@pytest.mark.parametrize("lens,new", [([0, 5, 700, 64, 3000], [0, 1, 7, 64, 200]), ([900] * 70 + [3000, 1], [3] * 70 + [150, 1])], ids=["5", "72"])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (4, 4), (5, 1)])
def test_states_of_short_parts(ext, gpu, lens, new, hq, hkv):
    """The same of calls whose rows of both classes are cut at a few tiles."""
    group, tokens, batch = hq // hkv, sum(new), len(lens)
    units = torch.cuda.get_device_properties(gpu).multi_processor_count
    cache = Cache(lens, new, hq, hkv, 16, BF16, seed=batch)
    floats, most, first = ext.paged_prefill_workspace_floats(batch, tokens, hq, hkv), states_at_most(tokens, group, units), plan_floats(batch)
    assert floats == first + 130 * most
    space = torch.full((floats,), float("nan"), device=gpu)
    run_chunk(ext, cache, gpu, workspace=space)
    want = written_states(lens, new, group, hkv, units)
    written = ~torch.isnan(space[first:first + 128 * most].view(most, 128)[:, 0]).cpu().numpy()
    assert want.any() and np.array_equal(written, np.concatenate([np.repeat(want, hkv), np.zeros(most - len(want) * hkv, dtype=bool)]))
