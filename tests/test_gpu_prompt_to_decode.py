"""The operators as a serving loop runs them: prompts admitted (pages and slots, attention over
the prompts, K/V into the cache), then decode steps (a page or slot each, the newest token
written, attention over the cache), over a 2-byte cache and a block-scaled fp8 cache."""
import numpy as np
import pytest
import torch

from oracle import prompt
from prompt_cases import U, assert_within, attention_tolerance

pytestmark = pytest.mark.gpu
F16, BF16, F8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("block_scaled", [False, True])
def test_prompts_then_decode_steps(ext, gpu, dtype, block_scaled):
    hq, hkv, ps, columns = 8, 2, 16, 12
    lengths = [33, 1, 150, 16]
    rows, pages = len(lengths), 40
    gen = torch.Generator().manual_seed(7)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    shape = (pages, hkv, ps, 128)
    pools = [torch.zeros(shape, dtype=dtype, device=gpu) for _ in range(2)]
    if block_scaled:
        pools = [x.to(F8) for x in pools]
    scales = torch.ones(pages, hkv, 2, device=gpu)
    table = torch.full((rows, columns), -1, dtype=torch.int32, device=gpu)
    free = torch.randperm(pages, generator=gen).to(torch.int32).to(gpu)
    counts = [i32([pages]), i32([0])]  # the number of free pages, in turn
    workspace = torch.empty(max(ext.fp8_block_workspace_floats(rows, hq, hkv),
                                ext.workspace_floats(rows, hq, 2)), device=gpu)
    cached, lens = i32([0] * rows), i32(lengths)
    keys, values = [[] for _ in lengths], [[] for _ in lengths]

    for step in range(20):  # the prompts, then 19 tokens each: every row crosses a page
        new = lengths if step == 0 else [1] * rows
        tokens = sum(new)
        qkv = (torch.randn(tokens, hq + 2 * hkv, 128, generator=gen) * (1 + step)).to(dtype)
        q, k, v = (x.to(gpu) for x in (qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]))
        q = q.contiguous()
        at = 0
        for b, n in enumerate(new):
            keys[b].append(qkv[at:at + n, hq:hq + hkv])
            values[b].append(qkv[at:at + n, hq + hkv:])
            at += n
        offsets, slots = i32([0] * (rows + 1)), i32([0] * tokens)
        ext.build_block_tables(cached, lens, free, counts[0], table, offsets, slots, counts[1], ps)
        counts.reverse()
        out = torch.empty_like(q)
        if step == 0:
            ext.prefill_attention(q, k, v, offsets, out)
        if block_scaled:
            ext.write_kv_fp8_block(k, v, *pools, scales, slots)
        else:
            ext.write_kv(k, v, *pools, slots)
        if step == 0:
            want, weight, vmax, score = prompt.prefill(*(x.double().cpu() for x in (q, k, v)), offsets.tolist())
            tiny = 150 * 2.0 ** -25 * vmax if dtype == F16 else 0.0
            assert_within(out, want, attention_tolerance(want, weight, score, 150, dtype, U[dtype], tiny), "prompts")
        elif block_scaled:
            ext.paged_attention_fp8_block(q, *pools, scales, table, lens, out, workspace, ps)
            # Every value in the cache lies within half an e4m3 step of its token's, under the
            # largest scale its page has had (each growth rounds subnormals once more: at most
            # 20 halves of 2^-9 of the scale in all).
            got = [torch.stack([p.cpu().float() * scales[:, :, i, None, None].cpu() for i, p in enumerate(pools)])]
            held = [keys, values]
            for b in range(rows):
                n = int(lens[b])
                ids = table[b, :-(-n // ps)].long().cpu()
                for i in range(2):
                    x = got[0][i][ids].permute(0, 2, 1, 3).reshape(-1, hkv, 128)[:n]
                    y = torch.cat(held[i][b]).float()
                    s = scales[ids, :, i].cpu().repeat_interleave(ps, 0)[:n, :, None]
                    assert ((x - y).abs() <= y.abs() * 2.0 ** -4 + 20 * s * 2.0 ** -10).all()
            want, weight, score, lead = prompt.fp8_block_decode(
                q.double().cpu(), *(p.double().cpu() for p in pools), scales.double().cpu(), table.cpu().numpy(), lens.tolist())
            tiny = 170 * 2.0 ** -25 * 448 * lead[..., None] if dtype == F16 else 0.0
            p_step = 2.0 ** -11 if dtype == F16 else 2.0 ** -16
            assert_within(out, want, attention_tolerance(want, weight, score, 170, dtype, p_step, tiny), f"step {step}")
        else:
            q0 = (q.float() / (1 + step) ** 2).to(dtype)  # scores of a usual size
            ext.paged_attention_masked(q0, *pools, table, lens, out, workspace, 170, ps, 2)
            for b in range(rows):
                kb, vb = (torch.cat(x[b]).double().transpose(0, 1) for x in (keys, values))
                x = torch.einsum("hgd,hnd->hgn", q0[b].double().cpu().view(hkv, -1, 128), kb) / 128 ** 0.5
                ref = torch.einsum("hgn,hnd->hgd", torch.softmax(x, -1), vb).reshape(hq, 128)
                # The decode ops' gate, 2e-3 beyond the output's rounding for values ~ N(0, 1),
                # grows with V's magnitude.
                diff = (out[b].double().cpu() - ref).abs()
                assert (diff <= U[dtype] * ref.abs() + 2e-3 * (1 + step)).all()
        cached = lens
        lens = lens + 1
    used = sum(-(-(n + 19) // ps) for n in lengths)
    assert counts[0].item() == pages - used
    ids = torch.cat([table[b, :-(-(n + 19) // ps)] for b, n in enumerate(lengths)])
    assert len(set(ids.tolist())) == used  # no page twice


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_captured_decode_step(ext, gpu, dtype):
    """One captured graph of a whole step (pages and slots, the write, attention, lengths one
    further), replayed 40 times with new tokens: as the same calls made one by one."""
    hq, hkv, ps, columns, lengths, pages = 8, 2, 16, 12, [33, 1, 127, 16], 40
    rows, gen = len(lengths), torch.Generator().manual_seed(17)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    free = torch.randperm(pages, generator=gen).to(torch.int32).to(gpu)
    prompts = [torch.randn(sum(lengths), hkv, 128, generator=gen).to(dtype).to(gpu) for _ in range(2)]

    class Loop:
        def __init__(self):
            self.pools = [torch.zeros(pages, hkv, ps, 128, device=gpu).to(F8) for _ in range(2)]
            self.scales = torch.ones(pages, hkv, 2, device=gpu)
            self.table = torch.full((rows, columns), -1, dtype=torch.int32, device=gpu)
            self.cached, self.lens, self.num_free, self.left = i32([0] * rows), i32(lengths), i32([pages]), i32([0])
            self.offsets = i32([0] * (rows + 1))
            self.qkv = torch.zeros(rows, hq + 2 * hkv, 128, dtype=dtype, device=gpu)
            self.out = torch.zeros(rows, hq, 128, dtype=dtype, device=gpu)
            self.workspace = torch.empty(ext.fp8_block_workspace_floats(rows, hq, hkv), device=gpu)
            self.admit(*prompts)

        def admit(self, k, v):
            slots = i32([0] * k.shape[0])
            ext.build_block_tables(self.cached, self.lens, free, self.num_free, self.table, self.offsets, slots, self.left, ps)
            ext.write_kv_fp8_block(k, v, *self.pools, self.scales, slots)
            self.slots = i32([0] * rows)
            self.further()

        def further(self):
            self.num_free.copy_(self.left)
            self.cached.copy_(self.lens)
            self.lens.add_(1)

        def step(self):
            ext.build_block_tables(self.cached, self.lens, free, self.num_free, self.table, self.offsets, self.slots, self.left, ps)
            ext.write_kv_fp8_block(self.qkv[:, hq:hq + hkv], self.qkv[:, hq + hkv:], *self.pools, self.scales, self.slots)
            ext.paged_attention_fp8_block(self.qkv[:, :hq].contiguous(), *self.pools, self.scales, self.table, self.lens,
                                          self.out, self.workspace, ps)
            self.further()

    eager, captured = Loop(), Loop()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # records, and runs nothing
        captured.step()
    for n in range(40):
        new = torch.randn(rows, hq + 2 * hkv, 128, generator=gen).to(dtype) * (1 + n % 7)
        for x in (eager, captured):
            x.qkv.copy_(new)
        eager.step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured.out, eager.out) and torch.isfinite(eager.out).all(), n
        assert torch.equal(captured.table, eager.table) and torch.equal(captured.num_free, eager.num_free)
        assert torch.equal(captured.scales, eager.scales)
    assert captured.num_free.item() == pages - sum(-(-(n + 40) // ps) for n in lengths)
