"""The operators together, as a serving loop runs them: prompts into the cache of two layers, rows
forked, a second turn over the shared prefixes, rows freed, the pool compacted, new prompts in the
rows that came free, decode steps; every attention against 64 bits over each row's own history."""
import numpy as np
import pytest
import torch

from oracle import turn
from prompt_cases import U, assert_within, attention_tolerance
from turn_cases import angles, i32, rope_tolerance

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
HQ, HKV, PS, COLUMNS, ROWS, PAGES, LAYERS, EPS = 8, 2, 16, 24, 7, 70, 2, 1e-6


class Loop:
    def __init__(self, ext, gpu, dtype, seed):
        gen = self.gen = torch.Generator().manual_seed(seed)
        self.ext, self.gpu, self.dtype = ext, gpu, dtype
        self.pools = [[torch.full((PAGES, HKV, PS, 128), float("nan"), dtype=dtype, device=gpu) for _ in range(2)] for _ in range(LAYERS)]
        self.table = torch.full((ROWS, COLUMNS), -1, dtype=torch.int32, device=gpu)
        self.free = torch.randperm(PAGES, generator=gen).to(torch.int32).to(gpu)
        self.num, self.left = i32([PAGES], gpu), i32([0], gpu)
        self.shares = torch.zeros(PAGES, dtype=torch.int32, device=gpu)
        self.lens = i32([0] * ROWS, gpu)
        self.weights = [1 + 0.2 * torch.randn(128, generator=gen) for _ in range(2)]
        self.angles = angles(400, 128)
        self.space = torch.empty(ext.page_workspace_ints(PAGES), dtype=torch.int32, device=gpu)
        self.history = [[[[], []] for _ in range(ROWS)] for _ in range(LAYERS)]  # K and V as stored

    def took(self):
        self.num, self.left = self.left, self.num

    def tokens(self, new):
        """`new` more tokens of every row, through both layers."""
        ext, gpu, dtype = self.ext, self.gpu, self.dtype
        total = sum(new)
        cached = self.lens.clone()
        self.lens += i32(new, gpu)
        offsets, slots = i32([0] * (ROWS + 1), gpu), i32([0] * total, gpu)
        ext.build_block_tables(cached, self.lens, self.free, self.num, self.table, offsets, slots, self.left, PS)
        self.took()
        assert self.num.item() >= 0
        pos = torch.cat([torch.arange(c, c + n) for c, n in zip(cached.tolist(), new)]).to(torch.int32)
        ws = torch.full((ext.paged_prefill_workspace_floats(ROWS, total, HQ, HKV),), float("nan"), device=gpu)
        for layer, (k_pages, v_pages) in enumerate(self.pools):
            qkv = torch.randn(total, HQ + 2 * HKV, 128, generator=self.gen).to(dtype)
            on = qkv.to(gpu)
            q, out = torch.empty(total, HQ, 128, dtype=dtype, device=gpu), torch.empty(total, HQ, 128, dtype=dtype, device=gpu)
            ext.norm_rope_write_kv(on[:, :HQ], on[:, HQ:HQ + HKV], on[:, HQ + HKV:], *(w.to(gpu) for w in self.weights), self.angles.to(gpu),
                                   pos.to(gpu), q, k_pages, v_pages, slots, EPS, False)
            ext.paged_prefill_attention(q, k_pages, v_pages, self.table, self.lens, offsets, out, ws, PS)
            # what went into the cache, and q, follow the formula
            at = slots.long()
            stored = [p[at // PS, :, at % PS].cpu() for p in (k_pages, v_pages)]
            for got, x, w in ((q, qkv[:, :HQ], self.weights[0]), (stored[0], qkv[:, HQ:HQ + HKV], self.weights[1])):
                want, size = turn.norm_rope(x.double().numpy(), w.double().numpy(), self.angles.double().numpy(), pos.tolist(), EPS, False)
                assert_within(got, want, rope_tolerance(want, size, dtype), "norm and rotation")
            assert torch.equal(stored[1], qkv[:, HQ + HKV:])
            start = 0
            for row, n in enumerate(new):
                for i in range(2):
                    self.history[layer][row][i].append(stored[i][start:start + n])
                if n:
                    self.check(layer, row, q[start:start + n], out[start:start + n])
                start += n
        return out

    def check(self, layer, row, q, out):
        k, v = (torch.cat(x).double().numpy()[None].transpose(0, 2, 1, 3) for x in self.history[layer][row])
        n = k.shape[2]
        want, weight, vmax, score = turn.paged_prefill(q.double().cpu().numpy(), k, v, np.zeros((1, 1), dtype=int), [n], [0, len(q)])
        tiny = n * 2.0 ** -25 * vmax if self.dtype == F16 else 0.0
        assert_within(out, want, attention_tolerance(want, weight, score, n, self.dtype, U[self.dtype], tiny), f"layer {layer} row {row}")

    def fork(self, parents, children):
        n = len(parents)
        src, dst = i32([0] * n, self.gpu), i32([0] * n, self.gpu)
        p, c = i32(parents, self.gpu), i32(children, self.gpu)
        self.ext.fork_rows(p, c, self.lens, self.table, self.shares, self.free, self.num, self.left, src, dst, PS)
        self.took()
        for k_pages, v_pages in self.pools:
            self.ext.copy_pages(src, dst, k_pages, v_pages)
        self.lens[c.long()] = self.lens[p.long()]
        for layer in self.history:
            for a, b in zip(parents, children):
                layer[b] = [list(x) for x in layer[a]]

    def release(self, rows):
        r = i32(rows, self.gpu)
        self.ext.free_rows(r, self.lens, self.table, self.shares, self.free, self.num, self.left, self.space, PS)
        self.took()
        self.lens[r.long()] = 0
        for layer in self.history:
            for row in rows:
                layer[row] = [[], []]

    def compact(self):
        gpu = self.gpu
        out = [torch.zeros_like(x) for x in (self.shares, self.table, self.shares, self.free)]
        src, dst = i32([0] * (PAGES // 2), gpu), i32([0] * (PAGES // 2), gpu)
        self.ext.compact_pages(self.table, self.shares, self.free, self.num, out[0], out[1], out[2], out[3], self.left, src, dst, self.space)
        for k_pages, v_pages in self.pools:
            self.ext.copy_pages(src, dst, k_pages, v_pages)
        self.table, self.shares, self.free = out[1:]
        self.took()
        used = PAGES - self.num.item()
        for k_pages, v_pages in self.pools:  # the rest could be given back
            k_pages[used:], v_pages[used:] = float("nan"), float("nan")

    def pages_add_up(self):
        lens, table = self.lens.tolist(), self.table.tolist()
        held = [p for row, n in zip(table, lens) for p in row[:-(-n // PS)]]
        free = self.free[:self.num.item()].tolist()
        assert sorted(set(held) | set(free)) == list(range(PAGES)) and not set(held) & set(free) and len(free) == len(set(free))
        assert self.shares.tolist() == [max(held.count(p) - 1, 0) for p in range(PAGES)]


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_conversation(ext, gpu, dtype):
    loop = Loop(ext, gpu, dtype, seed=3)
    loop.tokens([130, 45, 0, 0, 0, 0, 0])              # two prompts
    loop.pages_add_up()
    loop.fork([0, 0, 1], [2, 3, 4])                    # three more rows continue them
    loop.pages_add_up()
    loop.tokens([1, 37, 60, 1, 5, 0, 0])               # second turns and single tokens, of different lengths
    loop.fork([2, 4], [5, 6])                          # a fork of a fork
    loop.tokens([0, 1, 17, 1, 1, 90, 3])
    loop.pages_add_up()
    loop.release([0, 4])                               # their prefixes are held by others
    loop.pages_add_up()
    loop.compact()
    loop.pages_add_up()
    loop.tokens([33, 1, 1, 1, 0, 1, 20])               # a new prompt in a row that came free
    for _ in range(3):                                 # decode steps
        loop.tokens([1, 1, 1, 1, 0, 1, 1])
    loop.release([1, 2, 3, 5, 6, 0, 0])
    loop.pages_add_up()
    assert loop.num.item() == PAGES and not loop.shares.any()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_captured_step_over_forked_rows(ext, gpu, dtype):
    """Norm, rotation, write and attention of five tokens a row in one graph, replayed with new
    tokens and lengths, next to the same calls made one by one."""
    loop = Loop(ext, gpu, dtype, seed=4)
    loop.tokens([100, 31, 0, 0, 0, 0, 0])
    loop.fork([0, 1], [2, 3])
    total, step = 20, 5
    state = dict(cached=loop.lens.clone(), lens=loop.lens.clone(), num=loop.num.clone(), left=i32([0], gpu), table=loop.table.clone(),
                 pos=i32([0] * total, gpu), qkv=torch.zeros(total, HQ + 2 * HKV, 128, dtype=dtype, device=gpu),
                 q=torch.zeros(total, HQ, 128, dtype=dtype, device=gpu), out=torch.zeros(total, HQ, 128, dtype=dtype, device=gpu),
                 offsets=i32([0] * (ROWS + 1), gpu), slots=i32([0] * total, gpu), k=loop.pools[0][0].clone(), v=loop.pools[0][1].clone(),
                 ws=torch.empty(ext.paged_prefill_workspace_floats(ROWS, total, HQ, HKV), device=gpu))
    weights, table = [w.to(gpu) for w in loop.weights], loop.angles.to(gpu)
    grow = i32([step] * 4 + [0] * 3, gpu)

    def run(s):
        s["lens"].copy_(s["cached"]).add_(grow)
        ext.build_block_tables(s["cached"], s["lens"], loop.free, s["num"], s["table"], s["offsets"], s["slots"], s["left"], PS)
        s["pos"].copy_((s["cached"][:4, None] + torch.arange(step, device=gpu, dtype=torch.int32)).reshape(-1))
        x = s["qkv"]
        ext.norm_rope_write_kv(x[:, :HQ], x[:, HQ:HQ + HKV], x[:, HQ + HKV:], *weights, table, s["pos"], s["q"], s["k"], s["v"], s["slots"], EPS, True)
        ext.paged_prefill_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["offsets"], s["out"], s["ws"], PS)
        s["num"].copy_(s["left"])
        s["cached"].copy_(s["lens"])

    eager, captured = ({k: v.clone() for k, v in state.items()} for _ in range(2))
    warm = {k: v.clone() for k, v in state.items()}
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(warm)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(captured)
    for i in range(12):
        new = torch.randn(total, HQ + 2 * HKV, 128, generator=loop.gen).to(dtype)
        for s in (eager, captured):
            s["qkv"].copy_(new)
        run(eager)
        graph.replay()
        torch.cuda.synchronize()
        for name in ("out", "q", "table", "num", "lens"):
            assert torch.equal(captured[name], eager[name]), (i, name)
        assert torch.isfinite(eager["out"]).all()
    bits = lambda x: x.view(torch.int16)
    assert torch.equal(bits(captured["k"]), bits(eager["k"])) and torch.equal(bits(captured["v"]), bits(eager["v"]))
