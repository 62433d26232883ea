"""The calls that take a serving program through a second turn over rows that it has cached, with
their inputs, plain forms, results in 64 bits and necessary work.

  op "rope"     norms of q and k for each head and the rotation by position, in one pass; with
                ``write`` K and V go straight into the page pools by slot
  op "fork"     rows that continue another row's tokens: full pages shared, the part-filled last
                page copied (the metadata, and one layer's pools)
  op "free"     finished rows' pages back to the list of free ones, those still shared kept
  op "compact"  pages moved to the front of the pool: new ids, tables and list, and one layer's copies
  op "chunk"    attention of each row's newest tokens over its pages, causal from the row's end

Every case draws its rows' lengths from [lo, hi] with ``trace`` as the seed: "equal" (all hi),
"uniform", "bimodal" (every fourth row from the upper half of the range, the others below
hi / 32) or "zipf" (s = 1.1).
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

D = 128
EPS = 1e-6
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}


# ---------------------------------------------------------------------------------
# Cases.
# ---------------------------------------------------------------------------------
def _case(name, op, dtype, hq, hkv, page, family, rows, lo, hi, trace=20260624, **more):
    return {"name": name, "op": op, "dtype": dtype, "hq": hq, "hkv": hkv, "page": page,
            "family": family, "rows": rows, "lo": lo, "hi": hi, "trace": trace, **more}


def _rope(name, dtype, hq, hkv, page, family, rows, lo, hi, **more):
    """``step``: one token a row, at its end; else all of a row's.  ``rot``: dims that turn, in
    halves or in neighbouring ``pairs``.  ``norm``: both are normed, or only rotated."""
    return _case(name, "rope", dtype, hq, hkv, page, family, rows, lo, hi,
                 **{"step": False, "write": True, "rot": 128, "pairs": False, "norm": True, **more})


def listed():
    return [
        # The newest token of every row of a decode step, its K and V into the tail pages.
        _rope("rope_step", "bf16", 32, 8, 16, "zipf", 64, 128, 16384, step=True),
        # A batch of prompts on their way into the cache.
        _rope("rope_prompts", "bf16", 32, 8, 16, "bimodal", 8, 256, 32768),
        # Rotation alone of half the dims in neighbouring pairs, no K/V sharing, K kept packed.
        _rope("rope_pairs", "fp16", 32, 32, 16, "uniform", 16, 16, 1024, write=False, rot=64, pairs=True, norm=False),
        # Eight beams, each continued by another row.
        _case("fork_beams", "fork", "fp16", 32, 8, 16, "equal", 8, 1000, 1000, ways=1),
        # Four long prompts, sixteen samples of each, over an 8-bit cache with larger pages.
        _case("fork_samples", "fork", "fp8", 32, 8, 64, "uniform", 4, 16384, 65536, ways=16),
        # The rows that finish in one step of a batch.
        _case("free_step", "free", "fp16", 32, 8, 16, "zipf", 64, 128, 65536, gone=3, prefix=0),
        # A large batch abandoned but for a few rows, all of them behind a common prefix of 2000 tokens.
        _case("free_batch", "free", "fp16", 32, 8, 16, "uniform", 96, 4096, 65536, gone=90, prefix=2000),
        # A small pool, half empty.
        _case("compact_small", "compact", "bf16", 32, 8, 16, "uniform", 8, 16, 2048, fill=50),
        # A pool of 1 GB a layer, of whose pages less than half are in use.
        _case("compact_pool", "compact", "bf16", 32, 8, 16, "bimodal", 32, 256, 32768, fill=45),
        # Four guessed tokens of one row checked at once: the smallest call.
        _case("chunk_guesses", "chunk", "fp16", 32, 8, 16, "equal", 1, 2011, 2011, new=5, every=1),
        # A step of a server that mixes decoding rows with pieces of long prompts.
        _case("chunk_mixed", "chunk", "bf16", 32, 8, 16, "uniform", 32, 512, 8192, new=512, every=8),
        # The second turn of one long conversation.
        _case("chunk_turn", "chunk", "bf16", 32, 8, 16, "equal", 1, 32768, 32768, new=2048, every=1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["rope", "rope", "fork", "free", "compact", "chunk", "chunk", "chunk"])
    dtype = rng.choice(["fp16", "bf16"])
    hkv = rng.choice([1, 2, 4, 5, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 5, 8])
    page = rng.choice([8, 16, 24, 32, 64, 128])
    family = rng.choice(["equal", "uniform", "bimodal", "zipf"])
    trace = rng.randrange(1 << 30)
    if op == "rope":
        return _rope("", dtype, hq, hkv, page, family, _log_int(rng, 1, 200), 1, _log_int(rng, 64, 32768), trace=trace,
                     step=rng.random() < 0.4, write=rng.random() < 0.6, rot=rng.choice([16, 32, 64, 96, 128, 128]),
                     pairs=rng.random() < 0.3, norm=rng.random() < 0.7)
    if op == "fork":
        return _case("", op, rng.choice(["fp16", "bf16", "fp8"]), hq, hkv, page, family, _log_int(rng, 1, 64), 1,
                     _log_int(rng, 64, 65536), trace, ways=_log_int(rng, 1, 64))
    if op == "free":
        rows = _log_int(rng, 1, 200)
        return _case("", op, dtype, hq, hkv, page, family, rows, 1, _log_int(rng, 64, 65536), trace,
                     gone=_log_int(rng, 1, rows), prefix=rng.choice([0, 0, 100, 3000]))
    if op == "compact":
        return _case("", op, rng.choice(["fp16", "bf16", "fp8"]), hq, hkv, page, family, _log_int(rng, 1, 100), 1,
                     _log_int(rng, 64, 65536), trace, fill=rng.randint(15, 95))
    return _case("", op, dtype, hq, hkv, page, family, _log_int(rng, 1, 64), 1, _log_int(rng, 100, 32768), trace,
                 new=_log_int(rng, 1, 2048), every=rng.choice([1, 1, 2, 8]))


def _plain_values(case):
    """About how many values the plain form's largest array holds."""
    lengths = lengths_of(case)
    if case["op"] == "chunk":
        return case["rows"] * max(lengths) * (case["hq"] * max(new_of(case)) + case["hkv"] * D)
    if case["op"] == "rope":
        pool = _pool_pages(case) * case["hkv"] * case["page"] * D
        return max(sum(new_of(case)) * (case["hq"] + 2 * case["hkv"]) * D, pool)
    return _pool_pages(case) * case["hkv"] * case["page"] * D


def draw(rng):
    """One more case of the listed ones' ranges, that costs no more than the largest of its op."""
    while True:
        case = _draw(rng)
        del case["name"]
        alike = [c for c in listed() if c["op"] == case["op"]]
        w, most = work(case), [work(c) for c in alike]
        if all(w[k] <= max(m[k] for m in most) for k in w) and \
                _plain_values(case) <= max(map(_plain_values, alike)):
            return case


def lengths_of(case):
    """Each row's tokens."""
    rng = random.Random(case["trace"])
    lo, hi, n = case["lo"], case["hi"], case["rows"]
    if case["family"] == "equal":
        return [hi] * n
    if case["family"] == "uniform":
        return [rng.randint(lo, hi) for _ in range(n)]
    if case["family"] == "bimodal":
        return [rng.randint(hi // 2, hi) if i % 4 == 0 else rng.randint(lo, max(lo, hi // 32))
                for i in range(n)]
    # P(L) proportional to L^-1.1 on [lo, hi], by inversion
    a, b = lo ** -0.1, hi ** -0.1
    return [min(hi, max(lo, int((a + rng.random() * (b - a)) ** -10.0))) for _ in range(n)]


def new_of(case):
    """How many of each row's tokens are new."""
    lengths = lengths_of(case)
    if case["op"] == "chunk":
        return [min(n, case["new"] if i % case["every"] == 0 else 1) for i, n in enumerate(lengths)]
    return [1] * len(lengths) if case["step"] else lengths


def _gone_of(case):
    """The rows that are freed, in the order in which they finished."""
    return random.Random(case["trace"] + 1).sample(range(case["rows"]), case["gone"])


def _counts(case):
    return [-(-n // case["page"]) for n in lengths_of(case)]


def _shared_pages(case):
    """The leading pages of a row that are the same for all rows that reach as far."""
    return case.get("prefix", 0) // case["page"]


def _used_pages(case):
    counts, shared = _counts(case), _shared_pages(case)
    return sum(max(n - shared, 0) for n in counts) + min(max(counts), shared)


def _pool_pages(case):
    used = _used_pages(case)
    if case["op"] == "compact":
        return max(-(-100 * used // case["fill"]), used + 1)
    return math.ceil(1.25 * used) + (case["rows"] * case["ways"] if case["op"] == "fork" else 0)


def _page_bytes(case):
    """K, V and scales of one page of one layer."""
    elem = 1 if case["dtype"] == "fp8" else 2
    return 2 * case["hkv"] * case["page"] * D * elem + (8 * case["hkv"] if elem == 1 else 0)


def work(case):
    """Inputs read once, outputs written once, and the two products of attention."""
    lengths, counts = lengths_of(case), _counts(case)
    hq, hkv, page, rows = case["hq"], case["hkv"], case["page"], case["rows"]
    if case["op"] == "rope":
        new = sum(new_of(case))
        angles = sum(_first_read(case)) * 4 * case["rot"]
        heads = hq + hkv * (2 if case["write"] else 1)
        return {"bytes": new * (2 * 2 * D * heads + (8 if case["write"] else 4)) + angles, "flops": 0}
    if case["op"] == "fork":
        full = [n // page for n in lengths]
        tails = [(n % page) / page * _page_bytes(case) for n in lengths]
        return {"bytes": int(sum(4 * c + 8 * f + t for c, f, t in zip(counts, full, tails))
                             + case["ways"] * sum(4 * c + t for c, t in zip(counts, tails))), "flops": 0}
    if case["op"] == "free":
        held = [counts[i] for i in _gone_of(case)]
        own_pages = [max(n - _shared_pages(case), 0) for n in held]
        return {"bytes": 4 * sum(held) + 12 * sum(own_pages) + 8 * _shared_pages(case) + 8 * len(held), "flops": 0}
    if case["op"] == "compact":
        used, pool = _used_pages(case), _pool_pages(case)
        moves = used * (pool - used) // pool  # on the average of random pages
        return {"bytes": 2 * moves * (_page_bytes(case) + 4) + 8 * (pool - used) + 12 * pool + 8 * sum(counts), "flops": 0}
    new = new_of(case)
    return {"bytes": 2 * 2 * D * hkv * sum(lengths) + 4 * sum(counts) + 8 * rows + 2 * 2 * D * hq * sum(new),
            "flops": sum(4 * D * hq * (n * (n + 1) - (n - m) * (n - m + 1)) // 2 for n, m in zip(lengths, new))}


def _first_read(case):
    """How many positions of each row's new tokens no other row before it has: each position's
    angles are read once."""
    spans = sorted((n - m, n) for n, m in zip(lengths_of(case), new_of(case)))
    end, got = 0, []
    for first, last in spans:
        got.append(max(last - max(first, end), 0))
        end = max(end, last)
    return got


# ---------------------------------------------------------------------------------
# Inputs.
# ---------------------------------------------------------------------------------
def _ints(values):
    return torch.tensor(values, dtype=torch.int32).to("cuda:0")


def _tables(case, gen):
    """A block table of random pages of the pool, and the pool's pages in the order in which
    they were given out; its columns past a row's pages repeat the row's first page."""
    dev, counts, shared = gen.device, _counts(case), _shared_pages(case)
    order = torch.randperm(_pool_pages(case), generator=gen, device=dev)
    n = torch.tensor(counts, device=dev)
    alone = (n - shared).clamp(min=0)
    prefix = min(max(counts), shared)
    first = prefix + torch.cumsum(alone, 0) - alone
    cols = torch.arange(max(counts), device=dev)
    at = torch.where(cols[None] < shared, cols[None], first[:, None] + cols[None] - shared)
    at = torch.where(cols[None] < n[:, None], at, at[:, :1])
    return order[at].to(torch.int32), order.to(torch.int32)


def _offsets(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _positions(case):
    """Row and position of every new token, packed in row order."""
    rows, pos = [], []
    for b, (n, m) in enumerate(zip(lengths_of(case), new_of(case))):
        rows.append(torch.full((m,), b))
        pos.append(torch.arange(n - m, n))
    return torch.cat(rows).to("cuda:0"), torch.cat(pos).to("cuda:0")


def _shares(case, table):
    """For each page, the rows that hold it beyond the first."""
    n = torch.tensor(_counts(case), device=table.device)
    held = torch.arange(table.shape[1], device=table.device)[None] < n[:, None]
    holders = torch.zeros(_pool_pages(case), dtype=torch.int32, device=table.device)
    holders.scatter_add_(0, table.long().reshape(-1), held.to(torch.int32).reshape(-1))
    return (holders - 1).clamp(min=0).to(torch.int32)


def prepare(case, seed):
    dev, dt = torch.device("cuda:0"), DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    lengths, page, rows, hq, hkv = lengths_of(case), case["page"], case["rows"], case["hq"], case["hkv"]
    s = {"case": case}
    pages = _pool_pages(case)

    def normal(*shape):
        if dt == torch.float8_e4m3fn:
            return (torch.randn(*shape, generator=gen, device=dev, dtype=torch.float16) * 90.0).clamp(-448.0, 448.0).to(dt)
        return torch.randn(*shape, generator=gen, device=dev, dtype=dt)

    def pools():
        s["k_pages"], s["v_pages"] = normal(pages, hkv, page, D), normal(pages, hkv, page, D)
        if case["dtype"] == "fp8":
            s["kv_scales"] = torch.exp2(torch.randint(-9, -3, (pages, hkv, 2), generator=gen, device=dev).float())

    table, order = _tables(case, gen)
    if case["op"] == "rope":
        row, pos = _positions(case)
        # q, k and v are column ranges of one fused projection's output, whose size differs by head.
        qkv = normal(pos.numel(), hq + 2 * hkv, D)
        qkv *= torch.exp2(torch.randn(1, hq + 2 * hkv, 1, generator=gen, device=dev)).to(dt)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["positions"] = pos.to(torch.int32)
        for name in ("q_weight", "k_weight"):
            weight = 1.0 + 0.2 * torch.randn(D, generator=gen, device=dev)
            s[name] = weight if case["norm"] else weight[:0]
        # The angles as a model keeps them: computed in 64 bits for all positions, stored in 32.
        rate = 500000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device=dev) / case["rot"])
        angle = torch.arange(max(lengths), dtype=torch.float64, device=dev)[:, None] * rate
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        s["q_out"] = torch.empty(pos.numel(), hq, D, dtype=dt, device=dev)
        if case["write"]:
            pools()
            s["slot_mapping"] = (table[row, pos // page].long() * page + pos % page).to(torch.int32)
        else:
            s["k_out"] = torch.empty(pos.numel(), hkv, D, dtype=dt, device=dev)
        return s
    if case["op"] == "chunk":
        pools()
        offsets = _offsets(new_of(case))
        s["q"] = normal(offsets[-1], hq, D)
        s["block_table"], s["seq_lens"], s["token_offsets"] = table, _ints(lengths), _ints(offsets)
        s["output"] = torch.empty_like(s["q"])
        return s

    # The pages that no row holds are on the list of free ones.
    used = _used_pages(case)
    s["free_pages"] = torch.cat([order[used:], order[:used]])
    s["num_free"], s["num_free_out"] = _ints([pages - used]), _ints([0])
    s["page_shares"] = _shares(case, table)
    if case["op"] == "fork":
        children = rows * case["ways"]
        s["block_table"] = torch.cat([table, torch.full((children, table.shape[1]), -1, dtype=torch.int32, device=dev)])
        s["lens"] = _ints(lengths + [0] * children)
        s["parents"] = _ints([i // case["ways"] for i in range(children)])
        s["children"] = _ints([rows + i for i in range(children)])
        s["copy_src"], s["copy_dst"] = _ints([0] * children), _ints([0] * children)
        pools()
    elif case["op"] == "free":
        s["block_table"], s["lens"], s["rows"] = table, _ints(lengths), _ints(_gone_of(case))
    else:
        s["block_table"] = table
        s["page_map"] = torch.empty(pages, dtype=torch.int32, device=dev)
        s["block_table_out"], s["page_shares_out"] = torch.empty_like(table), torch.empty_like(s["page_shares"])
        s["free_pages_out"] = s["free_pages"].clone()
        s["copy_src"], s["copy_dst"] = _ints([0] * (pages // 2)), _ints([0] * (pages // 2))
        pools()
    return s


# ---------------------------------------------------------------------------------
# One pass.
# ---------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        _own(s, op)
    else:
        {"rope": _plain_rope, "fork": _plain_fork, "free": _plain_free, "compact": _plain_compact,
         "chunk": _plain_chunk}[op](s)
    if op == "rope":
        outputs = ("q_out", "k_pages", "v_pages") if case["write"] else ("q_out", "k_out")
    else:
        outputs = {"fork": ("block_table", "page_shares", "num_free_out", "copy_src", "copy_dst", "k_pages", "v_pages"),
                   "free": ("page_shares", "free_pages", "num_free_out"),
                   "compact": ("page_map", "block_table_out", "page_shares_out", "free_pages_out", "num_free_out",
                               "copy_src", "copy_dst", "k_pages", "v_pages"),
                   "chunk": ("output",)}[op]
        if "kv_scales" in s:
            outputs += ("kv_scales",)
    return {name: s[name] for name in outputs}


def _own(s, op):
    package = os.path.join(os.getcwd(), "persistentkv-attention_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import persistentkv_torch_ext as ext
    case = s["case"]
    page = case["page"]

    def workspace(size, dtype):  # kept, as a serving loop keeps it between steps
        if "workspace" not in s:
            s["workspace"] = torch.empty(size, dtype=dtype, device="cuda:0")
        return s["workspace"]

    if op == "rope":
        if case["write"]:
            ext.norm_rope_write_kv(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["cos_sin"], s["positions"],
                                   s["q_out"], s["k_pages"], s["v_pages"], s["slot_mapping"], EPS, case["pairs"])
        else:
            ext.norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["cos_sin"], s["positions"], s["q_out"],
                          s["k_out"], EPS, case["pairs"])
    elif op == "fork":
        ext.fork_rows(s["parents"], s["children"], s["lens"], s["block_table"], s["page_shares"], s["free_pages"],
                      s["num_free"], s["num_free_out"], s["copy_src"], s["copy_dst"], page)
        ext.copy_pages(s["copy_src"], s["copy_dst"], s["k_pages"], s["v_pages"], s.get("kv_scales"))
    elif op == "free":
        space = workspace(ext.page_workspace_ints(s["page_shares"].numel()), torch.int32)
        ext.free_rows(s["rows"], s["lens"], s["block_table"], s["page_shares"], s["free_pages"], s["num_free"],
                      s["num_free_out"], space, page)
    elif op == "compact":
        space = workspace(ext.page_workspace_ints(s["page_shares"].numel()), torch.int32)
        ext.compact_pages(s["block_table"], s["page_shares"], s["free_pages"], s["num_free"], s["page_map"],
                          s["block_table_out"], s["page_shares_out"], s["free_pages_out"], s["num_free_out"],
                          s["copy_src"], s["copy_dst"], space)
        ext.copy_pages(s["copy_src"], s["copy_dst"], s["k_pages"], s["v_pages"], s.get("kv_scales"))
    else:
        floats = ext.paged_prefill_workspace_floats(case["rows"], s["q"].shape[0], case["hq"], case["hkv"])
        ext.paged_prefill_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["seq_lens"],
                                    s["token_offsets"], s["output"], workspace(floats, torch.float32), page)


def _plain_rope_one(s, x, weight, out):
    case, x = s["case"], x.float()
    if weight.numel():
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    half = case["rot"] // 2
    angles = s["cos_sin"][s["positions"].long()][:, None]
    cos, sin = angles[..., :half], angles[..., half:]
    if case["pairs"]:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., 2 * half:]], -1).to(out)


def _plain_rope(s):
    dt = s["q"].dtype
    s["q_out"].copy_(_plain_rope_one(s, s["q"], s["q_weight"], dt))
    k = _plain_rope_one(s, s["k"], s["k_weight"], dt)
    if s["case"]["write"]:
        page, slot = s["case"]["page"], s["slot_mapping"].long()
        s["k_pages"][slot // page, :, slot % page] = k
        s["v_pages"][slot // page, :, slot % page] = s["v"]
    else:
        s["k_out"].copy_(k)


def _plain_copy(s):
    """Page dst becomes page src, where both are ids."""
    src, dst = s["copy_src"].long(), s["copy_dst"].long()
    both = (src >= 0) & (dst >= 0)
    src, dst = src[both], dst[both]
    k, v = s["k_pages"], s["v_pages"]
    if k.element_size() == 1:
        k, v = k.view(torch.uint8), v.view(torch.uint8)
    k[dst] = k[src]
    v[dst] = v[src]
    if "kv_scales" in s:
        s["kv_scales"][dst] = s["kv_scales"][src]


def _plain_fork(s):
    page, table, free = s["case"]["page"], s["block_table"], s["free_pages"]
    parents, children, avail = s["parents"].long(), s["children"].long(), s["num_free"].long()
    columns = table.shape[1]
    lens = s["lens"].long()[parents].clamp(0, columns * page)
    full, tail = lens // page, lens % page > 0
    taken = torch.cumsum(tail.long(), 0)
    fits = taken[-1:] <= avail
    at = avail - taken  # the i-th page from the list's end
    new = free.long()[at.clamp(0, free.numel() - 1)]
    old, column = table[parents].long(), torch.arange(columns, device=table.device)[None]
    shared, last = fits & (column < full[:, None]), fits & tail
    s["copy_src"].copy_(torch.where(last, old.gather(1, full.clamp(max=columns - 1)[:, None])[:, 0], -1))
    s["copy_dst"].copy_(torch.where(last, new, -1))
    here = torch.where(last[:, None] & (column == full[:, None]), new[:, None], table[children].long())
    table[children] = torch.where(shared, old, here).to(torch.int32)
    counted = shared & (old >= 0)
    s["page_shares"].scatter_add_(0, torch.where(counted, old, 0).reshape(-1), counted.to(torch.int32).reshape(-1))
    s["num_free_out"].copy_(avail - taken[-1:])
    _plain_copy(s)


def _plain_free(s):
    page, table, free, shares = s["case"]["page"], s["block_table"], s["free_pages"], s["page_shares"]
    rows, avail, pages = s["rows"].long(), s["num_free"].long(), s["page_shares"].numel()
    again = (rows[:, None] == rows[None]).tril(-1).any(1)
    held = (s["lens"].long()[rows].clamp(min=0) + page - 1) // page
    ids, column = table[rows].long(), torch.arange(table.shape[1], device=table.device)[None]
    mine = (column < held[:, None]) & (ids >= 0) & ~again[:, None]
    left = shares.long().scatter_add(0, torch.where(mine, ids, 0).reshape(-1), -mine.long().reshape(-1))
    gone = left < 0
    shares.copy_(left.clamp(min=0))
    at = torch.where(gone, avail + torch.cumsum(gone.long(), 0) - 1, free.numel())
    longer = torch.cat([free, free[:1]])
    longer.scatter_(0, at, torch.arange(pages, device=table.device).to(torch.int32))
    free.copy_(longer[:-1])
    s["num_free_out"].copy_(avail + gone.sum())


def _plain_compact(s):
    table, free, shares = s["block_table"], s["free_pages"], s["page_shares"]
    pages, dev = shares.numel(), shares.device
    p, listed_free = torch.arange(pages, device=dev), torch.arange(free.numel(), device=dev) < s["num_free"]
    used = torch.ones(pages + 1, dtype=torch.long, device=dev)
    used.scatter_(0, torch.where(listed_free, free.long(), pages), 0)
    used = used[:pages]
    total, before = used.sum(), torch.cumsum(used, 0) - used
    hole, mover = (used == 0) & (p < total), (used == 1) & (p >= total)
    none = torch.full((pages + 1,), -1, dtype=torch.long, device=dev)
    holes = none.scatter(0, torch.where(hole, p - before, pages), p)[:pages]
    turn = total - 1 - before  # the highest page takes the lowest place
    movers = none.scatter(0, torch.where(mover, turn, pages), p)[:pages]
    page_map = torch.where(mover, holes[turn.clamp(0, pages - 1)], torch.where(used == 1, p, -1))
    s["page_map"].copy_(page_map)
    known = (table >= 0) & (table < pages)
    s["block_table_out"].copy_(torch.where(known, page_map[table.long().clamp(0, pages - 1)], table.long()))
    moved = torch.zeros(pages + 1, dtype=torch.int32, device=dev)
    s["page_shares_out"].copy_(moved.scatter(0, torch.where(used == 1, page_map, pages), shares)[:pages])
    at = torch.arange(free.numel(), device=dev)
    s["free_pages_out"].copy_(torch.where(at < pages - total, pages - 1 - at, s["free_pages_out"].long()))
    s["num_free_out"].copy_((pages - total)[None])
    s["copy_src"].copy_(movers[:pages // 2])
    s["copy_dst"].copy_(torch.where(movers >= 0, holes, -1)[:pages // 2])
    _plain_copy(s)


def _plain_chunk(s):
    """Rows padded to the longest, softmax(q K^T / sqrt(128)) V over the keys up to each token."""
    case, table = s["case"], s["block_table"].long()
    hkv, group, page = case["hkv"], case["hq"] // case["hkv"], case["page"]
    offsets, lens, most = s["token_offsets"].long(), s["seq_lens"].long(), max(new_of(case))
    i = torch.arange(most, device=table.device)
    at = (offsets[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][at].float().reshape(-1, most, hkv, group, D).permute(0, 2, 3, 1, 4).reshape(-1, hkv, group * most, D)

    def tokens(pool):  # [rows, hkv, columns * page, D]
        return pool[table].permute(0, 2, 1, 3, 4).reshape(-1, hkv, table.shape[1] * page, D).float()

    x = torch.matmul(q, tokens(s["k_pages"]).transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(D))
    x = x.reshape(-1, hkv, group, most, x.shape[-1])
    last = lens[:, None] - (offsets[1:] - offsets[:-1])[:, None] + i  # [rows, most]
    hidden = torch.arange(x.shape[-1], device=x.device) > torch.minimum(last, lens[:, None] - 1)[..., None]
    x.masked_fill_(hidden[:, None, None], float("-inf"))
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.reshape(-1, hkv, group * most, x.shape[-1]), tokens(s["v_pages"]))
    o = o.reshape(-1, hkv, group, most, D) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(-1, most, case["hq"], D)
    t = torch.arange(s["q"].shape[0], device=table.device)
    row = torch.searchsorted(offsets[1:], t, right=True)
    s["output"].copy_(o[row, t - offsets[row]])


# ---------------------------------------------------------------------------------
# Results in 64 bits, row by row from the definitions.
# ---------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] not in ("rope", "chunk"):
        return None  # whole numbers and copies
    s = prepare(case, seed)
    return _exact_rope(s) if case["op"] == "rope" else _exact_chunk(s)


def _turn(x, weight, cos_sin, pairs):
    """x [tokens, heads, D] and the angles of its tokens [tokens, rot], in 64 bits: each pair of
    dims is a complex number, multiplied by the one of its angle."""
    if weight is not None:
        x = weight * x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + EPS)
    rot = cos_sin.shape[1]
    i = torch.arange(rot // 2, device=x.device)
    first, second = (2 * i, 2 * i + 1) if pairs else (i, i + rot // 2)
    turn = torch.complex(cos_sin[:, :rot // 2], cos_sin[:, rot // 2:])[:, None]
    z = torch.complex(x[..., first], x[..., second]) * turn
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_rope(s):
    case = s["case"]
    angles = s["cos_sin"].double()[s["positions"].long()]
    q, k = (_turn(s[n].double(), s[n + "_weight"].double() if case["norm"] else None, angles, case["pairs"]) for n in "qk")
    if not case["write"]:
        return {"q_out": q, "k_out": k}
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    place, offset = s["slot_mapping"].long() // case["page"], s["slot_mapping"].long() % case["page"]
    for h in range(case["hkv"]):
        k_pages[place, h, offset] = k[:, h]
        v_pages[place, h, offset] = s["v"][:, h].double()
    return {"q_out": q, "k_pages": k_pages, "v_pages": v_pages}


def _exact_chunk(s):
    case = s["case"]
    hkv, group = case["hkv"], case["hq"] // case["hkv"]
    out = torch.empty(s["output"].shape, dtype=torch.float64, device=s["q"].device)
    at = 0
    for b, (n, m) in enumerate(zip(lengths_of(case), new_of(case))):
        ids = s["block_table"][b, :-(-n // case["page"])].long()
        later = torch.arange(n, device=out.device) > torch.arange(n - m, n, device=out.device)[:, None]
        for h in range(hkv):
            k, v = (s[x][ids, h].double().reshape(-1, D)[:n] for x in ("k_pages", "v_pages"))
            for g in range(h * group, (h + 1) * group):
                x = (s["q"][at:at + m, g].double() @ k.T.contiguous()) / math.sqrt(D)
                out[at:at + m, g] = torch.softmax(x.masked_fill(later, -math.inf), -1) @ v
        at += m
    return {"output": out}
