"""write_kv and write_kv_fp8_block against plain loops.  Copies and roundings to e4m3 under
power-of-two scales have one right result: pools and scales must be equal bit for bit."""
import numpy as np
import pytest
import torch

from oracle import prompt

pytestmark = pytest.mark.gpu
F16, BF16, F8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def _slots(rows, page_size, pages, seed):
    """Slots of packed rows (cached, new): each row's pages drawn from one permutation."""
    order = np.random.default_rng(seed).permutation(pages).tolist()
    slots = []
    for cached, new in rows:
        need = -(-(cached + new) // page_size)
        mine, order = order[:need], order[need:]
        slots += [mine[p // page_size] * page_size + p % page_size for p in range(cached, cached + new)]
    return slots


def _new(tokens, hkv, dtype, seed, spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, 2 * hkv + 1, 128, generator=gen)
    x = (x * torch.exp2(spread * torch.randn(tokens, 2 * hkv + 1, 1, generator=gen))).to(dtype)
    return x[:, :hkv], x[:, hkv:2 * hkv]  # column ranges of a wider tensor


ROWS = [[(0, 1)], [(0, 16)], [(5, 1), (16, 1), (31, 1)], [(0, 40), (7, 9), (9, 30), (0, 3)], [(3, 200), (0, 130)]]


@pytest.mark.parametrize("rows", ROWS, ids=str)
@pytest.mark.parametrize("page_size,hkv,dtype", [(16, 2, F16), (5, 3, BF16), (64, 1, F16)])
def test_write_kv(ext, gpu, rows, page_size, hkv, dtype):
    pages = sum(-(-(c + n) // page_size) for c, n in rows) + 3
    slots = _slots(rows, page_size, pages, seed=1)
    slots[0] = -1 if len(slots) > 3 else slots[0]
    slots[-1] = pages * page_size if len(slots) > 3 else slots[-1]  # past the pool: skipped
    k, v = _new(len(slots), hkv, dtype, seed=2)
    k0, v0 = (torch.randn(pages, hkv, page_size, 128).to(dtype) for _ in range(2))
    kg, vg = k0.to(gpu), v0.to(gpu)
    wide = torch.cat([k, v], dim=1).to(gpu)
    ext.write_kv(wide[:, :hkv], wide[:, hkv:], kg, vg, torch.tensor(slots, dtype=torch.int32, device=gpu))
    assert torch.equal(kg.cpu(), torch.from_numpy(prompt.write_kv(k0.double().numpy(), k.double().numpy(), slots)).to(dtype))
    assert torch.equal(vg.cpu(), torch.from_numpy(prompt.write_kv(v0.double().numpy(), v.double().numpy(), slots)).to(dtype))


def _check_block(ext, gpu, k, v, slots, pages, page_size, seed=0, scales=None):
    hkv = k.shape[1]
    gen = torch.Generator().manual_seed(seed)
    k8, v8 = ((torch.randn(pages, hkv, page_size, 128, generator=gen) * 100).clamp(-448, 448).to(F8) for _ in range(2))
    if scales is None:
        scales = torch.exp2(torch.randint(-9, 3, (pages, hkv, 2), generator=gen).float())
    kg, vg, sg = k8.to(gpu), v8.to(gpu), scales.to(gpu)
    wide = torch.cat([k, v], dim=1).to(gpu)
    for again in range(2):  # writing the same tokens once more changes nothing
        ext.write_kv_fp8_block(wide[:, :hkv], wide[:, hkv:], kg, vg, sg,
                               torch.tensor(slots, dtype=torch.int32, device=gpu))
        torch.cuda.synchronize()
        for i, (pool, old, new) in enumerate(((kg, k8, k), (vg, v8, v))):
            want, s = prompt.write_kv_fp8_block(old.double().numpy(), scales[:, :, i].double().numpy(),
                                                new.double().numpy(), slots)
            got = pool.cpu().double().numpy()
            assert (np.isnan(got) == np.isnan(want)).all()
            assert (got[~np.isnan(want)] == want[~np.isnan(want)]).all(), (again, "KV"[i])
            assert (sg[:, :, i].cpu().double().numpy() == s).all()


@pytest.mark.parametrize("rows", ROWS, ids=str)
@pytest.mark.parametrize("page_size,hkv,dtype", [(16, 2, F16), (16, 3, BF16), (32, 1, F16), (48, 2, BF16), (64, 2, F16), (128, 1, BF16), (7, 2, F16)])
def test_write_block(ext, gpu, rows, page_size, hkv, dtype):
    pages = sum(-(-(c + n) // page_size) for c, n in rows) + 3
    slots = _slots(rows, page_size, pages, seed=3)
    k, v = _new(len(slots), hkv, dtype, seed=4)
    _check_block(ext, gpu, k, v, slots, pages, page_size, seed=5)


@pytest.mark.parametrize("tokens,hkv", [(3000, 8), (2100, 7)])
def test_write_block_many_tokens(ext, gpu, tokens, hkv):
    """Past the size from which a wave takes a window of tokens rather than one."""
    rows = [(3, tokens // 2), (0, 77), (16, 1), (30, 2), (0, tokens - tokens // 2 - 80)]
    pages = sum(-(-(c + n) // 16) for c, n in rows) + 3
    slots = _slots(rows, 16, pages, seed=6)
    k, v = _new(len(slots), hkv, F16, seed=7)
    _check_block(ext, gpu, k, v, slots, pages, 16, seed=8)


def test_write_block_skips_and_splits_runs(ext, gpu):
    """Slots outside the pool are skipped; runs end at them, at a jump and at a page's end."""
    slots = [5, 6, -1, 23, 24, 99999, 16 * 4, 16 * 4 + 1, 47, 16 * 9 + 15, 16 * 5, -3]
    k, v = _new(len(slots), 2, BF16, seed=9)
    _check_block(ext, gpu, k, v, slots, 10, 16, seed=10)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_write_block_values(ext, gpu, dtype):
    """Zeros, the borders of the scale, infinities, NaN, subnormals and every fp16 code."""
    inf, nan = float("inf"), float("nan")
    k = torch.zeros(40, 2, 128)
    k[1, 0, :8] = torch.tensor([448.0, -448.0, 0.0, -0.0, 1.0, 2.0 ** -9, 3 * 2.0 ** -10, 17.0])
    k[2, 0, :3] = torch.tensor([449.0, 1.0, -1.5])
    k[3, 1, :4] = torch.tensor([inf, -inf, nan, 5.0])
    k[4, 1, :2] = torch.tensor([nan, inf])
    k[5, 0, :2] = torch.tensor([2.0 ** -24, 2.0 ** -23])
    k[6, 0, :2] = torch.tensor([60000.0, 0.25])
    v = k.flip(0).contiguous()
    slots = [16 * i for i in range(16)] + [16 * i + 3 for i in range(16, 40)]
    _check_block(ext, gpu, k.to(dtype), v.to(dtype), slots, 40, 16, seed=11)
    codes = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(F16).view(512, 1, 128).to(dtype)
    _check_block(ext, gpu, codes, codes.flip(0).contiguous(), list(range(512)), 32, 16, seed=12)


def test_write_block_odd_old_scales(ext, gpu):
    """Earlier tokens under scales that are no powers of two, zero, negative, infinite, NaN."""
    scales = torch.tensor([0.3, 1.7, 0.0, -2.0, float("inf"), float("nan"), 1e-30, 1e30]).repeat(2, 1).t().reshape(8, 1, 2)
    slots = [16 * i + 4 for i in range(8)]
    k, v = _new(8, 1, F16, seed=13, spread=0.5)
    _check_block(ext, gpu, k, v, slots, 8, 16, seed=14, scales=scales.contiguous())


def test_write_nothing(ext, gpu):
    k = torch.zeros(0, 2, 128, dtype=F16, device=gpu)
    pool = torch.zeros(3, 2, 16, 128, dtype=F16, device=gpu)
    none = torch.zeros(0, dtype=torch.int32, device=gpu)
    ext.write_kv(k, k, pool, pool.clone(), none)
    p8, s = pool.to(F8), torch.ones(3, 2, 2, device=gpu)
    ext.write_kv_fp8_block(k, k, p8, p8.clone(), s, none)
    assert (s == 1).all()


def test_pools_past_32_bits(ext, gpu):
    """Pages at the end of pools of more than 2^32 bytes (and 2^31 elements)."""
    pages, hkv, ps = 2 ** 21 + 8, 1, 16
    near = [3, 0, 5]
    slots = {d: torch.tensor([(p + d) * ps + i for p in near for i in range(ps)], dtype=torch.int32, device=gpu)
             for d in (0, pages - 8)}
    k, v = (x.contiguous().to(gpu) for x in _new(48, hkv, F16, seed=15))
    small = [torch.zeros(8, hkv, ps, 128, dtype=F16, device=gpu) for _ in range(2)]
    ext.write_kv(k, v, *small, slots[0])
    big = [torch.empty(pages, hkv, ps, 128, dtype=F16, device=gpu) for _ in range(2)]
    for x in big:
        x[-8:] = 0
    ext.write_kv(k, v, *big, slots[pages - 8])
    assert all(torch.equal(b[-8:], s) for b, s in zip(big, small))
    del big
    small = [x.to(F8) for x in small]
    s0, s1 = torch.ones(8, hkv, 2, device=gpu), torch.ones(pages, hkv, 2, device=gpu)
    ext.write_kv_fp8_block(k, v, *small, s0, slots[0])
    big = [torch.empty(pages, hkv, ps, 128, dtype=F8, device=gpu) for _ in range(2)]
    for x in big:
        x.view(torch.uint8)[-8:] = 0
    ext.write_kv_fp8_block(k, v, *big, s1, slots[pages - 8])
    assert torch.equal(s1[-8:], s0)
    sel = torch.tensor(near, device=gpu)
    for b, s in zip(big, small):
        assert torch.equal(b.view(torch.uint8)[-8:][sel], s.view(torch.uint8)[sel])
    # and decode over them
    q = torch.randn(1, 4, 128, device=gpu).to(F16)
    table = torch.tensor([near], dtype=torch.int32, device=gpu)
    lens = torch.tensor([40], dtype=torch.int32, device=gpu)
    ws = torch.empty(ext.fp8_block_workspace_floats(1, 4, 1), device=gpu)
    a, b = torch.empty_like(q), torch.empty_like(q)
    ext.paged_attention_fp8_block(q, *small, s0, table, lens, a, ws, ps)
    ext.paged_attention_fp8_block(q, *big, s1, table + (pages - 8), lens, b, ws, ps)
    assert torch.equal(a, b) and torch.isfinite(a).all()
