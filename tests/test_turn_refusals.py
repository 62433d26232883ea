"""What the operators for a further turn over cached rows refuse, before any device work: through the
C ABI and through the op surface."""
import ctypes

import pytest
import torch

import pkv_native

F16, I32 = torch.float16, torch.int32
AT, OUT, NUM = 0x100000, 0x900000, 0x2000  # never dereferenced: validation fails first


def _rope(write=False, **o):
    a = dict(q=AT, qs=1024, k=0x200000, ks=256, v=0x300000, vs=256, qw=AT, qwh=1, kw=AT, kwh=1, table=AT, pos=AT, qo=OUT, qos=1024,
             ko=0xa00000, kos=256, kp=AT, vp=AT, slots=AT, tokens=4, hq=8, hkv=2, d=128, rot=128, most=100, pairs=0, eps=1e-6,
             pages=3, ps=16, dtype=0)
    a.update(o)
    for x in ("ko", "kos") if write else ("v", "vs", "kp", "vp", "slots", "pages", "ps"):
        del a[x]
    return getattr(pkv_native.lib(), "pkv_norm_rope_write_kv" if write else "pkv_norm_rope")(*a.values(), None)


def _fork(**o):
    a = dict(parents=AT, children=AT, lens=AT, table=AT, shares=AT, free=AT, num=NUM, left=AT, src=AT, dst=AT, n=2, batch=4, cols=3,
             pages=9, cap=9, ps=16)
    a.update(o)
    return pkv_native.lib().pkv_fork_rows(*a.values(), None)


def _free(**o):
    a = dict(rows=AT, lens=AT, table=AT, shares=AT, free=AT, num=NUM, left=AT, ws=AT, size=1 << 20, n=2, batch=4, cols=3, pages=9, cap=9, ps=16)
    a.update(o)
    return pkv_native.lib().pkv_free_rows(*a.values(), None)


def _compact(**o):
    a = dict(table=AT, shares=AT, free=AT, num=NUM, map=AT, to=AT, so=OUT, fo=OUT, left=AT, src=AT, dst=AT, ws=AT, size=1 << 20,
             batch=4, cols=3, pages=9, cap=9, copies=4)
    a.update(o)
    return pkv_native.lib().pkv_compact_pages(*a.values(), None)


def _copy(**o):
    a = dict(src=AT, dst=AT, k=AT, v=AT, scales=None, n=2, pages=9, hkv=2, ps=16, d=128, elem=2)
    a.update(o)
    return pkv_native.lib().pkv_copy_pages(*a.values(), None)


def _chunk(**o):
    a = dict(q=AT, qs=1024, k=AT, v=AT, table=AT, lens=AT, off=AT, out=OUT, ws=AT, size=1 << 40, batch=1, tokens=4, hq=8, hkv=2, d=128,
             pages=3, ps=16, cols=2, dtype=0)
    a.update(o)
    return pkv_native.lib().pkv_paged_prefill_attention(*a.values(), None)


def _write(**o):
    return _rope(write=True, **o)


@pytest.mark.parametrize("call,overrides,status,text", [
    (_rope, dict(d=64), 2, "head_dim"), (_rope, dict(tokens=-1), 1, "tokens"), (_rope, dict(hq=0), 1, "num_q_heads"),
    (_rope, dict(most=0), 1, "max_positions"), (_rope, dict(rot=8), 2, "rotary_dim"), (_rope, dict(rot=144), 2, "rotary_dim"),
    (_rope, dict(rot=72), 2, "rotary_dim"), (_rope, dict(dtype=7), 1, "dtype"), (_rope, dict(eps=0.0), 1, "eps"),
    (_rope, dict(eps=float("nan")), 1, "eps"), (_rope, dict(eps=-1.0), 1, "eps"), (_rope, dict(qs=1020), 1, "stride"),
    (_rope, dict(ks=128), 1, "stride"), (_rope, dict(qos=1016), 1, "stride"), (_rope, dict(kos=252), 1, "stride"),
    (_rope, dict(qwh=3), 1, "weights"), (_rope, dict(kwh=8), 1, "weights"), (_rope, dict(pos=None), 1, "null"), (_rope, dict(ko=None), 1, "null"),
    (_rope, dict(table=None), 1, "null"), (_rope, dict(q=AT + 8), 1, "aligned"), (_rope, dict(qw=AT + 4), 1, "aligned"),
    (_rope, dict(tokens=1 << 30), 2, "too many"), (_rope, dict(qo=0x200000), 1, "q_out must be its own"), (_rope, dict(qo=AT + 1024), 1, "q_out must be its own"),
    (_rope, dict(ko=AT + 2048), 1, "k_out must be its own"), (_rope, dict(ko=OUT + 256), 1, "q_out and k_out"),
    (_write, dict(vs=250), 1, "stride"), (_write, dict(ps=0), 1, "page_size"), (_write, dict(pages=1 << 30), 2, "int32"),
    (_write, dict(slots=None), 1, "null"), (_write, dict(vp=AT + 8), 1, "aligned"), (_write, dict(qo=0x300000), 1, "q_out must be its own"),
    (_write, dict(d=256), 2, "head_dim"), (_write, dict(kwh=5), 1, "weights"),
    (_fork, dict(n=-1), 1, "num_forks"), (_fork, dict(ps=0), 1, "page_size"), (_fork, dict(cols=0), 1, "max_pages"), (_fork, dict(n=8001), 2, "8000"),
    (_fork, dict(cols=1 << 28, ps=16), 2, "int32"), (_fork, dict(parents=None), 1, "null"), (_fork, dict(free=None), 1, "null"),
    (_fork, dict(left=NUM), 1, "num_free"), (_fork, dict(pages=0), 1, "num_pages"),
    (_fork, dict(cols=(1 << 30) + 1, ps=1), 2, "past 1073741824"), (_free, dict(cols=(1 << 30) + 1), 2, "at most 1073741824"),
    (_free, dict(n=8001), 2, "8000"), (_free, dict(cap=8), 1, "places"), (_free, dict(ws=None), 3, "workspace"), (_free, dict(size=7), 3, "workspace"),
    (_free, dict(ws=AT + 2), 3, "workspace"), (_free, dict(left=NUM), 1, "num_free"), (_free, dict(rows=None), 1, "null"), (_free, dict(batch=-1), 1, "batch"),
    (_compact, dict(copies=3), 1, "num_pages / 2"), (_compact, dict(cap=8), 1, "places"), (_compact, dict(so=AT), 1, "page_shares_out must not be"), (_compact, dict(fo=AT), 1, "free_pages_out must not be"),
    (_compact, dict(left=NUM), 1, "num_free_out must not be"), (_compact, dict(size=7), 3, "workspace"), (_compact, dict(map=None), 1, "null"),
    (_compact, dict(table=None), 1, "null"), (_compact, dict(pages=0), 1, "num_pages"),
    (_copy, dict(d=64), 2, "head_dim"), (_copy, dict(elem=4), 1, "1 or 2"), (_copy, dict(k=AT + 8), 1, "aligned"), (_copy, dict(dst=None), 1, "null"),
    (_copy, dict(ps=1 << 24), 2, "2 GiB"), (_copy, dict(hkv=0), 1, "num_kv_heads"), (_copy, dict(scales=AT + 2), 1, "aligned"),
    (_chunk, dict(d=64), 2, "head_dim"), (_chunk, dict(hq=9, qs=2048), 1, "divisible"), (_chunk, dict(hq=66, qs=16384), 2, "G="),
    (_chunk, dict(qs=1016), 1, "stride"), (_chunk, dict(dtype=5), 2, "dtype"), (_chunk, dict(tokens=-1), 1, "tokens"), (_chunk, dict(cols=0), 1, "max_pages"),
    (_chunk, dict(cols=1 << 27), 2, "2^31 - 32"), (_chunk, dict(ps=1 << 23), 2, "2 GiB"), (_chunk, dict(tokens=1 << 30), 2, "too many"),
    (_chunk, dict(batch=1 << 23), 2, "too many"), (_chunk, dict(ws=None), 3, "workspace"), (_chunk, dict(size=1000), 3, "workspace"),
    (_chunk, dict(ws=AT + 8), 3, "workspace"), (_chunk, dict(lens=None), 1, "null"), (_chunk, dict(v=AT + 8), 1, "aligned"),
    (_chunk, dict(out=AT + 2048), 1, "not overlap q"), (_chunk, dict(out=AT, qs=2048), 1, "not overlap q"),
])
def test_c_abi_refusals(call, overrides, status, text):
    assert call(**overrides) == status
    assert text in pkv_native.last_error()


def test_empty_calls_are_no_ops():
    assert _rope(tokens=0) == 0 and _write(tokens=0) == 0 and _copy(n=0) == 0 and _chunk(tokens=0) == 0 and _chunk(batch=0) == 0


def test_workspace_sizes():
    lib = pkv_native.lib()
    size = lib.pkv_paged_prefill_workspace_bytes
    assert 0 < size(1, 1, 32, 8) < size(1, 500, 32, 8) and size(0, 5, 32, 8) == size(1, 0, 32, 8) == size(1, 1, 9, 2) == 0
    assert size(65, 65, 32, 8) > 0 and size(8000, 1 << 20, 32, 8) < 1 << 29
    assert lib.pkv_page_workspace_bytes(1) == 8 and lib.pkv_page_workspace_bytes(1 << 20) == 4 * 1025 and lib.pkv_page_workspace_bytes(0) == 0


def test_op_refusals():
    import persistentkv_torch_ext as ext
    i = lambda *s: torch.zeros(*s, dtype=I32)
    h = lambda *s: torch.zeros(*s, dtype=F16)
    w = torch.zeros(0)
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        ext.norm_rope(h(4, 8, 128), h(4, 2, 128), w, w, torch.zeros(9, 128), i(4), h(4, 8, 128), h(4, 2, 128), 1e-6, False)
    with pytest.raises(RuntimeError, match="q has wrong dtype"):
        ext.norm_rope_write_kv(h(4, 8, 128).float(), h(4, 2, 128), h(4, 2, 128), w, w, torch.zeros(9, 128), i(4), h(4, 8, 128),
                               h(3, 2, 16, 128), h(3, 2, 16, 128), i(4), 1e-6, False)
    with pytest.raises(RuntimeError, match="parents must be a CUDA tensor"):
        ext.fork_rows(i(2), i(2), i(4), i(4, 3), i(9), i(9), i(1), i(1), i(2), i(2), 16)
    with pytest.raises(RuntimeError, match="rows must be a CUDA tensor"):
        ext.free_rows(i(2), i(4), i(4, 3), i(9), i(9), i(1), i(1), i(9), 16)
    with pytest.raises(RuntimeError, match="block_table must be a CUDA tensor"):
        ext.compact_pages(i(4, 3), i(9), i(9), i(1), i(9), i(4, 3), i(9), i(9), i(1), i(4), i(4), i(9))
    with pytest.raises(RuntimeError, match="k_pages must be a CUDA tensor"):
        ext.copy_pages(i(2), i(2), h(3, 2, 16, 128), h(3, 2, 16, 128))
    with pytest.raises(RuntimeError, match="k_pages has wrong dtype"):
        ext.copy_pages(i(2), i(2), h(3, 2, 16, 128).float(), h(3, 2, 16, 128))
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        ext.paged_prefill_attention(h(4, 8, 128), h(3, 2, 16, 128), h(3, 2, 16, 128), i(1, 2), i(1), i(2), h(4, 8, 128), torch.zeros(9), 16)


@pytest.mark.gpu
def test_op_refusals_on_the_gpu(ext, gpu):
    i = lambda *s: torch.zeros(*s, dtype=I32, device=gpu)
    h = lambda *s: torch.zeros(*s, dtype=F16, device=gpu)
    f = lambda *s: torch.zeros(*s, device=gpu)
    rope = lambda qw=f(0), kw=f(0), table=f(9, 128), pos=i(4), out=h(4, 8, 128), kout=h(4, 2, 128): ext.norm_rope(
        h(4, 8, 128), h(4, 2, 128), qw, kw, table, pos, out, kout, 1e-6, False)
    rope()
    for bad, text in ((dict(qw=f(127)), "q_weight must have shape"), (dict(qw=f(2, 128)), "q_weight must have shape"), (dict(kw=f(8, 128)), "k_weight must have shape"),
                      (dict(qw=h(128)), "q_weight has wrong dtype"), (dict(kw=torch.zeros(128)), "k_weight must be a CUDA"), (dict(table=f(9, 72)), "rotary_dim"),
                      (dict(table=f(9, 128).double()), "cos_sin has wrong dtype"), (dict(pos=i(5)), "one position a token"), (dict(out=h(5, 8, 128)), "q_out shape"),
                      (dict(kout=h(4, 3, 128)), "k_out shape"), (dict(table=f(0, 128)), "max_positions")):
        with pytest.raises(RuntimeError, match=text):
            rope(**bad)
    with pytest.raises(RuntimeError, match="one slot a token"):
        ext.norm_rope_write_kv(h(4, 8, 128), h(4, 2, 128), h(4, 2, 128), f(0), f(0), f(9, 128), i(4), h(4, 8, 128), h(3, 2, 16, 128), h(3, 2, 16, 128), i(5), 1e-6, False)
    with pytest.raises(RuntimeError, match="Hkv mismatch"):
        ext.norm_rope_write_kv(h(4, 8, 128), h(4, 2, 128), h(4, 2, 128), f(0), f(0), f(9, 128), i(4), h(4, 8, 128), h(3, 1, 16, 128), h(3, 1, 16, 128), i(4), 1e-6, False)
    n = i(1)
    with pytest.raises(RuntimeError, match="num_free_out must not be num_free"):
        ext.fork_rows(i(2), i(2), i(4), i(4, 3), i(9), i(9), n, n, i(2), i(2), 16)
    with pytest.raises(RuntimeError, match="one row a parent"):
        ext.fork_rows(i(2), i(3), i(4), i(4, 3), i(9), i(9), i(1), i(1), i(2), i(2), 16)
    with pytest.raises(RuntimeError, match="one entry a parent"):
        ext.fork_rows(i(2), i(2), i(4), i(4, 3), i(9), i(9), i(1), i(1), i(2), i(3), 16)
    with pytest.raises(RuntimeError, match="workspace of"):
        ext.free_rows(i(2), i(4), i(4, 3), i(9), i(9), i(1), i(1), i(0), 16)
    with pytest.raises(RuntimeError, match="batch mismatch"):
        ext.free_rows(i(2), i(5), i(4, 3), i(9), i(9), i(1), i(1), i(9), 16)
    with pytest.raises(RuntimeError, match="page_map must have"):
        ext.compact_pages(i(4, 3), i(9), i(9), i(1), i(8), i(4, 3), i(9), i(9), i(1), i(4), i(4), i(9))
    with pytest.raises(RuntimeError, match="kv_scales must have shape"):
        ext.copy_pages(i(2), i(2), h(3, 2, 16, 128), h(3, 2, 16, 128), f(3, 2, 1))
    with pytest.raises(RuntimeError, match="v_pages has wrong dtype"):
        ext.copy_pages(i(2), i(2), h(3, 2, 16, 128), h(3, 2, 16, 128).bfloat16())
    with pytest.raises(RuntimeError, match="workspace of"):
        ext.paged_prefill_attention(h(4, 8, 128), h(3, 2, 16, 128), h(3, 2, 16, 128), i(1, 2), i(1), i(2), h(4, 8, 128), f(9), 16)
    with pytest.raises(RuntimeError, match="contiguous heads"):
        ext.paged_prefill_attention(h(4, 8, 256)[..., ::2], h(3, 2, 16, 128), h(3, 2, 16, 128), i(1, 2), i(1), i(2), h(4, 8, 128), f(9), 16)
    with pytest.raises(RuntimeError, match="batch \\+ 1"):
        ext.paged_prefill_attention(h(4, 8, 128), h(3, 2, 16, 128), h(3, 2, 16, 128), i(1, 2), i(1), i(3), h(4, 8, 128), f(9), 16)
