"""What the operators between a prompt and the cache refuse, before any device work: through
the op surface (CPU tensors: the checks that come before the device) and through the C ABI."""
import ctypes

import pytest
import torch

import pkv_native

F16, F8, I32 = torch.float16, torch.float8_e4m3fn, torch.int32
FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first


OUT = ctypes.c_void_p(0x8000)


def _call(name, args):
    f = getattr(pkv_native.lib(), name)
    f.restype = ctypes.c_int
    conv = [ctypes.c_int64(a[1]) if isinstance(a, tuple) and a[0] == "i64" else
            ctypes.c_size_t(a[1]) if isinstance(a, tuple) else a for a in args]
    return f(*conv)


def _tables(**o):
    a = dict(cached=FAKE, lens=FAKE, free=FAKE, num=ctypes.c_void_p(0x2000), table=FAKE, off=FAKE, slots=FAKE,
             left=FAKE, batch=2, cap=4, cols=3, n=8, ps=16)
    a.update(o)
    return _call("pkv_build_block_tables", [*a.values(), None])


def _prefill(**o):
    a = dict(q=FAKE, qs=1024, k=FAKE, ks=256, v=FAKE, vs=256, off=FAKE, out=OUT, batch=1, tokens=4, hq=8, hkv=2, d=128, dtype=0)
    a.update(o)
    for s in ("qs", "ks", "vs"):
        a[s] = ("i64", a[s])
    return _call("pkv_prefill_attention", [*a.values(), None])


def _write(block=False, **o):
    a = dict(k=FAKE, ks=256, v=FAKE, vs=256, kp=FAKE, vp=FAKE, scales=FAKE, slots=FAKE, tokens=4, hkv=2, d=128, pages=3, ps=16, dtype=0)
    a.update(o)
    for s in ("ks", "vs"):
        a[s] = ("i64", a[s])
    if not block:
        del a["scales"]
    return _call("pkv_write_kv_fp8_block" if block else "pkv_write_kv", [*a.values(), None])


def _decode(**o):
    a = dict(q=FAKE, k=FAKE, v=FAKE, s=FAKE, table=FAKE, lens=FAKE, out=FAKE, ws=FAKE, size=1 << 30, batch=1, hq=8,
             hkv=2, d=128, pages=3, ps=16, cols=2, dtype=0)
    a.update(o)
    a["size"] = ("size", a["size"])
    return _call("pkv_paged_attention_fp8_block", [*a.values(), None])


@pytest.mark.parametrize("call,overrides,status,text", [
    (_tables, dict(ps=0), 1, "page_size"), (_tables, dict(cols=0), 1, "max_pages"), (_tables, dict(batch=-1), 1, "batch"),
    (_tables, dict(batch=8001), 2, "8000"), (_tables, dict(slots=None), 1, "null"), (_tables, dict(lens=None), 1, "null"),
    (_tables, dict(left=ctypes.c_void_p(0x2000)), 1, "num_free"),
    (_prefill, dict(d=64), 2, "head_dim"), (_prefill, dict(hq=9, qs=2048), 1, "divisible"), (_prefill, dict(hq=66, qs=16384), 2, "G="),
    (_prefill, dict(qs=1016), 1, "stride"), (_prefill, dict(ks=252), 1, "stride"), (_prefill, dict(vs=260), 1, "stride"),
    (_prefill, dict(ks=1 << 24), 2, "2^23"), (_prefill, dict(dtype=5), 2, "dtype"), (_prefill, dict(tokens=-1), 1, "tokens"),
    (_prefill, dict(tokens=1 << 30, hq=8), 2, "too many"), (_prefill, dict(out=None), 1, "null"),
    (_prefill, dict(k=ctypes.c_void_p(0x1008)), 1, "aligned"), (_prefill, dict(out=FAKE), 1, "must not be k or v"),
    (_write, dict(d=64), 2, "head_dim"), (_write, dict(ps=0), 1, "page_size"), (_write, dict(ks=128), 1, "stride"),
    (_write, dict(vs=260), 1, "stride"), (_write, dict(dtype=9), 1, "dtype"), (_write, dict(slots=None), 1, "null"),
    (_write, dict(pages=1 << 30), 2, "int32"), (_write, dict(tokens=-2), 1, "tokens"), (_write, dict(k=ctypes.c_void_p(0x1008)), 1, "aligned"),
    (_write, dict(block=True, scales=None), 1, "kv_scales"), (_write, dict(block=True, scales=ctypes.c_void_p(0x1004)), 1, "kv_scales"),
    (_decode, dict(d=64), 2, "d=128"), (_decode, dict(hq=9), 1, "divisible"), (_decode, dict(hq=66), 2, "G="),
    (_decode, dict(ps=8), 2, "multiple of 16"), (_decode, dict(ps=24), 2, "multiple of 16"), (_decode, dict(cols=0), 1, "max_pages"),
    (_decode, dict(ws=None), 3, "workspace"), (_decode, dict(size=1000), 3, "workspace"), (_decode, dict(dtype=3), 2, "dtype"),
    (_decode, dict(batch=16001), 2, "16000"), (_decode, dict(cols=1 << 28), 2, "too many"), (_decode, dict(s=None), 1, "null"),
    (_decode, dict(batch=15000, cols=1 << 20), 2, "too many"), (_decode, dict(q=ctypes.c_void_p(0x1002)), 1, "aligned"),
])
def test_c_abi_refusals(call, overrides, status, text):
    assert call(**overrides) == status
    assert text in pkv_native.last_error()


@pytest.mark.parametrize("call,overrides,status,text", [
    # Launches of 2^32 threads and more, which HIP does not take.
    (_prefill, dict(batch=1 << 23, tokens=1, hkv=2), 2, "too many"),
    (_prefill, dict(batch=1, tokens=(1 << 30) - 1, hq=2, qs=256, hkv=2), 2, "too many"),
    (_write, dict(tokens=1 << 28, hkv=1), 2, "2^28"), (_write, dict(tokens=1 << 27, hkv=2), 2, "2^28"),
    (_write, dict(block=True, ps=128, tokens=1 << 28, hkv=1), 2, "2^28"),
    (_decode, dict(batch=1 << 13, hq=1 << 11, hkv=1 << 11), 2, "2^24"),
])
def test_c_abi_refuses_launches_past_the_grid(call, overrides, status, text):
    assert call(**overrides) == status
    assert text in pkv_native.last_error()


FUSED = dict(qs=1536, ks=1536, vs=1536, k=ctypes.c_void_p(0x10800), v=ctypes.c_void_p(0x10a00), q=ctypes.c_void_p(0x10000))


@pytest.mark.parametrize("overrides,text", [
    # q, k, v: column ranges of four rows of 0xc00 bytes from 0x10000 on; the output takes 0x2000 bytes
    (dict(**FUSED, out=ctypes.c_void_p(0x10000)), "must not be k or v"),            # over the first rows
    (dict(**FUSED, out=ctypes.c_void_p(0x12ff0)), "must not be k or v"),            # the last 16 bytes of v
    (dict(**FUSED, out=ctypes.c_void_p(0xe010)), "not overlap q"),                  # the first 16 bytes of q
    (dict(**{**FUSED, "k": FAKE, "v": FAKE}, out=ctypes.c_void_p(0x10000)), "not overlap q"),  # at q, whose rows lie apart
    (dict(q=ctypes.c_void_p(0x10000), out=ctypes.c_void_p(0x10800)), "not overlap q"),   # a contiguous q, one row on
    (dict(q=ctypes.c_void_p(0x10800), out=ctypes.c_void_p(0x10000)), "not overlap q"),   # and one row before
    (dict(v=ctypes.c_void_p(0x9ff0)), "must not be k or v"), (dict(k=ctypes.c_void_p(0x7810)), "must not be k or v"),
])
def test_prefill_refuses_outputs_over_its_inputs(overrides, text):
    assert _prefill(**overrides) == 1
    assert text in pkv_native.last_error()


@pytest.mark.parametrize("out", [0x1100, 0x17f0, 0x810])
def test_decode_refuses_outputs_over_a_part_of_q(out):
    assert _decode(out=ctypes.c_void_p(out)) == 1
    assert "not overlap q" in pkv_native.last_error()


def test_c_abi_empty_calls_are_no_ops():
    assert _prefill(tokens=0) == 0 and _prefill(batch=0) == 0
    assert _write(tokens=0) == 0 and _write(block=True, tokens=0) == 0
    assert _decode(batch=0) == 0


def test_workspace_size():
    lib = pkv_native.lib()
    lib.pkv_fp8_block_workspace_bytes.restype = ctypes.c_size_t
    small, large = (lib.pkv_fp8_block_workspace_bytes(b, 32, 8) for b in (1, 100))
    assert 0 < small < large and lib.pkv_fp8_block_workspace_bytes(0, 32, 8) == 0


def test_op_refusals():
    import persistentkv_torch_ext as ext
    i = lambda *s: torch.zeros(*s, dtype=I32)
    h = lambda *s: torch.zeros(*s, dtype=F16)
    with pytest.raises(RuntimeError, match="cached_lens must be a CUDA tensor"):
        ext.build_block_tables(i(2), i(2), i(4), i(1), i(2, 3), i(3), i(8), i(1), 16)
    with pytest.raises(RuntimeError, match="q has wrong dtype"):
        ext.prefill_attention(h(4, 8, 128).float(), h(4, 2, 128), h(4, 2, 128), i(2), h(4, 8, 128))
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        ext.prefill_attention(h(4, 8, 128), h(4, 2, 128), h(4, 2, 128), i(2), h(4, 8, 128))
    with pytest.raises(RuntimeError, match="k_new must be a CUDA tensor"):
        ext.write_kv(h(4, 2, 128), h(4, 2, 128), h(3, 2, 16, 128), h(3, 2, 16, 128), i(4))
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        ext.paged_attention_fp8_block(h(1, 8, 128), h(3, 2, 16, 128).to(F8), h(3, 2, 16, 128).to(F8),
                                      torch.ones(3, 2, 2), i(1, 2), i(1), h(1, 8, 128), torch.zeros(9), 16)


@pytest.mark.gpu
def test_op_refusals_on_the_gpu(ext, gpu):
    i = lambda *s: torch.zeros(*s, dtype=I32, device=gpu)
    h = lambda *s: torch.zeros(*s, dtype=F16, device=gpu)
    with pytest.raises(RuntimeError, match="token_offsets must have"):
        ext.build_block_tables(i(2), i(2), i(4), i(1), i(2, 3), i(2), i(8), i(1), 16)
    n = i(1)
    with pytest.raises(RuntimeError, match="num_free_out must not be num_free"):
        ext.build_block_tables(i(2), i(2), i(4), n, i(2, 3), i(3), i(8), n, 16)
    with pytest.raises(RuntimeError, match="contiguous heads"):
        ext.prefill_attention(h(4, 8, 256)[..., ::2], h(4, 2, 128), h(4, 2, 128), i(2), h(4, 8, 128))
    with pytest.raises(RuntimeError, match="contiguous heads"):
        ext.prefill_attention(h(8, 4, 128).transpose(0, 1), h(4, 2, 128), h(4, 2, 128), i(2), h(4, 8, 128))
    with pytest.raises(RuntimeError, match="multiple of 8"):
        ext.prefill_attention(h(4, 1028)[:, :1024].view(4, 8, 128), h(4, 2, 128), h(4, 2, 128), i(2), h(4, 8, 128))
    with pytest.raises(RuntimeError, match="aligned"):
        ext.prefill_attention(h(4, 1032)[:, 4:1028].view(4, 8, 128), h(4, 2, 128), h(4, 2, 128), i(2), h(4, 8, 128))
    with pytest.raises(RuntimeError, match="output shape"):
        ext.prefill_attention(h(4, 8, 128), h(4, 2, 128), h(4, 2, 128), i(2), h(5, 8, 128))
    with pytest.raises(RuntimeError, match="divisible"):
        ext.prefill_attention(h(4, 8, 128), h(4, 3, 128), h(4, 3, 128), i(2), h(4, 8, 128))
    with pytest.raises(RuntimeError, match="one slot a token"):
        ext.write_kv(h(4, 2, 128), h(4, 2, 128), h(3, 2, 16, 128), h(3, 2, 16, 128), i(5))
    with pytest.raises(RuntimeError, match="kv_scales must have shape"):
        ext.write_kv_fp8_block(h(4, 2, 128), h(4, 2, 128), h(3, 2, 16, 128).to(F8), h(3, 2, 16, 128).to(F8),
                               torch.ones(3, 2, device=gpu).unsqueeze(-1), i(4))
    with pytest.raises(RuntimeError, match="slot_mapping is on cpu|must be a CUDA"):
        ext.write_kv(h(4, 2, 128), h(4, 2, 128), h(3, 2, 16, 128), h(3, 2, 16, 128), torch.zeros(4, dtype=I32))
    p8 = h(3, 2, 16, 128).to(F8)
    with pytest.raises(RuntimeError, match="workspace of"):
        ext.paged_attention_fp8_block(h(1, 8, 128), p8, p8, torch.ones(3, 2, 2, device=gpu), i(1, 2), i(1),
                                      h(1, 8, 128), torch.zeros(9, device=gpu), 16)
    p8 = h(3, 2, 8, 128).to(F8)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        ext.paged_attention_fp8_block(h(1, 8, 128), p8, p8, torch.ones(3, 2, 2, device=gpu), i(1, 2), i(1),
                                      h(1, 8, 128), torch.zeros(9, device=gpu), 8)
