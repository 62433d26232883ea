"""The ctypes declarations of the calls between a prompt and the cache follow include/pkv.h, so that
plain Python integers go out in the width that the library reads."""
import ctypes
import re

import pytest

import pkv_native

NAMES = ["pkv_build_block_tables", "pkv_prefill_attention", "pkv_write_kv", "pkv_write_kv_fp8_block",
         "pkv_paged_attention_fp8_block", "pkv_fp8_block_workspace_bytes"]
TYPES = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "size_t": ctypes.c_size_t, "int": ctypes.c_int}


def _prototype(name):
    with open(pkv_native.HEADER_PATH) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    result, args = re.search(rf"(\w+)\s+{name}\(([^)]*)\)", text).groups()
    kind = lambda a: ctypes.c_void_p if "*" in a else TYPES[a.split()[0]]
    return TYPES[result], [kind(a) for a in args.split(",")]


@pytest.mark.parametrize("name", NAMES)
def test_declared_as_in_the_header(name):
    f = getattr(pkv_native.lib(), name)
    assert (f.restype, f.argtypes) == _prototype(name)


def test_strides_go_out_in_64_bits():
    lib, at = pkv_native.lib(), 0x1000  # never dereferenced: validation fails first
    wide = (1 << 32) + 256  # 256 in its lower half, a valid stride
    assert lib.pkv_prefill_attention(at, 1024, at, wide, at, 256, at, 0x8000, 1, 4, 8, 2, 128, 0, None) == 2
    assert "2^23" in pkv_native.last_error()
    assert lib.pkv_write_kv(at, 256, at, 256 - (1 << 32), at, at, at, 4, 2, 128, 3, 16, 0, None) == 1
    assert "stride must hold" in pkv_native.last_error()
