"""The ctypes declarations of the calls for a further turn follow include/pkv.h, so that plain Python
numbers go out in the width that the library reads."""
import ctypes
import re

import pytest

import pkv_native

NAMES = ["pkv_norm_rope", "pkv_norm_rope_write_kv", "pkv_fork_rows", "pkv_free_rows", "pkv_compact_pages", "pkv_copy_pages",
         "pkv_page_workspace_bytes", "pkv_paged_prefill_attention", "pkv_paged_prefill_workspace_bytes"]
TYPES = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "size_t": ctypes.c_size_t, "int": ctypes.c_int, "float": ctypes.c_float}


@pytest.mark.parametrize("name", NAMES)
def test_declared_as_in_the_header(name):
    with open(pkv_native.HEADER_PATH) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    result, args = re.search(rf"(\w+)\s+{name}\(([^)]*)\)", text).groups()
    f = getattr(pkv_native.lib(), name)
    want = [ctypes.c_void_p if "*" in a else TYPES[a.split()[0]] for a in args.split(",")]
    assert f.restype == TYPES[result] and f.argtypes == want
