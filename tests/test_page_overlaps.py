"""The page operators refuse a call that writes what it reads, or two things in one place."""
import itertools

import pytest

import pkv_native
from test_turn_refusals import _compact, _fork, _free

# Every tensor apart from the others: 9 pages, 4 rows of 3 columns, 2 rows listed, 4 moves.
FORK = dict(zip("parents children lens table shares free num left src dst".split(), itertools.count(0x100000, 0x1000)))
FREE = dict(zip("rows lens table shares free num left ws".split(), itertools.count(0x100000, 0x1000)), size=8)
COMPACT = dict(zip("table shares free num map to so fo left src dst ws".split(), itertools.count(0x100000, 0x1000)), size=8)
NAMES = {"left": "num_free_out", "src": "copy_src", "dst": "copy_dst", "shares": "page_shares", "free": "free_pages", "num": "num_free",
         "ws": "workspace", "map": "page_map", "to": "block_table_out", "so": "page_shares_out", "fo": "free_pages_out", "table": "block_table"}
BYTES = {"parents": 8, "children": 8, "rows": 8, "lens": 16, "table": 48, "to": 48, "shares": 36, "free": 36, "num": 4, "left": 4,
         "map": 36, "so": 36, "fo": 36, "ws": 8}


def _bytes(name, call):
    return BYTES.get(name, 8 if call is _fork else 16)  # src, dst


CALLS = [(_fork, FORK, "left src dst table shares"), (_free, FREE, "ws left shares free"),
         (_compact, COMPACT, "ws map so fo left src dst to")]
PAIRS = [(call, a, w, o) for call, a, written in CALLS for w in written.split() for o in a if o not in (w, "size")
         and not (call is _compact and {w, o} == {"to", "table"})]


@pytest.mark.parametrize("call,args,w,o", PAIRS, ids=lambda x: x if isinstance(x, str) else "")
def test_overlaps(call, args, w, o):
    last = args[o] + _bytes(o, call) - 4  # the other's last entry
    assert call(**{**args, w: last}) == 1
    text = pkv_native.last_error()
    assert "must not" in text and all(NAMES.get(x, x) in text for x in (w, o)), text


@pytest.mark.parametrize("shift", [4, 44, -44])
def test_a_table_beside_itself(shift):
    assert _compact(**{**COMPACT, "to": COMPACT["table"] + shift}) == 1
    assert "block_table_out must not overlap block_table" in pkv_native.last_error()
