"""Sizes at the ends of 32 bits are refused before any device work."""
import pytest

import pkv_native
from test_turn_refusals import _rope, _write

MOST = 2 ** 31 - 1


@pytest.mark.parametrize("call", [_rope, _write])
@pytest.mark.parametrize("overrides", [
    dict(tokens=MOST), dict(tokens=MOST - 2), dict(tokens=MOST - 3), dict(tokens=1 << 30),
    dict(hq=MOST, qs=MOST * 128 + 128, qos=MOST * 128 + 128), dict(hkv=MOST, ks=MOST * 128 + 128, kos=MOST * 128 + 128, vs=MOST * 128 + 128),
    dict(tokens=1, hkv=MOST - 2, ks=MOST * 128 + 128, kos=MOST * 128 + 128, vs=MOST * 128 + 128),
])
def test_tokens_and_heads_of_norm_rope(call, overrides):
    if call is _write:
        overrides = {k: v for k, v in overrides.items() if k != "kos"}
    elif "vs" in overrides:
        overrides = {k: v for k, v in overrides.items() if k != "vs"}
    assert call(**overrides) == 2
    assert "too many tokens or heads" in pkv_native.last_error()
