"""Sizes at the ends of 32 bits are refused before any device work."""
import pytest

import pkv_native
from test_prompt_refusals import _write as _write_kv
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


@pytest.mark.parametrize("tokens", [MOST, MOST - 14, MOST - 40])
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("heads", [1, 2])
def test_tokens_of_block_scaled_writes(tokens, page, heads):
    assert _write_kv(block=True, tokens=tokens, hkv=heads, ps=page) == 2
    assert "too large" in pkv_native.last_error()
