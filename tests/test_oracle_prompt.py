"""Pins of oracle/prompt.py: hand-worked tables and slots, the decode oracle, torch's e4m3 cast."""
import numpy as np
import pytest
import torch

from oracle import attention, prompt
from prompt_cases import shortage_and_retry


def test_tables_by_hand():
    # pages of 4; row 0 holds 5 tokens (2 pages) and gets 4 more, row 1 is new with 3 tokens,
    # row 2 gets none, row 3 fills its two columns and goes past them
    table = [[7, 8, -5, -5], [-5] * 4, [9, -5, -5, -5], [-5] * 4]
    t, off, slots, left = prompt.build_block_tables(
        [5, 0, 2, 0], [9, 3, 2, 18], [10, 11, 12, 13, 14, 15, 16], 7, table, 32, 4)
    assert off.tolist() == [0, 4, 7, 7, 25]
    assert t.tolist() == [[7, 8, 16, -5], [15, -5, -5, -5], [9, -5, -5, -5], [14, 13, 12, 11]]
    assert left == 1
    assert slots[:7].tolist() == [33, 34, 35, 64, 60, 61, 62]
    assert slots[7:23].tolist() == [4 * p + i for p in (14, 13, 12, 11) for i in range(4)]
    assert slots[23:].tolist() == [-1] * 9


def test_tables_run_out():
    t, _, slots, left = prompt.build_block_tables([0, 0], [4, 9], [3, 4], 2, [[-7] * 3] * 2, 13, 4)
    assert t.tolist() == [[4, -7, -7], [3, -1, -1]] and left == -2
    assert slots.tolist() == [16, 17, 18, 19, 12, 13, 14, 15] + [-1] * 5


def test_tables_after_a_shortage():
    shortage_and_retry(lambda *a: [x.tolist() if hasattr(x, "tolist") else x for x in prompt.build_block_tables(*a)])


@pytest.mark.parametrize("lengths,hq,hkv", [([1, 5, 33], 4, 2), ([7], 3, 1)])
def test_prefill_last_token_is_a_decode_step(lengths, hq, hkv):
    rng = np.random.default_rng(0)
    n = sum(lengths)
    q, k, v = (rng.standard_normal((n, h, 128)) for h in (hq, hkv, hkv))
    off = np.concatenate([[0], np.cumsum(lengths)])
    out, *_ = prompt.prefill(q, k, v, off)
    for s, e in zip(off, off[1:]):
        for i in (s, e - 1):  # the first token attends to itself, the last to all
            ref = attention.attention_fp64(torch.tensor(q[i]), torch.tensor(k[s:i + 1]).transpose(0, 1),
                                           torch.tensor(v[s:i + 1]).transpose(0, 1))
            assert np.abs(out[i] - np.asarray(ref)).max() < 1e-12


def test_prefill_spreads_nonfinite_values_forward_only():
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal((6, 1, 128)) for _ in range(3))
    v[3, 0, 5], v[4, 0, 6], v[2, 0, 6] = np.nan, np.inf, -np.inf
    out, *_ = prompt.prefill(q, k, v, [0, 6])
    assert np.isfinite(out[:3, 0, 5]).all() and np.isnan(out[3:, 0, 5]).all()
    assert np.isfinite(out[:2, 0, 6]).all() and (out[2:4, 0, 6] == -np.inf).all() and np.isnan(out[4:, 0, 6]).all()


def test_e4m3_round_is_torchs_cast():
    codes = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    for scale in (1.0, 2.0 ** -5, 2.0 ** 7):
        x = codes.double() * scale
        want = x.float().clamp(-448, 448).to(torch.float8_e4m3fn).double().numpy()
        got = prompt.e4m3_round(x.numpy())
        assert (np.isnan(got) == np.isnan(want)).all()
        assert (got[~np.isnan(want)] == want[~np.isnan(want)]).all()


def test_power_of_two():
    assert [prompt.power_of_two(x) for x in (0.0, 1.0, 1.0001, 0.5, 3.0, 2.0 ** -70, 2.0 ** 70)] == \
        [2.0 ** -60, 1.0, 2.0, 0.5, 4.0, 2.0 ** -60, 2.0 ** 60]


def test_block_write_grows_a_scale():
    pages, scales = np.zeros((2, 1, 16, 128)), np.array([[1.0], [0.25]])
    pages[1, 0, 0, :2] = [448.0, 2.0 ** -9]
    new = np.zeros((1, 1, 128))
    new[0, 0, 0] = 449.0  # needs a scale of 2
    got, s = prompt.write_kv_fp8_block(pages, scales, new, [16 + 1])
    assert s.tolist() == [[1.0], [2.0]]
    assert got[1, 0, 0, :2].tolist() == [56.0, 0.0]  # an eighth; the smallest subnormal underflows
    assert got[1, 0, 1, 0] == 224.0  # 224.5 to a step of 16


@pytest.mark.parametrize("slots", [[5, 7], [7, 6], [3, 20, 4], [3, -1, 4], [3, 3]], ids=str)
def test_block_write_takes_a_page_as_one_run(slots):
    """Without gaps, in order and in one place: what the operator's header asks for."""
    with pytest.raises(ValueError, match="one run of consecutive slots"):
        prompt.write_kv_fp8_block(np.zeros((2, 1, 16, 128)), np.ones((2, 1)), np.ones((len(slots), 1, 128)), slots)
    prompt.write_kv_fp8_block(np.zeros((2, 1, 16, 128)), np.ones((2, 1)), np.ones((5, 1, 128)), [14, 15, -1, 16, 17])


def test_block_decode_matches_the_decode_oracle():
    rng = np.random.default_rng(2)
    k, v = (prompt.e4m3_round(rng.standard_normal((5, 2, 16, 128)) * 50) for _ in range(2))
    scales = 2.0 ** rng.integers(-8, 3, (5, 2, 2))
    q = rng.standard_normal((2, 4, 128))
    table = np.array([[4, 1, 0], [2, 3, 2]])
    out, *_ = prompt.fp8_block_decode(q, k, v, scales, table, [40, 17])
    kk, vv = k * scales[:, :, :1, None], v * scales[:, :, 1:, None]
    for b, n in ((0, 40), (1, 17)):
        kr, vr = attention.gather_row(torch.tensor(kk), torch.tensor(vv), torch.tensor(table[b]), n)
        ref = attention.attention_fp64(torch.tensor(q[b]), kr, vr)
        assert np.abs(out[b] - np.asarray(ref)).max() < 1e-12
