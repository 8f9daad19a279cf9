"""Which form a step over the 4-bit cache takes, by its sizes alone (CPU: the rules are host code of the kernels' libraries)."""
import ctypes

import pytest

from questwend_b200.kernels import ops


def plan(held, new, Hq=32, Hkv=8, hd=128, window=0):
    lens = [a + b for a, b in zip(held, new)]
    pages = [-(-n // 64) for n in lens]
    return ops._ask("attention_kv4", "qwb_kv4_plan", max(lens), max(new), window, max(pages), len(new), Hq, Hkv, hd, sum(new), sum(pages))


@pytest.mark.parametrize("held,new,read", [
    # one prompt beside single tokens: us on a B200, as rows / read back (32 query and 8 key heads of 128)
    ([0] + [4095] * 63, [4096] + [1] * 63, True),           # 10,711 / 864
    ([0] + [4095] * 63, [512] + [1] * 63, True),            # 1,187 / 470
    ([0] + [16383] * 31, [2048] + [1] * 31, True),          # 5,070 / 999
    ([0] + [4095] * 7, [512] + [1] * 7, True),              # 232 / 105
    ([0] + [1000] * 63, [128] + [1] * 63, True),            # 296 / 127
    ([0] + [500] * 31, [64] + [1] * 31, True),              # 50 / 36
    ([0] + [4095] * 15, [128] + [1] * 15, False),           # 95 / 124
    ([8000] * 8, [64] + [1] * 7, False),                    # 105 / 136
    # equal ones
    ([4095] * 8, [1] * 8, False), ([16383] * 32, [1] * 32, False), ([8192] * 4, [6] * 4, False), ([0], [4096], True), ([5000] * 3, [900] * 3, True)])
def test_a_step_goes_by_the_tokens_that_it_has(held, new, read):
    """Not by its longest sequence times their number."""
    assert bool(plan(held, new) & 1) is read


def pieces(T, B, max_new, max_len, Hq, Hkv, hd, window=0, most=64):
    ask = ops._lookup("attention_tc", "qwb_attn_tc_pieces")[1]
    ask.restype = ctypes.c_longlong
    tiles, n = divmod(ask(T, B, max_new, max_len, Hq, Hkv, hd, window, most), 2 ** 32)
    return n, tiles


def test_pieces_of_unequal_steps():
    """Single tokens beside a prompt leave SMs idle as few sequences do: keys are cut; a grid that is full cuts nothing; no grid is larger than it may be."""
    assert pieces(519, 8, 512, 4096, 32, 8, 128)[0] > 1 and pieces(4159, 64, 4096, 4096, 32, 8, 128)[0] == 1
    assert pieces(64, 1, 64, 60000, 32, 8, 128)[0] > 8
    for B in (1, 7, 60, 1100, 1183, 60000):
        for T in (B, 3 * B, B + 500):
            for max_new in (1, 3, T - B + 1):
                for hd in (64, 128):
                    n, tiles = pieces(T, B, max_new, 100000, 1, 1, hd)
                    assert n >= 1 and n * B <= 65535 and n * tiles >= 100000 // 64 + 1


@pytest.mark.parametrize("B,Hq,Hkv", [(0, 32, 8), (1, 0, 8), (1, 8, 0), (0, 0, 0), (1, 4, 8)])
def test_a_step_without_sequences_or_heads_is_no_division_by_0(B, Hq, Hkv):
    assert ops._ask("attention_kv4", "qwb_kv4_plan", 100, 50, 0, 2, B, Hq, Hkv, 64, 50, 3) & 7 == 4


def test_heads_go_a_few_at_a_time_where_memory_is_bounded(monkeypatch):
    monkeypatch.setattr(ops, "KV4_WORK_BYTES", 1000)
    assert [ops._heads_at_once(8, each) for each in (1, 125, 126, 250, 251, 333, 334, 500, 501, 1000, 1001, 10 ** 12)] == [8, 8, 4, 4, 3, 3, 2, 2, 1, 1, 1, 1]
    assert ops._heads_at_once(1, 10 ** 12) == 1 and ops._heads_at_once(7, 0) == 7
    assert pieces(64, 1, 64, 60000, 32, 8, 128, most=4)[0] <= 4 and pieces(64, 1, 64, 60000, 32, 8, 128, most=1)[0] == 1
