"""Which kernel the sizes of the GPU tests go by: each is reached by those that are there for it (no GPU: 256 compute units are counted with)."""
import pytest

import llm_simple_amd.bench_ops as bops
from tests import test_gpu_paged_attention as attention
from tests import test_gpu_paged_not_finite as not_finite
from tests import test_gpu_paged_runs as runs
from tests import test_gpu_paged_wide as wide

FEW, RUNS, TILES, WIDE, BOTH = range(5)


def kind(lengths, group, kv_heads, eight, window=0, sinks=0, max_q=None, max_kv=None):
    return bops.lib.llmhip_bench_paged_attn_kind(
        sum(m for _, m in lengths), len(lengths), max_q or max(1, max(m for _, m in lengths)), max(n for n, _ in lengths) if max_kv is None else max_kv, window, sinks, group,
        kv_heads, int(eight))


def cases(test, names):
    """The sizes that a test is parametrised with."""
    mark, = [m for m in test.pytestmark if m.name == "parametrize" and m.args[0] == names]
    return mark.args[1]


def test_decode():
    for group, kv_heads in cases(attention.test_decode, "group,kv_heads"):
        assert kind(attention.DECODE, group, kv_heads, False) == FEW
    assert kind(attention.LONG, 4, 2, True) == FEW


def test_runs():
    for kv_heads, lengths, window, sinks, eight in cases(attention.test_decode_in_runs, "kv_heads,lengths,window,sinks,eight"):
        assert kind(lengths, 1, kv_heads, eight, window, sinks) == RUNS
    assert kind([(runs.MOST, 1)] * runs.BATCH, 1, runs.KV_HEADS, True) == RUNS
    assert kind([(runs.MOST, 1)] * runs.BATCH, 1, runs.KV_HEADS, False) == RUNS


def test_tiles():
    for group, kv_heads, _ in cases(attention.test_chunks, "group,kv_heads,page_size"):
        assert kind(attention.CHUNKS, group, kv_heads, False) == (BOTH if group <= 16 else TILES)
    for lengths in cases(attention.test_chunks_in_splits, "lengths"):
        assert kind(lengths, 6, 1, False) == (TILES if len(lengths) == 1 else BOTH)


def test_wide():
    for eight in (False, True):
        for group, kv_heads, lengths in cases(wide.test_lengths, "group,kv_heads,lengths"):
            assert kind(lengths, group, kv_heads, eight, max_kv=wide.MANY) == WIDE
        for group, lengths, _ in cases(wide.test_values_that_are_not_finite_for_some_rows, "group,lengths,key"):
            assert kind(lengths, group, 2, eight, max_kv=wide.MANY) == WIDE
        assert kind([(1300, 30), (20, 30), (0, 30)], 5, 2, eight, max_kv=wide.MANY) == WIDE
        assert kind([(1500, 40), (900, 40)], 6, 1, eight, max_kv=wide.MANY) == WIDE
    (group, lengths, window, sinks), prompt = cases(wide.test_many_kv_heads, "group,lengths,window,sinks")
    assert kind(lengths, group, 128, False, window, sinks) == WIDE
    assert kind(prompt[1], prompt[0], 128, True) == WIDE and kind(prompt[1], prompt[0], 128, False) == TILES


def test_values_that_are_not_finite():
    seen = set()
    for lengths, group, kv_heads, window, sinks, max_kv, _ in not_finite.CASES:
        seen.add(kind(lengths, group, kv_heads, False, window, sinks, max_kv=max_kv))
    assert seen >= {FEW, TILES, WIDE, BOTH}


@pytest.mark.parametrize("bad", range(9))
def test_refused(bad):
    args = [1, 1, 1, 100, 0, 0, 1, 1, 0]
    args[bad] = -1
    # (a window below 1 is none, and 8 bits are any number but 0)
    assert (bops.lib.llmhip_bench_paged_attn_kind(*args) < 0) == (bad not in (4, 8))
