"""V that is not finite in some dims of some keys: what each row sees of them and no more, every other dim as it was, and in about the time of a call
without them."""
import numpy as np
import pytest
import torch

from tests.paged_gpu import Setup, po, to_host

pytestmark = pytest.mark.gpu
FP16, BF16 = po.DT_FLOAT16, po.DT_BFLOAT16
MANY = 1 << 16  # a bound on the keys that leads to wide tiles
BITS = {BF16: {"nan": 0x7FC0, "inf": 0x7F80, "-inf": 0xFF80}, FP16: {"nan": 0x7E00, "inf": 0x7C00, "-inf": 0xFC00}}


def poison(s, b, key, dims, what):
    page, row = po.place(s.table[b], s.num_pages, s.ps, key)
    if s.v.eight:
        s.v.rows_of(page)[:, row, dims] = 0x7F
    else:
        s.v.rows_of(page).view(np.uint16)[:, row, dims] = BITS[s.dt][what]


def visible(s, b, key, window, sinks):
    """[tokens]: whether each sees a key of sequence b."""
    sees = np.zeros(s.tokens, dtype=bool)
    for t in range(s.starts[b], s.starts[b + 1]):
        p = s.lens[b] - s.starts[b + 1] + t
        sees[t] = key <= p and (window == 0 or key > p - window or key < sinks)
    return sees


# lengths, group, kv heads, window, sinks, bound on the keys, keys with such a V
CASES = [
    ([(150, 150), (70, 70)], 3, 2, 0, 0, None, [(0, 0), (0, 77), (1, 69), (1, 31)]),          # prompts in tiles
    ([(300, 60), (200, 1), (64, 3)], 7, 1, 0, 0, None, [(0, 250), (0, 299), (1, 5), (2, 62)]),  # tiles and few rows in one launch
    ([(1500, 40)], 7, 1, 0, 0, None, [(0, 3), (0, 1470)]),                                     # tiles in parts
    ([(1500, 40)], 7, 1, 700, 20, None, [(0, 10), (0, 19), (0, 20), (0, 770), (0, 1480)]),      # the edges of a window and of sinks
    ([(400, 80)], 6, 1, 0, 0, MANY, [(0, 330), (0, 399)]),                                     # wide tiles
    ([(1300, 20), (900, 20)], 7, 1, 300, 0, MANY, [(0, 985), (0, 1295), (1, 590)]),
    ([(500, 4), (40, 4), (4, 4)], 4, 2, 0, 0, None, [(0, 0), (0, 498), (1, 38), (2, 1), (2, 3)]),  # few rows
    ([(2000, 3)], 5, 1, 0, 0, None, [(0, 100), (0, 1998)]),                                    # few rows in parts
    ([(700, 1), (1500, 1), (90, 2)], 3, 2, 200, 3, None, [(0, 2), (0, 3), (0, 499), (0, 500), (1, 1299), (1, 1300), (2, 88)]),
    ([(130, 1), (2500, 1)], 4, 2, 0, 0, None, [(0, 4), (1, 1111)]),                             # one row that sees all of them
]


# (8 bits have no infinities)
@pytest.mark.parametrize("dt,eight,what", [(dt, False, what) for dt in (BF16, FP16) for what in ("nan", "inf", "-inf")] + [(BF16, True, "nan"), (FP16, True, "nan")])
@pytest.mark.parametrize("lengths,group,kv_heads,window,sinks,max_kv,at", CASES)
def test_some_dims_of_some_keys(lengths, group, kv_heads, window, sinks, max_kv, at, dt, eight, what):
    s = Setup(1, lengths, group, kv_heads, dt, eight, 16)
    want, tol, _ = s.expected(window, sinks)
    bad = np.zeros((s.tokens, 128), dtype=bool)
    for i, (b, key) in enumerate(at):
        dims = [0, 31, 127] if i == 0 else [5 * i, 64 + i]
        poison(s, b, key, dims, what)
        bad[np.ix_(visible(s, b, key, window, sinks), dims)] = True
    assert bad.any() and not bad.all(-1).any()
    s.to_gpu()
    out = s.out()
    s.attend(out, window, sinks, max_kv=max_kv)
    got = po.orc.widen(to_host(out), dt).astype(np.float64)
    bad = np.broadcast_to(bad[:, None], got.shape)
    assert not np.isfinite(got[bad]).any()
    assert (np.abs(got - want)[~bad] <= tol[~bad]).all()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("lengths,group,window,first", [([(300, 200)], 3, 0, 170), ([(900, 8)], 2, 0, 896), ([(700, 100)], 2, 90, 650), ([(600, 3)], 4, 64, 598)])
def test_all_of_a_sequences_last_keys(lengths, group, window, first, eight):
    """What a model leaves that went wrong at some token: all of K and V from there on.  Nobody before it is concerned, nor is the next sequence."""
    s = Setup(2, lengths + [(150, 40), (80, 1)], group, 2, BF16, eight, 16)
    want, tol, _ = s.expected(window, 0)
    n = s.lens[0]
    for key in range(first, n):
        poison(s, 0, key, slice(None), "nan")
        page, row = po.place(s.table[0], s.num_pages, s.ps, key)
        if eight:
            s.k.rows_of(page)[:, row] = 0x7F
        else:
            s.k.rows_of(page).view(np.uint16)[:, row] = 0x7FC0
    sees = visible(s, 0, first, window, 0)
    for key in range(first, n):
        sees |= visible(s, 0, key, window, 0)
    assert sees.any() and not sees.all()
    s.to_gpu()
    out = s.out()
    s.attend(out, window, 0)
    got = po.orc.widen(to_host(out), BF16).astype(np.float64)
    assert np.isnan(got[sees]).all()
    assert (np.abs(got - want)[~sees] <= tol[~sees]).all()


@pytest.mark.parametrize("lengths,group,max_kv", [([(300, 1)], 4, None), ([(300, 300)], 3, None), ([(400, 60), (300, 2)], 3, MANY)])
def test_values_near_the_largest(lengths, group, max_kv):
    """Finite V whose weighted sum is within 32 bits, if no weight is above 1, and is not with a reference that trails the maximum."""
    s = Setup(3, lengths, group, 1, BF16, False, 16)
    for page in range(s.num_pages):
        rows = s.v.rows_of(page).view(np.uint16)
        rows[:] = po.orc.round_to((2.0 ** 122 * (1 + (np.abs(po.orc.widen(rows, BF16)) % 1))).astype(np.float32), BF16)
    most, trailing = 0.0, 0.0
    q = po.orc.widen(s.q, BF16).astype(np.float64)
    for b, n in enumerate(s.lens):
        k, _ = po.sequence_rows(s.k, s.table[b], n)
        v, _ = po.sequence_rows(s.v, s.table[b], n)
        for t in range(s.starts[b], s.starts[b + 1]):
            p = n - s.starts[b + 1] + t
            scores = q[t] @ k[:p + 1, 0].T / np.sqrt(128)
            sums = np.exp(scores - scores.max(-1, keepdims=True)) @ v[:p + 1, 0]
            most = max(most, sums.max())
            trailing = max(trailing, (sums * np.exp(scores.max(-1) - scores[:, :64].max(-1))[:, None]).max())
    assert most < 2.0 ** 127.9 and (trailing > 2.0 ** 128 or s.max_q == 1)
    expected = s.expected()
    s.to_gpu()
    out = s.out()
    s.attend(out, max_kv=max_kv)
    s.check(out, expected=expected)


def time_of(call, times):
    call()
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    start.record()
    for _ in range(times):
        call()
    end.record()
    torch.cuda.synchronize()
    return start.elapsed_time(end) / times


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("lengths,group,kv_heads,window", [([(1500, 700)], 7, 2, 0), ([(4000, 3)], 5, 2, 0), ([(4000, 40)], 7, 1, 0), ([(4000, 1)], 4, 2, 1000)])
def test_takes_no_more_than_some_calls(lengths, group, kv_heads, window, eight):
    """All rows see a key with a NaN in one dim.  A second pass of a wave by itself takes some of the first one's times; row by row and key by key, 32 or 16 rows one
    after the other, it was more than a hundred."""
    s = Setup(4, lengths, group, kv_heads, BF16, eight, 16).to_gpu()
    ws, out = s.workspace(window), s.out()
    clean = time_of(lambda: s.attend(out, window, ws=ws), 20)
    for key in range(s.lens[0] - 1000, s.lens[0], 10):
        poison(s, 0, key, [7], "nan")
    s.to_gpu()
    bad = time_of(lambda: s.attend(out, window, ws=ws), 3)
    assert np.isnan(po.orc.widen(to_host(out)[-1], BF16)[:, 7]).all()
    assert bad < 40 * clean, f"{bad * 1e3:.0f} us, without {clean * 1e3:.0f}"
