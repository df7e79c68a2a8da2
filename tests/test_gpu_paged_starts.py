"""Starts that run backwards: the sequences that are passed over take none of the others' tokens along."""
import numpy as np
import pytest
import torch

from tests.paged_gpu import Setup, dev_empty, f32_dev, i32, orc, po, to_dev, to_host

pytestmark = pytest.mark.gpu
BF16 = po.DT_BFLOAT16
ROWS = 400  # of the rotary table


def batch_of(seed, starts, lens, tokens, eight):
    """A sequence to each pair of neighbours in starts, in order or not; every one has its own pages."""
    s = Setup(seed, [(n, 1) for n in lens], 2, 2, BF16, eight, 16)
    s.starts, s.tokens = np.array(starts, dtype=np.int32), tokens
    s.lens = np.array([lens[b] for b in range(len(lens))], dtype=np.int32)
    s.q = orc.round_to(np.random.default_rng(seed).standard_normal((tokens, s.H, 128)).astype(np.float32), BF16)
    return s


def whole(s):
    """(sequence, its tokens) of those that are worked on"""
    pairs = [(b, int(s.starts[b]), int(s.starts[b + 1])) for b in range(s.batch)]
    return [(b, range(i0, i1)) for b, i0, i1 in pairs if 0 <= i0 <= i1 <= s.tokens and 0 <= s.lens[b] <= s.pps * s.ps]


# the lengths leave room behind them in a sequence's last page, where a token of another sequence would go
BATCHES = [([0, 2, 100, 4, 6, 8], [40, 41, 42, 43, 44], 8),             # an end far behind the tensors, and a start there
           ([0, 3, -7, 3, 9], [20, 33, 51, 60], 9),                     # a start before them
           ([2, 5, 0, 2], [20, 37, 18], 5),                             # two runs of tokens, the later first
           ([0, 1, 2, 1 << 30, 2, 3, 4], [17, 18, 19, 20, 21, 22], 4),
           ([0, *range(1, 90), 2 ** 31 - 1, *range(90, 150)], [20 + b % 9 for b in range(150)], 149)]  # past what a wave looks at at once


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("starts,lens,tokens", BATCHES)
def test_append(starts, lens, tokens, eight):
    s = batch_of(1, starts, lens, tokens, eight)
    table = orc.init_freq_cis(128, ROWS, 1e4, BF16)
    rng = np.random.default_rng(2)
    k, v = (orc.round_to(rng.standard_normal((tokens, 2, 128)).astype(np.float32), BF16) for _ in range(2))
    s.to_gpu()
    out = s.out()
    s.append(out, f32_dev(table), to_dev(s.q), to_dev(k), to_dev(v), True)
    want = np.full_like(s.q, 0x5A5A)
    for b, mine in whole(s):
        for t in mine:
            p = int(s.lens[b]) - mine.stop + t
            want[t] = orc.rope(s.q[t:t + 1], table, p, True, BF16)[0]
            at = po.place(s.table[b], s.num_pages, s.ps, p)
            s.k.put(*at, orc.rope(k[t:t + 1], table, p, True, BF16)[0])
            s.v.put(*at, v[t])
    assert np.array_equal(to_host(out), want)
    assert np.array_equal(s.d_k.cpu().numpy(), s.k.raw)
    assert np.array_equal(s.d_v.cpu().numpy(), s.v.raw)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("starts,lens,tokens", BATCHES)
@pytest.mark.parametrize("more", [0, 2500])  # rows that are no sequence's, behind the others: several tokens to a workgroup
def test_read(starts, lens, tokens, more, eight):
    if more and (np.array(starts) > tokens).any():
        starts = [2 ** 31 - 1 if x > tokens else x for x in starts]
    s = batch_of(3, starts, lens, tokens + more, eight)
    s.to_gpu()
    outs = [torch.full((s.tokens, 2, 128), 0x5A5A, dtype=torch.int16, device="cuda") for _ in range(2)]
    s.read(*outs)
    for out, pool in zip(outs, (s.k, s.v)):
        bits = to_host(out)
        mine = np.zeros(s.tokens, dtype=bool)
        for b, tokens_of in whole(s):
            for t in tokens_of:
                mine[t] = True
                got = orc.widen(bits[t], BF16).astype(np.float64)
                assert np.array_equal(got, pool.get(*po.place(s.table[b], s.num_pages, s.ps, int(s.lens[b]) - tokens_of.stop + t)))
        assert mine.any() and (bits[~mine] == 0x5A5A).all()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("starts,lens,tokens", BATCHES)
def test_append_then_attend(starts, lens, tokens, eight):
    """A step of the sequences that are whole is what it is without the others."""
    s = batch_of(4, starts, lens, tokens, eight)
    table = f32_dev(orc.init_freq_cis(128, ROWS, 1e4, BF16))
    rng = np.random.default_rng(5)
    k, v = (to_dev(orc.round_to(rng.standard_normal((tokens, 2, 128)).astype(np.float32), BF16)) for _ in range(2))
    s.to_gpu()
    rotated, out = s.out(), s.out()
    s.append(rotated, table, to_dev(s.q), k, v, True)
    s.attend(out, q=rotated, max_q=6)
    for b, mine in whole(s):
        if len(mine) == 0:
            continue
        alone = batch_of(4, starts, lens, tokens, eight).to_gpu()  # the pools as they were
        alone.batch = 1
        alone.d_starts, alone.d_lens, alone.d_table = i32([mine.start, mine.stop]), i32([alone.lens[b]]), i32(alone.table[b:b + 1])
        q_alone, o_alone = dev_empty(tuple(rotated.shape)), dev_empty(tuple(out.shape))
        alone.append(q_alone, table, to_dev(alone.q), k, v, True)
        alone.attend(o_alone, q=q_alone, max_q=6)
        part = slice(mine.start, mine.stop)
        assert torch.equal(rotated[part], q_alone[part]) and torch.equal(out[part], o_alone[part])
        if b > 20:
            break
