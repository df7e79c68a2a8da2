"""Wide tiles of the attention over pages: bounds that lead to them, with lengths that a test can work out."""
import numpy as np
import pytest
import torch

from tests.paged_gpu import Setup, po, to_host

pytestmark = pytest.mark.gpu
FP16, BF16 = po.DT_FLOAT16, po.DT_BFLOAT16
MANY = 1 << 16  # keys that the host counts with: enough for wide tiles of one kv head or two to be work for the chip


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("group,kv_heads,lengths", [
    (7, 2, [(1300, 20)]), (6, 1, [(1500, 80), (900, 80)]), (1, 2, [(300, 129), (130, 129), (129, 129)]), (130, 1, [(700, 1), (1, 1), (65, 1)]),
    (40, 1, [(90, 19)])])
def test_lengths(group, kv_heads, lengths, dt, eight):
    s = Setup(1, lengths, group, kv_heads, dt, eight, 16).to_gpu()
    out = s.out()
    s.attend(out, max_kv=MANY)
    s.check(out)


@pytest.mark.parametrize("eight", [False, True])
def test_pages_that_are_not_there_and_rows_before_the_first(eight):
    s = Setup(2, [(1300, 30), (20, 30), (0, 30)], 5, 2, BF16, eight, 16)
    s.table[0, 1], s.table[0, 4], s.table[0, 80], s.table[0, 33:39] = -1, s.num_pages, 2 ** 31 - 1, -2 ** 31
    s.to_gpu()
    out = s.out()
    s.attend(out, max_kv=MANY)
    s.check(out)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("group,lengths,key", [(7, [(1300, 20)], 1290), (3, [(200, 45)], 170)])
def test_values_that_are_not_finite_for_some_rows(group, lengths, key, eight):
    s = Setup(3, lengths, group, 2, BF16, eight, 16)
    want, tol, _ = s.expected()
    sees = s.lens[0] - s.tokens + np.arange(s.tokens) >= key
    assert sees.any() and not sees.all()
    page, row = po.place(s.table[0], s.num_pages, 16, key)
    if eight:
        s.v.rows_of(page)[:, row] = 0x7F
    else:
        s.v.rows_of(page)[:, row].view(np.uint16)[:] = 0x7FC0
    s.to_gpu()
    out = s.out()
    s.attend(out, max_kv=MANY)
    got = po.orc.widen(to_host(out), BF16).astype(np.float64)
    assert np.isnan(got[sees]).all()
    assert (np.abs(got - want)[~sees] <= tol[~sees]).all()


class Heads:
    """Some kv heads of a pool."""

    def __init__(self, pool, heads):
        self.pool, self.heads, self.h, self.n, self.ps = pool, heads, len(heads), pool.n, pool.ps

    def get(self, page, row):
        return self.pool.get(page, row)[self.heads]


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("group,lengths,window,sinks", [(1, [(1300, 130)], 800, 20), (2, [(380, 380)], 0, 0)])
def test_many_kv_heads(group, lengths, window, sinks, eight):
    """A window that hides keys, and a prompt (wide in 8 bits); two of the heads are looked at."""
    s = Setup(4, lengths, group, 128, BF16, eight, 64).to_gpu()
    out = s.out()
    s.attend(out, window, sinks)
    kv = [3, 127]
    heads = [h * group + i for h in kv for i in range(group)]
    want, tol, _ = po.attend(s.q[:, heads], Heads(s.k, kv), Heads(s.v, kv), s.table, s.starts, s.lens, s.dt, group, window, sinks)
    got = po.orc.widen(to_host(out)[:, heads], BF16).astype(np.float64)
    assert (np.abs(got - want) <= tol).all()


def test_captured_and_replayed_with_other_lengths():
    s = Setup(5, [(1500, 40), (900, 40)], 6, 1, BF16, True, 16).to_gpu()
    ws, out = s.workspace(max_kv=MANY), s.out()
    s.attend(out, max_kv=MANY, ws=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        s.attend(out, max_kv=MANY, ws=ws, stream=torch.cuda.current_stream().cuda_stream)
    for lens, middle in (((1500, 900), 40), ((40, 1), 40), ((1333, 800), 3), ((1500, 900), 80)):
        s.lens, s.starts = np.array(lens, dtype=np.int32), np.array([0, middle, 80], dtype=np.int32)
        if middle > 40 or 80 - middle > 40:  # (more tokens than the bound: passed over)
            keep = [b for b in (0, 1) if s.starts[b + 1] - s.starts[b] <= 40]
        else:
            keep = [0, 1]
        s.d_lens.copy_(torch.from_numpy(s.lens))
        s.d_starts.copy_(torch.from_numpy(s.starts))
        out.fill_(0x5A5A)
        graph.replay()
        torch.cuda.synchronize()
        want, tol, mine = s.expected()
        for b in (0, 1):
            if b not in keep:
                mine[s.starts[b]:s.starts[b + 1]] = False
        s.check(out, expected=(want, tol, mine))
