"""One graph of the kernel that takes few rows in runs over all sequences: lengths for runs, for equal parts and for neither in turn."""
import numpy as np
import pytest
import torch

from tests.paged_gpu import Setup, i32, po, to_host

pytestmark = pytest.mark.gpu
BF16 = po.DT_BFLOAT16
KV_HEADS, BATCH, MOST = 64, 5, 6400  # 4 workgroups of a kv head run at a time: runs from 96 units of 128 keys on, where equal parts do not come out even
# (lengths, which of the sequences have a new token, whether they are taken in runs)
TURNS = [([5000, 4000, 3000, 600, 17], [1, 1, 1, 1, 1], True), ([6400, 6400, 0, 0, 0], [1, 1, 0, 0, 0], False), ([3200, 3200, 3200, 3200, 9], [1, 1, 1, 1, 0], False),
         ([900, 40, 1, 0, 300], [1, 1, 1, 1, 1], False), ([1, 6400, 128, 6399, 5], [1, 1, 1, 1, 1], True), ([6400, 6400, 3000, 0, 0], [0, 1, 1, 0, 0], False),
         ([2600, 2600, 2600, 2600, 2600], [1, 1, 1, 1, 1], True)]


def in_runs(lengths, new):
    """What the kernel decides: too many units for one look at equal parts to come out within a fifth of an equal share."""
    units = [-(-n // 128) for n, m in zip(lengths, new) if m]
    parts, total = 256 // KV_HEADS, sum(units)
    fit, even = parts, False
    for _ in range(6):
        if 2 * fit <= parts or len(units) > parts:
            break
        chunk = max(total / fit, 3)
        over = sum(max(1, -(-u // chunk)) for u in units) - parts
        if over <= 0:
            even = chunk * parts <= 1.2 * total
            break
        fit -= int(over)
    return not even and total >= 24 * parts


class Heads:
    """Some kv heads of a pool."""

    def __init__(self, pool, heads):
        self.pool, self.heads, self.h, self.n, self.ps = pool, heads, len(heads), pool.n, pool.ps

    def get(self, page, row):
        return self.pool.get(page, row)[self.heads]


@pytest.mark.parametrize("eight", [False, True])
def test_captured_and_replayed(eight):
    s = Setup(1, [(640, 1)] * BATCH, 1, KV_HEADS, BF16, eight, 64)
    rng = np.random.default_rng(2)
    s.pps, s.max_kv = MOST // 64, MOST
    s.table = rng.integers(0, s.num_pages, (BATCH, s.pps)).astype(np.int32)  # (sequences may share pages)
    s.to_gpu()
    kv = [5, 63]
    k, v = Heads(s.k, kv), Heads(s.v, kv)
    ws, out = s.workspace(), s.out()
    s.attend(out, ws=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        s.attend(out, ws=ws, stream=torch.cuda.current_stream().cuda_stream)
    seen = {}
    for turn in [0, 1, 0, 2, 3, 4, 1, 5, 6, 3, 6, 4, 0]:
        lengths, new, runs = TURNS[turn]
        assert in_runs(lengths, new) == runs
        s.lens, s.starts = np.array(lengths), np.cumsum([0, *new])
        s.d_lens.copy_(i32(s.lens))
        s.d_starts.copy_(i32(s.starts))
        out.fill_(0x5A5A)
        graph.replay()
        torch.cuda.synchronize()
        if turn not in seen:
            seen[turn] = po.attend(s.q[:, kv], k, v, s.table, s.starts, s.lens, BF16, 1)
        want, tol, mine = seen[turn]
        bits = to_host(out)
        assert (bits[~mine] == 0x5A5A).all()
        got = po.orc.widen(bits[:, kv], BF16).astype(np.float64)
        assert (np.abs(got - want)[mine] <= tol[mine]).all()
        eager = s.out()
        s.attend(eager)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
