"""Further calls that the documentation allows: buffers in place, rows that are not finite among them; batches without a token; many short sequences."""
import numpy as np
import pytest
import torch

from tests import test_gpu_paged_not_finite as not_finite
from tests.paged_gpu import Setup, f32_dev, i32, orc, po, to_dev, to_host

pytestmark = pytest.mark.gpu
FP16, BF16 = po.DT_FLOAT16, po.DT_BFLOAT16


def random_rows(seed, shape, dt):
    return orc.round_to(np.random.default_rng(seed).standard_normal(shape).astype(np.float32), dt)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("neox", [False, True])
def test_append_with_q_in_place(neox, eight):
    s = Setup(1, [(200, 150), (31, 1), (90, 40), (500, 120)], 3, 2, FP16, eight, 16).to_gpu()  # (more tokens than compute units)
    table = f32_dev(orc.init_freq_cis(128, 600, 1e4, FP16))
    q, k, v = (to_dev(random_rows(2 + i, (s.tokens, h, 128), FP16)) for i, h in enumerate((s.H, 2, 2)))
    want = s.out()
    s.append(want, table, q, k, v, neox)
    pools = s.d_k.clone(), s.d_v.clone()
    s.to_gpu()
    s.append(q, table, q, k, v, neox)
    assert torch.equal(q, want) and torch.equal(s.d_k, pools[0]) and torch.equal(s.d_v, pools[1])


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("lengths,group,kv_heads,window,sinks,max_kv,at", not_finite.CASES)
def test_output_in_place_of_q_and_values_that_are_not_finite(lengths, group, kv_heads, window, sinks, max_kv, at, eight):
    s = Setup(3, lengths, group, kv_heads, BF16, eight, 16)
    for b, key in at:
        not_finite.poison(s, b, key, [1, 77], "nan")
    s.to_gpu()
    want = s.out()
    s.attend(want, window, sinks, max_kv=max_kv)
    s.attend(s.d_q, window, sinks, max_kv=max_kv)
    assert torch.equal(s.d_q, want)


def test_captured_and_replayed_with_values_that_come_and_go():
    """One graph over V that is not finite in some replays and is in others; the dims that it is not in have the same bits in all."""
    s = Setup(4, [(700, 50), (300, 2), (64, 1)], 5, 2, BF16, False, 16).to_gpu()
    ws, out, clean = s.workspace(), s.out(), s.out()
    s.attend(clean, ws=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        s.attend(out, ws=ws, stream=torch.cuda.current_stream().cuda_stream)
    good = s.d_v.clone()
    not_finite.poison(s, 0, 690, [9], "nan")
    not_finite.poison(s, 1, 299, [9], "nan")
    bad = torch.from_numpy(s.v.raw.copy()).cuda()
    expected = s.expected()
    want, tol, _ = expected
    sees = not_finite.visible(s, 0, 690, 0, 0) | not_finite.visible(s, 1, 299, 0, 0)
    others = np.arange(128) != 9
    for turn in range(6):
        s.d_v.copy_(bad if turn % 2 else good)
        out.fill_(0x5A5A)
        graph.replay()
        torch.cuda.synchronize()
        if turn % 2 == 0:
            assert torch.equal(out, clean)
            continue
        got = po.orc.widen(to_host(out), BF16).astype(np.float64)
        assert np.isnan(got[sees][..., 9]).all() and np.isfinite(got[~sees]).all()
        assert (np.abs(got - want)[..., others] <= tol[..., others]).all() and (np.abs(got - want)[~sees] <= tol[~sees]).all()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("lengths", [[(100, 1), (2000, 1)], [(300, 60), (20, 2)]])
def test_a_batch_without_a_token(lengths, eight):
    """Bounds of a batch that has some, starts that say there is none."""
    s = Setup(5, lengths, 3, 2, BF16, eight, 16).to_gpu()
    ws, out = s.workspace(), s.out()
    table = f32_dev(orc.init_freq_cis(128, 2100, 1e4, BF16))
    k, v = (to_dev(random_rows(6 + i, (s.tokens, 2, 128), BF16)) for i in range(2))
    for starts in ([0, 0, 0], [s.tokens] * 3, [1, 1, 1]):
        s.d_starts = i32(starts)
        s.attend(out, ws=ws)
        rotated, outs = s.out(), [torch.full((s.tokens, 2, 128), 0x5A5A, dtype=torch.int16, device="cuda") for _ in range(2)]
        s.append(rotated, table, s.d_q, k, v, True)
        s.read(*outs)
        for t in (out, rotated, *outs):
            assert (t == 0x5A5A).all()
        assert np.array_equal(s.d_k.cpu().numpy(), s.k.raw) and np.array_equal(s.d_v.cpu().numpy(), s.v.raw)


@pytest.mark.parametrize("eight", [False, True])
def test_read_of_many_short_sequences(eight):
    """Several tokens to a workgroup, of one sequence, of several, of none; pages that are not there; rows before the first."""
    rng = np.random.default_rng(7)
    lengths = [(int(n), int(min(m, n + 2))) for n, m in zip(rng.integers(0, 40, 700), rng.integers(0, 9, 700))]
    s = Setup(8, lengths, 1, 1, BF16, eight, 16, gap=5, tail=6)
    s.table[rng.random(s.table.shape) < 0.1] = -1
    s.table[rng.random(s.table.shape) < 0.05] = s.num_pages
    assert s.tokens >= 2048
    s.to_gpu()
    outs = [torch.full((s.tokens, 1, 128), 0x5A5A, dtype=torch.int16, device="cuda") for _ in range(2)]
    s.read(*outs)
    for out, pool in zip(outs, (s.k, s.v)):
        bits = to_host(out)
        got = orc.widen(bits, BF16).astype(np.float64)
        mine = np.zeros(s.tokens, dtype=bool)
        for b, (n, _) in enumerate(lengths):
            for t in range(s.starts[b], s.starts[b + 1]):
                mine[t] = True
                at = po.place(s.table[b], s.num_pages, s.ps, n - s.starts[b + 1] + t)
                assert np.array_equal(got[t], pool.get(*at) if at is not None else np.zeros((1, 128)))
        assert (bits[~mine] == 0x5A5A).all() and not mine.all()


@pytest.mark.parametrize("kv_heads,lengths", [(600, [(70, 1), (33, 1)]), (300, [(70, 20), (40, 1)])])
def test_more_kv_heads_than_places(kv_heads, lengths):
    """Nothing is split; two of the heads are looked at."""
    s = Setup(9, lengths, 2, kv_heads, BF16, False, 16).to_gpu()
    assert s.workspace()[1] == 0 or kv_heads < 512
    out = s.out()
    s.attend(out)
    whole = po.orc.widen(to_host(out), BF16).astype(np.float64)
    for h in (0, kv_heads - 1):
        class Head:
            def __init__(self, pool):
                self.pool, self.h, self.n, self.ps = pool, 1, pool.n, pool.ps

            def get(self, page, row):
                return self.pool.get(page, row)[h:h + 1]

        want, tol, _ = po.attend(s.q[:, 2 * h:2 * h + 2], Head(s.k), Head(s.v), s.table, s.starts, s.lens, BF16, 2)
        assert (np.abs(whole[:, 2 * h:2 * h + 2] - want) <= tol).all()
