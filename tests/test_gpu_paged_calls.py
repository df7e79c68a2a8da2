"""Calls over a cache in pages as programs make them: shared pages, slices of index arrays, graphs that take turns, bases anywhere."""
import numpy as np
import pytest
import torch

from tests.paged_gpu import Setup, dev_empty, f32_dev, i32, orc, po, to_dev, to_host

pytestmark = pytest.mark.gpu
FP16, BF16 = po.DT_FLOAT16, po.DT_BFLOAT16


@pytest.mark.parametrize("eight", [False, True])
def test_sequences_that_share_the_pages_of_a_prefix(eight):
    s = Setup(1, [(100, 1), (130, 20), (96, 1), (700, 1)], 3, 2, BF16, eight, 16)
    for b in (1, 2, 3):
        s.table[b, :6] = s.table[0, :6]
    s.to_gpu()
    out = s.out()
    s.attend(out)
    s.check(out)
    k_out, v_out = dev_empty((s.tokens, 2, 128)), dev_empty((s.tokens, 2, 128))
    s.read(k_out, v_out)
    assert np.array_equal(orc.widen(to_host(k_out), BF16)[21].astype(np.float64), s.k.get(*po.place(s.table[2], s.num_pages, 16, 95)))


def test_index_arrays_that_are_slices_and_bases_off_a_line():
    s = Setup(2, [(100, 1), (130, 20), (700, 3)], 3, 2, FP16, False, 16).to_gpu()
    want = s.out()
    s.attend(want)
    s.check(want)

    def moved(t, by, dtype):
        flat = torch.full((t.numel() + by + 64,), -7, dtype=dtype, device="cuda")
        flat[by:by + t.numel()] = t.reshape(-1)
        return flat[by:by + t.numel()].view(t.shape)

    s.d_table, s.d_starts, s.d_lens = (moved(t, by, torch.int32) for t, by in ((s.d_table, 1), (s.d_starts, 3), (s.d_lens, 5)))
    s.d_q, s.d_k, s.d_v = moved(s.d_q, 8, torch.int16), moved(s.d_k, 16, torch.uint8), moved(s.d_v, 48, torch.uint8)
    big = torch.full((s.out().numel() + 64,), 0x5A5A, dtype=torch.int16, device="cuda")
    out = big[24:24 + want.numel()].view(want.shape)
    s.attend(out)
    assert torch.equal(out, want)
    assert (big[:24] == 0x5A5A).all() and (big[24 + want.numel():] == 0x5A5A).all()
    # an append and the way back at such places
    table = orc.init_freq_cis(128, 800, 1e4, FP16)
    k, v = s.out()[:, :2].contiguous(), s.out()[:, :2].contiguous()
    s.append(moved(s.d_q, 8, torch.int16), f32_dev(table), s.d_q, moved(k, 8, torch.int16), moved(v, 24, torch.int16), True)
    k_out, v_out = moved(dev_empty(tuple(k.shape)), 8, torch.int16), moved(dev_empty(tuple(v.shape)), 40, torch.int16)
    s.read(k_out, v_out)
    assert torch.equal(v_out, v)


def test_graphs_that_share_a_workspace_in_turn():
    """Two graphs of different batches over one workspace, with eager calls of others in it between their replays."""
    a, b, c = (Setup(seed, lengths, 3, 2, BF16, eight, 16).to_gpu() for seed, lengths, eight in (
        (3, [(1500, 1), (900, 1)], True), (4, [(2000, 1), (100, 1), (600, 1)], False), (5, [(1200, 20), (1000, 1)], False)))
    expected = [s.expected() for s in (a, b, c)]
    ws = max((s.workspace() for s in (a, b, c)), key=lambda x: x[1])
    assert all(s.workspace()[1] > 0 for s in (a, b, c))
    outs, graphs = [s.out() for s in (a, b, c)], []
    for s, out in zip((a, b), outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            s.attend(out, ws=ws, stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(graph)
    torch.cuda.synchronize()
    for turn in range(6):
        for out in outs:
            out.fill_(0x5A5A)
        graphs[turn % 2].replay()
        c.attend(outs[2], ws=ws)
        if turn == 3:
            ws[0].fill_(0x7F)
        graphs[(turn + 1) % 2].replay()
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        for s, out, e in zip((a, b, c), outs, expected):
            s.check(out, expected=e)


def test_threads_that_call_at_once():
    import threading
    setups = [Setup(10 + i, [(900 + 50 * i, 1), (300, 7 + i)], 3, 2, BF16, bool(i & 1), 16).to_gpu() for i in range(4)]
    expected, outs, kept, errors = [s.expected() for s in setups], [s.out() for s in setups], [], []
    torch.cuda.synchronize()

    def work(s, out):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                ws = s.workspace()
                for _ in range(20):
                    s.attend(out, ws=ws, stream=stream.cuda_stream)
                stream.synchronize()
                kept.append(ws)
        except Exception as e:  # told by the main thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=x) for x in zip(setups, outs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for s, out, e in zip(setups, outs, expected):
        s.check(out, expected=e)


def test_append_then_attend_without_a_wait_between():
    """A step's calls queued back to back on a stream of their own, many steps, one wait at the end."""
    s = Setup(20, [(400, 1), (250, 1)], 3, 2, BF16, True, 16, pages_per_seq=40).to_gpu()
    table = orc.init_freq_cis(128, 600, 1e4, BF16)
    d_table, stream = f32_dev(table), torch.cuda.Stream()
    rng = np.random.default_rng(21)
    steps, keep, outs = [], [], []
    torch.cuda.synchronize()
    ws = s.workspace()
    with torch.cuda.stream(stream):
        for step in range(8):
            q, k, v = (orc.round_to(rng.standard_normal((2, h, 128), dtype=np.float32), BF16) for h in (6, 2, 2))
            lens = np.array([380 + step, 230 + step])
            s.d_lens = i32(lens)
            rotated, out = s.out(), s.out()
            d = [to_dev(x) for x in (q, k, v)]
            s.append(rotated, d_table, *d, True, stream.cuda_stream)
            s.attend(out, q=rotated, ws=ws, stream=stream.cuda_stream)
            keep.append((d, s.d_lens, rotated))
            steps.append((lens, k, v))
            outs.append(out)
    torch.cuda.synchronize()
    for (lens, k, v), (_, _, rotated), out in zip(steps, keep, outs):
        for b, n in enumerate(lens):
            at = po.place(s.table[b], s.num_pages, 16, int(n) - 1)
            s.k.put(*at, orc.rope(k[b:b + 1], table, int(n) - 1, True, BF16)[0])
            s.v.put(*at, v[b])
        s.lens, s.q = lens, to_host(rotated)
        s.check(out)


def test_a_batch_of_overlapping_sequences_leaves_nothing_behind():
    """Replays of one graph: a right batch, one whose starts run back and forth (not allowed; nothing of it is looked at), the right one."""
    s = Setup(30, [(1990, 1), (1100, 1)], 3, 8, BF16, True, 16).to_gpu()
    ws, want = s.workspace(), s.out()
    s.attend(want, ws=ws)
    s.check(want)
    # 200 sequences over these pages, of which the others have no tokens; the launch is shaped for two tokens
    s.batch = 200
    s.d_table, s.d_lens = i32(np.tile(s.table, (100, 1))), i32(np.tile(s.lens, 100))
    s.d_starts = i32(np.minimum(np.arange(201), 2))
    ws, out = s.workspace(), s.out()
    s.attend(out, ws=ws)
    s.check(out)
    s.attend(want, ws=ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        s.attend(out, ws=ws, stream=torch.cuda.current_stream().cuda_stream)
    right, wrong = s.d_starts.clone(), i32(np.arange(201) % 2)
    for turn in range(6):
        s.d_starts.copy_(wrong if turn % 2 == 0 else right)
        out.fill_(0x5A5A)
        graph.replay()
        torch.cuda.synchronize()
        assert turn % 2 == 0 or torch.equal(out, want)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("tokens,unit,each", [(1, 128, 32), (20, 64, 16)])
@pytest.mark.parametrize("more", [(0, 0), (0, 1), (1, -1), (1, 7), (2, 0)])
def test_one_workgroup_past_what_it_looks_up_at_a_time(tokens, unit, each, more, eight):
    """A bound of a few keys: nothing is split, and a workgroup takes all of a sequence, about as many units as it looks up at once, or twice."""
    s = Setup(40, [(unit * (each + each * (more[0] > 0) + more[0] - 1) + more[1], tokens), (unit * each - 3, tokens)], 1, 2, BF16, eight, 32).to_gpu()
    assert s.workspace(max_kv=unit)[1] == 0
    out = s.out()
    s.attend(out, max_kv=unit)
    s.check(out)
