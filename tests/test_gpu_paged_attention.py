"""Attention over a cache in pages against plain arithmetic in 64 bits, within what the roundings of a kernel may make (paged_oracle)."""
import numpy as np
import pytest
import torch

from tests.paged_gpu import Setup, i32, po, to_host

pytestmark = pytest.mark.gpu
FP16, BF16 = po.DT_FLOAT16, po.DT_BFLOAT16

# (rows, new tokens) of the sequences
DECODE = [(1, 1), (2, 1), (15, 1), (16, 1), (17, 1), (33, 1), (128, 1), (129, 1), (300, 1)]
LONG = [(2500, 1), (700, 1), (3, 1)]
CHUNKS = [(70, 40), (200, 1), (129, 129), (64, 64), (65, 2), (1, 1)]


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("group,kv_heads", [(1, 3), (5, 2), (7, 4), (16, 1)])
def test_decode(group, kv_heads, dt, eight):
    s = Setup(1, DECODE, group, kv_heads, dt, eight, 16).to_gpu()
    out = s.out()
    s.attend(out)
    s.check(out)


@pytest.mark.parametrize("page_size", [16, 48, 1024])
@pytest.mark.parametrize("eight", [False, True])
def test_decode_in_splits(page_size, eight):
    s = Setup(2, LONG, 4, 2, BF16, eight, page_size).to_gpu()
    assert s.workspace()[1] > 0
    out = s.out()
    s.attend(out)
    s.check(out)


@pytest.mark.parametrize("kv_heads,lengths,window,sinks,eight", [
    (256, [(1500, 1), (3, 0), (700, 1), (0, 1), (900, 1)], 0, 0, False), (128, [(2600, 1), (1500, 1), (900, 1), (1, 1), (1300, 1)], 0, 0, True),
    (128, [(2100, 1), (40, 1), (1900, 1), (2000, 1), (1, 1), (1700, 1)], 1500, 40, False)])
def test_decode_in_runs(kv_heads, lengths, window, sinks, eight):
    """Workgroups that end one sequence and begin another: one or two to a kv head, with 24 units of 128 keys or more each."""
    s = Setup(22, lengths, 1, kv_heads, BF16, eight, 16).to_gpu()
    out = s.out()
    s.attend(out, window, sinks)
    s.check(out, window, sinks)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("group,kv_heads,page_size", [(1, 2, 16), (7, 1, 48), (3, 2, 32), (17, 1, 16), (40, 1, 64)])
def test_chunks(group, kv_heads, page_size, dt, eight):
    s = Setup(3, CHUNKS, group, kv_heads, dt, eight, page_size).to_gpu()
    out = s.out()
    s.attend(out)
    s.check(out)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("lengths", [[(1500, 30)], [(1100, 25), (900, 2), (40, 3)]])
def test_chunks_in_splits(lengths, eight):
    s = Setup(4, lengths, 6, 1, BF16, eight, 16).to_gpu()
    assert s.workspace()[1] > 0
    out = s.out()
    s.attend(out)
    s.check(out)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (17, 0), (100, 70), (64, 1000), (1 << 30, 3), (5000, 0)])
@pytest.mark.parametrize("lengths", [[(1, 1), (40, 1), (700, 1), (1500, 1)], [(300, 150), (90, 90), (513, 1), (260, 7)], [(1400, 20)]])
def test_window_and_sinks(lengths, window, sinks, eight):
    s = Setup(5, lengths, 3, 2, BF16, eight, 16).to_gpu()
    out = s.out()
    s.attend(out, window, sinks)
    s.check(out, window, sinks)


def test_sequences_without_tokens_rows_of_none_and_lengths_of_zero():
    # no new tokens; no rows at all; more tokens than rows: the first of them see nothing
    s = Setup(6, [(20, 0), (0, 0), (5, 9), (0, 3), (200, 60), (1, 4), (33, 1)], 4, 2, BF16, False, 16, gap=3, tail=5).to_gpu()
    out = s.out()
    s.attend(out)
    s.check(out)
    got = to_host(out)
    assert not got[3:3 + 4].any() and not got[3 + 9:3 + 12].any(), "a row that sees no key is zeros"


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("lengths", [[(100, 1), (200, 1)], [(100, 30), (200, 90)], [(2000, 1)], [(2000, 40)]])
def test_pages_that_are_not_there(lengths, eight):
    s = Setup(7, lengths, 4, 2, BF16, eight, 16)
    s.table[0, 1], s.table[0, 4] = -1, s.num_pages
    s.table[-1, 0], s.table[-1, 3] = 2 ** 31 - 1, -2 ** 31
    s.to_gpu()
    out = s.out()
    s.attend(out)
    s.check(out)


def test_sequence_whose_pages_are_all_gone():
    s = Setup(8, [(50, 1), (50, 20), (60, 1)], 4, 2, BF16, False, 16)
    s.table[0] = -1
    s.table[1] = s.num_pages
    s.to_gpu()
    out = s.out()
    s.attend(out)
    s.check(out)
    assert not to_host(out)[:21].any()


def bad_rows(s, name, rows):
    """Rows of the pool become NaN, infinities and the type's lowest value."""
    pool = s.k if name == "k" else s.v
    for i, (b, key) in enumerate(rows):
        page, row = po.place(s.table[b], s.num_pages, s.ps, key)
        if pool.eight:
            pool.rows_of(page)[:, row] = 0x7F if i % 2 else 0xFF
            pool.bytes_of(page)[:, row] = 255 if i % 3 == 0 else 130
        else:
            bits = [0x7FC0, 0x7F80, 0xFF80, 0xFF7F] if s.dt == BF16 else [0x7E00, 0x7C00, 0xFC00, 0xFBFF]
            pool.rows_of(page)[:, row].view(np.uint16)[:] = bits[i % 4]


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("lengths,window,sinks", [([(40, 1), (135, 1)], 0, 0), ([(45, 20), (140, 140), (9, 1)], 0, 0), ([(700, 3), (1500, 1)], 90, 5),
                                                  ([(600, 100)], 130, 3), ([(1300, 20)], 0, 0), ([(1300, 20)], 700, 20)])
def test_values_that_are_not_finite_where_nobody_looks(lengths, window, sinks, dt, eight):
    s = Setup(9, lengths, 3, 2, dt, eight, 16)
    expected = s.expected(window, sinks)
    hidden = []  # behind the last row, and what no row of the sequence sees
    for b, (n, m) in enumerate(lengths):
        hidden += [(b, key) for key in range(n, -(-n // 16) * 16)]
        if window:
            hidden += [(b, key) for key in range(sinks, max(sinks, n - m + 1 - window))]
    bad_rows(s, "k", hidden)
    bad_rows(s, "v", hidden[::-1])
    s.to_gpu()
    out = s.out()
    s.attend(out, window, sinks)
    s.check(out, window, sinks, expected)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("group", [1, 3])
@pytest.mark.parametrize("lengths,window,sinks,at", [([(20, 5), (70, 2)], 0, 0, [(0, 17), (1, 69)]), ([(200, 150), (64, 64)], 0, 0, [(0, 120), (1, 40), (1, 63)]),
                                                     ([(400, 200)], 60, 2, [(0, 250), (0, 255)]), ([(1300, 20)], 0, 0, [(0, 1290)])])
def test_values_that_are_not_finite_for_some_rows(lengths, window, sinks, at, group, eight):
    """A row that sees such a key is NaN, a row that does not is as if it were not there."""
    s = Setup(10, lengths, group, 2, BF16, eight, 16)
    want, tol, mine = s.expected(window, sinks)
    sees = np.zeros(s.tokens, dtype=bool)
    for b, key in at:
        for t in range(s.starts[b], s.starts[b + 1]):
            p = s.lens[b] - s.starts[b + 1] + t
            sees[t] |= key <= p and (window == 0 or key > p - window or key < sinks)
    assert sees.any() and not sees.all()
    for b, key in at:
        page, row = po.place(s.table[b], s.num_pages, s.ps, key)
        if eight:
            s.v.rows_of(page)[:, row] = 0x7F
        else:
            s.v.rows_of(page)[:, row].view(np.uint16)[:] = 0x7FC0
    s.to_gpu()
    out = s.out()
    s.attend(out, window, sinks)
    got = po.orc.widen(to_host(out), BF16).astype(np.float64)
    assert np.isnan(got[sees]).all()
    assert (np.abs(got - want)[~sees] <= tol[~sees]).all()


def test_scores_of_equal_and_of_far_apart_size():
    for scale in (0.0, 30.0):
        s = Setup(11, [(300, 1), (200, 70)], 2, 2, BF16, False, 16)
        s.q = po.orc.round_to((po.orc.widen(s.q, BF16) * np.float32(scale)).astype(np.float32), BF16)
        s.to_gpu()
        out = s.out()
        s.attend(out)
        s.check(out)


def test_output_in_place_of_q():
    for lengths in (DECODE, CHUNKS, LONG, [(1500, 30)]):
        s = Setup(12, lengths, 3, 2, BF16, False, 16).to_gpu()
        out = s.out()
        s.attend(out)
        kept = s.d_q.clone()
        s.attend(s.d_q)
        assert torch.equal(s.d_q, out)
        s.d_q = kept


def test_bounds_that_are_larger_or_smaller_than_the_lengths():
    for lengths in (DECODE, CHUNKS, LONG, [(1500, 30)]):
        s = Setup(13, lengths, 3, 2, BF16, False, 16).to_gpu()
        expected = s.expected()
        for max_q, max_kv in ((s.max_q, 1 << 20), (4096, s.max_kv), (1 << 28, 1 << 30), (s.max_q, 0), (s.max_q, s.max_kv // 3)):
            out = s.out()
            s.attend(out, max_q=max_q, max_kv=max_kv)
            s.check(out, expected=expected)


@pytest.mark.parametrize("change", ["starts backwards", "start before the tensor", "end behind it", "length below zero", "length past the table", "too many tokens"])
def test_sequences_that_are_passed_over(change):
    s = Setup(14, [(100, 20), (60, 1), (90, 30)], 4, 2, BF16, False, 16).to_gpu()
    want = s.out()
    s.attend(want)
    starts, lens, max_q = s.starts.copy(), s.lens.copy(), s.max_q
    left = slice(20, 21)
    if change == "starts backwards":
        starts[2] = starts[1] - 5  # sequence 1 ends before it begins, sequence 2 has 35 tokens, past the bound
        left = slice(20, 51)
    elif change == "start before the tensor":
        starts[0] = -3
        left = slice(0, 20)
    elif change == "end behind it":
        starts[3] += 1
        left = slice(21, 51)
    elif change == "length below zero":
        lens[1] = -1
    elif change == "length past the table":
        lens[1] = s.pps * s.ps + 1
    else:
        max_q, left = 29, slice(21, 51)
    s.d_starts, s.d_lens = i32(starts), i32(lens)
    out = s.out()
    s.attend(out, max_q=max_q)
    whole = torch.ones(s.tokens, dtype=torch.bool)
    whole[left] = False
    assert torch.equal(out[whole], want[whole])
    assert (out[left] == 0x5A5A).all()


def test_pools_page_by_page_in_one_allocation():
    for eight in (False, True):
        s = Setup(15, CHUNKS, 3, 2, BF16, eight, 32)
        expected = s.expected()
        both = np.stack([s.k.raw, s.v.raw], 1)  # [page][K, V][bytes]
        s.to_gpu()
        d = torch.from_numpy(both).cuda()
        s.d_k, s.d_v, s.k.stride = d[:, 0], d[:, 1], 2 * s.k.page_bytes
        out = s.out()
        s.attend(out)
        s.check(out, expected=expected)


def test_pool_past_4_gib():
    """Pages at both ends of a pool of 9 GiB: byte offsets of more than 32 bits (and, in 256-byte rows, of 33)."""
    s = Setup(16, [(200, 1), (150, 60)], 4, 2, BF16, False, 16, extra_pages=0)
    expected = s.expected()
    s.to_gpu()
    pages = (9 << 30) // s.k.page_bytes
    far = np.where(np.arange(s.num_pages) % 2 == 0, np.arange(s.num_pages), pages - 1 - np.arange(s.num_pages))
    for name in ("d_k", "d_v"):
        pool = torch.empty(pages, s.k.page_bytes, dtype=torch.uint8, device="cuda")
        pool[torch.from_numpy(far).cuda()] = getattr(s, name)
        setattr(s, name, pool)
    s.d_table = i32(np.where(s.table >= 0, far[s.table], -1))
    s.num_pages = pages
    out = s.out()
    s.attend(out)
    s.check(out, expected=expected)


def test_many_sequences():
    """More sequences than a wave looks at at once, some without tokens."""
    rng = np.random.default_rng(17)
    lengths = [(int(rng.integers(1, 60)), int(rng.choice([0, 1, 1, 1, 2, 9]))) for _ in range(150)]
    s = Setup(17, lengths, 5, 1, BF16, False, 16).to_gpu()
    out = s.out()
    s.attend(out)
    s.check(out)


def test_same_call_same_bits():
    for lengths in (LONG, CHUNKS, [(1500, 30)]):
        s = Setup(18, lengths, 3, 2, BF16, True, 16).to_gpu()
        first = s.out()
        s.attend(first)
        for _ in range(5):
            out = s.out()
            s.attend(out)
            assert torch.equal(out, first)


def test_captured_and_replayed_with_other_lengths():
    """One graph over lengths, starts and tables that change between replays, shaped by bounds."""
    s = Setup(19, [(900, 1), (40, 1), (300, 12)], 3, 2, BF16, True, 16, pages_per_seq=64).to_gpu()
    stream = torch.cuda.Stream()
    out = s.out()
    ws = s.workspace(max_q=16, max_kv=1024)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        s.attend(out, max_q=16, max_kv=1024, ws=ws, stream=torch.cuda.current_stream().cuda_stream)
    for lens, starts in (([900, 40, 300], [0, 1, 2, 14]), ([17, 1, 130], [0, 1, 2, 14]), ([899, 33, 290], [0, 0, 1, 6]), ([900, 40, 300], [0, 1, 2, 14])):
        s.d_lens.copy_(i32(lens))
        s.d_starts.copy_(i32(starts))
        s.lens, s.starts = np.array(lens), np.array(starts)
        out.fill_(0x5A5A)
        graph.replay()
        torch.cuda.synchronize()
        s.check(out)
        eager = s.out()
        s.attend(eager, max_q=16, max_kv=1024)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_two_streams_at_once():
    a, b = (Setup(seed, lengths, 3, 2, BF16, False, 16).to_gpu() for seed, lengths in ((20, LONG), (21, CHUNKS)))
    streams, outs, kept = [torch.cuda.Stream(), torch.cuda.Stream()], [a.out(), b.out()], []
    torch.cuda.synchronize()
    for _ in range(10):
        for s, stream, out in zip((a, b), streams, outs):
            with torch.cuda.stream(stream):
                kept.append(s.attend(out, stream=stream.cuda_stream, ws=s.workspace()))
    torch.cuda.synchronize()
    a.check(outs[0])
    b.check(outs[1])
