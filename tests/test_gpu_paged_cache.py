"""Rows into a cache in pages and back: bit for bit what plain arithmetic gives."""
import numpy as np
import pytest
import torch

from tests.paged_gpu import Setup, dev_empty, f32_dev, i32, normal_bits, orc, po, to_dev, to_host

pytestmark = pytest.mark.gpu
FP16, BF16 = po.DT_FLOAT16, po.DT_BFLOAT16
ROWS = 400  # of the rotary table


def tensors(s, seed):
    rng = np.random.default_rng(seed)
    k, v = (orc.round_to((rng.standard_normal((s.tokens, s.hkv, 128)) * np.exp(rng.uniform(-8, 3, (s.tokens, s.hkv, 1)))).astype(np.float32), s.dt)
            for _ in range(2))
    return s.q, k, v


def expected(s, table, q, k, v, neox):
    """(rotated q with the rows of no sequence as they were, the pools after)."""
    out = np.full_like(q, 0x5A5A)
    for b, (n, m) in enumerate(s.lengths):
        for t in range(s.starts[b], s.starts[b + 1]):
            p = n - s.starts[b + 1] + t
            if not 0 <= p < table.shape[0]:
                continue
            out[t] = orc.rope(q[t:t + 1], table, int(p), neox, s.dt)[0]
            at = po.place(s.table[b], s.num_pages, s.ps, p)
            if at is not None:
                s.k.put(*at, orc.rope(k[t:t + 1], table, int(p), neox, s.dt)[0])
                s.v.put(*at, v[t])
    return out


def run_append(s, seed, neox, table_rows=ROWS):
    table = orc.init_freq_cis(128, table_rows, 1e4, s.dt)
    q, k, v = tensors(s, seed)
    s.to_gpu()
    out = s.out()
    s.append(out, f32_dev(table), to_dev(q), to_dev(k), to_dev(v), neox)
    want = expected(s, table, q, k, v, neox)
    assert np.array_equal(to_host(out), want)
    assert np.array_equal(s.d_k.cpu().numpy(), s.k.raw)
    assert np.array_equal(s.d_v.cpu().numpy(), s.v.raw)


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("group,kv_heads,page_size,lengths", [
    (1, 1, 16, [(1, 1)]), (5, 2, 16, [(17, 1), (1, 1), (16, 1), (200, 1)]), (7, 4, 48, [(100, 60), (30, 30), (5, 0), (31, 1)]), (1, 32, 128, [(150, 21), (1, 1)])])
def test_append(group, kv_heads, page_size, lengths, neox, dt, eight):
    run_append(Setup(1, lengths, group, kv_heads, dt, eight, page_size, gap=2, tail=3), 2, neox)


@pytest.mark.parametrize("eight", [False, True])
def test_append_where_there_is_no_page_or_no_row_of_the_table(eight):
    s = Setup(3, [(100, 60), (3, 9), (390, 1), (404, 8), (40, 3)], 2, 2, BF16, eight, 16)
    s.table[0, 5], s.table[4, 2] = -1, s.num_pages
    run_append(s, 4, True)


@pytest.mark.parametrize("eight", [False, True])
def test_append_of_sequences_that_are_passed_over(eight):
    s = Setup(5, [(40, 2), (40, 3), (40, 4)], 2, 2, BF16, eight, 16)
    q, k, v = tensors(s, 6)
    table = orc.init_freq_cis(128, ROWS, 1e4, BF16)
    for lens, starts in (([40, -1, 40], None), ([40, s.pps * 16 + 1, 40], None), ([40, 40, 40], [-1, 2, 5, 9]),
                         ([40, 40, 40], [0, 2, 5, 10])):
        s.to_gpu()
        s.d_lens = i32(lens)
        if starts:
            s.d_starts = i32(starts)
        out = s.out()
        s.append(out, f32_dev(table), to_dev(q), to_dev(k), to_dev(v), True)
        starts = starts or list(s.starts)
        left = torch.zeros(s.tokens, dtype=torch.bool)
        for b in range(3):
            if not 0 <= lens[b] <= s.pps * 16 or not 0 <= starts[b] <= starts[b + 1] <= s.tokens:
                left[max(0, starts[b]):starts[b + 1]] = True
        assert left.any()
        assert (out[left] == 0x5A5A).all() and (out[~left] != 0x5A5A).any(-1).all()


@pytest.mark.parametrize("dt", [FP16, BF16])
def test_eight_bits_of_every_kind_of_value(dt):
    """Every bit pattern of the type as values, in rows of one size and of all sizes; zero rows; rows with infinities and NaN."""
    every = np.arange(1 << 16, dtype=np.uint16)
    size = np.abs(orc.widen(every, dt).astype(np.float64))
    by_size = every[np.argsort(np.where(np.isnan(size), np.inf, size), kind="stable")]
    rows = np.concatenate([by_size.reshape(-1, 128), np.random.default_rng(7).permutation(every).reshape(-1, 128), np.zeros((2, 128), np.uint16)])
    m = rows.shape[0] // 2
    s = Setup(8, [(m, m)], 1, 2, dt, True, 64)
    v = rows.reshape(m, 2, 128)
    table = np.zeros((m, 64, 2), np.float32)
    table[..., 0] = 1.0  # no turn (but infinities and NaN, times 0, become NaN: they go in as v)
    s.to_gpu()
    out = s.out()
    s.append(out, f32_dev(table), to_dev(s.q), to_dev(np.zeros_like(v)), to_dev(v), True)
    for t in range(m):
        s.v.put(*po.place(s.table[0], s.num_pages, s.ps, t), v[t])
    got = s.d_v.cpu().numpy()
    for page in s.table[0]:
        a, b = got[page, :s.v.values], s.v.raw[page, :s.v.values]
        assert np.array_equal(a & 127, b & 127) and (((a ^ b) & 128 == 0) | (a & 127 == 127)).all()  # (a NaN has either sign)
        assert np.array_equal(got[page, s.v.values:], s.v.raw[page, s.v.values:])
    # and back: what the 8 bits stand for, exactly
    k_out, v_out = dev_empty((m, 2, 128)), dev_empty((m, 2, 128))
    s.read(k_out, v_out)
    back = orc.widen(to_host(v_out), dt).astype(np.float64)
    want = np.stack([s.v.get(*po.place(s.table[0], s.num_pages, s.ps, t)) for t in range(m)])
    assert np.array_equal(back, want, equal_nan=True)
    finite = np.isfinite(orc.widen(v, dt))
    assert np.isnan(back[~finite]).all() and np.isfinite(back[finite]).all()


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dt", [FP16, BF16])
@pytest.mark.parametrize("kv_heads,page_size,lengths", [(1, 16, [(1, 1)]), (8, 16, [(50, 50), (20, 3), (0, 0), (17, 0), (33, 1)]), (3, 48, [(200, 190), (4, 9)])])
def test_read(kv_heads, page_size, lengths, dt, eight):
    s = Setup(9, lengths, 1, kv_heads, dt, eight, page_size, gap=1, tail=2)
    if len(lengths) > 2:
        s.table[0, 1], s.table[1, 1] = -1, s.num_pages
    s.to_gpu()
    outs = [torch.full((s.tokens, kv_heads, 128), 0x5A5A, dtype=torch.int16, device="cuda") for _ in range(2)]
    s.read(*outs)
    for out, pool in zip(outs, (s.k, s.v)):
        bits = to_host(out)
        got = orc.widen(bits, dt).astype(np.float64)
        mine = np.zeros(s.tokens, dtype=bool)
        for b, (n, m) in enumerate(lengths):
            for t in range(s.starts[b], s.starts[b + 1]):
                mine[t] = True
                at = po.place(s.table[b], s.num_pages, s.ps, n - s.starts[b + 1] + t)
                assert np.array_equal(got[t], pool.get(*at) if at is not None else np.zeros((kv_heads, 128)))
        assert (bits[~mine] == 0x5A5A).all()


@pytest.mark.parametrize("eight", [False, True])
def test_conversation(eight):
    """Prompts, then tokens one by one, then a second turn: append, attention and the way back as they are used, the lengths on the device;
    in 16 bits beside the contiguous cache's operators."""
    import llm_simple_amd.ops as ops
    group, hkv, dt, rows = 3, 2, BF16, 256
    H = group * hkv
    table = orc.init_freq_cis(128, rows, 1e4, dt)
    d_table = f32_dev(table)
    s = Setup(10, [(192, 1), (192, 1)], group, hkv, dt, eight, 16)
    s.to_gpu()
    flat = [tuple(torch.zeros(rows, hkv, 128, dtype=torch.int16, device="cuda") for _ in "kv") for _ in range(2)]
    lens = np.zeros(2, dtype=np.int64)
    for step, new in enumerate([(70, 33), (1, 1), (1, 1), (1, 0), (40, 1), (1, 60)]):
        lens = lens + new
        s.lengths, s.lens, s.starts = list(zip(lens.tolist(), new)), lens, np.cumsum([0, *new])
        s.tokens, s.max_q, s.max_kv = int(s.starts[-1]), max(new), int(lens.max())
        s.d_lens, s.d_starts = i32(lens), i32(s.starts)
        s.q = normal_bits(100 + step, (s.tokens, H, 128), dt)
        q, k, v = tensors(s, 200 + step)
        rotated, out = s.out(), s.out()
        s.append(rotated, d_table, to_dev(q), to_dev(k), to_dev(v), True)
        s.attend(out, q=rotated)
        assert np.array_equal(to_host(rotated), expected(s, table, q, k, v, True))
        s.q = to_host(rotated)
        s.check(out)
        k_out, v_out = dev_empty((s.tokens, hkv, 128)), dev_empty((s.tokens, hkv, 128))
        s.read(k_out, v_out)
        for t, pool in ((k_out, s.k), (v_out, s.v)):
            got = orc.widen(to_host(t), dt)
            for b in range(2):
                for i in range(s.starts[b], s.starts[b + 1]):
                    assert np.array_equal(got[i], pool.get(*po.place(s.table[b], s.num_pages, 16, int(lens[b] - s.starts[b + 1] + i))))
        if eight:
            continue
        for b in range(2):
            if new[b] == 0:
                continue
            i0, i1, past = int(s.starts[b]), int(s.starts[b + 1]), int(lens[b] - new[b])
            q_rot, o = dev_empty((new[b], H, 128)), dev_empty((new[b], H, 128))
            ops.hip_rope_kv_append_layer(q_rot, *flat[b], d_table, to_dev(q[i0:i1]), to_dev(k[i0:i1]), to_dev(v[i0:i1]), past, new[b], H, hkv, 128, True, dt)
            ops.hip_flash_attn_gqa_layer(o, q_rot, *flat[b], new[b], int(lens[b]), past, group, hkv, 128, dt)
            assert torch.equal(q_rot, rotated[i0:i1])
            a, c = orc.widen(to_host(o), dt).astype(np.float64), orc.widen(to_host(out[i0:i1]), dt).astype(np.float64)
            want, tol, _ = s.expected()
            assert (np.abs(a - c) <= 2 * tol[i0:i1]).all()


def test_captured_append_and_read_with_other_lengths():
    s = Setup(11, [(60, 1), (200, 1), (30, 1)], 2, 2, BF16, True, 16, pages_per_seq=16).to_gpu()
    table = orc.init_freq_cis(128, ROWS, 1e4, BF16)
    q, k, v = tensors(s, 12)
    d_table, d_q, d_k, d_v = f32_dev(table), to_dev(q), to_dev(k), to_dev(v)
    out, k_out, v_out = s.out(), dev_empty((3, 2, 128)), dev_empty((3, 2, 128))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        stream = torch.cuda.current_stream().cuda_stream
        s.append(out, d_table, d_q, d_k, d_v, True, stream)
        s.read(k_out, v_out, stream)
    for lens in ([60, 200, 30], [61, 193, 31], [1, 64, 17]):
        s.lens, s.lengths = np.array(lens), [(n, 1) for n in lens]
        s.d_lens.copy_(i32(lens))
        out.fill_(0x5A5A)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(to_host(out), expected(s, table, q, k, v, True))
        assert np.array_equal(s.d_k.cpu().numpy(), s.k.raw) and np.array_equal(s.d_v.cpu().numpy(), s.v.raw)
        for t, pool in ((k_out, s.k), (v_out, s.v)):
            assert np.array_equal(orc.widen(to_host(t), BF16), np.stack([pool.get(*po.place(s.table[b], s.num_pages, 16, n - 1)) for b, n in enumerate(lens)]))
