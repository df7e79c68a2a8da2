"""Dense tensors of more rows than one dimension of a launch takes workgroups of: few of the rows are a sequence's, the rest is not looked at."""
import numpy as np
import pytest
import torch

from tests.paged_gpu import Setup, f32_dev, orc, po, to_dev, to_host

pytestmark = pytest.mark.gpu
BF16 = po.DT_BFLOAT16


def setup(seed, tokens, eight):
    """Sequences at the tensors' beginning and at their end; the one between, of all other rows, is passed over."""
    s = Setup(seed, [(20, 3), (40, 2), (31, 0), (50, 4)], 1, 1, BF16, eight, 16)
    s.starts, s.tokens = np.array([0, 3, 5, tokens - 4, tokens], dtype=np.int32), tokens
    s.lens[2] = -1
    return s.to_gpu()


def free_gib():
    return torch.cuda.mem_get_info()[0] >> 30


@pytest.mark.parametrize("eight", [False, True])
def test_append(eight):
    """2^24 tokens and some: a workgroup of 256 to each would be 2^32 threads."""
    tokens = (1 << 24) + 5
    if free_gib() < 24:
        pytest.skip("needs 24 GiB")
    s = setup(1, tokens, eight)
    table = orc.init_freq_cis(128, 64, 1e4, BF16)
    rng = np.random.default_rng(2)
    mine = [*range(5), *range(tokens - 4, tokens)]
    q, k, v = (orc.round_to(rng.standard_normal((len(mine), 1, 128)).astype(np.float32), BF16) for _ in range(3))
    at = torch.tensor(mine, device="cuda")
    full = []
    for x in (q, k, v):
        t = torch.empty(tokens, 1, 128, dtype=torch.int16, device="cuda")
        t[at] = to_dev(x)
        full.append(t)
    out = torch.full((tokens, 1, 128), 0x5A5A, dtype=torch.int16, device="cuda")
    s.append(out, f32_dev(table), *full, True)
    want = np.empty_like(q)
    for b in (0, 1, 3):
        for t in range(s.starts[b], s.starts[b + 1]):
            i, p = mine.index(t), int(s.lens[b] - s.starts[b + 1] + t)
            want[i] = orc.rope(q[i:i + 1], table, p, True, BF16)[0]
            place = po.place(s.table[b], s.num_pages, s.ps, p)
            s.k.put(*place, orc.rope(k[i:i + 1], table, p, True, BF16)[0])
            s.v.put(*place, v[i])
    assert np.array_equal(to_host(out[at]), want)
    assert (out[5:tokens - 4:99991] == 0x5A5A).all() and (out[tokens - 99:tokens - 4] == 0x5A5A).all()
    assert np.array_equal(s.d_k.cpu().numpy(), s.k.raw) and np.array_equal(s.d_v.cpu().numpy(), s.v.raw)


@pytest.mark.parametrize("eight", [False, True])
def test_read(eight):
    """2^26 tokens and some, four of which a workgroup has."""
    tokens = (1 << 26) + 7
    if free_gib() < 48:
        pytest.skip("needs 48 GiB")
    s = setup(3, tokens, eight)
    outs = [torch.full((tokens, 1, 128), 0x5A5A, dtype=torch.int16, device="cuda") for _ in range(2)]
    s.read(*outs)
    for out, pool in zip(outs, (s.k, s.v)):
        for b in (0, 1, 3):
            for t in range(s.starts[b], s.starts[b + 1]):
                got = orc.widen(to_host(out[t]), BF16).astype(np.float64)
                assert np.array_equal(got, pool.get(*po.place(s.table[b], s.num_pages, s.ps, int(s.lens[b] - s.starts[b + 1] + t))))
        assert (out[5:tokens - 4:99991] == 0x5A5A).all() and (out[tokens - 99:tokens - 4] == 0x5A5A).all()
