"""A batch over a cache in pages on the GPU and on the host, for the tests."""
import numpy as np
import torch

from oracle import oracle as orc
from tests import paged_oracle as po
from tests.helpers import dev_empty, f32_dev, normal_bits, to_dev, to_host


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


class Setup:
    """lengths: (rows of the sequence, its new tokens).  The pools begin with normal rows of differing size."""

    def __init__(self, seed, lengths, group, kv_heads, dt, eight, page_size, extra_pages=2, gap=0, stride=None, tail=0, pages_per_seq=None):
        import llm_simple_amd.ops as ops
        self.ops, self.lengths, self.g, self.hkv, self.dt, self.ps = ops, lengths, group, kv_heads, dt, page_size
        self.H, self.batch = group * kv_heads, len(lengths)
        self.cache_dt = po.DT_FLOAT8 if eight else dt
        rng = np.random.default_rng(seed)
        counts = [-(-n // page_size) for n, _ in lengths]
        self.pps = pages_per_seq or max(1, max(counts))
        self.num_pages = sum(counts) + extra_pages
        order = rng.permutation(self.num_pages)
        self.table = np.full((self.batch, self.pps), -1, dtype=np.int32)
        at = 0
        for b, c in enumerate(counts):
            self.table[b, :c] = order[at:at + c]
            at += c
        self.starts = np.cumsum([gap] + [m for _, m in lengths]).astype(np.int32)
        self.lens = np.array([n for n, _ in lengths], dtype=np.int32)
        self.tokens = int(self.starts[-1]) + tail
        self.max_q, self.max_kv = max(1, max(m for _, m in lengths)), int(self.lens.max())
        self.k, self.v = (po.Pool(self.num_pages, page_size, kv_heads, self.cache_dt, dt, stride) for _ in range(2))
        for name, pool in (("k", self.k), ("v", self.v)):
            for page in range(self.num_pages):
                x = normal_bits(rng.integers(1 << 30), (kv_heads, page_size, 128), dt)
                x = orc.round_to((orc.widen(x, dt) * np.exp(0.5 * rng.standard_normal((kv_heads, page_size, 1)))).astype(np.float32), dt)
                if eight:
                    codes, byte = po.eight_bits(orc.widen(x, dt).astype(np.float64), dt)
                    pool.rows_of(page)[:] = codes
                    pool.bytes_of(page)[:] = byte
                else:
                    pool.rows_of(page)[:] = x.view(np.uint8).reshape(kv_heads, page_size, 256)
        self.q = normal_bits(rng.integers(1 << 30), (self.tokens, self.H, 128), dt)

    def to_gpu(self):
        self.d_k, self.d_v = (torch.from_numpy(pool.raw.copy()).cuda() for pool in (self.k, self.v))
        self.d_table, self.d_starts, self.d_lens, self.d_q = i32(self.table), i32(self.starts), i32(self.lens), to_dev(self.q)
        return self

    def workspace(self, window=0, sinks=0, max_q=None, max_kv=None):
        size = self.ops.paged_flash_attn_workspace_bytes(self.tokens, self.batch, max_q or self.max_q, self.max_kv if max_kv is None else max_kv,
                                                         window, sinks, self.g, self.hkv, 128)
        return torch.full((max(16, size),), 0xFF, dtype=torch.uint8, device="cuda"), size  # (NaN wherever it is read before it is written)

    def attend(self, out, window=0, sinks=0, max_q=None, max_kv=None, q=None, ws=None, stream=0):
        ws, size = ws or self.workspace(window, sinks, max_q, max_kv)
        self.ops.hip_paged_flash_attn_gqa_layer(
            out, self.d_q if q is None else q, self.d_k, self.d_v, self.d_table, self.d_starts, self.d_lens, ws, size, self.tokens, self.batch,
            max_q or self.max_q, self.max_kv if max_kv is None else max_kv, self.pps, self.num_pages, self.ps, self.k.stride, window, sinks,
            self.g, self.hkv, 128, self.cache_dt, self.dt, stream)
        return ws  # (to be kept until the work is done)

    def append(self, out_q, table, q, k, v, neox, stream=0, table_rows=None):
        self.ops.hip_paged_rope_kv_append_layer(
            out_q, self.d_k, self.d_v, self.d_table, self.d_starts, self.d_lens, table, q, k, v, self.tokens, self.batch, self.pps, self.num_pages,
            self.ps, self.k.stride, table_rows or table.shape[0], self.H, self.hkv, 128, neox, self.cache_dt, self.dt, stream)

    def read(self, out_k, out_v, stream=0):
        self.ops.hip_paged_kv_read_layer(out_k, out_v, self.d_k, self.d_v, self.d_table, self.d_starts, self.d_lens, self.tokens, self.batch, self.pps,
                                         self.num_pages, self.ps, self.k.stride, self.hkv, 128, self.cache_dt, self.dt, stream)

    def out(self, fill=0x5A5A):
        return torch.full((self.tokens, self.H, 128), fill, dtype=torch.int16, device="cuda")

    def expected(self, window=0, sinks=0):
        return po.attend(self.q, self.k, self.v, self.table, self.starts, self.lens, self.dt, self.g, window, sinks)

    def check(self, out, window=0, sinks=0, expected=None):
        want, tol, mine = expected or self.expected(window, sinks)
        bits = to_host(out)
        got = orc.widen(bits, self.dt).astype(np.float64)
        assert (bits[~mine] == 0x5A5A).all(), "rows of no sequence"
        assert np.isfinite(got[mine]).all()
        off = np.abs(got - want)[mine] / np.maximum(tol[mine], 1e-30)
        assert off.size == 0 or off.max() <= 1, f"{off.max()} of the bound at {np.unravel_index(off.argmax(), off.shape)}"


__all__ = ["Setup", "i32", "dev_empty", "f32_dev", "normal_bits", "to_dev", "to_host", "po", "orc"]
