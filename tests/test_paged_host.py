"""A KV cache in pages: arguments that are refused before any launch, sizes, and the host's own arithmetic of 8 bits.  No GPU."""
import ctypes

import numpy as np
import pytest

from tests import paged_oracle as po


def pointer():
    buf = ctypes.create_string_buffer(256)
    return buf, (ctypes.addressof(buf) + 15) & ~15


APPEND = dict(out_q=0, k_pages=0, v_pages=0, page_table=0, q_starts=0, kv_lens=0, freq_cis=0, in_q=0, in_k=0, in_v=0, tokens=4, batch=2,
              pages_per_seq=3, num_pages=8, page_size=16, page_stride=16 * 2 * 256, table_rows=64, n_heads=4, n_kv_heads=2, head_dim=128,
              neox=1, cache_dt=5, dt=5, stream=None)
ATTEND = dict(out=0, q=0, k_pages=0, v_pages=0, page_table=0, q_starts=0, kv_lens=0, workspace=0, workspace_bytes=1 << 40, tokens=4, batch=2,
              max_q_len=2, max_kv_len=40, pages_per_seq=3, num_pages=8, page_size=16, page_stride=16 * 2 * 256, window=0, sinks=0,
              group_size=2, kv_head_num=2, head_dim=128, cache_dt=5, dt=5, stream=None)
READ = dict(out_k=0, out_v=0, k_pages=0, v_pages=0, page_table=0, q_starts=0, kv_lens=0, tokens=4, batch=2, pages_per_seq=3, num_pages=8,
            page_size=16, page_stride=16 * 2 * 256, kv_head_num=2, head_dim=128, cache_dt=5, dt=5, stream=None)
CALLS = {"llmhip_paged_rope_kv_append": APPEND, "llmhip_paged_flash_attn_gqa": ATTEND, "llmhip_paged_kv_read": READ}
COMMON = [("tokens", 0, -1), ("batch", 0, -1), ("pages_per_seq", 0, -1), ("num_pages", 0, -1), ("page_size", 0, -1), ("page_size", 8, -2),
          ("page_size", 24, -2), ("page_size", 1040, -2), ("page_stride", 16 * 2 * 256 - 16, -1), ("page_stride", 16 * 2 * 256 + 8, -1),
          ("page_stride", -16 * 2 * 256, -1), ("head_dim", 64, -2), ("cache_dt", 4, -1), ("cache_dt", 0, -1), ("dt", 6, -1), ("dt", 16, -1),
          ("pages_per_seq", (1 << 26) + 1, -2), ("q_starts", 2, -1), ("kv_lens", 1, -1), ("page_table", 2, -1), ("k_pages", 8, -1),
          ("v_pages", 4, -1), ("k_pages", None, -1), ("v_pages", None, -1), ("page_table", None, -1), ("q_starts", None, -1),
          ("kv_lens", None, -1), ("batch", 65536, -2), ("tokens", (1 << 30) + 1, -2)]
OWN = [("llmhip_paged_rope_kv_append", *x) for x in [
           ("table_rows", 0, -1), ("n_heads", 0, -1), ("n_kv_heads", 0, -1), ("n_kv_heads", 65536, -2), ("n_heads", 65536, -2),
           ("out_q", None, -1), ("in_q", 2, -1), ("in_k", None, -1), ("in_v", 8, -1), ("freq_cis", 4, -1)]] + \
      [("llmhip_paged_flash_attn_gqa", *x) for x in [
           ("max_q_len", 0, -1), ("max_kv_len", -1, -1), ("sinks", -1, -1), ("group_size", 0, -1), ("kv_head_num", 0, -1),
           ("group_size", 40000, -2), ("workspace", 8, -1), ("out", None, -1), ("q", 2, -1), ("tokens", 1 << 30, -2)]] + \
      [("llmhip_paged_kv_read", *x) for x in [("kv_head_num", 0, -1), ("out_k", None, -1), ("out_v", 4, -1)]]


def call(name, **changed):
    import llm_simple_amd.ops as ops
    buf, p = pointer()
    args = dict(CALLS[name])
    for key, value in args.items():
        if value == 0 and key not in ("window", "sinks"):
            args[key] = p
    for key, value in changed.items():
        if args[key] == p and value is not None:
            value += p  # an offset
        args[key] = value
    return getattr(ops.lib, name)(*args.values())


@pytest.mark.parametrize("name", sorted(CALLS))
@pytest.mark.parametrize("what,value,status", COMMON)
def test_refused(name, what, value, status):
    assert call(name, **{what: value}) == status


@pytest.mark.parametrize("name,what,value,status", OWN)
def test_refused_of_its_own(name, what, value, status):
    assert call(name, **{what: value}) == status


@pytest.mark.parametrize("name", sorted(CALLS))
def test_eight_bits_need_the_larger_page(name):
    sixteen_rows = 16 * 2 * 129
    assert call(name, cache_dt=16, page_stride=sixteen_rows - 16) == -1


def test_workspace_is_asked_for():
    import llm_simple_amd.ops as ops
    need = ops.paged_flash_attn_workspace_bytes(1, 1, 1, 32768, 0, 0, 5, 8, 128)
    assert need > 0
    sizes = dict(tokens=1, batch=1, max_q_len=1, max_kv_len=32768, pages_per_seq=2048, group_size=5, kv_head_num=8, page_stride=16 * 8 * 256)
    assert call("llmhip_paged_flash_attn_gqa", **sizes, workspace_bytes=need - 1) == -3
    assert call("llmhip_paged_flash_attn_gqa", **sizes, workspace=None) == -3
    # a short cache is one workgroup's for each kv head
    assert ops.paged_flash_attn_workspace_bytes(1, 1, 1, 100, 0, 0, 5, 8, 128) == 0
    # a window bounds it
    assert ops.paged_flash_attn_workspace_bytes(1, 1, 1, 32768, 64, 4, 5, 8, 128) == 0
    for bad in [(0, 1, 1, 1, 0, 0, 1, 1, 128), (1, 1, 1, 1, 0, -1, 1, 1, 128), (1, 1, 1, 1, 0, 0, 1, 1, 64), (1, 1, 1, 1, 0, 0, 1 << 16, 1, 128)]:
        assert ops.paged_flash_attn_workspace_bytes(*bad) == 0


def test_page_bytes():
    import llm_simple_amd.ops as ops
    assert ops.paged_page_bytes(16, 8, 128, 5) == ops.paged_page_bytes(16, 8, 128, 4) == 16 * 8 * 256
    assert ops.paged_page_bytes(64, 4, 128, ops.DT_FLOAT8_E4M3) == 64 * 4 * 129
    for bad in [(0, 8, 128, 5), (8, 8, 128, 5), (1040, 8, 128, 5), (16, 0, 128, 5), (16, 8, 64, 5), (16, 8, 128, 6)]:
        assert ops.paged_page_bytes(*bad) == 0


def test_python_face():
    import llm_simple_amd.ops as ops
    with pytest.raises(ops.LlmHipError, match="invalid argument"):
        ops.hip_paged_kv_read_layer(*[None] * 7, 1, 1, 1, 1, 16, 16 * 256, 1, 128, 5, 5)
    with pytest.raises(TypeError, match="missing argument 'dt'"):
        ops.hip_paged_kv_read_layer(*[None] * 7, 1, 1, 1, 1, 16, 16 * 256, 1, 128, 5)
    with pytest.raises(TypeError, match="unexpected"):
        ops.hip_paged_flash_attn_gqa_layer(*[None] * 8, 0, *[1] * 16, windows=3)


# the oracle's own arithmetic

def test_oracle_eight_bits():
    import torch
    x = np.random.default_rng(0).standard_normal(100000) * np.exp(np.random.default_rng(1).uniform(-12, 6, 100000))
    x = np.clip(x.astype(np.float32), -448, 448)
    x = np.concatenate([x, po.E4M3, (po.E4M3[1:] + po.E4M3[:-1]) / 2]).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn)
    assert np.array_equal(po.narrow(x), want.view(torch.uint8).numpy())
    assert np.array_equal(po.widen8(po.narrow(x)), want.double().numpy())
    rows = np.zeros((4, 128))
    rows[0, 3] = 448.0   # the largest of e4m3: 2^0
    rows[1, 3] = 449.0   # 2^1
    rows[2, 3] = 2.0 ** -90
    codes, byte = po.eight_bits(rows, po.DT_BFLOAT16)
    assert list(byte) == [127, 128, 64, 64]
    assert po.widen8(codes[0])[3] == 448 and po.widen8(codes[1])[3] * 2 == 448 and not codes[2].any() and not codes[3].any()
