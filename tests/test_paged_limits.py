"""More workgroups than a launch takes: the attention over pages says so, before it asks for anything of the device.  No GPU."""
import pytest

from tests.test_paged_host import call


# (tokens, batch, max_q_len, group, kv heads): single tokens; tiles; both in one launch
@pytest.mark.parametrize("tokens,batch,max_q_len,group,kv_heads", [
    (16384, 16384, 1, 1, 1024), (65535, 65535, 1, 1, 257), (65535, 65535, 1, 1, 65535), (1 << 26, 1, 1 << 26, 1, 65), (1 << 30, 1, 1 << 30, 1, 2),
    (1 << 24, 65535, 4096, 8, 128)])
def test_refused(tokens, batch, max_q_len, group, kv_heads):
    sizes = dict(tokens=tokens, batch=batch, max_q_len=max_q_len, group_size=group, kv_head_num=kv_heads, page_stride=16 * kv_heads * 256)
    assert call("llmhip_paged_flash_attn_gqa", **sizes, max_kv_len=64) == -2
