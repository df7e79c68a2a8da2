"""A batch over a cache in pages through the C++ face (tests/cpp/op_test_paged.cpp), beside the contiguous path."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu
EXE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "bin", "op_test_paged")


@pytest.mark.parametrize("flags", [
    ("--head_num", 28, "--kv_head_num", 4, "--batch", 3, "--prompt", 100, "--steps", 3, "--dtype", "bf16"),
    ("--head_num", 8, "--kv_head_num", 8, "--batch", 2, "--prompt", 200, "--steps", 2, "--dtype", "fp16", "--is_neox", 0, "--page_size", 48),
    ("--head_num", 12, "--kv_head_num", 2, "--batch", 4, "--prompt", 300, "--steps", 2, "--dtype", "bf16", "--eight", 1),
])
def test_op_test_paged(flags):
    print("running", EXE, *flags, flush=True)
    r = subprocess.run([EXE, *map(str, flags)], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "PASS" in r.stdout, r.stdout + r.stderr
