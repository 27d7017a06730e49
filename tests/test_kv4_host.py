"""Host checks of what the attention over the 4-bit cache takes from the caller's data, and of its refusals (no GPU)."""
import os
import subprocess

import pytest

import ternary_llm_amd as tl
from tests.test_kv4 import _attend_call, _kv4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rows_and_positions_of_any_starts(tmp_path):
    """Starts that descend, lie out of range or are as far apart as 32 bits allow."""
    exe = tmp_path / "kv4_rows_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover=all",
                    "-I", os.path.join(ROOT, "ternary-llm_amd", "csrc"), os.path.join(ROOT, "tests", "kv4_rows_check.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and "bad=0" in out.stdout, out.stdout + out.stderr


def test_attention_takes_all_sizes_that_it_can_count():
    """Calls within the header's limits are taken, on both sides of what 32 bits count."""
    def size(heads, kv, max_query, max_length, **sizes):
        return tl.lib().tllm_attention_kv4_workspace_bytes(*_kv4(heads=kv, **sizes), heads, max_query, max_length)

    many = dict(pages=1000, page=64, width=2048)
    assert size(4, 1, 1, 131072, batch=40000, n=40000, **many) > 0                       # single tokens of many users
    assert size(32, 8, 32768, 131072, batch=512, n=1 << 23, **many) > 0                  # prompts and single tokens, long ones among them
    assert size(32, 8, 4096, 131072, batch=64, n=64 * 4096, **many) == 0                 # prompts, a row tile a workgroup
    wide = dict(pages=1000, page=16, batch=65535)
    assert size(8, 1, 1, 1 << 18, n=65535, width=1 << 17, **wide) > 0                    # batch * max_length just below 2^34
    assert size(64, 1, 1, 1 << 18, n=65535, width=1 << 17, **wide) > 0
    assert size(8, 1, 1, 1 << 30, n=65535, width=1 << 17, **wide) == -4                  # ... and 2^21 positions each: 2^32 steps
    assert size(64, 1, 1 << 15, 16, n=1 << 23, width=1, **wide) >= 0                     # batch * rows 2^37
    assert size(64, 1, 1 << 21, 16, n=1 << 23, width=1, **wide) == -4                    # 2^43: 2^35 row tiles
    # the call itself refuses them too, before it looks at anything on the device
    assert _attend_call(heads=8, kv_heads=1, qs=512, os_=512, mq=1, ml=1 << 30, n=65535, width=1 << 17, pages=1000, page=16, batch=65535) == -4


def test_numbers_beyond_32_bits():
    """A window of 2^32 is not none, a bound of 2^32 + 1 not one position."""
    import torch
    q = torch.zeros(3, 4, 64, dtype=torch.float16)
    pos = torch.zeros(3, dtype=torch.int32)
    cache = tl.kv4_cache(4, 16, 4, 64, device="cpu")
    batch = (torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32))
    for wrong in (2 ** 31, 2 ** 32 + 1, -2 ** 31 - 1):
        with pytest.raises(ValueError, match="window"):
            tl.attention_kv4(q, q.clone(), *cache, *batch, 3, 32, window=wrong)
        with pytest.raises(ValueError, match="max_length"):
            tl.attention_kv4(q, q.clone(), *cache, *batch, 3, wrong)
        with pytest.raises(ValueError, match="max_query"):
            tl.attention_kv4(q, q.clone(), *cache, *batch, wrong, 32)
        for name, numbers in (("n_heads", (wrong, 3, 3, 32)), ("n_rows", (4, wrong, 3, 32)), ("max_query", (4, 3, wrong, 32)), ("max_length", (4, 3, 3, wrong))):
            with pytest.raises(ValueError, match=name):
                tl.attention_kv4_workspace_bytes(numbers[0], *cache, *batch, *numbers[1:])
        with pytest.raises(ValueError, match="rotary_dim"):
            tl.rotary(q, None, q, None, pos, wrong, 1e4)
        with pytest.raises(ValueError, match="original_length"):
            tl.rotary(q, None, q, None, pos, 64, 1e4, scaling="yarn", original_length=wrong)
