"""What the attention launchers say about their scratch, from argument blocks
alone: no GPU is reached."""

import ctypes as C
import subprocess
import sys
from pathlib import Path

import pytest

from test_decoder_cpu import P, cross

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.parametrize("sizes", [dict(query_tokens=1, key_tokens=5000), dict(query_tokens=1, key_tokens=10),
                                   dict(batch=64, query_tokens=700, key_tokens=1370), dict(key_tokens=0),
                                   dict(batch=7, key_tokens=33, dtype=1)])
def test_cross_scratch_by_sizes_alone(pkg, lib, sizes):
    # a block without pointers, as the operator surface takes it, asks for what a call with a mask needs
    bare = dict(query=None, keys=None, values=None, output=None)
    need = lib.dav2_hip_cross_attention_scratch_bytes(C.byref(cross(pkg, **bare, **sizes)))
    for pointers in (dict(key_mask=P), dict(key_lengths=P), dict(key_mask=P, key_lengths=P), {}):
        a = cross(pkg, **pointers, **sizes)
        assert lib.dav2_hip_cross_attention_scratch_bytes(C.byref(a)) == need
    # a mask's list of keys is always part of it
    a = cross(pkg, key_mask=P, **sizes)
    assert need >= 4 * a.batch * a.key_tokens
    if need:
        for scratch, size in ((None, need), (P, need - 1), (P + 8, need)):
            a.scratch, a.scratch_bytes = scratch, size
            assert lib.dav2_hip_cross_attention(C.byref(a), None) == 1


@pytest.mark.parametrize("sizes", [dict(batch=1 << 28, heads=1 << 28, kv_heads=1 << 28, query_tokens=256 * 128),
                                   dict(batch=1 << 31, heads=1 << 31, kv_heads=1 << 31, query_tokens=1 << 31),
                                   dict(batch=0xffffffff, heads=0xffffffff, kv_heads=0xffffffff, query_tokens=0xffffffff,
                                        key_tokens=0xffffffff, head_dim=0xffffffff)])
def test_scratch_of_impossible_sizes(pkg, sizes):
    # the question alone must not end the process, in a process of its own
    code = f"""
import ctypes as C, sys
sys.path.insert(0, {str(ROOT / 'tests')!r})
from conftest import load_package
from test_decoder_cpu import attend, cross
pkg = load_package()
lib = pkg.load()
sizes = {sizes!r}
lib.dav2_hip_cross_attention_scratch_bytes(C.byref(cross(pkg, **sizes)))
assert lib.dav2_hip_cross_attention(C.byref(cross(pkg, **sizes)), None) == 1
cache = dict(kv_heads=sizes["kv_heads"])
a = attend(pkg, cache, heads=sizes["heads"], sequences=sizes["batch"], tokens=sizes["query_tokens"], max_query=0xffffffff)
lib.dav2_hip_attention_cache_i8_scratch_bytes(C.byref(a))
assert lib.dav2_hip_attention_cache_i8(C.byref(a), None) == 1
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, (run.returncode, run.stderr)
