"""What the attention launchers say about their scratch, from argument blocks
alone: no GPU is reached."""

import ctypes as C

import pytest

from test_decoder_cpu import P, attend, cross


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
