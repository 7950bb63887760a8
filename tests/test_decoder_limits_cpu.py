"""Calls of the decoder operators whose answer would depend on which workgroup
comes last: refused, without reaching a GPU."""

import ctypes as C

import pytest

from test_decoder_cpu import cross


@pytest.mark.parametrize("stride", [0, 248])
def test_cross_attention_batches_on_one_output(pkg, lib, stride):
    a = cross(pkg, output_batch_stride=stride, query_tokens=1)
    need = lib.dav2_hip_cross_attention_scratch_bytes(C.byref(a))
    a.scratch, a.scratch_bytes = 1 << 20, need
    assert lib.dav2_hip_cross_attention(C.byref(a), None) == 1
