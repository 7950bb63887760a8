"""Calls of the decoder operators at the edges of what their argument blocks say:
sequences that get nothing, hints larger than any launch, norms near the ends of
fp32, scratch sized from a block without pointers."""

import ctypes as C
import math

import pytest

import decoder_ref as ref
from gpu_util import db
from test_gpu_decoder import (cross_args, ints, launch, ops, qk_args, qk_want, rand, random_cache,  # noqa: F401
                              store_args, surface)

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f16", "bf16"]


# ---- storing ------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 48])
def test_store_of_nothing_leaves_the_page(gpu, pkg, lib, dtype, d):
    # sequences without new rows whose last page is begun: its scale, below 1e-8 or none, and its codes stay
    torch = gpu
    cache = random_cache(torch, 3, 8, 2, 16, d)
    for scales in cache[2:]:
        scales[0], scales[1], scales[2], scales[3] = 0.0, 1e-9, math.nan, -1.0
    before = [t.clone() for t in cache]
    table = ints(torch, [[4, 0], [5, 1], [6, 2], [7, 3]])
    k = rand(torch, 1, 6, 2, d, dtype=dtype)
    launch(torch, lib, "dav2_hip_cache_store_i8",
           store_args(pkg, cache, k, k, table, ints(torch, [2, 2, 2, 2, 2]), ints(torch, [17, 21, 31, 25]), 3, dtype))
    torch.cuda.synchronize()
    for a, b in zip(cache, before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
def test_store_beside_idle_sequences(gpu, pkg, lib, dtype):
    # lengths and table entries of idle sequences are stale: their pages belong to those that store now
    torch = gpu
    sequences, page_size = 96, 32
    cache = random_cache(torch, 3, 8, 2, page_size, 64)
    table = ints(torch, [[i % 4, 4 + i % 4] for i in range(sequences)])
    lengths = [33 + i % 31 for i in range(sequences)]
    busy = {40: (0, 6), 41: (6, 7), 42: (7, 40), 43: (40, 43)}
    starts, at = [], 0
    for i in range(sequences + 1):
        starts.append(at)
        at = busy.get(i, (0, at))[1]
    k, v = rand(torch, 1, 43, 2, 64, dtype=dtype), rand(torch, 2, 43, 2, 64, dtype=dtype, scale=3.0)
    starts, lengths = ints(torch, starts), ints(torch, lengths)
    want = ref.store(*cache, k, v, table, starts, lengths)
    launch(torch, lib, "dav2_hip_cache_store_i8", store_args(pkg, cache, k, v, table, starts, lengths, 33, dtype))
    torch.cuda.synchronize()
    for got, w in zip(cache, want):
        assert torch.equal(got.cpu(), w)


def test_store_of_more_pages_than_a_launch_has(gpu, pkg, lib):
    # room for 2^29 new tokens in pages of 16; five come, at the end of a table of 2^25 pages
    torch = gpu
    tokens, d = 1 << 29, 16
    cache = random_cache(torch, 3, 4, 1, 16, d)
    small = [t.clone() for t in cache]
    rows = torch.empty((tokens, 1, d), dtype=torch.float16, device="cuda")
    rows[:5] = rand(torch, 1, 5, 1, d, dtype="f16", scale=2.0)
    table = torch.full((1, 1 << 25), 2, dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    starts = ints(torch, [0, 5])
    launch(torch, lib, "dav2_hip_cache_store_i8",
           store_args(pkg, cache, rows, rows, table, starts, ints(torch, [tokens - 3]), tokens, "f16"))
    launch(torch, lib, "dav2_hip_cache_store_i8",
           store_args(pkg, small, rows[:5], rows[:5], ints(torch, [[2, 1]]), starts, ints(torch, [29]), 5, "f16"))
    torch.cuda.synchronize()
    for a, b in zip(cache, small):
        assert torch.equal(a, b)


# ---- norms ------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("head_dim", [64, 33])
@pytest.mark.parametrize("epsilon", [1e-40, 1.2e-38, 1e-30])
def test_norm_near_the_ends_of_fp32(gpu, pkg, lib, dtype, norm, head_dim, epsilon):
    # an epsilon that is subnormal in fp32, heads of zeros and of 1e-18 and 1e17 beside it
    torch = gpu
    epsilon = float(torch.tensor(epsilon, dtype=torch.float32))
    q = rand(torch, 1, 6, 2, head_dim, dtype=dtype)
    q[0] = 0.0
    q[1:3] *= 1e-18
    q[3:5] *= 1e17
    k = q.flip(0).contiguous()
    w = 1 + 0.3 * rand(torch, 2, head_dim)
    positions, freq = ints(torch, [0] * 6), None
    q_out, k_out = torch.full_like(q, math.nan), torch.full_like(k, math.nan)
    launch(torch, lib, "dav2_hip_qk_norm_rotary",
           qk_args(pkg, q, k, q_out, k_out, w, w, positions, freq, 0, "halves", norm, dtype, epsilon))
    torch.cuda.synchronize()
    for x, out in ((q, q_out), (k, k_out)):
        want, bound = qk_want(x, w, norm, epsilon, positions, freq, 0, "halves", dtype)
        ref.assert_within(out, want, bound)


# ---- cross attention through the surface -------------------------------------------------


def cross_case(torch, pkg, lib, dtype, queries, keys, masked=True, batch=3, heads=4, kv=2, d=64):
    """Tensors of a call, its buffers in the surface's order without scratch, and a block without pointers."""
    q = rand(torch, 1, batch, queries, heads, d, dtype=dtype)
    k, v = (rand(torch, i, batch, keys, kv, d, dtype=dtype) for i in (2, 3))
    mask = (torch.rand((batch, keys), device="cuda") < 0.5).to(torch.uint8) if masked else None
    out = torch.full_like(q, math.nan)
    a, _ = cross_args(torch, pkg, lib, q, k, v, out, None, None, dtype, 0.125)
    for name, kind in a._fields_:
        if kind is C.c_void_p:
            setattr(a, name, None)
    a.scratch_bytes = 0
    buffers = [db(pkg, t) for t in (out, q, k, v, None, mask)]
    want, bound = ref.cross(q, k, v, None, mask, 0.125, dtype)
    torch.cuda.synchronize()
    return (q, k, v, mask), out, buffers, a, want, bound


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries,keys", [(1, 1370), (600, 200), (5, 0)])
def test_surface_mask_with_scratch_of_a_bare_block(gpu, pkg, lib, ops, dtype, queries, keys):  # noqa: F811
    torch = gpu
    held, out, buffers, a, want, bound = cross_case(torch, pkg, lib, dtype, queries, keys)
    need = lib.dav2_hip_cross_attention_scratch_bytes(C.byref(a))
    scratch = torch.full((max(need, 1),), 255, dtype=torch.uint8, device="cuda")
    for given in (db(pkg, scratch, need), db(pkg, None)):
        out.fill_(math.nan)
        torch.cuda.synchronize()
        surface(lib, lib.dav2_ops_cross_attention(ops, *buffers, given, C.byref(a)))
        surface(lib, lib.dav2_ops_synchronize(ops))
        ref.assert_within(out, want, bound)
    if need:
        assert lib.dav2_ops_cross_attention(ops, *buffers, db(pkg, scratch, need - 1), C.byref(a)) == 1
        assert b"scratch" in lib.dav2_ops_last_error()


def test_surface_mask_captured(gpu, pkg, lib, ops):  # noqa: F811
    # a mask or split keys under capture bring a scratch; a call that touches none needs none
    torch = gpu
    masked = cross_case(torch, pkg, lib, "f16", 1, 1370)
    whole = cross_case(torch, pkg, lib, "bf16", 300, 60, masked=False)
    need = lib.dav2_hip_cross_attention_scratch_bytes(C.byref(masked[3]))
    scratch = torch.empty(need, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.ExternalStream(lib.dav2_ops_stream(ops))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        refused = lib.dav2_ops_cross_attention(ops, *masked[2], db(pkg, None), C.byref(masked[3]))
        text = lib.dav2_ops_last_error()
        rc = [lib.dav2_ops_cross_attention(ops, *masked[2], db(pkg, scratch), C.byref(masked[3])),
              lib.dav2_ops_cross_attention(ops, *whole[2], db(pkg, None), C.byref(whole[3]))]
    assert refused == 1 and b"scratch" in text and rc == [0, 0]
    for replay in range(4):
        for case in (masked, whole):
            case[1].fill_(math.nan)
        scratch.fill_(255)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
        for case in (masked, whole):
            ref.assert_within(case[1], case[4], case[5], str(replay))
        eager = torch.full_like(masked[1], math.nan)
        torch.cuda.synchronize()
        surface(lib, lib.dav2_ops_cross_attention(ops, db(pkg, eager), *masked[2][1:], db(pkg, None), C.byref(masked[3])))
        surface(lib, lib.dav2_ops_synchronize(ops))
        assert torch.equal(eager, masked[1])
