"""Calls of the decoder operators at the edges of what their argument blocks say:
sequences that get nothing, hints larger than any launch, norms near the ends of
fp32, scratch sized from a block without pointers."""

import ctypes as C
import math

import pytest

import decoder_ref as ref
from test_gpu_decoder import ints, launch, ptr, rand, random_cache, store_args

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
