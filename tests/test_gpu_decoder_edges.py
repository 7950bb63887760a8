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
