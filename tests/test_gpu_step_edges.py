"""Calls of a decoding step's operators at the edges of what their argument blocks
say: sequences that get nothing, more rows than a launch has, temperatures without
end."""

import math

import pytest

import step_ref
from test_gpu_step import check_sample, ints, launch, norm_args, rand, random_cache, store_args

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f16", "bf16"]


# ---- storing ------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 48])
def test_store_of_nothing_leaves_the_page(gpu, pkg, lib, dtype, d):
    # sequences without new rows, or whose rows are behind the last one, whose last page is begun
    torch = gpu
    cache = random_cache(torch, 3, 8, 2, 16, d)
    for scales in cache[2:]:
        scales[0], scales[1], scales[2], scales[3] = 0.0, 1e-9, math.nan, -1.0
    before = [t.clone() for t in cache]
    table = ints(torch, [[4, 0], [5, 1], [6, 2], [7, 3]])
    k = rand(torch, 1, 6, 2, d, dtype=dtype)
    for starts in ([2, 2, 2, 2, 2], [6, 9, 9, 11, 20]):
        launch(torch, lib, "dav2_hip_cache_store_i4",
               store_args(pkg, cache, k, k, table, ints(torch, starts), ints(torch, [17, 21, 31, 25]), 9, dtype))
        torch.cuda.synchronize()
        for a, b in zip(cache, before):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("behind", [0, 3])
def test_store_beside_idle_sequences(gpu, pkg, lib, dtype, behind):
    # lengths and table entries of idle sequences are stale: their pages belong to those that store now; the rows of
    # those behind the last busy one, if they have any, do not exist
    torch = gpu
    sequences, page_size = 96, 32
    cache = random_cache(torch, 3, 8, 2, page_size, 64)
    table = ints(torch, [[i % 4, 4 + i % 4] for i in range(sequences)])
    lengths = [33 + i % 31 for i in range(sequences)]
    busy = {40: (0, 6), 41: (6, 7), 42: (7, 40), 43: (40, 43)}
    starts, at = [], 0
    for i in range(sequences + 1):
        starts.append(at)
        at = busy.get(i, (0, at))[1] + (behind if i > 43 else 0)
    k, v = rand(torch, 1, 43, 2, 64, dtype=dtype), rand(torch, 2, 43, 2, 64, dtype=dtype, scale=3.0)
    starts, lengths = ints(torch, starts), ints(torch, lengths)
    want = step_ref.store(*cache, k, v, table, starts, lengths)
    launch(torch, lib, "dav2_hip_cache_store_i4", store_args(pkg, cache, k, v, table, starts, lengths, 33, dtype))
    torch.cuda.synchronize()
    for got, w in zip(cache, want):
        assert torch.equal(got.cpu(), w)


# ---- the norm ---------------------------------------------------------------------------


def test_norm_of_more_rows_than_a_launch_has(gpu, pkg, lib):
    # 2^27 rows and five more, of 4096 different ones
    torch = gpu
    rows, columns = (1 << 27) + 5, 8
    x, r = rand(torch, 1, 4096, columns, dtype="bf16"), rand(torch, 2, 4096, columns, dtype="bf16", scale=3.0)
    w = 1 + 0.3 * rand(torch, 3, columns)
    h, y, s, c = (t.cuda() for t in step_ref.add_rms_norm(x, r, w, 1e-6))
    c = torch.cat([c, torch.zeros((4096, 64 - columns), dtype=torch.int8, device="cuda")], dim=1)

    def repeated(t):
        return torch.cat([t[None].expand(rows // 4096, *t.shape).flatten(0, 1), t[:5]])

    total, out = repeated(x), repeated(r)  # in place
    codes, scales = torch.empty((rows, 64), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    launch(torch, lib, "dav2_hip_add_rms_norm",
           norm_args(pkg, total, out, w, total, out, codes, scales, "bf16"))
    torch.cuda.synchronize()
    for got, want in ((total, h), (out, y.to(x.dtype)), (codes, c), (scales, s)):
        assert (got[:rows - 5].unflatten(0, (-1, 4096)) == want).all() and torch.equal(got[rows - 5:], want[:5])


# ---- sampling ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary", [70, 5000, 40000, 270000])
def test_sample_high_temperatures(gpu, pkg, lib, dtype, vocabulary):
    # temperatures at which any finite logit has a weight, infinite ones too: beside logits further apart than fp32
    # holds, masks of the lowest value, infinities; in lists, counted by value, with rows shared and not
    torch = gpu
    n = 12
    x = rand(torch, vocabulary, n, vocabulary, dtype=dtype, scale=3.0)
    f = torch.finfo(x.dtype)
    x[1, 5] = x[1, vocabulary - 1] = math.inf
    x[2, vocabulary // 2:] = f.min
    x[3, ::2], x[3, 1::2] = f.max, f.min
    x[4, : vocabulary // 3] = -math.inf
    x[5, ::2] = math.nan
    x[6] = f.min
    x[7] = f.max
    x[8] = f.min
    x[8, vocabulary // 2] = f.max
    x[9] = f.min
    x[9, ::3] = math.inf
    x[10] = (torch.linspace(-1.0, 1.0, vocabulary, device="cuda", dtype=torch.float64) * f.max).to(x.dtype)
    x[11] = -math.inf
    x[11, 7], x[11, 9] = f.min, f.max
    hot = [math.inf, 3e38, 1e38, 1e37, 1e36]
    for turn in range(len(hot)):
        t = [hot[(i + turn) % len(hot)] for i in range(n)]
        u = [(0.0, 0.31, 0.5, 0.77, 0.9999999)[(3 * i + turn) % 5] for i in range(n)]
        check_sample(torch, pkg, lib, x, u, dtype, temperature=t)
        check_sample(torch, pkg, lib, x, u, dtype, temperature=t, top_p=[0.6] * n)
        check_sample(torch, pkg, lib, x, u, dtype, temperature=t, top_k=[vocabulary // 2] * n, top_p=[0.83] * n,
                     min_p=[0.01] * n)
        check_sample(torch, pkg, lib, x, u, dtype, temperature=t, top_k=[33] * n)
