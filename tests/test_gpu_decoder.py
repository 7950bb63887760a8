"""The decoder operators (rotary positions, query/key norms, the int8 cache,
attention over it, cross attention) against float64, through the launcher
layer, the operator surface, captured graphs, and together."""

import ctypes as C
import math

import pytest

import decoder_ref as ref
from gpu_util import db

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def ops(gpu, lib):
    h = lib.dav2_ops_create(0)
    assert h, lib.dav2_ops_last_error()
    yield h
    lib.dav2_ops_destroy(h)


def ptr(t):
    return None if t is None else t.data_ptr()


def launch(torch, lib, entry, args, stream=None):
    s = (stream or torch.cuda.current_stream()).cuda_stream
    rc = getattr(lib, entry)(C.byref(args), s)
    assert rc == 0, f"{entry}: {rc}"


def rand(torch, seed, *shape, dtype="f32", scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(ref.DTYPES[dtype])


def ints(torch, values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- rotary ---------------------------------------------------------------------


def rotary_args(pkg, x, out, positions, freq, rotary_dim, layout, dtype, amplitude=1.0):
    return pkg.RotaryArgs(input=ptr(x), output=ptr(out), input_stride=x.stride(0), output_stride=out.stride(0),
                          positions=ptr(positions), frequencies=ptr(freq), tokens=x.shape[0], heads=x.shape[1],
                          head_dim=x.shape[2], rotary_dim=rotary_dim, layout=pkg.ROTARY_LAYOUT[layout],
                          dtype=pkg.DTYPE[dtype], amplitude=amplitude)


def rotary_bound(want, size, dtype):
    # cos and sin within 8 steps of fp32, their products and sum three roundings
    return size * 12 * ref.U + want.abs() * ref.half_step(dtype) + ref.floor_of(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("tokens,heads,head_dim,rotary_dim", [(1, 1, 2, 2), (5, 3, 64, 64), (7, 2, 80, 20),
                                                              (33, 5, 128, 64), (2, 9, 96, 96), (3, 1, 256, 128),
                                                              (130, 16, 64, 32), (3, 2, 7, 4), (2, 3, 1024, 1024)])
def test_rotary(gpu, pkg, lib, dtype, layout, tokens, heads, head_dim, rotary_dim):
    torch = gpu
    x = rand(torch, tokens + head_dim, tokens, heads, head_dim, dtype=dtype)
    positions = torch.randint(-1000, 1000000, (tokens,), dtype=torch.int32, device="cuda")
    freq = ref.frequencies(rotary_dim)
    out = torch.full_like(x, math.nan)
    launch(torch, lib, "dav2_hip_rotary", rotary_args(pkg, x, out, positions, freq, rotary_dim, layout, dtype, 1.25))
    want, size = ref.rotary(x.double(), positions, freq, rotary_dim, layout, 1.25)
    ref.assert_within(out, want, rotary_bound(want, size, dtype))
    # in place
    launch(torch, lib, "dav2_hip_rotary", rotary_args(pkg, x, x, positions, freq, rotary_dim, layout, dtype, 1.25))
    assert torch.equal(x, out)


@pytest.mark.parametrize("offset,stride_more", [(0, 8), (1, 3), (8, 1), (4, 4)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rotary_strides_and_alignment(gpu, pkg, lib, dtype, offset, stride_more):
    torch = gpu
    tokens, heads, head_dim = 19, 3, 64
    stride = heads * head_dim + stride_more
    store = rand(torch, 5, offset + tokens * stride, dtype=dtype)
    x = store[offset:].as_strided((tokens, heads, head_dim), (stride, head_dim, 1), offset)
    whole = torch.full((tokens * stride + 16,), 7.0, dtype=ref.DTYPES[dtype], device="cuda")
    out = whole.as_strided((tokens, heads, head_dim), (stride, head_dim, 1), offset)
    positions, freq = torch.arange(tokens, dtype=torch.int32, device="cuda"), ref.frequencies(head_dim)
    launch(torch, lib, "dav2_hip_rotary", rotary_args(pkg, x, out, positions, freq, head_dim, "halves", dtype))
    want, size = ref.rotary(x.double(), positions, freq, head_dim, "halves")
    ref.assert_within(out, want, rotary_bound(want, size, dtype))
    rest = torch.ones_like(whole, dtype=torch.bool)
    rest.as_strided((tokens, heads, head_dim), (stride, head_dim, 1), offset).fill_(False)
    assert (whole[rest] == 7.0).all()  # nothing beside the heads is written


def test_rotary_not_finite(gpu, pkg, lib):
    torch = gpu
    x = rand(torch, 1, 4, 2, 64)
    x[1, 0, 3], x[2, 1, 40] = math.nan, math.inf
    positions, freq = ints(torch, [1, 2, 3, 4]), ref.frequencies(64)
    out = torch.empty_like(x)
    launch(torch, lib, "dav2_hip_rotary", rotary_args(pkg, x, out, positions, freq, 64, "halves", "f32"))
    touched = torch.zeros_like(x, dtype=torch.bool)
    touched[1, 0, 3] = touched[1, 0, 35] = touched[2, 1, 8] = touched[2, 1, 40] = True
    assert torch.equal(~out.isfinite(), touched)


# ---- query / key norm ----------------------------------------------------------------


def qk_args(pkg, q, k, q_out, k_out, qw, kw, positions, freq, rotary_dim, layout, norm, dtype, epsilon=1e-6):
    return pkg.QkNormRotaryArgs(
        query=ptr(q), key=ptr(k), query_out=ptr(q_out), key_out=ptr(k_out), query_stride=q.stride(0),
        key_stride=k.stride(0), query_out_stride=q_out.stride(0), key_out_stride=k_out.stride(0), query_weight=ptr(qw),
        key_weight=ptr(kw), positions=ptr(positions), frequencies=ptr(freq), tokens=q.shape[0],
        query_heads=q.shape[1], key_heads=k.shape[1], head_dim=q.shape[2], rotary_dim=rotary_dim,
        layout=pkg.ROTARY_LAYOUT[layout], dtype=pkg.DTYPE[dtype], norm=pkg.QK_NORM[norm], epsilon=epsilon,
        amplitude=1.0)


def qk_want(x, weight, norm, epsilon, positions, freq, rotary_dim, layout, dtype):
    y, most = ref.norm(x.double(), weight, norm, epsilon)
    want, _ = (y, None) if rotary_dim == 0 else ref.rotary(y, positions, freq, rotary_dim, layout)
    # mean and variance are sums of head_dim / 64 terms per lane and 6 joins; with the root, the
    # quotient, the weight and the rotation fewer than 40 + head_dim / 32 roundings of at most
    # `most`, two values of which a rotation adds
    bound = 2 * most * (40 + x.shape[-1] / 32) * ref.U + want.abs() * ref.half_step(dtype) + ref.floor_of(dtype)
    return want, bound


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm,layout", [("rms", "halves"), ("layer", "pairs"), ("rms", "pairs")])
@pytest.mark.parametrize("tokens,heads,kv,head_dim,rotary_dim", [(1, 4, 2, 64, 64), (9, 8, 1, 128, 128),
                                                                 (3, 3, 3, 80, 40), (5, 2, 1, 256, 64),
                                                                 (70, 6, 2, 96, 96), (4, 2, 2, 33, 16),
                                                                 (2, 1, 1, 64, 0), (2, 2, 1, 1024, 512)])
def test_qk_norm_rotary(gpu, pkg, lib, dtype, norm, layout, tokens, heads, kv, head_dim, rotary_dim):
    torch = gpu
    rows = rand(torch, tokens * 3 + head_dim, tokens, (heads + 2 * kv) * head_dim, dtype=dtype, scale=3.0)
    rows[0] = 0.0  # a head of zeros
    q = rows[:, :heads * head_dim].unflatten(1, (heads, head_dim))
    k = rows[:, heads * head_dim:(heads + kv) * head_dim].unflatten(1, (kv, head_dim))
    qw, kw = 1 + 0.3 * rand(torch, 1, head_dim), None if tokens == 3 else 1 + 0.3 * rand(torch, 2, head_dim)
    positions = torch.randint(0, 200000, (tokens,), dtype=torch.int32, device="cuda")
    freq = ref.frequencies(rotary_dim) if rotary_dim else None
    q_out, k_out = (torch.full(x.shape, math.nan, dtype=x.dtype, device="cuda") for x in (q, k))
    launch(torch, lib, "dav2_hip_qk_norm_rotary",
           qk_args(pkg, q, k, q_out, k_out, qw, kw, positions, freq, rotary_dim, layout, norm, dtype))
    for x, w, out in ((q, qw, q_out), (k, kw, k_out)):
        want, bound = qk_want(x, w, norm, 1e-6, positions, freq, rotary_dim, layout, dtype)
        ref.assert_within(out, want, bound)
    # in place within the packed rows; the values' part stays
    before = rows.clone()
    launch(torch, lib, "dav2_hip_qk_norm_rotary",
           qk_args(pkg, q, k, q, k, qw, kw, positions, freq, rotary_dim, layout, norm, dtype))
    assert torch.equal(q, q_out) and torch.equal(k, k_out)
    assert torch.equal(rows[:, (heads + kv) * head_dim:], before[:, (heads + kv) * head_dim:])


# ---- the cache -------------------------------------------------------------------------


def random_cache(torch, seed, pages, heads, page_size, head_dim):
    g = torch.Generator(device="cuda").manual_seed(seed)
    keys = torch.randint(-127, 128, (pages, heads, page_size, head_dim), generator=g, dtype=torch.int8, device="cuda")
    values = torch.randint(-127, 128, (pages, heads, head_dim, page_size), generator=g, dtype=torch.int8,
                           device="cuda")
    ks = 0.005 + 0.02 * torch.rand((pages, heads), generator=g, device="cuda")
    vs = 0.005 + 0.02 * torch.rand((pages, heads), generator=g, device="cuda")
    return [keys, values, ks, vs]


def cache_struct(pkg, cache):
    keys = cache[0]
    return pkg.CacheI8(keys=ptr(cache[0]), values=ptr(cache[1]), key_scales=ptr(cache[2]), value_scales=ptr(cache[3]),
                       pages=keys.shape[0], kv_heads=keys.shape[1], page_size=keys.shape[2], head_dim=keys.shape[3])


def shuffled_table(torch, seed, sequences, most, pages):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[:sequences * most].to(torch.int32).view(sequences, most).cuda()


def store_args(pkg, cache, k, v, table, starts, lengths, max_new, dtype):
    return pkg.CacheStoreI8Args(cache=cache_struct(pkg, cache), keys=ptr(k), values=ptr(v), key_stride=k.stride(0),
                                value_stride=v.stride(0), page_table=ptr(table), starts=ptr(starts),
                                lengths=ptr(lengths), sequences=lengths.numel(), table_pages=table.shape[1],
                                tokens=k.shape[0], max_new=max_new, dtype=pkg.DTYPE[dtype])


def check_store(torch, pkg, lib, cache, k, v, table, starts, lengths, max_new, dtype):
    want = ref.store(*cache, k, v, table, starts, lengths)
    for again in range(2):  # the second call stores the same rows again
        launch(torch, lib, "dav2_hip_cache_store_i8",
               store_args(pkg, cache, k, v, table, starts, lengths, max_new, dtype))
        torch.cuda.synchronize()
        for name, got, w in zip(("keys", "values", "key scales", "value scales"), cache, want):
            assert torch.equal(got.cpu(), w), (name, again)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page_size", [16, 32, 128, 208])
@pytest.mark.parametrize("heads,head_dim", [(1, 64), (3, 80), (2, 128), (5, 16)])
def test_cache_store(gpu, pkg, lib, dtype, page_size, heads, head_dim):
    torch = gpu
    # one token into a full table, none, some that end inside a page, some that cross pages, a first token
    new, total = [1, 0, 5, 2 * page_size + 3, 1, page_size], [page_size + 4, 7, 11, 3 * page_size + 1, 1, page_size]
    starts = ints(torch, [sum(new[:i]) for i in range(len(new) + 1)])
    cache = random_cache(torch, page_size + heads, 6 * 4 + 3, heads, page_size, head_dim)
    table = shuffled_table(torch, 3, 6, 4, 6 * 4 + 3)
    # rows wider than their heads, some larger than the pages' old values
    wide = rand(torch, 9, sum(new) + 2, heads * head_dim + 8, dtype=dtype)
    wide[::3] *= 3.0
    k = wide[:, :heads * head_dim].unflatten(1, (heads, head_dim))
    v = rand(torch, 8, sum(new) + 2, heads, head_dim, dtype=dtype, scale=0.7)
    check_store(torch, pkg, lib, cache, k, v, table, starts, ints(torch, total), max(new), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,more", [(1, 0), (0, 1), (3, 5)])
def test_cache_store_alignment(gpu, pkg, lib, dtype, offset, more):
    torch = gpu
    tokens, heads, d, page_size = 45, 3, 48, 32
    stride = heads * d + more
    k, v = (rand(torch, i, offset + tokens * stride, dtype=dtype).as_strided((tokens, heads, d), (stride, d, 1), offset)
            for i in (1, 2))
    cache = random_cache(torch, 3, 8, heads, page_size, d)
    table = shuffled_table(torch, 4, 2, 4, 8)
    check_store(torch, pkg, lib, cache, k, v, table, ints(torch, [0, 5, 45]), ints(torch, [37, 100]), 40, dtype)


def test_cache_store_one_by_one(gpu, pkg, lib):
    # growing values: every token of a page makes its scale larger and its older codes smaller
    torch = gpu
    cache = random_cache(torch, 1, 4, 2, 16, 64)
    table = ints(torch, [[2, 0, 3]])
    for t in range(37):
        k = rand(torch, t, 1, 2, 64, scale=1.2 ** t)
        v = rand(torch, 100 + t, 1, 2, 64, scale=0.8 ** t)
        check_store(torch, pkg, lib, cache, k, v, table, ints(torch, [0, 1]), ints(torch, [t + 1]), 1, "f32")


def test_cache_store_bad_pages_and_ranges(gpu, pkg, lib):
    # pages that do not exist, rows and positions outside, a hint that is too small
    torch = gpu
    cache = random_cache(torch, 4, 8, 2, 16, 32)
    table = ints(torch, [[0, 8, 1], [-1, 2, 3], [4, 5, 2 ** 31 - 1], [6, 7, -2 ** 31]])
    k, v = rand(torch, 1, 130, 2, 32), rand(torch, 2, 130, 2, 32)
    starts = ints(torch, [-3, 40, 70, 110, 400])
    check_store(torch, pkg, lib, cache, k, v, table, starts, ints(torch, [40, 47, 60, 10]), 1, "f32")


def test_cache_store_small_and_not_finite(gpu, pkg, lib):
    torch = gpu
    cache = random_cache(torch, 6, 3, 1, 16, 32)
    table = ints(torch, [[1, 2]])
    tiny = rand(torch, 1, 16, 1, 32, scale=1e-7)
    tiny[3] = 0.0
    check_store(torch, pkg, lib, cache, tiny, torch.zeros_like(tiny), table, ints(torch, [0, 16]), ints(torch, [16]),
                16, "f32")
    bad = rand(torch, 2, 2, 1, 32)
    bad[1, 0, 5] = math.nan
    worse = rand(torch, 3, 2, 1, 32)
    worse[0, 0, 31] = -math.inf
    launch(torch, lib, "dav2_hip_cache_store_i8",
           store_args(pkg, cache, bad, worse, table, ints(torch, [0, 2]), ints(torch, [18]), 2, "f32"))
    torch.cuda.synchronize()
    assert cache[2][2, 0].isnan() and cache[3][2, 0].isinf()  # the page says so
    assert cache[2][1].isfinite().all()
    fine = rand(torch, 4, 1, 1, 32)  # begun anew, the page is sound again
    check_store(torch, pkg, lib, cache, fine, fine, table, ints(torch, [0, 1]), ints(torch, [17]), 1, "f32")


# ---- attention over the cache -------------------------------------------------------------


def attend_args(torch, pkg, lib, cache, q, out, table, starts, lengths, causal, dtype, scale, max_query=None,
                max_length=None):
    a = pkg.AttentionCacheI8Args(
        cache=cache_struct(pkg, cache), query=ptr(q), output=ptr(out), query_stride=q.stride(0),
        output_stride=out.stride(0), page_table=ptr(table), starts=ptr(starts), lengths=ptr(lengths),
        sequences=lengths.numel(), table_pages=table.shape[1], tokens=q.shape[0], heads=q.shape[1],
        max_query=max_query or int(starts.diff().max()), max_length=max_length or max(int(lengths.max()), 1),
        causal=int(causal), dtype=pkg.DTYPE[dtype], scale=scale)
    size = lib.dav2_hip_attention_cache_i8_scratch_bytes(C.byref(a))
    scratch = None
    if size:
        scratch = torch.full((size,), 255, dtype=torch.uint8, device="cuda")  # NaN, if any of it were read unwritten
        a.scratch, a.scratch_bytes = ptr(scratch), size
    return a, scratch


LONG = 2 ** 22  # as max_length: many rows take the way of a long cache, whatever the lengths are


def check_attend(torch, pkg, lib, cache, q, table, starts, lengths, causal, dtype, scale=None, **hints):
    scale = scale or 1 / math.sqrt(q.shape[2])
    want, bound = ref.attend(q, cache, table, starts, lengths, causal, scale, dtype)
    nobody = want.isnan()
    for hint in (hints, dict(max_length=LONG)) if "max_length" not in hints else (hints,):
        out = torch.full(q.shape, 3.0, dtype=q.dtype, device="cuda")
        a, keep = attend_args(torch, pkg, lib, cache, q, out, table, starts, lengths, causal, dtype, scale, **hint)
        launch(torch, lib, "dav2_hip_attention_cache_i8", a)
        torch.cuda.synchronize()
        assert (out[nobody] == 3.0).all()  # rows of no sequence are left alone
        ref.assert_within(torch.where(nobody, want, out.double()), want, bound, str(hint))
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,head_dim,page_size", [(1, 1, 64, 16), (8, 2, 128, 16), (6, 6, 80, 48),
                                                         (16, 1, 128, 64), (5, 1, 96, 256), (40, 2, 64, 32),
                                                         (3, 3, 16, 16)])
def test_cache_attention_single_tokens(gpu, pkg, lib, dtype, heads, kv, head_dim, page_size):
    torch = gpu
    lengths = [1, 0, 15, 16, 17, 63, 64, 65, 257, 1370]
    most = -(-max(lengths) // page_size)
    cache = random_cache(torch, heads + head_dim, len(lengths) * most + 1, kv, page_size, head_dim)
    table = shuffled_table(torch, 2, len(lengths), most, len(lengths) * most + 1)
    q = rand(torch, 5, len(lengths), heads, head_dim, dtype=dtype)
    check_attend(torch, pkg, lib, cache, q, table, ints(torch, list(range(len(lengths) + 1))), ints(torch, lengths),
                 True, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,head_dim,page_size", [(4, 2, 64, 16), (8, 1, 128, 32), (3, 3, 80, 64),
                                                         (10, 2, 112, 144)])
def test_cache_attention_prompts(gpu, pkg, lib, dtype, causal, heads, kv, head_dim, page_size):
    torch = gpu
    # a whole prompt, a chunk behind older tokens, more rows than tokens (the first see nothing), none, one
    new, total = [70, 33, 9, 0, 1, 130], [70, 333, 5, 40, 200, 131]
    starts = ints(torch, [sum(new[:i]) for i in range(len(new) + 1)])
    most = -(-max(total) // page_size)
    cache = random_cache(torch, 17 + heads, len(new) * most, kv, page_size, head_dim)
    table = shuffled_table(torch, 7, len(new), most, len(new) * most)
    q = rand(torch, 6, sum(new) + 3, heads, head_dim, dtype=dtype)  # three rows of no sequence
    check_attend(torch, pkg, lib, cache, q, table, starts, ints(torch, total), causal, dtype)


def test_cache_attention_long(gpu, pkg, lib):
    # the keys are split over many workgroups
    torch = gpu
    lengths = [40000, 3, 12345]
    cache = random_cache(torch, 3, 1600, 2, 64, 128)
    table = shuffled_table(torch, 4, 3, 625, 1600) if 3 * 625 <= 1600 else None
    table = torch.randint(0, 1600, (3, 625), dtype=torch.int32, device="cuda") if table is None else table
    for dtype in DTYPES:
        q = rand(torch, 8, 3, 8, 128, dtype=dtype)
        check_attend(torch, pkg, lib, cache, q, table, ints(torch, [0, 1, 2, 3]), ints(torch, lengths), True, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sequences,queries,heads,kv,head_dim,page_size", [(64, 20, 16, 8, 64, 16), (8, 256, 32, 32, 80, 32),
                                                                           (8, 250, 32, 32, 128, 16)])
def test_cache_attention_whole(gpu, pkg, lib, dtype, sequences, queries, heads, kv, head_dim, page_size):
    # tiles enough to fill the chip: the keys are not split
    torch = gpu
    total = [queries - 1 + 37 * (i % 5) for i in range(sequences)]
    most = -(-max(total) // page_size)
    cache = random_cache(torch, 5 + heads, 200, kv, page_size, head_dim)
    table = torch.randint(0, 200, (sequences, most), dtype=torch.int32, device="cuda")  # pages that several have
    q = rand(torch, 6, sequences * queries, heads, head_dim, dtype=dtype)
    starts = ints(torch, [queries * i for i in range(sequences + 1)])
    check_attend(torch, pkg, lib, cache, q, table, starts, ints(torch, total), True, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cache_attention_more_tiles_than_said(gpu, pkg, lib, dtype):
    # max_query 1 with 40 heads of one cache head: a workgroup goes through all tiles of rows
    torch = gpu
    cache = random_cache(torch, 5, 40, 1, 16, 128)
    table = shuffled_table(torch, 6, 2, 20, 40)
    q = rand(torch, 6, 71, 40, 128, dtype=dtype)
    check_attend(torch, pkg, lib, cache, q, table, ints(torch, [0, 40, 71]), ints(torch, [300, 31]), True, dtype,
                 max_query=1, max_length=LONG)


@pytest.mark.parametrize("queries", [1, 40])
def test_far_pages(gpu, pkg, lib, queries):
    # pages past 2^32 bytes of a cache: stored and read as in a small one
    torch = gpu
    heads, page_size, d, count = 2, 256, 128, 3
    pages = 2 ** 32 // (heads * page_size * d) + 4
    near = random_cache(torch, 1, count, heads, page_size, d)
    far = [torch.empty((pages, *t.shape[1:]), dtype=t.dtype, device="cuda") for t in near]
    for a, b in zip(near, far):
        b[-count:].copy_(a)
    order = ints(torch, [[2, 0, 1]])
    k, v = rand(torch, 2, queries, heads, d), rand(torch, 3, queries, heads, d)
    q = rand(torch, 4, queries, 2 * heads, d)
    starts, lengths = ints(torch, [0, queries]), ints(torch, [530])
    outs = []
    for cache, table in ((near, order), (far, order + pages - count)):
        launch(torch, lib, "dav2_hip_cache_store_i8", store_args(pkg, cache, k, v, table, starts, lengths, queries, "f32"))
        for hint in (None, LONG):
            out = torch.full_like(q, math.nan)
            a, keep = attend_args(torch, pkg, lib, cache, q, out, table, starts, lengths, True, "f32", 0.1, max_length=hint)
            launch(torch, lib, "dav2_hip_attention_cache_i8", a)
            outs.append(out)
            torch.cuda.synchronize()
    for a, b in zip(near, far):
        assert torch.equal(a, b[-count:])
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3]) and outs[0].isfinite().all()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_far_strides(gpu, pkg, lib, dtype):
    # rows and batches past 2^32 bytes of their tensor
    torch = gpu
    apart, d, heads = 2 ** 31 + 64, 64, 2
    store = torch.empty(apart + 512 * heads * d, dtype=ref.DTYPES[dtype], device="cuda")

    def far(x, stride):  # x with its first axis apart
        y = store.as_strided(x.shape, (apart, *stride[1:]), 0)
        y.copy_(x)
        return y

    q, k, v = (rand(torch, i, 2, n, heads, d, dtype=dtype) for i, n in ((1, 5), (2, 200), (3, 200)))
    mask = torch.ones((2, 200), dtype=torch.uint8, device="cuda")
    mask[:, ::3] = 0
    outs = []
    for tensors in ((q, k, v), (far(q, q.stride()), k, v), (q, far(k, k.stride()), v), (q, k, far(v, v.stride()))):
        for m in (None, mask):
            out = torch.full_like(q, math.nan)
            # the buffer holds one of them at a time: written here, read before the next is written
            if tensors[0] is not q:
                tensors[0].copy_(q)
            if tensors[1] is not k:
                tensors[1].copy_(k)
            if tensors[2] is not v:
                tensors[2].copy_(v)
            a, keep = cross_args(torch, pkg, lib, *tensors, out, None, m, dtype, 0.125)
            launch(torch, lib, "dav2_hip_cross_attention", a)
            torch.cuda.synchronize()
            outs.append(out)
    for i in range(2, len(outs)):
        assert torch.equal(outs[i], outs[i % 2])
    assert outs[0].isfinite().all()
    x = rand(torch, 5, 2, heads, d, dtype=dtype)
    positions, freq = ints(torch, [3, 70000]), ref.frequencies(d)
    y, z = torch.empty_like(x), far(x, x.stride())
    launch(torch, lib, "dav2_hip_rotary", rotary_args(pkg, x, y, positions, freq, d, "halves", dtype))
    launch(torch, lib, "dav2_hip_rotary", rotary_args(pkg, z, z, positions, freq, d, "halves", dtype))
    torch.cuda.synchronize()
    assert torch.equal(y, z)


@pytest.mark.parametrize("queries", [1, 40])
def test_cache_attention_hints_too_small(gpu, pkg, lib, queries):
    # max_query and max_length size the launch; sequences beyond them are computed all the same
    torch = gpu
    cache = random_cache(torch, 3, 60, 2, 32, 64)
    table = shuffled_table(torch, 4, 2, 30, 60)
    q = rand(torch, 8, 2 * queries, 4, 64, dtype="f16")
    check_attend(torch, pkg, lib, cache, q, table, ints(torch, [0, queries, 2 * queries]), ints(torch, [900, 77]), True,
                 "f16", max_query=1, max_length=1)


@pytest.mark.parametrize("queries", [1, 50])
def test_cache_attention_bad_pages(gpu, pkg, lib, queries):
    torch = gpu
    cache = random_cache(torch, 3, 9, 1, 16, 64)
    table = ints(torch, [[0, -1, 2, 9, 4], [-5, 100, 2 ** 31 - 1, -2 ** 31, 9], [5, 6, 7, 8, 1]])
    q = rand(torch, 8, 3 * queries, 2, 64)
    starts = ints(torch, [0, queries, 2 * queries, 3 * queries])
    out = check_attend(torch, pkg, lib, cache, q, table, starts, ints(torch, [70, 80, 100000]), False, "f32")
    assert (out[queries:2 * queries] == 0).all()  # nothing to see


@pytest.mark.parametrize("queries", [1, 65])
@pytest.mark.parametrize("dtype", DTYPES)
def test_cache_attention_unequal_scales(gpu, pkg, lib, queries, dtype):
    # the page that carries the weight has values a million times smaller than a page that carries none;
    # large scores; pages of zeros (scale 1e-8)
    torch = gpu
    cache = random_cache(torch, 3, 8, 2, 16, 64)
    cache[3][:] = 1e-6 * cache[3]
    cache[3][2], cache[3][5] = 1.0, 1e-8
    cache[2][:] *= 20.0
    cache[2][2], cache[2][4] = 1e-8, 1e-8
    table = ints(torch, [[0, 2, 1, 3, 5], [2, 5, 4, 6, 7]])
    q = rand(torch, 8, 2 * queries, 2, 64, dtype=dtype, scale=2.0)
    check_attend(torch, pkg, lib, cache, q, table, ints(torch, [0, queries, 2 * queries]), ints(torch, [77, 80]), True,
                 dtype)


@pytest.mark.parametrize("queries", [1, 33])
def test_cache_attention_range_of_queries(gpu, pkg, lib, queries):
    # values that binary16 does not hold, in the types that do, and subnormal ones
    torch = gpu
    cache = random_cache(torch, 3, 8, 1, 16, 64)
    table = ints(torch, [[0, 1, 2, 3]])
    for dtype, size in (("f32", 1e9), ("bf16", 1e9), ("f32", 1e-12), ("bf16", 1e-12), ("f16", 3e-6)):
        q = rand(torch, 8, queries, 4, 64, dtype=dtype, scale=size)
        check_attend(torch, pkg, lib, cache, q, table, ints(torch, [0, queries]), ints(torch, [60]), True, dtype,
                     scale=0.125 / size)


@pytest.mark.parametrize("queries", [1, 40])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("most", [None, LONG])
def test_cache_attention_not_finite(gpu, pkg, lib, queries, dtype, most):
    # NaN and infinity in a query, NaN pages behind the last token and in pages of nobody stay where they are
    torch = gpu
    cache = random_cache(torch, 3, 8, 2, 32, 64)
    table = ints(torch, [[0, 1, 6], [3, 4, 7]])
    cache[2][6], cache[3][6], cache[2][7, 0], cache[3][5] = math.nan, math.nan, math.nan, math.inf
    q = rand(torch, 8, 2 * queries, 4, 64, dtype=dtype)
    starts, lengths = ints(torch, [0, queries, 2 * queries]), ints(torch, [64, 64])
    check_attend(torch, pkg, lib, cache, q, table, starts, lengths, True, dtype)
    q[0, 1, 3] = math.nan
    q[0, 2, 7] = math.inf
    out = torch.zeros_like(q)
    a, keep = attend_args(torch, pkg, lib, cache, q, out, table, starts, lengths, True, dtype, 0.125, max_length=most)
    launch(torch, lib, "dav2_hip_attention_cache_i8", a)
    torch.cuda.synchronize()
    assert out[0, 1].isnan().all() and out[0, 2].isnan().any()
    assert out[0, 0].isfinite().all() and out[0, 3].isfinite().all() and out[1:].isfinite().all()
    # a page that is seen and not finite
    out.zero_()
    q = rand(torch, 8, 2 * queries, 4, 64, dtype=dtype)
    a, keep = attend_args(torch, pkg, lib, cache, q, out, table, starts, ints(torch, [65 + queries, 64]), False, dtype,
                          0.125, max_length=most)
    launch(torch, lib, "dav2_hip_attention_cache_i8", a)
    torch.cuda.synchronize()
    assert out[:queries].isnan().all() and out[queries:].isfinite().all()


@pytest.mark.parametrize("queries", [3, 60])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("most", [None, LONG])
def test_cache_attention_not_finite_ahead(gpu, pkg, lib, queries, dtype, most):
    # a page that only the later rows of a tile see is not finite: the earlier rows are untouched
    torch = gpu
    cache = random_cache(torch, 3, 8, 2, 16, 64)
    table = ints(torch, [[0, 1, 2, 3, 4, 5]])
    total, last = 80, 64  # the page of tokens 64 .. 79
    cache[2][4, 0], cache[3][4, 1] = math.nan, math.inf
    q = rand(torch, 8, queries, 4, 64, dtype=dtype)
    out = torch.zeros_like(q)
    total = last + 2  # the last two rows see into it
    starts, lengths = ints(torch, [0, queries]), ints(torch, [total])
    a, keep = attend_args(torch, pkg, lib, cache, q, out, table, starts, lengths, True, dtype, 0.125, max_length=most)
    launch(torch, lib, "dav2_hip_attention_cache_i8", a)
    torch.cuda.synchronize()
    assert out[-2:].isnan().all() and out[:-2].isfinite().all()
    fine = [t.clone() for t in cache]
    fine[2][4], fine[3][4] = 0.01, 0.01
    want, bound = ref.attend(q, fine, table, starts, lengths, True, 0.125, dtype)
    ref.assert_within(out[:-2], want[:-2], bound[:-2])


# ---- cross attention -------------------------------------------------------------------------


def cross_args(torch, pkg, lib, q, k, v, out, lengths, mask, dtype, scale):
    a = pkg.CrossAttentionArgs(
        query=ptr(q), keys=ptr(k), values=ptr(v), output=ptr(out), query_stride=q.stride(1), key_stride=k.stride(1),
        value_stride=v.stride(1), output_stride=out.stride(1), query_batch_stride=q.stride(0),
        key_batch_stride=k.stride(0), value_batch_stride=v.stride(0), output_batch_stride=out.stride(0),
        key_lengths=ptr(lengths), key_mask=ptr(mask), batch=q.shape[0], query_tokens=q.shape[1],
        key_tokens=k.shape[1], heads=q.shape[2], kv_heads=k.shape[2], head_dim=q.shape[3], dtype=pkg.DTYPE[dtype],
        scale=scale)
    size = lib.dav2_hip_cross_attention_scratch_bytes(C.byref(a))
    scratch = None
    if size:
        scratch = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
        a.scratch, a.scratch_bytes = ptr(scratch), size
    return a, scratch


def check_cross(torch, pkg, lib, q, k, v, lengths, mask, dtype, scale=None, out=None):
    scale = scale or 1 / math.sqrt(q.shape[3])
    out = torch.full(q.shape, math.nan, dtype=q.dtype, device="cuda") if out is None else out
    a, keep = cross_args(torch, pkg, lib, q, k, v, out, lengths, mask, dtype, scale)
    launch(torch, lib, "dav2_hip_cross_attention", a)
    want, bound = ref.cross(q, k, v, lengths, mask, scale, dtype)
    torch.cuda.synchronize()
    ref.assert_within(out, want, bound)
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,head_dim", [(3, 3, 64), (8, 2, 128), (5, 1, 80), (2, 2, 16), (6, 3, 112)])
@pytest.mark.parametrize("queries,keys", [(1, 1), (1, 1370), (2, 65), (17, 64), (100, 333), (33, 31), (129, 700)])
def test_cross_attention(gpu, pkg, lib, dtype, heads, kv, head_dim, queries, keys):
    torch = gpu
    q = rand(torch, 1, 2, queries, heads, head_dim, dtype=dtype)
    k = rand(torch, 2, 2, keys, kv, head_dim, dtype=dtype)
    v = rand(torch, 3, 2, keys, kv, head_dim, dtype=dtype)
    check_cross(torch, pkg, lib, q, k, v, None, None, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("batch,queries,keys,heads,kv,head_dim", [(2, 200, 1370, 16, 8, 128), (8, 250, 130, 16, 16, 80),
                                                                  (2, 129, 999, 32, 16, 112), (9, 130, 64, 15, 15, 96)])
def test_cross_attention_wide(gpu, pkg, lib, dtype, masked, batch, queries, keys, heads, kv, head_dim):
    # tiles of 256 rows, with splits of the keys and without; a batch that sees one key, one that sees none
    torch = gpu
    q = rand(torch, 1, batch, queries, heads, head_dim, dtype=dtype)
    k, v = (rand(torch, i, batch, keys, kv, head_dim, dtype=dtype) for i in (2, 3))
    lengths = ints(torch, [keys - 7 * i for i in range(batch)])
    lengths[1] = 0 if masked else 1
    mask = (torch.rand((batch, keys), device="cuda") < 0.6).to(torch.uint8) if masked else None
    check_cross(torch, pkg, lib, q, k, v, lengths, mask, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [1, 21, 150])
def test_cross_attention_lengths_and_masks(gpu, pkg, lib, dtype, queries):
    # lengths of zero, one, all, too much; masks that leave nothing, one key, whole tiles out; anything in masked places
    torch = gpu
    keys, heads = 200, 4
    lengths = ints(torch, [0, 1, 200, 70, 1000, -3, 129, 200])
    b = lengths.numel()
    q = rand(torch, 1, b, queries, heads, 64, dtype=dtype)
    k = rand(torch, 2, b, keys, 2, 64, dtype=dtype)
    v = rand(torch, 3, b, keys, 2, 64, dtype=dtype)
    mask = (torch.rand((b, keys), device="cuda") < 0.6).to(torch.uint8) * 255
    mask[2] = 0
    mask[4] = 0
    mask[4, 131] = 1
    mask[6, :64] = 0
    mask[7, 64:] = 0
    for m in (mask, None):
        for n in (lengths, None):
            if m is None and n is None:
                continue
            hidden = torch.zeros((b, keys), dtype=torch.bool, device="cuda")
            if m is not None:
                hidden |= m == 0
            if n is not None:
                hidden |= torch.arange(keys, device="cuda") >= n[:, None]
            kk, vv = k.clone(), v.clone()
            low = torch.finfo(k.dtype).min
            for where, fill in ((hidden, math.nan), (hidden & (torch.arange(keys, device="cuda") % 3 == 0), math.inf),
                                (hidden & (torch.arange(keys, device="cuda") % 3 == 1), low)):
                kk[where] = fill
                vv[where] = fill
            out = check_cross(torch, pkg, lib, q, kk, vv, n, m, dtype)
            assert (out[hidden.all(1)] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [3, 90])
def test_cross_attention_strides(gpu, pkg, lib, dtype, queries):
    # keys and values packed in one row, batches apart, queries of a packed row, head-major output rows
    torch = gpu
    heads, kv, d, keys = 4, 2, 64, 150
    qrow = rand(torch, 1, 3, queries, heads * d + 24, dtype=dtype)
    kvrow = rand(torch, 2, 3, keys + 5, 2 * kv * d + 8, dtype=dtype)
    q = qrow[:, :, 16:16 + heads * d].unflatten(2, (heads, d))
    k = kvrow[:, 5:, :kv * d].unflatten(2, (kv, d))
    v = kvrow[:, 5:, kv * d:2 * kv * d].unflatten(2, (kv, d))
    whole = torch.full((3, queries + 1, heads * d + 8), 5.0, dtype=ref.DTYPES[dtype], device="cuda")
    check_cross(torch, pkg, lib, q, k, v, None, None, dtype,
                out=whole[:, :queries, :heads * d].unflatten(2, (heads, d)))
    assert (whole[:, queries] == 5).all() and (whole[:, :, heads * d:] == 5).all()
    # one batch's keys for all: a batch stride of zero
    shared = k[:1].expand(3, -1, -1, -1)
    check_cross(torch, pkg, lib, q, shared, v[:1].expand(3, -1, -1, -1), None, None, dtype)


@pytest.mark.parametrize("queries", [1, 64])
@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_attention_large_scores(gpu, pkg, lib, queries, dtype):
    # scores of several hundred, and weights of one key only
    torch = gpu
    q = rand(torch, 1, 1, queries, 2, 64, dtype=dtype, scale=12.0)
    k = rand(torch, 2, 1, 500, 2, 64, dtype=dtype, scale=6.0)
    v = rand(torch, 3, 1, 500, 2, 64, dtype=dtype)
    check_cross(torch, pkg, lib, q, k, v, None, None, dtype)


@pytest.mark.parametrize("queries", [1, 70])
@pytest.mark.parametrize("dtype", DTYPES)
def test_cross_attention_not_finite(gpu, pkg, lib, queries, dtype):
    # NaN in a seen value reaches that feature of its batch and head, NaN in a query its row, and nothing else
    torch = gpu
    q = rand(torch, 1, 2, queries, 2, 64, dtype=dtype)
    k = rand(torch, 2, 2, 130, 2, 64, dtype=dtype)
    v = rand(torch, 3, 2, 130, 2, 64, dtype=dtype)
    v[0, 77, 1, 9] = math.nan
    q[1, 0, 0, 4] = math.nan
    out = torch.zeros_like(q)
    a, keep = cross_args(torch, pkg, lib, q, k, v, out, None, None, dtype, 0.125)
    launch(torch, lib, "dav2_hip_cross_attention", a)
    torch.cuda.synchronize()
    where = torch.zeros_like(q, dtype=torch.bool)
    where[0, :, 1, 9] = True
    where[1, 0, 0] = True
    assert torch.equal(out.isnan(), where)


# ---- the operator surface, graphs, and all together --------------------------------------------


def surface(lib, rc):
    assert rc == 0, lib.dav2_ops_last_error().decode()


def ops_cache(pkg, cache):
    return pkg.OpsCacheInt8(*[db(pkg, t) for t in cache])




class Step:
    """One layer's step of a decoder behind the encoder: norm and rotation, the cache, attention, cross attention."""

    def __init__(self, torch, pkg, dtype, sequences, queries, older, heads=8, kv=2, d=64, page=16, image=197, seed=0):
        self.torch, self.pkg, self.dtype, self.d, self.heads, self.kv = torch, pkg, dtype, d, heads, kv
        n = sequences * queries
        self.rows = rand(torch, seed + 1, n, (heads + 2 * kv) * d, dtype=dtype)
        self.qw, self.kw = 1 + 0.2 * rand(torch, seed + 2, d), 1 + 0.2 * rand(torch, seed + 3, d)
        self.freq = ref.frequencies(d)
        self.positions = (older + torch.arange(queries, device="cuda", dtype=torch.int32)).repeat(sequences)
        most = -(-(older + queries) // page)
        self.cache = random_cache(torch, seed + 4, sequences * most, kv, page, d)
        self.before = [t.clone() for t in self.cache]
        self.table = shuffled_table(torch, seed + 5, sequences, most, sequences * most)
        self.starts = ints(torch, [i * queries for i in range(sequences + 1)])
        self.lengths = ints(torch, [older + queries] * sequences)
        self.image = rand(torch, seed + 6, sequences, image, 2 * kv * d, dtype=dtype)
        self.image_lengths = ints(torch, [image - 3 * i for i in range(sequences)])
        t = ref.DTYPES[dtype]
        self.q, self.k, self.o, self.x = (torch.full((n, h, d), math.nan, dtype=t, device="cuda")
                                          for h in (heads, kv, heads, heads))
        self.queries, self.sequences, self.older, self.n = queries, sequences, older, n
        split = heads * d
        self.q_in = self.rows[:, :split].unflatten(1, (heads, d))
        self.k_in = self.rows[:, split:split + kv * d].unflatten(1, (kv, d))
        self.v = self.rows[:, split + kv * d:].unflatten(1, (kv, d))
        self.ik = self.image[:, :, :kv * d].unflatten(2, (kv, d))
        self.iv = self.image[:, :, kv * d:].unflatten(2, (kv, d))
        self.scale = 1 / math.sqrt(d)

    def blocks(self, lib):
        torch, pkg, dtype = self.torch, self.pkg, self.dtype
        qk = qk_args(pkg, self.q_in, self.k_in, self.q, self.k, self.qw, self.kw, self.positions, self.freq, self.d,
                     "halves", "rms", dtype)
        st = store_args(pkg, self.cache, self.k, self.v, self.table, self.starts, self.lengths, self.queries, dtype)
        at, keep = attend_args(torch, pkg, lib, self.cache, self.q, self.o, self.table, self.starts, self.lengths, True,
                               dtype, self.scale)
        by_batch = self.o.view(self.sequences, self.queries, self.heads, self.d)
        xa, keep2 = cross_args(torch, pkg, lib, by_batch, self.ik, self.iv, self.x.view(by_batch.shape),
                               self.image_lengths, None, dtype, self.scale)
        return [("dav2_hip_qk_norm_rotary", qk), ("dav2_hip_cache_store_i8", st), ("dav2_hip_attention_cache_i8", at),
                ("dav2_hip_cross_attention", xa)], (keep, keep2)

    def by_surface(self, lib, ops):
        pkg = self.pkg
        none = db(pkg, None)
        (_, qk), (_, st), (_, at), (_, xa) = self.blocks(lib)[0]
        self.torch.cuda.synchronize()

        def rows_of(first):  # the packed rows from one part's first feature on
            return pkg.DeviceBuffer(first.data_ptr(), self.rows.data_ptr() + self.rows.numel() *
                                    self.rows.element_size() - first.data_ptr())

        image = pkg.DeviceBuffer(self.iv.data_ptr(), self.image.data_ptr() + self.image.numel() *
                                 self.image.element_size() - self.iv.data_ptr())
        surface(lib, lib.dav2_ops_qk_norm_rotary(ops, db(pkg, self.q), db(pkg, self.k), rows_of(self.q_in),
                                                 rows_of(self.k_in), db(pkg, self.qw), db(pkg, self.kw),
                                                 db(pkg, self.positions), db(pkg, self.freq), C.byref(qk)))
        surface(lib, lib.dav2_ops_cache_store_int8(ops, ops_cache(pkg, self.cache), db(pkg, self.k), rows_of(self.v),
                                                   db(pkg, self.table), db(pkg, self.starts), db(pkg, self.lengths),
                                                   C.byref(st)))
        surface(lib, lib.dav2_ops_attention_cache_int8(ops, db(pkg, self.o), db(pkg, self.q), ops_cache(pkg, self.cache),
                                                       db(pkg, self.table), db(pkg, self.starts), db(pkg, self.lengths),
                                                       none, C.byref(at)))
        surface(lib, lib.dav2_ops_cross_attention(ops, db(pkg, self.x), db(pkg, self.o), db(pkg, self.image), image,
                                                  db(pkg, self.image_lengths), none, none, C.byref(xa)))
        surface(lib, lib.dav2_ops_synchronize(ops))

    def check(self):
        """Every operator against float64 on what the one before it gave."""
        torch = self.torch
        torch.cuda.synchronize()
        for x, w, out in ((self.q_in, self.qw, self.q), (self.k_in, self.kw, self.k)):
            want, bound = qk_want(x, w, "rms", 1e-6, self.positions, self.freq, self.d, "halves", self.dtype)
            ref.assert_within(out, want, bound, "norm")
        want = ref.store(*self.before, self.k, self.v, self.table, self.starts, self.lengths)
        for got, w in zip(self.cache, want):
            assert torch.equal(got.cpu(), w)
        want, bound = ref.attend(self.q, self.cache, self.table, self.starts, self.lengths, True, self.scale, self.dtype)
        ref.assert_within(self.o, want, bound, "cache attention")
        by_batch = self.o.view(self.sequences, self.queries, self.heads, self.d)
        want, bound = ref.cross(by_batch, self.ik, self.iv, self.image_lengths, None, self.scale, self.dtype)
        ref.assert_within(self.x.view(by_batch.shape), want, bound, "cross attention")

    def outputs(self):
        return [t.clone() for t in (self.q, self.k, self.o, self.x, *self.cache)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sequences,queries,older", [(3, 1, 100), (2, 45, 0), (2, 20, 600), (1, 1, 0)])
def test_decoder_step(gpu, pkg, lib, ops, dtype, sequences, queries, older):
    torch = gpu
    step = Step(torch, pkg, dtype, sequences, queries, older)
    calls, keep = step.blocks(lib)
    for entry, args in calls:
        launch(torch, lib, entry, args)
    step.check()
    by_launchers = step.outputs()
    other = Step(torch, pkg, dtype, sequences, queries, older)
    other.by_surface(lib, ops)
    for a, b in zip(by_launchers, other.outputs()):
        assert torch.equal(a, b)  # the same kernels


def test_decoder_step_on_another_stream(gpu, pkg, lib):
    # behind work of that stream that the default stream knows nothing of
    torch = gpu
    side = torch.cuda.Stream()
    step = Step(torch, pkg, "f16", 3, 11, 50, seed=9)
    blocks, keep = step.blocks(lib)
    rows = step.rows.clone()
    step.rows.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        burn = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            burn = burn @ burn
        step.rows.copy_(rows)
        for entry, args in blocks:
            launch(torch, lib, entry, args)
    side.synchronize()
    step.check()


def test_decoder_step_captured(gpu, pkg, lib):
    # two graphs with a workspace each, replayed on two streams at once and beside eager calls
    torch = gpu
    steps = [Step(torch, pkg, "bf16", 3, 1, 500, seed=1), Step(torch, pkg, "f16", 2, 17, 900, seed=2)]
    want, graphs, held = [], [], []
    for step in steps:
        calls, keep = step.blocks(lib)
        held.append((calls, keep))
        for entry, args in calls:
            launch(torch, lib, entry, args)
        step.check()
        want.append(step.outputs())
    for step, (calls, _) in zip(steps, held):
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            for entry, args in calls:
                launch(torch, lib, entry, args)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in steps]
    eager = Step(torch, pkg, "f32", 2, 3, 40, seed=3)
    calls, keep = eager.blocks(lib)
    for replay in range(4):
        for step in steps:
            for t in (step.q, step.k, step.o, step.x):
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        for entry, args in calls:
            launch(torch, lib, entry, args)
        torch.cuda.synchronize()
        for step, w in zip(steps, want):
            for a, b in zip(step.outputs(), w):
                assert torch.equal(a, b), replay
    eager.check()


def test_surface_scratch(gpu, pkg, lib, ops):
    # the instance's scratch grows between calls; a scratch that is too small is refused; none under capture
    torch = gpu
    cache = random_cache(torch, 3, 400, 2, 64, 64)
    for length in (2000, 20000, 300):
        table = torch.randint(0, 400, (2, -(-length // 64)), dtype=torch.int32, device="cuda")
        starts, lengths = ints(torch, [0, 1, 2]), ints(torch, [length, length // 2])
        q = rand(torch, 8, 2, 4, 64, dtype="f16")
        out = torch.zeros_like(q)
        a, keep = attend_args(torch, pkg, lib, cache, q, out, table, starts, lengths, True, "f16", 0.125)
        torch.cuda.synchronize()
        fixed = [db(pkg, t) for t in (table, starts, lengths)]
        surface(lib, lib.dav2_ops_attention_cache_int8(ops, db(pkg, out), db(pkg, q), ops_cache(pkg, cache), *fixed,
                                                       db(pkg, None), C.byref(a)))
        surface(lib, lib.dav2_ops_synchronize(ops))
        want, bound = ref.attend(q, cache, table, starts, lengths, True, 0.125, "f16")
        ref.assert_within(out, want, bound)
        if keep is not None:
            small = db(pkg, keep, keep.numel() - 1)
            assert lib.dav2_ops_attention_cache_int8(ops, db(pkg, out), db(pkg, q), ops_cache(pkg, cache), *fixed,
                                                     small, C.byref(a)) == 1
            assert b"scratch" in lib.dav2_ops_last_error()


def test_surface_refusals(gpu, pkg, lib, ops):
    torch = gpu
    s = Step(torch, pkg, "f16", 2, 3, 20)
    calls, keep = s.blocks(lib)
    (_, qk), (_, st), (_, at), (_, xa) = calls
    none = db(pkg, None)
    short = lambda t: db(pkg, t, t.numel() * t.element_size() - 1)  # noqa: E731
    cache = ops_cache(pkg, s.cache)
    sequences = [db(pkg, t) for t in (s.table, s.starts, s.lengths)]

    def refused(rc, text):
        assert rc == 1, rc
        assert text in lib.dav2_ops_last_error(), lib.dav2_ops_last_error()

    x, pos, freq = s.q, db(pkg, s.positions), db(pkg, s.freq)
    ro = rotary_args(pkg, x, s.x, s.positions, s.freq, s.d, "halves", "f16")
    refused(lib.dav2_ops_rotary(ops, short(s.x), db(pkg, x), pos, freq, C.byref(ro)), b"output")
    refused(lib.dav2_ops_rotary(ops, db(pkg, s.x), short(x), pos, freq, C.byref(ro)), b"input")
    refused(lib.dav2_ops_rotary(ops, db(pkg, s.x), db(pkg, x), short(s.positions), freq, C.byref(ro)), b"positions")
    refused(lib.dav2_ops_rotary(ops, db(pkg, s.x), db(pkg, x), pos, short(s.freq), C.byref(ro)), b"frequencies")
    refused(lib.dav2_ops_rotary(ops, db(pkg, s.x), db(pkg, x), pos, freq, None), b"argument block")
    ro.rotary_dim = 63
    refused(lib.dav2_ops_rotary(ops, db(pkg, s.x), db(pkg, x), pos, freq, C.byref(ro)), b"rotary")
    ro.rotary_dim, ro.dtype = 64, 3
    refused(lib.dav2_ops_rotary(ops, db(pkg, s.x), db(pkg, x), pos, freq, C.byref(ro)), b"type")
    ro.dtype, ro.tokens = 1, 0
    refused(lib.dav2_ops_rotary(ops, db(pkg, s.x), db(pkg, x), pos, freq, C.byref(ro)), b"dimensions")

    rows = db(pkg, s.rows)
    args = [db(pkg, s.q), db(pkg, s.k), rows, rows, db(pkg, s.qw), db(pkg, s.kw), pos, freq]
    for i, t in enumerate((s.q, s.k, None, None, s.qw, s.kw, s.positions, s.freq)):
        if t is not None:
            refused(lib.dav2_ops_qk_norm_rotary(ops, *args[:i], short(t), *args[i + 1:], C.byref(qk)), b"too small")
    args = [db(pkg, s.k), db(pkg, s.k), *sequences]
    st.value_stride = st.key_stride
    for i, t in enumerate((s.k, s.k, s.table, s.starts, s.lengths)):
        refused(lib.dav2_ops_cache_store_int8(ops, cache, *args[:i], short(t), *args[i + 1:], C.byref(st)), b"too small")
    for i, t in enumerate(s.cache):
        parts = [db(pkg, c) for c in s.cache]
        parts[i] = short(t)
        refused(lib.dav2_ops_cache_store_int8(ops, pkg.OpsCacheInt8(*parts), *args, C.byref(st)), b"cache")
        refused(lib.dav2_ops_attention_cache_int8(ops, db(pkg, s.o), db(pkg, s.q), pkg.OpsCacheInt8(*parts),
                                                  *sequences, none, C.byref(at)), b"cache")
    for i, t in enumerate((s.o, s.q)):
        parts = [db(pkg, s.o), db(pkg, s.q)]
        parts[i] = short(t)
        refused(lib.dav2_ops_attention_cache_int8(ops, *parts, cache, *sequences, none, C.byref(at)), b"too small")
    image = db(pkg, s.image)
    parts = [db(pkg, s.x), db(pkg, s.o), image, image, db(pkg, s.image_lengths), none, none]
    for i, t in ((0, s.x), (1, s.o), (4, s.image_lengths)):
        refused(lib.dav2_ops_cross_attention(ops, *parts[:i], short(t), *parts[i + 1:], C.byref(xa)), b"too small")
    half = pkg.DeviceBuffer(s.image.data_ptr(), s.image.numel())
    for i in (2, 3):
        refused(lib.dav2_ops_cross_attention(ops, *parts[:i], half, *parts[i + 1:], C.byref(xa)), b"too small")
    xa.heads = 7
    refused(lib.dav2_ops_cross_attention(ops, *parts, C.byref(xa)), b"cross attention")
    torch.cuda.synchronize()
