"""The operators of a decoding step around a 4-bit cache: the cache and attention
over it, the plan of a step, residual addition with RMS norm and 8-bit rows,
sampling; each alone, through the operator surface, captured, and together."""

import ctypes as C
import math

import numpy as np
import pytest

import decoder_ref as ref
import step_ref
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


def with_scratch(torch, lib, entry, args):
    """The call's workspace, filled with what would show if it were read unwritten."""
    size = getattr(lib, entry + "_scratch_bytes")(C.byref(args))
    if not size:
        return None
    scratch = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    args.scratch, args.scratch_bytes = ptr(scratch), size
    return scratch


# ---- the 4-bit cache ----------------------------------------------------------------------


def random_cache(torch, seed, pages, heads, page_size, head_dim, spread=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    # every half byte, the one that is never stored among them
    keys = torch.randint(0, 256, (pages, heads, page_size, head_dim // 2), generator=g, dtype=torch.uint8, device="cuda")
    values = torch.randint(0, 256, (pages, heads, page_size // 16, head_dim, 8), generator=g, dtype=torch.uint8,
                           device="cuda")
    ks, vs = (0.05 + 0.3 * torch.rand((pages, heads, page_size), generator=g, device="cuda") for _ in range(2))
    if spread:  # scales of tokens far apart
        vs *= 10.0 ** torch.randint(-9, 10, vs.shape, generator=g, device="cuda")
    return [keys, values, ks, vs]


def cache_struct(pkg, cache):
    pages, heads, page_size, half = cache[0].shape
    return pkg.CacheI4(keys=ptr(cache[0]), values=ptr(cache[1]), key_scales=ptr(cache[2]), value_scales=ptr(cache[3]),
                       pages=pages, kv_heads=heads, page_size=page_size, head_dim=2 * half)


def shuffled_table(torch, seed, sequences, most, pages):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[:sequences * most].to(torch.int32).view(sequences, most).cuda()


def store_args(pkg, cache, k, v, table, starts, lengths, max_new, dtype):
    return pkg.CacheStoreI4Args(cache=cache_struct(pkg, cache), keys=ptr(k), values=ptr(v), key_stride=k.stride(0),
                                value_stride=v.stride(0), page_table=ptr(table), starts=ptr(starts),
                                lengths=ptr(lengths), sequences=lengths.numel(), table_pages=table.shape[1],
                                tokens=k.shape[0], max_new=max_new, dtype=pkg.DTYPE[dtype])


def check_store(torch, pkg, lib, cache, k, v, table, starts, lengths, max_new, dtype):
    want = step_ref.store(*cache, k, v, table, starts, lengths)
    for again in range(2):  # the second call stores the same rows again
        launch(torch, lib, "dav2_hip_cache_store_i4",
               store_args(pkg, cache, k, v, table, starts, lengths, max_new, dtype))
        torch.cuda.synchronize()
        for name, got, w in zip(("keys", "values", "key scales", "value scales"), cache, want):
            assert torch.equal(got.cpu(), w), (name, again)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page_size", [16, 32, 128, 208])
@pytest.mark.parametrize("heads,head_dim", [(1, 64), (3, 80), (2, 128), (5, 16)])
def test_store(gpu, pkg, lib, dtype, page_size, heads, head_dim):
    # one token into a full table, none, some that end inside a page, some that cross pages, a first token
    torch = gpu
    new, total = [1, 0, 5, 2 * page_size + 3, 1, page_size], [page_size + 4, 7, 11, 3 * page_size + 1, 1, page_size]
    starts = ints(torch, [sum(new[:i]) for i in range(len(new) + 1)])
    cache = random_cache(torch, page_size + heads, 6 * 4 + 3, heads, page_size, head_dim)
    table = shuffled_table(torch, 3, 6, 4, 6 * 4 + 3)
    # rows wider than their heads; the last two rows belong to nobody
    wide = rand(torch, 9, sum(new) + 2, heads * head_dim + 8, dtype=dtype)
    wide[::3] *= 3.0
    k = wide[:, :heads * head_dim].unflatten(1, (heads, head_dim))
    v = rand(torch, 8, sum(new) + 2, heads, head_dim, dtype=dtype, scale=0.7)
    check_store(torch, pkg, lib, cache, k, v, table, starts, ints(torch, total), max(new), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,more", [(1, 0), (0, 1), (3, 5)])
def test_store_alignment(gpu, pkg, lib, dtype, offset, more):
    torch = gpu
    tokens, heads, d, page_size = 45, 3, 48, 32
    stride = heads * d + more
    k, v = (rand(torch, i, offset + tokens * stride, dtype=dtype).as_strided((tokens, heads, d), (stride, d, 1), offset)
            for i in (1, 2))
    cache = random_cache(torch, 3, 8, heads, page_size, d)
    table = shuffled_table(torch, 4, 2, 4, 8)
    check_store(torch, pkg, lib, cache, k, v, table, ints(torch, [0, 5, 45]), ints(torch, [37, 100]), 40, dtype)


def test_store_one_by_one(gpu, pkg, lib):
    # older tokens keep their codes, whatever comes after them
    torch = gpu
    cache = random_cache(torch, 1, 4, 2, 16, 64)
    table = ints(torch, [[2, 0, 3]])
    for t in range(37):
        k, v = rand(torch, t, 1, 2, 64, scale=1.2 ** t), rand(torch, 100 + t, 1, 2, 64, scale=0.8 ** t)
        check_store(torch, pkg, lib, cache, k, v, table, ints(torch, [0, 1]), ints(torch, [t + 1]), 1, "f32")


def test_store_bad_pages_and_ranges(gpu, pkg, lib):
    # pages that do not exist, rows and positions outside, a hint that is too small
    torch = gpu
    cache = random_cache(torch, 4, 8, 2, 16, 32)
    table = ints(torch, [[0, 8, 1], [-1, 2, 3], [4, 5, 2 ** 31 - 1], [6, 7, -2 ** 31]])
    k, v = rand(torch, 1, 130, 2, 32), rand(torch, 2, 130, 2, 32)
    starts = ints(torch, [-3, 40, 70, 110, 400])
    check_store(torch, pkg, lib, cache, k, v, table, starts, ints(torch, [40, 47, 60, 10]), 1, "f32")


def test_store_borders(gpu, pkg, lib):
    # quotients next to a half, zeros, values below the smallest scale
    torch = gpu
    x = torch.zeros((40, 1, 64), device="cuda")
    half = torch.arange(-7, 7, device="cuda") + 0.5
    for i in range(40):
        scale = 1.0 + i / 40
        x[i, 0, :14] = half * scale * (1.0 + (i % 5 - 2) * 2.0 ** -23)
        x[i, 0, 14] = 7.0 * scale
    x[7] = 0.0
    x[8] *= 1e-9
    cache = random_cache(torch, 6, 3, 1, 16, 64)
    check_store(torch, pkg, lib, cache, x, -x, ints(torch, [[1, 2, 0]]), ints(torch, [0, 40]), ints(torch, [40]), 40,
                "f32")


def test_store_not_finite(gpu, pkg, lib):
    # a NaN or infinity spoils its head and token alone
    torch = gpu
    cache = random_cache(torch, 6, 3, 2, 16, 32)
    k, v = rand(torch, 2, 20, 2, 32), rand(torch, 3, 20, 2, 32)
    k[3, 0, 5], v[7, 1, 31], v[8, 0, 0] = math.nan, -math.inf, math.nan
    table, starts, lengths = ints(torch, [[1, 2]]), ints(torch, [0, 20]), ints(torch, [20])
    want = step_ref.store(*cache, torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0), table, starts, lengths)
    launch(torch, lib, "dav2_hip_cache_store_i4", store_args(pkg, cache, k, v, table, starts, lengths, 20, "f32"))
    torch.cuda.synchronize()
    ks, vs = cache[2].cpu(), cache[3].cpu()
    assert ks[1, 0, 3].isnan() and vs[1, 1, 7].isinf() and vs[1, 0, 8].isnan()
    kc, vc = step_ref.key_codes(cache[0].cpu()), step_ref.value_codes(cache[1].cpu())
    wk, wv = step_ref.key_codes(want[0]), step_ref.value_codes(want[1])
    spoilt_k, spoilt_v = torch.zeros_like(ks, dtype=torch.bool), torch.zeros_like(vs, dtype=torch.bool)
    spoilt_k[1, 0, 3] = spoilt_v[1, 1, 7] = spoilt_v[1, 0, 8] = True
    assert torch.equal(ks[~spoilt_k], want[2][~spoilt_k]) and torch.equal(vs[~spoilt_v], want[3][~spoilt_v])
    assert torch.equal(kc[~spoilt_k], wk[~spoilt_k]) and torch.equal(vc[~spoilt_v], wv[~spoilt_v])


# ---- attention over it ---------------------------------------------------------------------


def attend_args(torch, pkg, lib, cache, q, out, table, starts, lengths, causal, dtype, scale, max_query=None,
                max_length=None):
    a = pkg.AttentionCacheI4Args(
        cache=cache_struct(pkg, cache), query=ptr(q), output=ptr(out), query_stride=q.stride(0),
        output_stride=out.stride(0), page_table=ptr(table), starts=ptr(starts), lengths=ptr(lengths),
        sequences=lengths.numel(), table_pages=table.shape[1], tokens=q.shape[0], heads=q.shape[1],
        max_query=max_query or int(starts.diff().max()), max_length=max_length or max(int(lengths.max()), 1),
        causal=int(causal), dtype=pkg.DTYPE[dtype], scale=scale)
    return a, with_scratch(torch, lib, "dav2_hip_attention_cache_i4", a)


LONG = 2 ** 22  # as max_length: many rows take the way of a long cache, whatever the lengths are


def check_attend(torch, pkg, lib, cache, q, table, starts, lengths, causal, dtype, scale=None, **hints):
    scale = scale or 1 / math.sqrt(q.shape[2])
    want, bound = step_ref.attend(q, cache, table, starts, lengths, causal, scale, dtype)
    nobody = want.isnan() if not hints.pop("nan", False) else torch.zeros_like(want, dtype=torch.bool)
    for hint in (hints, dict(max_length=LONG)) if "max_length" not in hints else (hints,):
        out = torch.full(q.shape, 3.0, dtype=q.dtype, device="cuda")
        a, keep = attend_args(torch, pkg, lib, cache, q, out, table, starts, lengths, causal, dtype, scale, **hint)
        launch(torch, lib, "dav2_hip_attention_cache_i4", a)
        torch.cuda.synchronize()
        assert (out[nobody] == 3.0).all()  # rows of no sequence are left alone
        ref.assert_within(torch.where(nobody, want, out.double()), want, bound, str(hint))
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,head_dim,page_size", [(1, 1, 64, 16), (8, 2, 128, 16), (6, 6, 80, 48),
                                                         (16, 1, 128, 64), (5, 1, 96, 256), (40, 2, 64, 32),
                                                         (3, 3, 16, 16), (16, 2, 112, 32), (4, 2, 48, 16)])
def test_attention_single_tokens(gpu, pkg, lib, dtype, heads, kv, head_dim, page_size):
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
                                                         (10, 2, 112, 144), (2, 2, 32, 16)])
def test_attention_prompts(gpu, pkg, lib, dtype, causal, heads, kv, head_dim, page_size):
    # sequences with few and many new rows, one with more rows than tokens, one with none, rows of nobody
    torch = gpu
    new, total = [3, 150, 0, 70, 1, 40], [400, 150, 9, 333, 200, 25]
    starts = ints(torch, [sum(new[:i]) for i in range(len(new) + 1)])
    most = -(-max(total) // page_size)
    cache = random_cache(torch, 7, 6 * most, kv, page_size, head_dim)
    table = shuffled_table(torch, 8, 6, most, 6 * most)
    q = rand(torch, 9, sum(new) + 2, heads, head_dim, dtype=dtype)
    check_attend(torch, pkg, lib, cache, q, table, starts, ints(torch, total), causal, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [1, 2, 5, 40])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 7, 8, 16])
def test_attention_groups(gpu, pkg, lib, dtype, queries, group):
    # rows of a cache head from 1 to 640, over a cache long enough to be split
    torch = gpu
    cache = random_cache(torch, 21, 2 * 60, 2, 16, 64)
    table = shuffled_table(torch, 22, 2, 60, 120)
    q = rand(torch, 23, 2 * queries, 2 * group, 64, dtype=dtype)
    check_attend(torch, pkg, lib, cache, q, table, ints(torch, [0, queries, 2 * queries]), ints(torch, [957, 511]),
                 True, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [1, 80])
def test_attention_missing_pages(gpu, pkg, lib, dtype, queries):
    # entries that are no page inside and at the end; a table shorter than the sequence; no page at all
    torch = gpu
    cache = random_cache(torch, 3, 40, 2, 32, 64)
    table = shuffled_table(torch, 4, 4, 10, 40)
    table[0, 3], table[0, 9], table[1, 0], table[2, 4:7] = -1, 40, 2 ** 31 - 1, -2 ** 31
    table[3] = -1
    q = rand(torch, 5, 4 * queries, 4, 64, dtype=dtype)
    check_attend(torch, pkg, lib, cache, q, table, ints(torch, [i * queries for i in range(5)]),
                 ints(torch, [320, 300, 900, 100]), True, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [1, 3, 90])
def test_attention_hidden_tokens(gpu, pkg, lib, dtype, queries):
    # what lies behind a sequence's last token, or a row's, may have any scale
    torch = gpu
    cache = random_cache(torch, 13, 12, 2, 32, 64)
    table = shuffled_table(torch, 14, 2, 6, 12)
    lengths = ints(torch, [101, 150])
    for s, total in enumerate((101, 150)):
        for t in range(total, 192):
            page, slot = int(table[s, t // 32]), t % 32
            for scales in cache[2:]:
                scales[page, :, slot] = (math.nan, math.inf, 1e38)[t % 3]
    q = rand(torch, 15, 2 * queries, 4, 64, dtype=dtype)
    starts = ints(torch, [0, queries, 2 * queries])
    check_attend(torch, pkg, lib, cache, q, table, starts, lengths, True, dtype)
    if queries > 1:  # the last token is seen by the last row alone
        page, slot = int(table[0, 100 // 32]), 100 % 32
        cache[2][page, 0, slot] = math.nan
        cache[3][page, 1, slot] = math.inf
        out = torch.zeros_like(q)
        for hint in (None, LONG):
            a, keep = attend_args(torch, pkg, lib, cache, q, out, table, starts, lengths, True, dtype, 0.125,
                                  max_length=hint)
            launch(torch, lib, "dav2_hip_attention_cache_i4", a)
            torch.cuda.synchronize()
            where = torch.zeros_like(q, dtype=torch.bool)
            where[queries - 1] = True
            assert torch.equal(~out.isfinite(), where), hint


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [1, 70])
def test_attention_scales_apart(gpu, pkg, lib, dtype, queries):
    # value scales from 1e-10 to 1e8 among neighbours: each key's share is as exact as alone
    torch = gpu
    cache = random_cache(torch, 31, 20, 1, 16, 64, spread=True)
    if dtype == "f16":
        cache[3].clamp_(max=30.0)  # what the output's type holds
    table = shuffled_table(torch, 32, 2, 10, 20)
    q = rand(torch, 33, 2 * queries, 2, 64, dtype=dtype, scale=0.3)
    check_attend(torch, pkg, lib, cache, q, table, ints(torch, [0, queries, 2 * queries]), ints(torch, [160, 97]),
                 True, dtype)
    # small values where the weights are, large ones where none is left
    cache[2].fill_(0.2)
    near = torch.rand(cache[3].shape, device="cuda") < 0.5
    cache[3][:] = torch.where(near, 1e-3, 20.0)
    cache[2][:] = torch.where(near, 0.01, 0.8)
    check_attend(torch, pkg, lib, cache, q * 4, table, ints(torch, [0, queries, 2 * queries]), ints(torch, [160, 97]),
                 True, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries", [1, 70])
@pytest.mark.parametrize("scale", [40.0, -3.0, 1e-6, 3e7])
def test_attention_large_and_negative_scales(gpu, pkg, lib, dtype, queries, scale):
    torch = gpu
    cache = random_cache(torch, 41, 40, 2, 16, 64)
    table = shuffled_table(torch, 42, 1, 40, 40)
    q = rand(torch, 43, queries, 4, 64, dtype=dtype)
    if scale > 1e6:  # scores past 2^30: the largest alone is left, its bound is all of the output
        out = torch.zeros_like(q)
        starts, lengths = ints(torch, [0, queries]), ints(torch, [633])
        want, _ = step_ref.attend(q, cache, table, starts, lengths, False, scale, dtype)
        for hint in (None, LONG):
            a, keep = attend_args(torch, pkg, lib, cache, q, out, table, starts, lengths, False, dtype, scale,
                                  max_length=hint)
            launch(torch, lib, "dav2_hip_attention_cache_i4", a)
            torch.cuda.synchronize()
            assert out.isfinite().all() and (out.double().abs() <= 8 * 0.36).all()
            # 64 bits and fp32 may differ in which of two near scores is the largest, rarely
            same = ((out.double() - want).abs().amax(-1) <= 0.02).double().mean()
            assert same > 0.95, float(same)
        return
    check_attend(torch, pkg, lib, cache, q, table, ints(torch, [0, queries]), ints(torch, [633]), True, dtype,
                 scale=scale)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_long_and_mixed(gpu, pkg, lib, dtype):
    # a long cache in splits, another sequence's few tokens, a prompt, in one call with wrong hints
    torch = gpu
    cache = random_cache(torch, 51, 2600, 2, 16, 128)
    table = torch.randint(0, 2600, (3, 2500), dtype=torch.int32, device="cuda")
    starts, lengths = ints(torch, [0, 1, 3, 203]), ints(torch, [39999, 5, 500])
    q = rand(torch, 52, 203, 8, 128, dtype=dtype)
    check_attend(torch, pkg, lib, cache, q, table, starts, lengths, True, dtype)
    check_attend(torch, pkg, lib, cache, q, table, starts, lengths, True, dtype, max_query=1, max_length=300)


def test_attention_far_pages(gpu, pkg, lib):
    # a cache whose bytes pass 2^32: the last pages
    torch = gpu
    pages, page_size, d = 262200, 256, 128  # 4.3 GB of codes a side
    keys = torch.zeros((pages, 1, page_size, d // 2), dtype=torch.uint8, device="cuda")
    values = torch.zeros((pages, 1, page_size // 16, d, 8), dtype=torch.uint8, device="cuda")
    ks, vs = (torch.ones((pages, 1, page_size), device="cuda") for _ in range(2))
    table = ints(torch, [[pages - 1, 3, pages - 2]])
    small = [t[[3, pages - 2, pages - 1]].contiguous() for t in (keys, values, ks, vs)]
    k, v = rand(torch, 1, 600, 1, d, dtype="f16"), rand(torch, 2, 600, 1, d, dtype="f16")
    starts, lengths = ints(torch, [0, 600]), ints(torch, [600])
    launch(torch, lib, "dav2_hip_cache_store_i4",
           store_args(pkg, [keys, values, ks, vs], k, v, table, starts, lengths, 600, "f16"))
    near = ints(torch, [[2, 0, 1]])
    launch(torch, lib, "dav2_hip_cache_store_i4", store_args(pkg, small, k, v, near, starts, lengths, 600, "f16"))
    torch.cuda.synchronize()
    for t, w in zip((keys, values, ks, vs), small):
        assert torch.equal(t[[3, pages - 2, pages - 1]], w)
    for n in (1, 600):
        q = rand(torch, 3, n, 2, d, dtype="f16")
        one = ints(torch, [0, n])
        out, want = torch.zeros_like(q), torch.zeros_like(q)
        for cache, t, o in (([keys, values, ks, vs], table, out), (small, near, want)):
            a, keep = attend_args(torch, pkg, lib, cache, q, o, t, one, lengths, True, "f16", 0.1, max_length=LONG)
            launch(torch, lib, "dav2_hip_attention_cache_i4", a)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and out.abs().sum() > 0


# ---- the plan ---------------------------------------------------------------------------------


def run_plan(torch, pkg, lib, held, added, table, ring, state, tokens, page_size, optional=True, in_place=False):
    d = dict(held=ints(torch, held), added=ints(torch, added), page_table=ints(torch, table),
             free_pages=ints(torch, ring), free_state=ints(torch, state))
    n = len(held)
    out = {x: torch.full((m,), -77, dtype=torch.int32, device="cuda")
           for x, m in (("held_out", n), ("free_state_out", 2), ("starts", n + 1), ("lengths", n))}
    if in_place:
        out["held_out"], out["free_state_out"] = d["held"], d["free_state"]
    if optional:
        out.update(positions=torch.full((tokens,), -77, dtype=torch.int32, device="cuda"),
                   owners=torch.full((tokens,), -77, dtype=torch.int32, device="cuda"),
                   slots=torch.full((tokens,), -77, dtype=torch.int64, device="cuda"))
    a = pkg.CachePlanArgs(**{x: ptr(t) for x, t in {**d, **out}.items()}, sequences=n, table_pages=len(table[0]),
                          tokens=tokens, pages=len(ring), page_size=page_size)
    keep = with_scratch(torch, lib, "dav2_hip_cache_plan", a)
    launch(torch, lib, "dav2_hip_cache_plan", a)
    torch.cuda.synchronize()
    got = {x: t.tolist() for x, t in out.items()}
    got.update(table=d["page_table"].tolist(), ring=d["free_pages"].tolist(), state_out=got.pop("free_state_out"))
    return got


def check_plan(torch, pkg, lib, held, added, table, ring, state, tokens, page_size):
    want = step_ref.plan(held, added, table, ring, state, tokens, page_size)
    for optional, in_place in ((True, False), (False, True)):
        got = run_plan(torch, pkg, lib, held, added, table, ring, state, tokens, page_size, optional, in_place)
        for name, x in got.items():
            assert x == want[name], (name, optional)
    return want


def random_plan(seed, sequences, most_new, most_held, page_size, share=1.0, ends=0.15):
    r = np.random.default_rng(seed)
    held = r.integers(0, most_held + 1, sequences).tolist()
    added = np.where(r.random(sequences) < ends, -1, r.integers(0, most_new + 1, sequences)).tolist()
    most = -(-(most_held + most_new) // page_size)
    owned = [-(-h // page_size) for h in held]
    pages = sum(owned) + int(sequences * most * share) + 1
    order = r.permutation(pages).tolist()
    table = r.integers(-5, pages + 5, (sequences, most)).tolist()
    for i, o in enumerate(owned):
        table[i][:o], order = order[:o], order[o:]
    ring = r.integers(-5, pages + 5, pages).tolist()
    first = int(r.integers(0, pages))
    for i, p in enumerate(order):
        ring[(first + i) % pages] = p
    return held, added, table, ring, [first, len(order)]


@pytest.mark.parametrize("sequences,most_new,most_held,page_size", [
    (1, 1, 40, 16), (7, 1, 100, 16), (48, 1, 600, 32), (3, 200, 64, 16), (20, 33, 90, 48), (1025, 2, 50, 16),
    (2500, 7, 30, 16), (130, 400, 500, 256)])
@pytest.mark.parametrize("share", [1.0, 0.02])
def test_plan(gpu, pkg, lib, sequences, most_new, most_held, page_size, share):
    torch = gpu
    held, added, table, ring, state = random_plan(sequences + most_new, sequences, most_new, most_held, page_size, share)
    rows = sum(max(a, 0) for a in added)
    want = check_plan(torch, pkg, lib, held, added, table, ring, state, rows + 5, page_size)
    if share == 1.0:
        assert all(n == h + a for n, h, a in zip(want["lengths"], held, added) if a >= 0)
    if rows > 1:  # rows for some of the sequences only
        check_plan(torch, pkg, lib, held, added, table, ring, state, rows - 1, page_size)
        check_plan(torch, pkg, lib, held, added, table, ring, state, rows // 2, page_size)


def test_plan_edges(gpu, pkg, lib):
    torch = gpu
    table = [[5, -1], [6, 7], [-1, -1]]
    ring = [0, 1, 2, 3, 4, 8]
    # no rows at all, none asked for, everything ends, negative counts, a state outside the ring
    check_plan(torch, pkg, lib, [3, 20, 0], [0, 0, 0], table, ring, [0, 5], 0, 16)
    check_plan(torch, pkg, lib, [3, 20, 0], [-1, -5, -1], table, ring, [4, 2], 4, 16)
    check_plan(torch, pkg, lib, [-9, 20, 0], [3, 1, 1], table, ring, [9, 3], 6, 16)
    check_plan(torch, pkg, lib, [16, 32, 0], [1, 1, 33], table, ring, [-4, 99], 60, 16)  # two do not fit their table
    check_plan(torch, pkg, lib, [16, 17, 0], [16, 15, 32], table, ring, [5, 3], 63, 16)  # all full
    check_plan(torch, pkg, lib, [16, 17, 0], [2 ** 31 - 1, 1, 2], table, ring, [5, 3], 63, 16)
    check_plan(torch, pkg, lib, [16, 17, 0], [1, 1, 2], table, ring, [5, 0], 63, 16)  # no page is free
    # more given back than the ring has room for
    check_plan(torch, pkg, lib, [16, 32, 0], [-1, -1, 3], table, ring, [5, 5], 63, 16)
    check_plan(torch, pkg, lib, [2 ** 31 - 1, 32, 0], [-1, -1, 3], table, ring, [1, 1], 63, 16)


@pytest.mark.parametrize("sequences", [1023, 1024, 65535])
def test_plan_many_sequences(gpu, pkg, lib, sequences):
    torch = gpu
    held, added, table, ring, state = random_plan(3, sequences, 2, 20, 16)
    rows = sum(max(a, 0) for a in added)
    want = step_ref.plan(held, added, table, ring, state, rows, 16)
    got = run_plan(torch, pkg, lib, held, added, table, ring, state, rows, 16)
    for name, x in got.items():
        assert x == want[name], name


def test_plan_pages_come_back(gpu, pkg, lib):
    # many steps: no page is in two places, none is lost
    torch = gpu
    r = np.random.default_rng(5)
    n, most, pages, size = 12, 6, 40, 16
    held, table = [0] * n, [[-1] * most for _ in range(n)]
    ring, state = list(range(pages)), [17, pages]
    ring = ring[-17:] + ring[:-17]
    for step in range(40):
        added = [int(r.choice([-1, 0, 1, 5, 30])) if h < 60 else -1 for h in held]
        got = run_plan(torch, pkg, lib, held, added, table, ring, state, 400, size)
        want = step_ref.plan(held, added, table, ring, state, 400, size)
        for name, x in got.items():
            assert x == want[name], (name, step)
        held, table, ring, state = got["held_out"], got["table"], got["ring"], got["state_out"]
        used = [p for h, row in zip(held, table) for p in row[:-(-h // size)]]
        free = [ring[(state[0] + i) % pages] for i in range(state[1])]
        assert sorted(used + free) == list(range(pages)), step


# ---- the norm ---------------------------------------------------------------------------------


def norm_args(pkg, x, residual, weight, total, output, codes, scales, dtype, epsilon=1e-6):
    def stride(t):
        return t.stride(0) if t is not None else 0

    return pkg.AddRmsNormArgs(
        input=ptr(x), residual=ptr(residual), weight=ptr(weight), sum=ptr(total), output=ptr(output), codes=ptr(codes),
        scales=ptr(scales), input_stride=stride(x), residual_stride=stride(residual), sum_stride=stride(total),
        output_stride=stride(output), code_stride=stride(codes), rows=x.shape[0], columns=x.shape[1],
        dtype=pkg.DTYPE[dtype], epsilon=epsilon)


def check_norm(torch, pkg, lib, x, residual, weight, dtype, epsilon=1e-6, which=(True, True, True), more=0):
    rows, columns = x.shape
    h, y, s, c = step_ref.add_rms_norm(x, residual, weight, epsilon)
    total, output = (torch.full_like(x, 7.0) if w else None for w in which[:2])
    width = -(-columns // 64) * 64 + 64 * more
    codes = torch.full((rows, width), 77, dtype=torch.int8, device="cuda") if which[2] else None
    scales = torch.full((rows,), 7.0, device="cuda") if which[2] else None
    launch(torch, lib, "dav2_hip_add_rms_norm",
           norm_args(pkg, x, residual, weight, total, output, codes, scales, dtype, epsilon))
    torch.cuda.synchronize()
    if which[0]:
        assert torch.equal(total.cpu(), h)
    if which[1]:
        assert torch.equal(output.cpu(), y.to(x.dtype))
    if which[2]:
        assert torch.equal(scales.cpu(), s)
        assert torch.equal(codes[:, :columns].cpu(), c)
        assert (codes[:, columns:] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 7), (2, 64), (5, 130), (33, 384), (7, 1024), (2, 1025), (3, 2048),
                                          (4, 4099), (2, 8192), (1, 16384), (2, 16400), (1, 70001), (700, 96),
                                          (300, 1500)])
def test_norm(gpu, pkg, lib, dtype, rows, columns):
    torch = gpu
    x, r = rand(torch, 1, rows, columns, dtype=dtype), rand(torch, 2, rows, columns, dtype=dtype, scale=3.0)
    x[0], r[0] = 0.0, 0.0  # a row of zeros
    w = 1 + 0.3 * rand(torch, 3, columns)
    check_norm(torch, pkg, lib, x, r, w, dtype)
    check_norm(torch, pkg, lib, x, None, w, dtype, which=(False, True, False))
    check_norm(torch, pkg, lib, x, r, None, dtype, which=(False, False, True), more=2)
    check_norm(torch, pkg, lib, x, r, w, dtype, which=(True, False, True), epsilon=0.3)


@pytest.mark.parametrize("dtype,rows,columns", [("bf16", 1100, 5003), ("f16", 1100, 8192), ("bf16", 600, 16384),
                                                ("f32", 300, 16384), ("f16", 20000, 520), ("f32", 8203, 1024)])
def test_norm_rows_in_turns(gpu, pkg, lib, dtype, rows, columns):
    # more rows than are worked on at once
    torch = gpu
    x, r = rand(torch, 1, rows, columns, dtype=dtype), rand(torch, 2, rows, columns, dtype=dtype, scale=3.0)
    check_norm(torch, pkg, lib, x, r, 1 + 0.3 * rand(torch, 3, columns), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("columns", [100, 1024, 5000, 40000])
def test_norm_in_place(gpu, pkg, lib, dtype, columns):
    # the sum into the residual and the norm into the input, each way round; rows apart; nothing beside them is written
    torch = gpu
    for swap in (False, True):
        wide = rand(torch, 5, 6, 2 * columns + 11, dtype=dtype)
        before = wide.clone()
        x, r = wide[:, 1:1 + columns], wide[:, columns + 3:2 * columns + 3]
        w = 1 + 0.3 * rand(torch, 3, columns)
        h, y, s, c = step_ref.add_rms_norm(x, r, w, 1e-5)
        codes = torch.empty((6, -(-columns // 64) * 64), dtype=torch.int8, device="cuda")
        scales = torch.empty(6, device="cuda")
        total, output = (x, r) if swap else (r, x)
        launch(torch, lib, "dav2_hip_add_rms_norm",
               norm_args(pkg, x, r, w, total, output, codes, scales, dtype, 1e-5))
        torch.cuda.synchronize()
        assert torch.equal(total.cpu(), h) and torch.equal(output.cpu(), y.to(x.dtype))
        assert torch.equal(codes[:, :columns].cpu(), c) and torch.equal(scales.cpu(), s)
        rest = torch.ones(wide.shape[1], dtype=torch.bool)
        rest[1:1 + columns] = False
        rest[columns + 3:2 * columns + 3] = False
        assert torch.equal(wide[:, rest], before[:, rest])
        # the norm alone over one of its inputs
        wide.copy_(before)
        launch(torch, lib, "dav2_hip_add_rms_norm",
               norm_args(pkg, x, r, w, None, output, codes, scales, dtype, 1e-5))
        torch.cuda.synchronize()
        assert torch.equal(output.cpu(), y.to(x.dtype)) and torch.equal(codes[:, :columns].cpu(), c)


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_extremes(gpu, pkg, lib, dtype):
    # the type's largest and smallest values: squares that pass fp32; sums that pass the type
    torch = gpu
    f = torch.finfo(ref.DTYPES[dtype])
    x = rand(torch, 1, 5, 300, dtype=dtype)
    x[0] = f.max / 4
    x[1] = f.tiny * 4
    x[2, :150] = f.max / 2
    x[3, 7] = 0.0
    r = torch.zeros_like(x)
    check_norm(torch, pkg, lib, x, r, None, dtype, epsilon=1e-30)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("columns", [200, 9000])
def test_norm_not_finite(gpu, pkg, lib, dtype, columns):
    torch = gpu
    x, r = rand(torch, 1, 5, columns, dtype=dtype), rand(torch, 2, 5, columns, dtype=dtype)
    x[1, 3], r[2, columns - 1], x[3, 0] = math.nan, math.inf, -math.inf
    out, codes = torch.zeros_like(x), torch.zeros((5, 9024), dtype=torch.int8, device="cuda")
    scales = torch.zeros(5, device="cuda")
    launch(torch, lib, "dav2_hip_add_rms_norm", norm_args(pkg, x, r, None, None, out, codes, scales, dtype))
    torch.cuda.synchronize()
    assert out[[1, 2, 3]].isnan().any(1).all() and scales[[1, 2, 3]].isnan().all()
    h, y, s, c = step_ref.add_rms_norm(x[[0, 4]], r[[0, 4]], None, 1e-6)
    assert torch.equal(out[[0, 4]].cpu(), y.to(x.dtype)) and torch.equal(codes[[0, 4], :columns].cpu(), c)


def test_norm_into_product(gpu, pkg, lib):
    # the codes are rows of the int8 product
    torch = gpu
    rows, columns, n = 37, 200, 96
    x, r = rand(torch, 1, rows, columns, dtype="bf16"), rand(torch, 2, rows, columns, dtype="bf16")
    w = 1 + 0.1 * rand(torch, 3, columns)
    codes = torch.empty((rows, 256), dtype=torch.int8, device="cuda")
    scales, out = torch.empty(rows, device="cuda"), torch.empty((rows, n), device="cuda")
    b = torch.zeros((n, 256), dtype=torch.int8, device="cuda")
    b[:, :columns] = torch.randint(-127, 128, (n, columns), dtype=torch.int8, device="cuda")
    bs = torch.rand(n, device="cuda")
    launch(torch, lib, "dav2_hip_add_rms_norm", norm_args(pkg, x, r, w, None, None, codes, scales, "bf16"))
    g = pkg.GemmArgs(a=ptr(codes), lda=256, b=ptr(b), ldb=256, m=rows, n=n, k=256, epilogue=1, a_scales=ptr(scales),
                     b_scales=ptr(bs), out=ptr(out))
    assert lib.dav2_hip_gemm_i8(C.byref(g), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    _, _, s, c = step_ref.add_rms_norm(x, r, w, 1e-6)
    want = (c.double() @ b[:, :columns].cpu().double().T) * s.double()[:, None] * bs.cpu().double()
    # acc is exact, two products of fp32
    assert ((out.cpu().double() - want).abs() <= want.abs() * 4 * ref.U).all()


# ---- sampling -----------------------------------------------------------------------------------


def sample_args(torch, pkg, lib, logits, uniform, tokens, probabilities, dtype, temperature=None, top_k=None,
                top_p=None, min_p=None):
    a = pkg.SampleArgs(logits=ptr(logits), logit_stride=logits.stride(0), temperature=ptr(temperature),
                       top_k=ptr(top_k), top_p=ptr(top_p), min_p=ptr(min_p), uniform=ptr(uniform), tokens=ptr(tokens),
                       probabilities=ptr(probabilities), rows=logits.shape[0], vocabulary=logits.shape[1],
                       dtype=pkg.DTYPE[dtype])
    return a, with_scratch(torch, lib, "dav2_hip_sample", a)


def floats(torch, values):
    return None if values is None else torch.tensor(values, dtype=torch.float32, device="cuda")


def check_sample(torch, pkg, lib, logits, uniform, dtype, temperature=None, top_k=None, top_p=None, min_p=None):
    """Lists of parameters, or None for what is left out."""
    n = logits.shape[0]
    tokens = torch.full((n,), -77, dtype=torch.int32, device="cuda")
    shares = torch.full((n,), -77.0, device="cuda")
    given = dict(temperature=floats(torch, temperature), top_k=None if top_k is None else ints(torch, top_k),
                 top_p=floats(torch, top_p), min_p=floats(torch, min_p))
    u = floats(torch, uniform)
    a, keep = sample_args(torch, pkg, lib, logits, u, tokens, shares, dtype, **given)
    launch(torch, lib, "dav2_hip_sample", a)
    torch.cuda.synchronize()
    host = logits.float().cpu().numpy()
    at = {x: None if t is None else t.tolist() for x, t in given.items()}
    for i, r in enumerate(u.tolist()):
        token, share = step_ref.sample(host[i], 1.0 if at["temperature"] is None else at["temperature"][i],
                                       0 if at["top_k"] is None else at["top_k"][i],
                                       1.0 if at["top_p"] is None else at["top_p"][i],
                                       0.0 if at["min_p"] is None else at["min_p"][i], r)
        assert int(tokens[i]) == token, (i, int(tokens[i]), token)
        # weights in units of 2^-42 of the largest at the least, their sum, one rounding to fp32
        assert abs(float(shares[i]) - share) <= share * 2 ** -23 + 2 ** -40, (i, float(shares[i]), share)
    a.probabilities = None
    again = tokens.clone()
    tokens.fill_(-77)
    launch(torch, lib, "dav2_hip_sample", a)
    torch.cuda.synchronize()
    assert torch.equal(tokens, again)
    return tokens


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocabulary", [(1, 1), (3, 2), (5, 63), (4, 64), (3, 65), (9, 1000), (2, 1024), (2, 1025),
                                             (8, 4097), (5, 32000), (3, 100003), (2, 131072), (1, 1 << 20)])
def test_sample(gpu, pkg, lib, dtype, rows, vocabulary):
    torch = gpu
    logits = rand(torch, vocabulary, rows, vocabulary, dtype=dtype, scale=2.5)
    r = np.random.default_rng(rows)
    u = r.random(rows).tolist()
    t = (0.5 + r.random(rows)).tolist()
    k = r.integers(1, 2 + vocabulary // 2, rows).tolist()
    few = r.integers(1, 60, rows).tolist()
    p = (0.3 + 0.7 * r.random(rows)).tolist()
    m = (0.3 * r.random(rows)).tolist()
    check_sample(torch, pkg, lib, logits, u, dtype)
    check_sample(torch, pkg, lib, logits, u, dtype, temperature=t, top_k=k)
    check_sample(torch, pkg, lib, logits, u, dtype, temperature=t, top_p=p)
    check_sample(torch, pkg, lib, logits, u, dtype, temperature=t, min_p=m)
    check_sample(torch, pkg, lib, logits, u, dtype, temperature=t, top_k=few, top_p=p, min_p=m)
    check_sample(torch, pkg, lib, logits, u, dtype, temperature=t, top_k=k, top_p=p)
    check_sample(torch, pkg, lib, logits, u, dtype, temperature=[0.0] * rows, top_k=k, top_p=p)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_parameters(gpu, pkg, lib, dtype):
    # ends of every range and beyond, each in a row of its own
    torch = gpu
    nan, inf = math.nan, math.inf
    cases = ([(t, 0, 1.0, 0.0, 0.4) for t in (0.0, -1.0, nan, 1e-30, 1e-4, 0.02, 50.0, 1e30, inf)] +
             [(1.0, k, 1.0, 0.0, 0.7) for k in (-5, 0, 1, 2, 1999, 2000, 2 ** 31 - 1)] +
             [(1.0, 0, p, 0.0, 0.7) for p in (-1.0, 0.0, 1e-9, 1e-3, 0.5, 0.999999, 1.0, 1.5, nan, inf)] +
             [(1.0, 0, 1.0, m, 0.7) for m in (-1.0, 0.0, 1e-30, 1e-4, 0.5, 0.9999999, 1.0, 1.1, nan)] +
             [(0.7, 40, 0.9, 0.02, u) for u in (0.0, 1e-30, 0.25, 0.99999994, 1.0, 7.0, -3.0, nan)] +
             [(5.0, 0, 0.99, 0.0, u) for u in (0.0, 0.5, 0.99999994)])
    logits = rand(torch, 4, len(cases), 2000, dtype=dtype, scale=3.0)
    t, k, p, m, u = map(list, zip(*cases))
    check_sample(torch, pkg, lib, logits, u, dtype, t, k, p, m)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary", [70, 5000, 40000])
def test_sample_ties_and_masks(gpu, pkg, lib, dtype, vocabulary):
    # equal logits in bulk, tokens masked out by -infinity, NaN and the type's lowest value, infinities, nothing left
    torch = gpu
    n = 14
    x = rand(torch, 4, n, vocabulary, dtype=dtype, scale=2.0)
    low = torch.finfo(x.dtype).min
    x[0] = 0.0
    x[1] = -3.5
    x[2] = torch.round(x[2])
    x[3] = torch.round(x[3] / 4) * 4
    x[4, vocabulary // 3:] = -math.inf
    x[5] = -math.inf
    x[6] = math.nan
    x[7] = low
    x[8] = low
    x[8, vocabulary - 2] = 1.0
    x[9, ::2] = math.nan
    x[10, 5], x[10, vocabulary - 1] = math.inf, math.inf
    x[11] = -math.inf
    x[11, vocabulary // 2] = -2.0
    x[12, ::3] = -0.0
    x[12, 1::3] = 0.0
    x[12, 2::3] = -1.0
    x[13, vocabulary // 2:] = low
    for i, u in enumerate((0.0, 0.31, 0.77, 0.9999999)):
        us = [u] * n
        tokens = check_sample(torch, pkg, lib, x, us, dtype)
        assert tokens[5] == -1 and tokens[6] == -1
        check_sample(torch, pkg, lib, x, us, dtype, top_k=[33] * n)
        check_sample(torch, pkg, lib, x, us, dtype, top_p=[0.6] * n)
        check_sample(torch, pkg, lib, x, us, dtype, temperature=[0.0, 1.0] * (n // 2), top_k=[vocabulary // 2] * n,
                     top_p=[0.83] * n, min_p=[0.01] * n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocabulary", [(97, 4097), (130, 16390), (100, 40000), (98, 70001),
                                             (40, 40970)])
def test_sample_many_rows(gpu, pkg, lib, dtype, rows, vocabulary):
    # rows that have a workgroup each; some of equal logits, masked, or of one number in bulk
    torch = gpu
    x = rand(torch, rows, rows, vocabulary, dtype=dtype, scale=2.5)
    x[1] = 0.5
    x[2] = -math.inf
    x[3, 7:] = math.nan
    x[4, 2:] = -30000.0
    x[5] = torch.round(x[5])
    x[6, :60] = math.inf
    x[7] = torch.where(torch.arange(vocabulary, device="cuda") % 3 == 0, -0.0, 0.0)
    x[8, : vocabulary // 2] = torch.finfo(x.dtype).min
    x[9, 1:] = 0.0
    x[10, 500:] = -math.inf
    r = np.random.default_rng(rows)
    u = r.random(rows).tolist()
    t = (0.4 + r.random(rows)).tolist()
    t[11], t[12], t[13], t[14] = 0.0, math.nan, 1e-20, 1e30
    p = (0.3 + 0.69 * r.random(rows)).tolist()
    check_sample(torch, pkg, lib, x, u, dtype)
    check_sample(torch, pkg, lib, x, u, dtype, temperature=t, top_p=p)
    check_sample(torch, pkg, lib, x, u, dtype, temperature=t, min_p=[0.02 * (i % 4) for i in range(rows)])
    check_sample(torch, pkg, lib, x, u, dtype, temperature=t, top_k=[(1, 50, 2048, 3000, 0)[i % 5] for i in range(rows)],
                 top_p=p)
    check_sample(torch, pkg, lib, x[:, 1:vocabulary - 2], u, dtype, temperature=t, top_p=p)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_strides(gpu, pkg, lib, dtype):
    # rows of a wider matrix at an odd address, in any order of the rows' requests
    torch = gpu
    wide = rand(torch, 6, 12, 3007, dtype=dtype, scale=2.0)
    wide[:, :3] = 50.0
    wide[:, 2900:] = 50.0
    logits = wide[:, 3:2900]
    r = np.random.default_rng(3)
    check_sample(torch, pkg, lib, logits, r.random(12).tolist(), dtype, top_p=[0.9] * 12, top_k=[100, 0] * 6)


def test_sample_frequencies(gpu, pkg, lib):
    # a grid of random numbers draws every token as often as its share says, to one step of the grid
    torch = gpu
    n = 4096
    x = rand(torch, 2, 1, 50, scale=1.5)
    u = ((np.arange(n) + 0.5) / n).tolist()
    tokens = check_sample(torch, pkg, lib, x.expand(n, 50).contiguous(), u, "f32", temperature=[0.8] * n)
    share = torch.softmax(x[0].double().cpu() / np.float64(np.float32(0.8)), 0)
    counts = torch.bincount(tokens.cpu().long(), minlength=50)
    assert ((counts / n - share).abs() <= 1.0 / n).all()


# ---- the operator surface, streams, graphs, and all together -------------------------------------------


def surface(lib, rc):
    assert rc == 0, lib.dav2_ops_last_error().decode()


class Model:
    """A small decoder on the 4-bit cache, one token for each sequence a step, held whole on the device: a step reads
    the last tokens and what the sequences hold, and writes the next ones."""

    def __init__(self, torch, pkg, lib, dtype="f32", sequences=5, heads=4, kv=2, d=32, page=16, vocabulary=300, seed=0,
                 most=6):
        self.torch, self.pkg, self.lib, self.dtype = torch, pkg, lib, dtype
        n, width = sequences, heads * d
        self.n, self.width, self.kv, self.d, self.heads = n, width, kv, d, heads
        t = ref.DTYPES[dtype]
        self.embedding = rand(torch, seed + 1, vocabulary, width, dtype=dtype)
        rows = (heads + 2 * kv) * d
        self.qkv_weight, self.out_weight = (
            torch.randint(-127, 128, (m, width), generator=torch.Generator(device="cuda").manual_seed(seed + i),
                          dtype=torch.int8, device="cuda") for i, m in ((2, rows), (3, vocabulary)))
        self.qkv_scales = torch.full((rows,), 0.02 / width ** 0.5, device="cuda")
        self.out_scales = torch.full((vocabulary,), 0.06 / width ** 0.5, device="cuda")
        self.weight = 1 + 0.1 * rand(torch, seed + 4, width)
        self.freq = ref.frequencies(d)
        pages = n * most + 3
        self.cache = random_cache(torch, seed + 5, pages, kv, page, d)
        self.table = torch.full((n, most), -1, dtype=torch.int32, device="cuda")
        self.ring = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32).cuda()
        self.free = ints(torch, [pages - 2, pages])
        self.held, self.added = ints(torch, [0] * n), ints(torch, [1] * n)
        self.lengths, self.starts = ints(torch, [0] * n), ints(torch, [0] * (n + 1))
        self.positions, self.owners = ints(torch, [0] * n), ints(torch, [0] * n)
        self.slots = torch.zeros(n, dtype=torch.int64, device="cuda")
        self.tokens = ints(torch, list(range(n)))
        self.uniform, self.shares = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        self.top_p = floats(torch, [0.9] * n)
        self.x, self.h = (torch.zeros((n, width), dtype=t, device="cuda") for _ in range(2))
        self.codes = torch.zeros((n, width), dtype=torch.int8, device="cuda")
        self.scales = torch.zeros(n, device="cuda")
        self.qkv32, self.qkv = (torch.zeros((n, rows), dtype=x, device="cuda") for x in (torch.float32, t))
        self.q, self.o = (torch.zeros((n, heads, d), dtype=t, device="cuda") for _ in range(2))
        self.k = torch.zeros((n, kv, d), dtype=t, device="cuda")
        self.logits = torch.zeros((n, vocabulary), device="cuda")
        self.calls, self.keep = self.blocks()

    def blocks(self):
        torch, pkg, lib = self.torch, self.pkg, self.lib
        n, kv, d, heads = self.n, self.kv, self.d, self.heads
        plan = pkg.CachePlanArgs(
            held=ptr(self.held), added=ptr(self.added), page_table=ptr(self.table), free_pages=ptr(self.ring),
            free_state=ptr(self.free), held_out=ptr(self.held), free_state_out=ptr(self.free), starts=ptr(self.starts),
            lengths=ptr(self.lengths), positions=ptr(self.positions), owners=ptr(self.owners), slots=ptr(self.slots),
            sequences=n, table_pages=self.table.shape[1], tokens=n, pages=self.ring.numel(),
            page_size=self.cache[0].shape[2])
        split = heads * d
        q_in = self.qkv[:, :split].unflatten(1, (heads, d))
        k_in = self.qkv[:, split:split + kv * d].unflatten(1, (kv, d))
        v = self.qkv[:, split + kv * d:].unflatten(1, (kv, d))
        first = norm_args(pkg, self.x, None, self.weight, None, None, self.codes, self.scales, self.dtype)

        def product(b, scales, out):
            return pkg.GemmArgs(a=ptr(self.codes), lda=self.width, b=ptr(b), ldb=self.width, m=n, n=b.shape[0],
                                k=self.width, epilogue=1, a_scales=ptr(self.scales), b_scales=ptr(scales),
                                out=ptr(out))

        qk = pkg.QkNormRotaryArgs(
            query=ptr(q_in), key=ptr(k_in), query_out=ptr(self.q), key_out=ptr(self.k), query_stride=q_in.stride(0),
            key_stride=k_in.stride(0), query_out_stride=split, key_out_stride=kv * d, positions=ptr(self.positions),
            frequencies=ptr(self.freq), tokens=n, query_heads=heads, key_heads=kv, head_dim=d, rotary_dim=d,
            dtype=pkg.DTYPE[self.dtype], epsilon=1e-6, amplitude=1.0)
        store = store_args(pkg, self.cache, self.k, v, self.table, self.starts, self.lengths, 1, self.dtype)
        span = self.table.shape[1] * self.cache[0].shape[2]
        attend, s1 = attend_args(torch, pkg, lib, self.cache, self.q, self.o, self.table, self.starts, self.lengths,
                                 True, self.dtype, d ** -0.5, max_query=1, max_length=span)
        second = norm_args(pkg, self.o.view(n, -1), self.x, self.weight, self.h, None, self.codes, self.scales,
                           self.dtype)
        draw, s2 = sample_args(torch, pkg, lib, self.logits, self.uniform, self.tokens, self.shares, "f32",
                               top_p=self.top_p)
        s3 = with_scratch(torch, lib, "dav2_hip_cache_plan", plan)
        return [("dav2_hip_cache_plan", plan), ("embed", None), ("dav2_hip_add_rms_norm", first),
                ("dav2_hip_gemm_i8", product(self.qkv_weight, self.qkv_scales, self.qkv32)), ("cast", None),
                ("dav2_hip_qk_norm_rotary", qk), ("dav2_hip_cache_store_i4", store),
                ("dav2_hip_attention_cache_i4", attend), ("dav2_hip_add_rms_norm", second),
                ("dav2_hip_gemm_i8", product(self.out_weight, self.out_scales, self.logits)),
                ("dav2_hip_sample", draw)], (s1, s2, s3)

    def step(self, check=False):
        torch = self.torch
        for entry, args in self.calls:
            if entry == "embed":
                torch.index_select(self.embedding, 0, self.tokens, out=self.x)
            elif entry == "cast":
                self.qkv.copy_(self.qkv32)
            else:
                launch(torch, self.lib, entry, args)
            if check and entry == "dav2_hip_attention_cache_i4":
                want, bound = step_ref.attend(self.q, self.cache, self.table, self.starts, self.lengths, True,
                                              self.d ** -0.5, self.dtype)
                ref.assert_within(torch.where(want.isnan(), want, self.o.double()), want, bound)  # NaN: rows of nobody

    def request(self, step, r):
        """What comes from outside: random numbers, and that a sequence ends or begins."""
        self.uniform.copy_(floats(self.torch, r.random(self.n).tolist()))
        self.added.copy_(ints(self.torch, [-1 if step % 7 == 5 and i == step % self.n else 1 for i in range(self.n)]))

    def state(self):
        return [t.clone() for t in (self.tokens, self.shares, self.logits, self.h, self.o, self.q, *self.cache, self.table,
                                    self.ring, self.free, self.held, self.lengths, self.positions, self.slots)]


@pytest.mark.parametrize("dtype", DTYPES)
def test_decoding(gpu, pkg, lib, dtype):
    # steps of the whole, captured once and replayed, give the bits of eager ones; attention holds in each
    torch = gpu
    eager, captured = (Model(torch, pkg, lib, dtype) for _ in range(2))
    for m in (eager, captured):  # a first step outside the graph
        m.request(0, np.random.default_rng(9))
        m.step()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        captured.step()
    r, r2 = np.random.default_rng(1), np.random.default_rng(1)
    seen = set()
    for step in range(1, 40):
        eager.request(step, r)
        eager.step(check=step % 6 == 0)
        captured.request(step, r2)
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(eager.state(), captured.state())):
            assert torch.equal(a, b), (step, i)
        seen |= set(eager.tokens.tolist())
    assert len(seen) > 20 and int(eager.held.max()) > 16


def test_two_graphs_and_streams(gpu, pkg, lib):
    # two captured decoders with workspaces of their own, replayed at once on two streams
    torch = gpu
    models = [Model(torch, pkg, lib, "bf16", seed=3), Model(torch, pkg, lib, "f16", sequences=3, heads=8, kv=1, d=64, seed=4)]
    plain = [Model(torch, pkg, lib, "bf16", seed=3), Model(torch, pkg, lib, "f16", sequences=3, heads=8, kv=1, d=64, seed=4)]
    graphs, streams = [], [torch.cuda.Stream() for _ in models]
    for m, p in zip(models, plain):
        for x in (m, p):
            x.request(0, np.random.default_rng(2))
            x.step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            m.step()
        graphs.append(graph)
    for step in range(1, 6):
        for m, p in zip(models, plain):
            m.request(step, np.random.default_rng(step))
            p.request(step, np.random.default_rng(step))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        for p in plain:
            p.step()
        torch.cuda.synchronize()
        for m, p in zip(models, plain):
            for i, (a, b) in enumerate(zip(m.state(), p.state())):
                assert torch.equal(a, b), (step, i)


def test_long_calls_captured(gpu, pkg, lib):
    # the calls of several launches with a workspace: each replay on other inputs gives the bits of the eager call
    torch = gpu
    rows, wide = rand(torch, 1, 3, 100003, scale=2.5), rand(torch, 2, 100, 42000, dtype="bf16", scale=2.5)
    u = torch.zeros(100, device="cuda")
    top_p = floats(torch, [0.9] * 100)
    cache = random_cache(torch, 3, 200, 2, 32, 64)
    table = shuffled_table(torch, 4, 2, 100, 200)
    q = rand(torch, 5, 2 * 200, 8, 64, dtype="f16")
    starts, lengths = ints(torch, [0, 200, 400]), ints(torch, [3001, 2500])
    held, added = ints(torch, [0] * 300), ints(torch, [7] * 300)
    x = rand(torch, 6, 70, 5000, dtype="f16")

    def make():
        t = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (3, 100)]
        p = [torch.zeros(n, device="cuda") for n in (3, 100)]
        o, y = torch.zeros_like(q), torch.zeros_like(x)
        codes, scales = torch.zeros((70, 5056), dtype=torch.int8, device="cuda"), torch.zeros(70, device="cuda")
        pages = torch.zeros((300, 4), dtype=torch.int32, device="cuda")
        ring = torch.arange(1000, dtype=torch.int32, device="cuda")
        state = ints(torch, [3, 1000])
        plan_out = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (300, 2, 301, 300, 2500, 2500)]
        slots = torch.zeros(2500, dtype=torch.int64, device="cuda")
        calls = []
        for logits, tokens, share, dtype in ((rows, t[0], p[0], "f32"), (wide, t[1], p[1], "bf16")):
            a, s = sample_args(torch, pkg, lib, logits, u, tokens, share, dtype, top_p=top_p)
            calls.append(("dav2_hip_sample", a, s))
        a, s = attend_args(torch, pkg, lib, cache, q, o, table, starts, lengths, True, "f16", 0.125)
        calls.append(("dav2_hip_attention_cache_i4", a, s))
        plan = pkg.CachePlanArgs(held=ptr(held), added=ptr(added), page_table=ptr(pages), free_pages=ptr(ring),
                                 free_state=ptr(state), held_out=ptr(plan_out[0]), free_state_out=ptr(plan_out[1]),
                                 starts=ptr(plan_out[2]), lengths=ptr(plan_out[3]), positions=ptr(plan_out[4]),
                                 owners=ptr(plan_out[5]), slots=ptr(slots), sequences=300, table_pages=4, tokens=2500,
                                 pages=1000, page_size=16)
        calls.append(("dav2_hip_cache_plan", plan, with_scratch(torch, lib, "dav2_hip_cache_plan", plan)))
        calls.append(("dav2_hip_add_rms_norm", norm_args(pkg, x, None, None, None, y, codes, scales, "f16"), None))
        return calls, [*t, *p, o, y, codes, scales, pages, ring, *plan_out, slots, state]

    (eager, want), (captured, got) = make(), make()
    assert all(c[2] is not None for c in (captured[0], captured[2], captured[3]))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        for entry, args, _ in captured:
            launch(torch, lib, entry, args)
    for replay in range(4):
        u.copy_(floats(torch, np.random.default_rng(replay).random(100).tolist()))
        rows.mul_(-1.0)
        wide.copy_(wide.flip(1))
        q.mul_(0.9)
        x.copy_(x.flip(0) * 1.1)
        added.copy_(ints(torch, [(i * (replay + 3)) % 9 - 1 for i in range(300)]))
        held.copy_(ints(torch, [(i * 5) % 30 for i in range(300)]))
        torch.cuda.synchronize()
        graph.replay()
        for entry, args, _ in eager:
            launch(torch, lib, entry, args)
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(want, got)):
            assert torch.equal(a, b), (replay, i)


def test_decoding_by_surface(gpu, pkg, lib, ops):
    # the same kernels through the operator surface, with the instance's own scratch
    torch = gpu
    by_launchers, m = (Model(torch, pkg, lib, "f32", seed=8) for _ in range(2))
    r, r2 = np.random.default_rng(1), np.random.default_rng(1)
    none = db(pkg, None)
    blocks = dict((e, a) for e, a in m.calls if e != "dav2_hip_add_rms_norm")
    norms = [a for e, a in m.calls if e == "dav2_hip_add_rms_norm"]
    table = [db(pkg, t) for t in (m.table, m.starts, m.lengths)]
    cache = pkg.OpsCacheInt4(*[db(pkg, t) for t in m.cache])
    split = m.heads * m.d + m.kv * m.d
    values = pkg.DeviceBuffer(m.qkv[:, split:].data_ptr(), (m.qkv.numel() - split) * 4)
    plan = pkg.OpsCachePlanBuffers(*[db(pkg, t) for t in (m.held, m.added, m.table, m.ring, m.free, m.held, m.free,
                                                          m.starts, m.lengths, m.positions, m.owners, m.slots)])
    for step in range(4):
        by_launchers.request(step, r)
        by_launchers.step()
        m.request(step, r2)
        torch.cuda.synchronize()
        surface(lib, lib.dav2_ops_cache_plan(ops, C.byref(plan), none, C.byref(blocks["dav2_hip_cache_plan"])))
        m.x.copy_(m.embedding[m.tokens])
        torch.cuda.synchronize()
        surface(lib, lib.dav2_ops_add_rms_norm(ops, none, none, db(pkg, m.codes), db(pkg, m.scales), db(pkg, m.x), none,
                                               db(pkg, m.weight), C.byref(norms[0])))
        surface(lib, lib.dav2_ops_synchronize(ops))
        for e, a in m.calls[3:6]:
            m.qkv.copy_(m.qkv32) if e == "cast" else launch(torch, lib, e, a)
        torch.cuda.synchronize()
        surface(lib, lib.dav2_ops_cache_store_int4(ops, cache, db(pkg, m.k), values, *table,
                                                   C.byref(blocks["dav2_hip_cache_store_i4"])))
        surface(lib, lib.dav2_ops_attention_cache_int4(ops, db(pkg, m.o), db(pkg, m.q), cache, *table, none,
                                                       C.byref(blocks["dav2_hip_attention_cache_i4"])))
        surface(lib, lib.dav2_ops_add_rms_norm(ops, db(pkg, m.h), none, db(pkg, m.codes), db(pkg, m.scales),
                                               db(pkg, m.o), db(pkg, m.x), db(pkg, m.weight), C.byref(norms[1])))
        surface(lib, lib.dav2_ops_synchronize(ops))
        launch(torch, lib, *m.calls[9])
        torch.cuda.synchronize()
        surface(lib, lib.dav2_ops_sample(ops, db(pkg, m.tokens), db(pkg, m.shares), db(pkg, m.logits), none, none,
                                         db(pkg, m.top_p), none, db(pkg, m.uniform), none,
                                         C.byref(blocks["dav2_hip_sample"])))
        surface(lib, lib.dav2_ops_synchronize(ops))
        for i, (a, b) in enumerate(zip(by_launchers.state(), m.state())):
            assert torch.equal(a, b), (step, i)


def test_surface_refusals(gpu, pkg, lib, ops):
    torch = gpu
    m = Model(torch, pkg, lib, "f32", seed=8)
    torch.cuda.synchronize()
    none = db(pkg, None)
    short = lambda t: db(pkg, t, t.numel() * t.element_size() - 1)  # noqa: E731
    blocks = dict((e, a) for e, a in m.calls if e != "dav2_hip_add_rms_norm")

    def refused(rc, text):
        assert rc == 1, rc
        assert text in lib.dav2_ops_last_error(), lib.dav2_ops_last_error()

    names = ("held", "added", "table", "ring", "free", "held", "free", "starts", "lengths", "positions", "owners", "slots")
    args = blocks["dav2_hip_cache_plan"]
    for i, name in enumerate(names):
        parts = [db(pkg, getattr(m, x)) for x in names]
        parts[i] = short(getattr(m, name))
        refused(lib.dav2_ops_cache_plan(ops, C.byref(pkg.OpsCachePlanBuffers(*parts)), none, C.byref(args)), b"too small")
    whole = pkg.OpsCachePlanBuffers(*[db(pkg, getattr(m, x)) for x in names])
    refused(lib.dav2_ops_cache_plan(ops, None, none, C.byref(args)), b"argument block")
    refused(lib.dav2_ops_cache_plan(ops, C.byref(whole), none, None), b"argument block")
    refused(lib.dav2_ops_cache_plan(ops, C.byref(whole), db(pkg, m.scales, 8), C.byref(args)), b"scratch")
    args.page_size = 24
    refused(lib.dav2_ops_cache_plan(ops, C.byref(whole), none, C.byref(args)), b"cache plan")
    args.page_size = 0
    refused(lib.dav2_ops_cache_plan(ops, C.byref(whole), none, C.byref(args)), b"dimensions")

    fixed = [db(pkg, t) for t in (m.table, m.starts, m.lengths)]
    for i in range(4):
        parts = [db(pkg, t) for t in m.cache]
        parts[i] = short(m.cache[i])
        refused(lib.dav2_ops_cache_store_int4(ops, pkg.OpsCacheInt4(*parts), db(pkg, m.k), db(pkg, m.qkv), *fixed,
                                              C.byref(blocks["dav2_hip_cache_store_i4"])), b"cache")
        refused(lib.dav2_ops_attention_cache_int4(ops, db(pkg, m.o), db(pkg, m.q), pkg.OpsCacheInt4(*parts), *fixed, none,
                                                  C.byref(blocks["dav2_hip_attention_cache_i4"])), b"cache")

    norm = [a for e, a in m.calls if e == "dav2_hip_add_rms_norm"][1]
    good = [db(pkg, t) for t in (m.h, None, m.codes, m.scales, m.o, m.x, m.weight)]
    for i, t in enumerate((m.h, None, m.codes, m.scales, m.o, m.x, m.weight)):
        if t is not None:
            refused(lib.dav2_ops_add_rms_norm(ops, *good[:i], short(t), *good[i + 1:], C.byref(norm)), b"too small")
    refused(lib.dav2_ops_add_rms_norm(ops, none, none, none, none, *good[4:], C.byref(norm)), b"norm")
    norm.dtype = 3
    refused(lib.dav2_ops_add_rms_norm(ops, *good, C.byref(norm)), b"type")

    draw = blocks["dav2_hip_sample"]
    all_of = (m.tokens, m.shares, m.logits, m.shares, m.tokens, m.top_p, m.shares, m.uniform)
    good = [db(pkg, t) for t in all_of]
    for i, t in enumerate(all_of):
        refused(lib.dav2_ops_sample(ops, *good[:i], short(t), *good[i + 1:], none, C.byref(draw)), b"too small")
    draw.vocabulary = 0
    refused(lib.dav2_ops_sample(ops, *good, none, C.byref(draw)), b"dimensions")


def test_surface_under_capture(gpu, pkg, lib, ops):
    # a call under capture has to bring its scratch
    torch = gpu
    m = Model(torch, pkg, lib, "f32", seed=8)
    names = ("held", "added", "table", "ring", "free", "held", "free", "starts", "lengths", "positions", "owners", "slots")
    plan = pkg.OpsCachePlanBuffers(*[db(pkg, getattr(m, x)) for x in names])
    args = m.calls[0][1]
    scratch = m.keep[2]
    stream = torch.cuda.ExternalStream(lib.dav2_ops_stream(ops))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        assert lib.dav2_ops_cache_plan(ops, C.byref(plan), db(pkg, None), C.byref(args)) == 1
        message = lib.dav2_ops_last_error()
        surface(lib, lib.dav2_ops_cache_plan(ops, C.byref(plan), db(pkg, scratch), C.byref(args)))
    assert b"capture" in message
    held = m.held.clone()
    for replay in range(3):
        graph.replay()
        torch.cuda.synchronize()
        held += 1
        assert torch.equal(m.held, held) and torch.equal(m.positions, held - 1)
