"""What the operators of a decoding step refuse. Nothing here reaches a GPU:
every launcher checks its argument block before its first HIP call."""

import ctypes as C
import math
import re
from pathlib import Path

import pytest

P = 1 << 20  # an address that is never read


def cache(pkg, **kw):
    a = dict(keys=P, values=P, key_scales=P, value_scales=P, pages=10, kv_heads=2, page_size=16, head_dim=64)
    return pkg.CacheI4(**{**a, **kw})


def store(pkg, cache_kw=None, **kw):
    a = dict(cache=cache(pkg, **(cache_kw or {})), keys=P, values=P, key_stride=128, value_stride=128, page_table=P,
             starts=P, lengths=P, sequences=2, table_pages=4, tokens=5, max_new=3, dtype=0)
    return pkg.CacheStoreI4Args(**{**a, **kw})


def attend(pkg, cache_kw=None, **kw):
    a = dict(cache=cache(pkg, **(cache_kw or {})), query=P, output=P, query_stride=256, output_stride=256,
             page_table=P, starts=P, lengths=P, sequences=2, table_pages=4, tokens=5, heads=4, max_query=3,
             max_length=60, causal=1, dtype=0, scale=0.125)
    return pkg.AttentionCacheI4Args(**{**a, **kw})


def plan(pkg, **kw):
    a = dict(held=P, added=P, page_table=P, free_pages=P, free_state=P, held_out=P, free_state_out=P, starts=P,
             lengths=P, sequences=3, table_pages=4, tokens=9, pages=12, page_size=16, scratch=P, scratch_bytes=1 << 16)
    return pkg.CachePlanArgs(**{**a, **kw})


def norm(pkg, **kw):
    a = dict(input=P, residual=2 * P, weight=P, sum=3 * P, output=4 * P, codes=5 * P, scales=P, input_stride=100,
             residual_stride=100, sum_stride=100, output_stride=100, code_stride=128, rows=3, columns=100, dtype=0,
             epsilon=1e-6)
    return pkg.AddRmsNormArgs(**{**a, **kw})


def sample(pkg, **kw):
    a = dict(logits=P, logit_stride=1000, uniform=P, tokens=P, rows=3, vocabulary=1000, dtype=0, scratch=P,
             scratch_bytes=1 << 30)
    return pkg.SampleArgs(**{**a, **kw})


CACHE = [dict(keys=None), dict(values=None), dict(key_scales=None), dict(value_scales=None), dict(keys=P + 8),
         dict(values=P + 1), dict(pages=0), dict(pages=1 << 31), dict(kv_heads=0), dict(page_size=0),
         dict(page_size=8), dict(page_size=24), dict(page_size=272), dict(head_dim=0), dict(head_dim=8),
         dict(head_dim=72), dict(head_dim=144), dict(kv_heads=32768)]
STORE = [dict(keys=None), dict(values=None), dict(page_table=None), dict(starts=None), dict(lengths=None),
         dict(table_pages=0), dict(dtype=3), dict(sequences=65536), dict(tokens=1 << 31), dict(key_stride=127),
         dict(value_stride=0)]
ATTEND = [dict(query=None), dict(output=None), dict(query=P + 8), dict(output=P + 2), dict(page_table=None),
          dict(starts=None), dict(lengths=None), dict(table_pages=0), dict(dtype=3), dict(heads=0), dict(heads=3),
          dict(query_stride=255), dict(query_stride=248), dict(output_stride=260), dict(sequences=65536),
          dict(tokens=1 << 31), dict(tokens=1 << 20, heads=1 << 12, query_stride=1 << 19, output_stride=1 << 19)]
PLAN = [dict([(x, None)]) for x in ("held", "added", "page_table", "free_pages", "free_state", "held_out",
                                    "free_state_out", "starts", "lengths", "scratch")] + [
    dict(sequences=65536), dict(table_pages=0), dict(table_pages=1 << 31), dict(tokens=1 << 31), dict(pages=0),
    dict(pages=1 << 31), dict(page_size=0), dict(page_size=8), dict(page_size=24), dict(page_size=272),
    dict(scratch=P + 4), dict(scratch_bytes=8)]
NORM = [dict(input=None), dict(sum=None, output=None, codes=None), dict(dtype=3), dict(epsilon=0.0),
        dict(epsilon=-1.0), dict(epsilon=math.nan), dict(rows=1 << 31), dict(columns=1 << 20, input_stride=1 << 20),
        dict(input_stride=99), dict(residual_stride=99), dict(sum_stride=0), dict(output_stride=99),
        dict(scales=None), dict(codes=P + 4), dict(code_stride=120), dict(code_stride=64), dict(sum=P, sum_stride=104),
        dict(output=2 * P, output_stride=101), dict(sum=4 * P)]
SAMPLE = [dict(logits=None), dict(uniform=None), dict(tokens=None), dict(rows=65536), dict(vocabulary=0),
          dict(vocabulary=(1 << 20) + 1, logit_stride=1 << 21), dict(dtype=3), dict(logit_stride=999)]


@pytest.mark.parametrize("bad", CACHE)
def test_cache_refuses(pkg, lib, bad):
    assert lib.dav2_hip_cache_store_i4(C.byref(store(pkg, bad)), None) == 1
    assert lib.dav2_hip_attention_cache_i4(C.byref(attend(pkg, bad)), None) == 1
    assert lib.dav2_hip_attention_cache_i4_scratch_bytes(C.byref(attend(pkg, bad))) < 1 << 40


@pytest.mark.parametrize("block,entry,bad", [(b, e, x) for b, e, many in (
    (store, "dav2_hip_cache_store_i4", STORE), (attend, "dav2_hip_attention_cache_i4", ATTEND),
    (plan, "dav2_hip_cache_plan", PLAN), (norm, "dav2_hip_add_rms_norm", NORM),
    (sample, "dav2_hip_sample", SAMPLE)) for x in many])
def test_refuses(pkg, lib, block, entry, bad):
    assert getattr(lib, entry)(C.byref(block(pkg, **bad)), None) == 1


def test_nothing_to_do_is_no_error(pkg, lib):
    assert lib.dav2_hip_cache_store_i4(C.byref(store(pkg, tokens=0)), None) == 0
    assert lib.dav2_hip_cache_store_i4(C.byref(store(pkg, sequences=0)), None) == 0
    assert lib.dav2_hip_cache_store_i4(C.byref(store(pkg, max_new=0)), None) == 0
    assert lib.dav2_hip_attention_cache_i4(C.byref(attend(pkg, tokens=0)), None) == 0
    assert lib.dav2_hip_attention_cache_i4(C.byref(attend(pkg, max_query=0)), None) == 0
    assert lib.dav2_hip_cache_plan(C.byref(plan(pkg, sequences=0)), None) == 0
    assert lib.dav2_hip_add_rms_norm(C.byref(norm(pkg, rows=0)), None) == 0
    assert lib.dav2_hip_add_rms_norm(C.byref(norm(pkg, columns=0)), None) == 0
    assert lib.dav2_hip_sample(C.byref(sample(pkg, rows=0)), None) == 0


@pytest.mark.parametrize("entry", ["dav2_hip_cache_store_i4", "dav2_hip_attention_cache_i4", "dav2_hip_cache_plan",
                                   "dav2_hip_add_rms_norm", "dav2_hip_sample"])
def test_no_argument_block(lib, entry):
    assert getattr(lib, entry)(None, None) == 1


@pytest.mark.parametrize("block,entry", [
    (lambda pkg: attend(pkg, max_query=1, tokens=2, max_length=30000, table_pages=2000), "dav2_hip_attention_cache_i4"),
    (plan, "dav2_hip_cache_plan"), (sample, "dav2_hip_sample"),
    (lambda pkg: sample(pkg, rows=2, vocabulary=200000, logit_stride=200000), "dav2_hip_sample")])
def test_scratch_is_checked(pkg, lib, block, entry):
    a = block(pkg)
    size_of = getattr(lib, entry + "_scratch_bytes")
    need = size_of(C.byref(a))
    a.scratch, a.scratch_bytes = P, need + 16
    assert size_of(C.byref(a)) == need  # by the sizes alone
    assert size_of(None) == 0
    if need:
        for scratch, size in ((None, need), (P, need - 1), (P + 8, need)):
            a.scratch, a.scratch_bytes = scratch, size
            assert getattr(lib, entry)(C.byref(a), None) == 1


def test_sample_scratch_by_sizes_alone(pkg, lib):
    for dtype in (0, 1, 2):
        for rows in (1, 2, 7, 16, 31, 32, 33, 64, 96, 97, 200):
            for vocabulary in (1, 4096, 4097, 25088, 32000, 65536, 69632, 100003, 131072, 200000, 1 << 20):
                sizes = [lib.dav2_hip_sample_scratch_bytes(C.byref(pkg.SampleArgs(
                    rows=rows, vocabulary=vocabulary, dtype=dtype, top_k=k))) for k in (None, P)]
                assert sizes[0] == sizes[1], (dtype, rows, vocabulary)


def test_argument_blocks_match_the_headers(pkg):
    include = Path(__file__).resolve().parents[1] / "include"
    for file, names in (("dav2_hip.h", {"dav2_cache_i4": pkg.CacheI4, "dav2_cache_store_i4_args": pkg.CacheStoreI4Args,
                                        "dav2_attention_cache_i4_args": pkg.AttentionCacheI4Args,
                                        "dav2_cache_plan_args": pkg.CachePlanArgs,
                                        "dav2_add_rms_norm_args": pkg.AddRmsNormArgs,
                                        "dav2_sample_args": pkg.SampleArgs}),
                        ("dav2_ops.h", {"dav2_ops_cache_int4": pkg.OpsCacheInt4,
                                        "dav2_ops_cache_plan_buffers": pkg.OpsCachePlanBuffers})):
        text = re.sub(r"/\*.*?\*/", "", (include / file).read_text(), flags=re.S)
        for name, struct in names.items():
            body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
            fields = []
            for line in body.split(";"):
                m = re.match(r"\s*(?:const\s+)?(\w+)(\s*\*)?\s*(.+)", line, re.S)
                if m:
                    kind = {"uint32_t": C.c_uint32, "uint64_t": C.c_uint64, "float": C.c_float,
                            "dav2_cache_i4": pkg.CacheI4, "dav2_device_buffer": pkg.DeviceBuffer}.get(m.group(1))
                    kind = C.c_void_p if m.group(2) else kind
                    fields += [(n.strip(), kind) for n in m.group(3).split(",")]
            assert [(n, t) for n, t in struct._fields_] == fields, name
