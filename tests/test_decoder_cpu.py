"""What the decoder operators refuse, and the host helper for rotary
frequencies. Nothing here reaches a GPU: every launcher checks its argument
block before its first HIP call."""

import ctypes as C
import math

import pytest

P = 1 << 20  # an address that is never read


def rotary(pkg, **kw):
    a = dict(input=P, output=P + (1 << 16), input_stride=128, output_stride=128, positions=P, frequencies=P, tokens=3,
             heads=2, head_dim=64, rotary_dim=64, layout=0, dtype=0, amplitude=1.0)
    return pkg.RotaryArgs(**{**a, **kw})


def qk(pkg, **kw):
    a = dict(query=P, key=P, query_out=P + (1 << 16), key_out=P + (2 << 16), query_stride=128, key_stride=64,
             query_out_stride=128, key_out_stride=64, positions=P, frequencies=P, tokens=3, query_heads=2, key_heads=1,
             head_dim=64, rotary_dim=64, layout=0, dtype=0, norm=0, epsilon=1e-6, amplitude=1.0)
    return pkg.QkNormRotaryArgs(**{**a, **kw})


def cache(pkg, **kw):
    a = dict(keys=P, values=P, key_scales=P, value_scales=P, pages=10, kv_heads=2, page_size=16, head_dim=64)
    return pkg.CacheI8(**{**a, **kw})


def store(pkg, cache_kw=None, **kw):
    a = dict(cache=cache(pkg, **(cache_kw or {})), keys=P, values=P, key_stride=128, value_stride=128, page_table=P,
             starts=P, lengths=P, sequences=2, table_pages=4, tokens=5, max_new=3, dtype=0)
    return pkg.CacheStoreI8Args(**{**a, **kw})


def attend(pkg, cache_kw=None, **kw):
    a = dict(cache=cache(pkg, **(cache_kw or {})), query=P, output=P, query_stride=256, output_stride=256,
             page_table=P, starts=P, lengths=P, sequences=2, table_pages=4, tokens=5, heads=4, max_query=3,
             max_length=60, causal=1, dtype=0, scale=0.125)
    return pkg.AttentionCacheI8Args(**{**a, **kw})


def cross(pkg, **kw):
    a = dict(query=P, keys=P, values=P, output=P, query_stride=256, key_stride=128, value_stride=128,
             output_stride=256, query_batch_stride=2560, key_batch_stride=1280, value_batch_stride=1280,
             output_batch_stride=2560, batch=2, query_tokens=10, key_tokens=10, heads=4, kv_heads=2, head_dim=64,
             dtype=0, scale=0.125)
    return pkg.CrossAttentionArgs(**{**a, **kw})


ROTARY = [dict(input=None), dict(output=None), dict(positions=None), dict(frequencies=None), dict(head_dim=0),
          dict(head_dim=1025, rotary_dim=64, input_stride=4096, output_stride=4096), dict(rotary_dim=0),
          dict(rotary_dim=33), dict(rotary_dim=66), dict(layout=2), dict(dtype=3), dict(input_stride=127),
          dict(output_stride=127), dict(output=P, output_stride=136), dict(heads=65536, input_stride=1 << 32),
          dict(tokens=1 << 31)]
QK = [dict(query=None), dict(key=None), dict(query_out=None), dict(key_out=None), dict(positions=None),
      dict(frequencies=None), dict(norm=2), dict(epsilon=0.0), dict(epsilon=-1.0), dict(epsilon=math.nan),
      dict(layout=7), dict(dtype=9), dict(rotary_dim=65), dict(rotary_dim=128), dict(head_dim=0, rotary_dim=0),
      dict(query_stride=64), dict(key_stride=63), dict(query_out_stride=0), dict(key_out_stride=0),
      dict(key_out=P, key_out_stride=72)]
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
CROSS = [dict(query=None), dict(keys=None), dict(values=None), dict(output=None), dict(query=P + 4), dict(keys=P + 8),
         dict(values=P + 2), dict(output=P + 1), dict(heads=0), dict(heads=3), dict(kv_heads=0), dict(head_dim=0),
         dict(head_dim=72), dict(head_dim=8), dict(head_dim=144), dict(dtype=3), dict(query_stride=248),
         dict(key_stride=120), dict(value_stride=132), dict(output_stride=0), dict(query_batch_stride=2561),
         dict(key_batch_stride=4), dict(batch=65536), dict(query_tokens=1 << 31), dict(key_tokens=1 << 31),
         dict(batch=60000, query_tokens=1 << 16)]


@pytest.mark.parametrize("bad", ROTARY)
def test_rotary_refuses(pkg, lib, bad):
    assert lib.dav2_hip_rotary(C.byref(rotary(pkg, **bad)), None) == 1


@pytest.mark.parametrize("bad", QK)
def test_qk_norm_refuses(pkg, lib, bad):
    assert lib.dav2_hip_qk_norm_rotary(C.byref(qk(pkg, **bad)), None) == 1


@pytest.mark.parametrize("bad", CACHE)
def test_cache_refuses(pkg, lib, bad):
    assert lib.dav2_hip_cache_store_i8(C.byref(store(pkg, bad)), None) == 1
    assert lib.dav2_hip_attention_cache_i8(C.byref(attend(pkg, bad)), None) == 1
    assert lib.dav2_hip_attention_cache_i8_scratch_bytes(C.byref(attend(pkg, bad))) < 1 << 40


@pytest.mark.parametrize("bad", STORE)
def test_cache_store_refuses(pkg, lib, bad):
    assert lib.dav2_hip_cache_store_i8(C.byref(store(pkg, **bad)), None) == 1


@pytest.mark.parametrize("bad", ATTEND)
def test_cache_attention_refuses(pkg, lib, bad):
    assert lib.dav2_hip_attention_cache_i8(C.byref(attend(pkg, **bad)), None) == 1


@pytest.mark.parametrize("bad", CROSS)
def test_cross_attention_refuses(pkg, lib, bad):
    assert lib.dav2_hip_cross_attention(C.byref(cross(pkg, **bad)), None) == 1


def test_nothing_to_do_is_no_error(pkg, lib):
    assert lib.dav2_hip_rotary(C.byref(rotary(pkg, tokens=0, input=None)), None) == 0
    assert lib.dav2_hip_rotary(C.byref(rotary(pkg, heads=0)), None) == 0
    assert lib.dav2_hip_qk_norm_rotary(C.byref(qk(pkg, tokens=0)), None) == 0
    assert lib.dav2_hip_cache_store_i8(C.byref(store(pkg, tokens=0)), None) == 0
    assert lib.dav2_hip_cache_store_i8(C.byref(store(pkg, sequences=0)), None) == 0
    assert lib.dav2_hip_attention_cache_i8(C.byref(attend(pkg, tokens=0)), None) == 0
    assert lib.dav2_hip_cross_attention(C.byref(cross(pkg, batch=0)), None) == 0
    assert lib.dav2_hip_cross_attention(C.byref(cross(pkg, query_tokens=0)), None) == 0


@pytest.mark.parametrize("entry", ["dav2_hip_rotary", "dav2_hip_qk_norm_rotary", "dav2_hip_cache_store_i8",
                                   "dav2_hip_attention_cache_i8", "dav2_hip_cross_attention"])
def test_no_argument_block(lib, entry):
    assert getattr(lib, entry)(None, None) == 1


@pytest.mark.parametrize("block,entry,size_of", [
    (lambda pkg: attend(pkg, max_query=1, tokens=2, max_length=30000, table_pages=2000), "dav2_hip_attention_cache_i8",
     "dav2_hip_attention_cache_i8_scratch_bytes"),
    (lambda pkg: cross(pkg, query_tokens=1, key_tokens=5000), "dav2_hip_cross_attention",
     "dav2_hip_cross_attention_scratch_bytes")])
def test_scratch_is_checked(pkg, lib, block, entry, size_of):
    a = block(pkg)
    need = getattr(lib, size_of)(C.byref(a))
    a.scratch, a.scratch_bytes = P, need + 16
    assert getattr(lib, size_of)(C.byref(a)) == need  # by the sizes alone
    if need:
        for scratch, size in ((None, need), (P, need - 1), (P + 8, need)):
            a.scratch, a.scratch_bytes = scratch, size
            assert getattr(lib, entry)(C.byref(a), None) == 1


def table(pkg, lib, n, base=10000.0, **scaling):
    out = (C.c_double * (n // 2))()
    s = C.byref(pkg.RotaryScaling(**scaling)) if scaling else None
    rc = lib.dav2_ops_rotary_frequencies(out, n, base, s)
    return rc, list(out)


def test_rotary_frequencies(pkg, lib):
    n, base = 64, 500000.0
    plain = [base ** (-2 * i / n) for i in range(n // 2)]
    close = lambda a, b: all(abs(x - y) <= 4 * 2.0 ** -52 * y for x, y in zip(a, b))  # noqa: E731
    assert close(table(pkg, lib, n, base)[1], plain)
    kinds = pkg.ROTARY_SCALING
    assert close(table(pkg, lib, n, base, kind=kinds["none"])[1], plain)
    assert close(table(pkg, lib, n, base, kind=kinds["linear"], factor=4.0)[1], [f / 4 for f in plain])
    rc, got = table(pkg, lib, n, base, kind=kinds["base"], factor=8.0)
    assert rc == 0 and got[0] == 1.0 and abs(got[-1] * 8 / plain[-1] - 1) < 1e-13
    rc, got = table(pkg, lib, n, base, kind=kinds["wavelength"], factor=8.0, original_length=8192.0, low_turns=1.0,
                    high_turns=4.0)
    assert rc == 0
    for f, g in zip(plain, got):
        r = 8192 * f / (2 * math.pi)
        kept = min(1.0, max(0.0, (r - 1) / 3))
        assert abs(g - f * (kept + (1 - kept) / 8)) <= 1e-14 * f
    assert got[0] == plain[0] and abs(got[-1] * 8 / plain[-1] - 1) < 1e-13


@pytest.mark.parametrize("n,base,scaling", [
    (0, 1e4, {}), (3, 1e4, {}), (4, 1.0, {}), (4, math.nan, {}), (4, math.inf, {}), (4, 1e4, dict(kind=4)),
    (4, 1e4, dict(kind=1, factor=0.5)), (4, 1e4, dict(kind=1, factor=math.nan)),
    (4, 1e4, dict(kind=1, factor=math.inf)), (2, 1e4, dict(kind=2, factor=2.0)),
    (4, 1e4, dict(kind=3, factor=2.0, original_length=0.0, low_turns=1.0, high_turns=4.0)),
    (4, 1e4, dict(kind=3, factor=2.0, original_length=64.0, low_turns=4.0, high_turns=4.0)),
    (4, 1e4, dict(kind=3, factor=2.0, original_length=64.0, low_turns=-1.0, high_turns=4.0))])
def test_rotary_frequencies_refuses(pkg, lib, n, base, scaling):
    out = (C.c_double * 4)()
    s = C.byref(pkg.RotaryScaling(**scaling)) if scaling else None
    assert lib.dav2_ops_rotary_frequencies(out, n, base, s) == 1
    assert len(lib.dav2_ops_last_error()) > 0
    assert lib.dav2_ops_rotary_frequencies(None, 64, 1e4, None) == 1


def test_argument_blocks_match_the_header(pkg):
    # fields and sizes as the C compiler lays them out
    import re
    from pathlib import Path
    text = (Path(__file__).resolve().parents[1] / "include" / "dav2_hip.h").read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, struct in (("dav2_rotary_args", pkg.RotaryArgs), ("dav2_qk_norm_rotary_args", pkg.QkNormRotaryArgs),
                         ("dav2_cache_i8", pkg.CacheI8), ("dav2_cache_store_i8_args", pkg.CacheStoreI8Args),
                         ("dav2_attention_cache_i8_args", pkg.AttentionCacheI8Args),
                         ("dav2_cross_attention_args", pkg.CrossAttentionArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
        fields = []
        for line in body.split(";"):
            m = re.match(r"\s*(?:const\s+)?(\w+)(\s*\*)?\s*(.+)", line, re.S)
            if m:
                kind = {"uint32_t": C.c_uint32, "uint64_t": C.c_uint64, "float": C.c_float,
                        "dav2_cache_i8": pkg.CacheI8}.get(m.group(1))
                kind = C.c_void_p if m.group(2) else kind
                fields += [(n.strip(), kind) for n in m.group(3).split(",")]
        assert [(n, t) for n, t in struct._fields_] == fields, name
