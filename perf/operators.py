"""The operators of a decoder behind the encoder, as cases that can be timed and checked.

  rotary      dav2_hip_rotary: rotary positions of the heads of a matrix of tokens
  qk_norm     dav2_hip_qk_norm_rotary: norm of each query and key head and the rotation in one pass
  store       dav2_hip_cache_store_i8: new keys and values into a paged int8 cache, one scale per page and head
  attend      dav2_hip_attention_cache_i8: attention over such a cache, single tokens and prompts
  cross       dav2_hip_cross_attention: queries against an encoder's keys and values

`own` false: the operators in elementary torch operations. `own` true: the library's kernels, on torch's
current stream, as a program calls them (include/dav2_hip.h).
"""

from __future__ import annotations

import ctypes
import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
EPSILON = 1e-6


def listed():
    return [
        # one token of a small decoder: the latency of a call
        dict(name="rotary_token", kind="rotary", tokens=1, heads=16, head_dim=64, rotary_dim=64, layout="halves",
             dtype="f32", last=1370),
        # a prompt whose heads are rotated in half their width, far positions
        dict(name="rotary_prompt_partial", kind="rotary", tokens=8191, heads=32, head_dim=128, rotary_dim=64,
             layout="pairs", dtype="bf16", last=131071),
        # one decoding step of a batch, 4 query heads per key head
        dict(name="qk_norm_step", kind="qk_norm", tokens=48, heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             layout="halves", norm="rms", dtype="bf16", last=32767),
        # a long prompt
        dict(name="qk_norm_prompt", kind="qk_norm", tokens=16411, heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             layout="halves", norm="rms", dtype="f16", last=16410),
        # one new token for each of 64 sequences, small pages
        dict(name="store_step", kind="store", sequences=64, max_new=1, max_length=64, kv_heads=8, head_dim=128,
             page_size=16, dtype="bf16"),
        # eight prompts of different lengths
        dict(name="store_prompts", kind="store", sequences=8, max_new=2048, max_length=2048, kv_heads=8, head_dim=128,
             page_size=64, dtype="f16"),
        # a token looks at one 518x518 image's 1370 encoder tokens
        dict(name="attend_token_image", kind="attend", sequences=1, max_query=1, max_length=1370, heads=16,
             kv_heads=16, head_dim=64, page_size=16, causal=True, dtype="f32"),
        # a decoding step of 32 sequences, up to 32768 tokens each
        dict(name="attend_step_long", kind="attend", sequences=32, max_query=1, max_length=32768, heads=32,
             kv_heads=8, head_dim=128, page_size=32, causal=True, dtype="bf16"),
        # the last quarter of two prompts
        dict(name="attend_prompt_chunk", kind="attend", sequences=2, max_query=2048, max_length=8192, heads=32,
             kv_heads=8, head_dim=128, page_size=64, causal=True, dtype="f16"),
        # a decoding step that looks at four images
        dict(name="cross_token", kind="cross", batch=4, queries=1, keys=1370, heads=16, kv_heads=16, head_dim=64,
             lengths=False, mask=False, dtype="f16"),
        # a resampler's queries in the float mode, images of different sizes in one batch
        dict(name="cross_f32", kind="cross", batch=2, queries=577, keys=1370, heads=16, kv_heads=16, head_dim=64,
             lengths=True, mask=False, dtype="f32"),
        # prompts against 1036x1036 images with masked patches
        dict(name="cross_prompts", kind="cross", batch=4, queries=2048, keys=5477, heads=32, kv_heads=8, head_dim=128,
             lengths=True, mask=True, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["rotary", "qk_norm", "store", "attend", "attend", "cross", "cross"])
        case = dict(kind=kind, dtype=rng.choice(list(DTYPES)))
        if kind in ("rotary", "qk_norm"):
            d = rng.choice([32, 64, 80, 96, 128, 256])
            case.update(tokens=_log_int(rng, 1, 16500), heads=_log_int(rng, 1, 48), head_dim=d,
                        rotary_dim=rng.choice([d, d, d // 2, d // 4]), layout=rng.choice(["halves", "pairs"]),
                        last=_log_int(rng, 17000, 1000000))
            if kind == "qk_norm":
                case.update(kv_heads=_log_int(rng, 1, 16), norm=rng.choice(["rms", "rms", "layer"]))
        elif kind == "store":
            most_new = rng.choice([1, 1, _log_int(rng, 2, 2048)])
            case.update(sequences=_log_int(rng, 1, 64), max_new=most_new, max_length=most_new + _log_int(rng, 1, 256),
                        kv_heads=_log_int(rng, 1, 16), head_dim=rng.choice([64, 80, 96, 128]),
                        page_size=rng.choice([16, 32, 64, 128]))
        elif kind == "attend":
            queries = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 2048)])
            kv = _log_int(rng, 1, 16)
            case.update(sequences=_log_int(rng, 1, 48 if queries < 9 else 4), max_query=queries,
                        max_length=queries + _log_int(rng, 1, 32768 if queries < 9 else 8192), kv_heads=kv,
                        heads=kv * rng.choice([1, 2, 4, 5, 8]), head_dim=rng.choice([64, 80, 96, 128]),
                        page_size=rng.choice([16, 32, 64, 128]), causal=rng.random() < 0.7)
        else:
            kv = _log_int(rng, 1, 16)
            case.update(batch=_log_int(rng, 1, 16), queries=rng.choice([1, _log_int(rng, 2, 2048)]),
                        keys=_log_int(rng, 1, 5477), kv_heads=kv, heads=kv * rng.choice([1, 1, 2, 4]),
                        head_dim=rng.choice([64, 80, 96, 128]), lengths=rng.random() < 0.5, mask=rng.random() < 0.4)
        if _cost(case) <= most and _plain_floats(case) <= 3e9:
            return case


def _plain_floats(case):
    """Values that the plain form holds at a time."""
    if case["kind"] == "attend":
        return (case["sequences"] * case["max_length"] * (case["heads"] * case["max_query"] +
                                                          2 * case["kv_heads"] * case["head_dim"]))
    if case["kind"] == "cross":
        return case["batch"] * case["heads"] * case["queries"] * case["keys"]
    return 0


def _cost(case):
    w = work(case)
    # the float mode's products run at the rate of 32-bit matrix instructions
    return w["flops"] * (16.0 if case["dtype"] == "f32" else 1.0) + 100.0 * w["bytes"]


# ---- inputs --------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _sizes(case):
    """Lengths of a case's sequences (in all, and new ones): the first has the most, the others are spread."""
    r = random.Random("%d %d %d" % (case["sequences"], case["max_length"], case.get("max_new", 0)))
    if case["kind"] == "attend":
        new = [case["max_query"]] * case["sequences"]
        total = [max(n, round(case["max_length"] * (r.uniform(0.25, 1.0) if i else 1.0))) for i, n in enumerate(new)]
        return total, new
    new = [max(1, round(case["max_new"] * (r.uniform(0.1, 1.0) if i else 1.0))) for i in range(case["sequences"])]
    before = case["max_length"] - case["max_new"]
    return [n + (r.randint(0, before) if before else 0) for n in new], new


def _key_counts(case):
    r = random.Random("%d %d" % (case["batch"], case["keys"]))
    if not case["lengths"]:
        return [case["keys"]] * case["batch"]
    return [round(case["keys"] * (r.uniform(0.3, 1.0) if i else 1.0)) or 1 for i in range(case["batch"])]


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _frequencies(case):
    """Radians per position of each rotated pair, base 10000, in 64 bits."""
    i = torch.arange(case["rotary_dim"] // 2, dtype=torch.float64, device="cuda")
    return torch.exp(i * (-2.0 * math.log(10000.0) / case["rotary_dim"]))


def _pages(case):
    """A page table over shuffled pages: [sequences][most pages of one], and how many pages there are."""
    most = -(-case["max_length"] // case["page_size"])
    count = case["sequences"] * most
    order = torch.randperm(count, generator=torch.Generator().manual_seed(count + case["page_size"]))
    return order.to(torch.int32).view(case["sequences"], most).cuda(), count


def _quantized(x):
    """Codes of x [..][a][b] with one scale for its last two axes, and the scales."""
    s = torch.clamp_min((x.abs().amax(dim=(-2, -1)).double() / 127.0).float(), 1e-8)
    return torch.round((x.double() / s.double()[..., None, None]).float()).to(torch.int8), s


def _random_cache(case, pages, g):
    """Keys and values of a decoder, quantized: some features of the keys are large, values differ from page to page."""
    h, p, d = case["kv_heads"], case["page_size"], case["head_dim"]
    wide = 1.0 + 3.0 * (torch.rand((h, 1, d), generator=g, device="cuda") < 0.05)
    keys = torch.empty((pages, h, p, d), dtype=torch.int8, device="cuda")
    values = torch.empty((pages, h, d, p), dtype=torch.int8, device="cuda")
    ks, vs = (torch.empty((pages, h), device="cuda") for _ in range(2))
    step = max(1, int(2 ** 26 // (h * p * d)))
    for a in range(0, pages, step):
        n = min(step, pages - a)
        keys[a:a + n], ks[a:a + n] = _quantized(torch.randn((n, h, p, d), generator=g, device="cuda") * wide)
        v = torch.randn((n, h, d, p), generator=g, device="cuda")
        v *= 0.25 + torch.rand((n, h, 1, 1), generator=g, device="cuda")
        values[a:a + n], vs[a:a + n] = _quantized(v)
    return keys, values, ks, vs


def prepare(case, seed):
    g = _generator(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)

    state = {"case": case}
    if kind == "rotary":
        t, h, d = case["tokens"], case["heads"], case["head_dim"]
        state.update(x=normal(t, h, d), frequencies=_frequencies(case),
                     positions=_int32(list(range(case["last"] + 1 - t, case["last"] + 1))),
                     out=torch.empty((t, h, d), dtype=dtype, device="cuda"))
    elif kind == "qk_norm":
        t, h, k, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
        rows = normal(t, (h + 2 * k) * d, scale=2.0)  # the packed product that queries and keys are parts of
        state.update(rows=rows, q=rows[:, :h * d].view(t, h, d), k=rows[:, h * d:(h + k) * d].view(t, k, d),
                     q_weight=1.0 + 0.2 * torch.randn(d, generator=g, device="cuda"),
                     k_weight=1.0 + 0.2 * torch.randn(d, generator=g, device="cuda"), frequencies=_frequencies(case),
                     positions=torch.randint(0, case["last"] + 1, (t,), generator=g, device="cuda", dtype=torch.int32),
                     q_out=torch.empty((t, h, d), dtype=dtype, device="cuda"),
                     k_out=torch.empty((t, k, d), dtype=dtype, device="cuda"))
    elif kind in ("store", "attend"):
        total, new = _sizes(case)
        table, pages = _pages(case)
        keys, values, ks, vs = _random_cache(case, pages, g)
        starts = [sum(new[:i]) for i in range(len(new) + 1)]
        state.update(keys=keys, values=values, key_scales=ks, value_scales=vs, table=table, starts=_int32(starts),
                     lengths=_int32(total))
        n, h, d = starts[-1], case["kv_heads"], case["head_dim"]
        if kind == "store":
            state.update(new_keys=normal(n, h, d, scale=1.1), new_values=normal(n, h, d, scale=0.6),
                         stored=[torch.empty(keys.shape, device="cuda"), torch.empty(values.shape, device="cuda")])
        else:
            state.update(q=normal(n, case["heads"], d),
                         out=torch.zeros((n, case["heads"], d), dtype=dtype, device="cuda"))
    else:
        b, tq, tk = case["batch"], case["queries"], case["keys"]
        h, k, d = case["heads"], case["kv_heads"], case["head_dim"]
        counts = _key_counts(case)
        state.update(q=normal(b, tq, h, d, scale=1.2), k=normal(b, tk, k, d, scale=1.2), v=normal(b, tk, k, d),
                     lengths=_int32(counts) if case["lengths"] else None,
                     mask=(torch.rand((b, tk), generator=g, device="cuda") < 0.8).to(torch.uint8)
                     if case["mask"] else None, out=torch.empty((b, tq, h, d), dtype=dtype, device="cuda"))
    return state


# ---- the operators in elementary operations -----------------------------------------


def _rotated(x, state):
    """x [tokens][heads][head_dim] in 32 bits, rotated."""
    case = state["case"]
    r = case["rotary_dim"]
    angle = state["positions"].double()[:, None] * state["frequencies"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if case["layout"] == "halves":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([y, x[..., r:]], dim=-1)


def _normed(x, weight, kind):
    if kind == "layer":
        x = x - x.mean(dim=-1, keepdim=True)
    return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPSILON) * weight


def _stored(state):
    """The cache with the new tokens in it, in place: every page that gets one is computed anew."""
    case = state["case"]
    p = case["page_size"]
    starts, lengths = state["starts"].long(), state["lengths"].long()
    first = (lengths - starts.diff())[:, None]  # the first new token's position
    touched = (case["max_new"] + p - 2) // p + 1
    # past a sequence's last page: that page again
    place = torch.minimum(first // p + torch.arange(touched, device="cuda"), (lengths[:, None] - 1) // p)
    page = state["table"].long().gather(1, place)  # [sequences][touched]
    pos = place[..., None] * p + torch.arange(p, device="cuda")
    fresh = ((pos >= first[..., None]) & (pos < lengths[:, None, None]))[:, :, None, :, None]
    older = (pos < first[..., None])[:, :, None, :, None]
    begun = older[..., :1, :]  # the page holds older tokens
    row = (starts[:-1, None, None] + pos - first[..., None]).clamp(0, state["new_keys"].shape[0] - 1)
    for new, codes, scales, turn in ((state["new_keys"], state["keys"], state["key_scales"], False),
                                     (state["new_values"], state["values"], state["value_scales"], True)):
        c = codes.transpose(2, 3) if turn else codes  # [pages][heads][page_size][head_dim]
        held, old = c[page], scales[page][..., None, None]
        x = new[row].float().transpose(2, 3)  # [sequences][touched][heads][page_size][head_dim]
        most = (x.abs() * fresh).amax(dim=(-2, -1), keepdim=True)
        s = torch.maximum(old * begun, torch.clamp_min((most.double() / 127.0).float(), 1e-8))
        again = torch.round(((held.double() * old.double()).float().double() / s.double()).float())
        coded = torch.round((x.double() / s.double()).float())
        c[page] = torch.where(fresh, coded, torch.where(older, again, held.float())).to(torch.int8)
        scales[page] = s[..., 0, 0]


def _softmax_values(q, k, v, visible):
    """softmax(q k^T) v in 32 bits; rows that see no key give zeros. q [..][rows][d], k, v [..][keys][d]."""
    scores = torch.matmul(q, k.transpose(-1, -2).contiguous())
    scores.masked_fill_(~visible, -math.inf)
    most = scores.amax(dim=-1, keepdim=True)
    scores.sub_(torch.where(most == -math.inf, torch.zeros_like(most), most)).exp_()
    total = scores.sum(dim=-1, keepdim=True)
    return torch.matmul(scores, v) / torch.where(total == 0, torch.ones_like(total), total)


def _attended(state):
    case = state["case"]
    b, h, d, nq = case["sequences"], case["kv_heads"], case["head_dim"], case["max_query"]
    group = case["heads"] // h
    table = state["table"].long()
    span = table.shape[1] * case["page_size"]
    k = state["keys"][table].float() * state["key_scales"][table][..., None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(b, h, span, d)
    v = state["values"][table].float() * state["value_scales"][table][..., None, None]
    v = v.permute(0, 2, 1, 4, 3).reshape(b, h, span, d)
    q = state["q"].float().view(b, nq, h, group, d).permute(0, 2, 1, 3, 4).reshape(b, h, nq * group, d) / math.sqrt(d)
    key = torch.arange(span, device="cuda")
    lengths = state["lengths"].long()
    if case["causal"]:
        seen = lengths[:, None] - nq + 1 + torch.arange(nq, device="cuda")
    else:
        seen = lengths[:, None].expand(b, nq)
    visible = (key < seen[..., None]).repeat_interleave(group, dim=1)[:, None]
    o = _softmax_values(q, k, v, visible)
    o = o.view(b, h, nq, group, d).permute(0, 2, 1, 3, 4).reshape(b * nq, h * group, d)
    return o.to(DTYPES[case["dtype"]])


def _crossed(state):
    case = state["case"]
    b, tq, tk, h, d = case["batch"], case["queries"], case["keys"], case["kv_heads"], case["head_dim"]
    group = case["heads"] // h
    q = state["q"].float().view(b, tq, h, group, d).permute(0, 2, 1, 3, 4).reshape(b, h, tq * group, d) / math.sqrt(d)
    k = state["k"].float().permute(0, 2, 1, 3).contiguous()
    v = state["v"].float().permute(0, 2, 1, 3).contiguous()
    visible = torch.ones((b, 1, 1, tk), dtype=torch.bool, device="cuda")
    if state["lengths"] is not None:
        visible = visible & (torch.arange(tk, device="cuda") < state["lengths"].long()[:, None])[:, None, None]
    if state["mask"] is not None:
        visible = visible & (state["mask"] != 0)[:, None, None]
    o = _softmax_values(q, k, v, visible)
    o = o.view(b, h, tq, group, d).permute(0, 2, 1, 3, 4).reshape(b, tq, h * group, d)
    return o.to(DTYPES[case["dtype"]])


def _plain(state):
    case = state["case"]
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "rotary":
        return _rotated(state["x"].float(), state).to(dtype)
    if kind == "qk_norm":
        return [_rotated(_normed(state[x].float(), state[x + "_weight"], case["norm"]), state).to(dtype)
                for x in ("q", "k")]
    if kind == "store":
        _stored(state)
        return _cache_values(state)
    return _attended(state) if kind == "attend" else _crossed(state)


def _cache_values(state):
    for out, codes, scales in zip(state["stored"], (state["keys"], state["values"]),
                                  (state["key_scales"], state["value_scales"])):
        torch.mul(codes, scales[..., None, None], out=out)
    return {"keys": state["stored"][0], "values": state["stored"][1], "key_scales": state["key_scales"],
            "value_scales": state["value_scales"]}


# ---- the library's calls --------------------------------------------------------------


def _package():
    if "dav2_amd" not in sys.modules:
        spec = importlib.util.spec_from_file_location("dav2_amd", ROOT / "depth-anything-v2_amd" / "__init__.py")
        mod = importlib.util.module_from_spec(spec)
        sys.modules["dav2_amd"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["dav2_amd"]


def _at(t):
    return None if t is None else t.data_ptr()


def _cache_of(pkg, state):
    case = state["case"]
    return pkg.CacheI8(keys=_at(state["keys"]), values=_at(state["values"]), key_scales=_at(state["key_scales"]),
                       value_scales=_at(state["value_scales"]), pages=state["key_scales"].shape[0],
                       kv_heads=case["kv_heads"], page_size=case["page_size"], head_dim=case["head_dim"])


def _scratch(state, args, size):
    """The workspace that a program keeps for calls of this size."""
    if size:
        state["scratch"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        args.scratch, args.scratch_bytes = _at(state["scratch"]), size


def _arguments(state):
    """The entry point and the argument block of a case's call; a program that calls in a loop keeps them."""
    pkg = _package()
    lib = pkg.load()
    case = state["case"]
    kind, code = case["kind"], CODES[case["dtype"]]
    if kind in ("rotary", "qk_norm"):
        d = case["head_dim"]
        shared = dict(positions=_at(state["positions"]), frequencies=_at(state["frequencies"]), tokens=case["tokens"],
                      head_dim=d, rotary_dim=case["rotary_dim"], layout=pkg.ROTARY_LAYOUT[case["layout"]], dtype=code,
                      amplitude=1.0)
        if kind == "rotary":
            args = pkg.RotaryArgs(input=_at(state["x"]), output=_at(state["out"]), input_stride=case["heads"] * d,
                                  output_stride=case["heads"] * d, heads=case["heads"], **shared)
            return lib.dav2_hip_rotary, args, state["out"]
        args = pkg.QkNormRotaryArgs(
            query=_at(state["q"]), key=_at(state["k"]), query_out=_at(state["q_out"]), key_out=_at(state["k_out"]),
            query_stride=state["q"].stride(0), key_stride=state["k"].stride(0),
            query_out_stride=case["heads"] * d, key_out_stride=case["kv_heads"] * d,
            query_weight=_at(state["q_weight"]), key_weight=_at(state["k_weight"]), query_heads=case["heads"],
            key_heads=case["kv_heads"], norm=pkg.QK_NORM[case["norm"]], epsilon=EPSILON, **shared)
        return lib.dav2_hip_qk_norm_rotary, args, [state["q_out"], state["k_out"]]
    if kind in ("store", "attend"):
        shared = dict(cache=_cache_of(pkg, state), page_table=_at(state["table"]), starts=_at(state["starts"]),
                      lengths=_at(state["lengths"]), sequences=case["sequences"], table_pages=state["table"].shape[1],
                      dtype=code)
        if kind == "store":
            x = state["new_keys"]
            args = pkg.CacheStoreI8Args(keys=_at(x), values=_at(state["new_values"]), key_stride=x.stride(0),
                                        value_stride=x.stride(0), tokens=x.shape[0], max_new=case["max_new"], **shared)
            return lib.dav2_hip_cache_store_i8, args, None
        q = state["q"]
        args = pkg.AttentionCacheI8Args(query=_at(q), output=_at(state["out"]), query_stride=q.stride(0),
                                        output_stride=q.stride(0), tokens=q.shape[0], heads=case["heads"],
                                        max_query=case["max_query"], max_length=case["max_length"],
                                        causal=int(case["causal"]), scale=1.0 / math.sqrt(case["head_dim"]), **shared)
        _scratch(state, args, lib.dav2_hip_attention_cache_i8_scratch_bytes(ctypes.byref(args)))
        return lib.dav2_hip_attention_cache_i8, args, state["out"]
    q, k, v, out = state["q"], state["k"], state["v"], state["out"]
    args = pkg.CrossAttentionArgs(
        query=_at(q), keys=_at(k), values=_at(v), output=_at(out), query_stride=q.stride(1), key_stride=k.stride(1),
        value_stride=v.stride(1), output_stride=out.stride(1), query_batch_stride=q.stride(0),
        key_batch_stride=k.stride(0), value_batch_stride=v.stride(0), output_batch_stride=out.stride(0),
        key_lengths=_at(state["lengths"]), key_mask=_at(state["mask"]), batch=case["batch"],
        query_tokens=case["queries"], key_tokens=case["keys"], heads=case["heads"], kv_heads=case["kv_heads"],
        head_dim=case["head_dim"], dtype=code, scale=1.0 / math.sqrt(case["head_dim"]))
    _scratch(state, args, lib.dav2_hip_cross_attention_scratch_bytes(ctypes.byref(args)))
    return lib.dav2_hip_cross_attention, args, out


def _own(state):
    if "call" not in state:
        state["call"] = _arguments(state)
    entry, args, out = state["call"]
    status = entry(ctypes.byref(args), torch.cuda.current_stream().cuda_stream)
    if status:
        raise RuntimeError("%s: status %d" % (state["case"]["kind"], status))
    return _cache_values(state) if out is None else out


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without -------------------------------------------------------


def work(case):
    kind, e = case["kind"], 4.0 if case["dtype"] == "f32" else 2.0
    if kind in ("rotary", "qk_norm"):
        heads = case["heads"] + case.get("kv_heads", 0)
        n = case["tokens"] * heads * case["head_dim"]
        turned = case["tokens"] * heads * case["rotary_dim"]
        return {"bytes": 2.0 * e * n + 4.0 * case["tokens"], "flops": 3.0 * turned + (4.0 * n if kind == "qk_norm" else 0.0)}
    if kind == "store":
        total, new = _sizes(case)
        rows = sum(new) * case["kv_heads"] * case["head_dim"]
        span = -(-case["max_length"] // case["page_size"]) * case["page_size"] * case["sequences"]
        cache = span * case["kv_heads"] * case["head_dim"]
        # the new rows, their codes, and the values that the whole cache stands for
        return {"bytes": 2.0 * rows * (e + 1.0) + 2.0 * cache * (1.0 + 4.0), "flops": 4.0 * rows + 2.0 * cache}
    if kind == "attend":
        total, new = _sizes(case)
        pairs = sum(sum(t - n + 1 + i for i in range(n)) if case["causal"] else t * n for t, n in zip(total, new))
        pages = sum(-(-t // case["page_size"]) for t in total)
        return {"bytes": 2.0 * case["kv_heads"] * (sum(total) * case["head_dim"] + 4.0 * pages) +
                2.0 * e * sum(new) * case["heads"] * case["head_dim"],
                "flops": 4.0 * case["heads"] * case["head_dim"] * pairs}
    keys = sum(_key_counts(case))
    return {"bytes": 2.0 * e * case["head_dim"] * (keys * case["kv_heads"] + case["batch"] * case["queries"] *
                                                   case["heads"]),
            "flops": 4.0 * case["heads"] * case["head_dim"] * case["queries"] * keys * (0.8 if case["mask"] else 1.0)}


# ---- the same in 64 bits ---------------------------------------------------------------


def _turn64(x, case, positions):
    r, last = case["rotary_dim"], x.shape[-1]
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    phase = positions.double().view(-1, 1, 1) * torch.exp(i * (-2.0 * math.log(10000.0) / r))
    z = torch.polar(torch.ones_like(phase), phase)
    if case["layout"] == "pairs":
        w = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous()) * z
        y = torch.view_as_real(w).reshape(*x.shape[:-1], r)
    else:
        w = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * z
        y = torch.cat([w.real, w.imag], -1)
    return torch.cat([y, x[..., r:last]], -1)


def _attention64(q, k, v):
    """One head: q [rows][d], k, v [keys][d]; -inf has been put nowhere: all keys are seen."""
    return torch.softmax(q @ k.T, dim=-1) @ v


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        return _turn64(state["x"].double(), case, state["positions"])
    if kind == "qk_norm":
        out = []
        for x, w in ((state["q"], state["q_weight"]), (state["k"], state["k_weight"])):
            x = x.double()
            if case["norm"] == "layer":
                x = x - x.mean(-1, keepdim=True)
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPSILON) * w.double()
            out.append(_turn64(x, case, state["positions"]))
        return out
    if kind == "store":
        return _store64(case, state)
    d = case["head_dim"]
    group = case["heads"] // case["kv_heads"]
    if kind == "cross":
        out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(_key_counts(case)):
            seen = torch.arange(n, device="cuda")
            if state["mask"] is not None:
                seen = seen[state["mask"][b, :n] != 0]
            if seen.numel() == 0:
                continue
            for h in range(case["heads"]):
                out[b, :, h] = _attention64(state["q"][b, :, h].double() / math.sqrt(d),
                                            state["k"][b, seen, h // group].double(),
                                            state["v"][b, seen, h // group].double())
        return out
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    total, new = _sizes(case)
    at = 0
    for b, (t, n) in enumerate(zip(total, new)):
        pages = state["table"][b, :-(-t // case["page_size"])].long()
        for h in range(case["kv_heads"]):
            k = state["keys"][pages, h].double() * state["key_scales"][pages, h].double()[:, None, None]
            v = state["values"][pages, h].double() * state["value_scales"][pages, h].double()[:, None, None]
            k, v = k.reshape(-1, d)[:t], v.transpose(1, 2).reshape(-1, d)[:t]
            for j in range(group):
                q = state["q"][at:at + n, h * group + j].double() / math.sqrt(d)
                s = q @ k.T
                if case["causal"]:
                    s = s + torch.full((n, t), -math.inf, dtype=torch.float64, device="cuda").triu(t - n + 1)
                out[at:at + n, h * group + j] = torch.softmax(s, dim=-1) @ v
        at += n
    return out


def _store64(case, state):
    """Sequence by sequence and page by page, in 64 bits; a quotient is rounded to 32 bits before it becomes a code."""
    p = case["page_size"]
    total, new = _sizes(case)
    if sum(-(-n // p) + 1 for n in new) > 4000:
        return None
    table = state["table"].tolist()
    sides = [(state["new_keys"].double(), state["keys"].double(), state["key_scales"].double()),
             (state["new_values"].double(), state["values"].double().transpose(2, 3), state["value_scales"].double())]
    row = 0
    for b, (t, n) in enumerate(zip(total, new)):
        pos = t - n
        while pos < t:
            page, slot = table[b][pos // p], pos % p
            take = min(p - slot, t - pos)
            for x, codes, scales in sides:
                part = x[row:row + take].transpose(0, 1)  # [heads][take][head_dim]
                s = (part.abs().amax(dim=(1, 2)) / 127.0).float().double().clamp_min(float(torch.tensor(1e-8)))
                old = scales[page].clone()
                if slot:
                    s = torch.maximum(s, old)
                    held = (codes[page, :, :slot] * old[:, None, None]).float().double()
                    codes[page, :, :slot] = torch.round((held / s[:, None, None]).float().double())
                codes[page, :, slot:slot + take] = torch.round((part / s[:, None, None]).float().double())
                scales[page] = s
            pos, row = pos + take, row + take
    (_, k, ks), (_, v, vs) = sides
    return {"keys": k * ks[..., None, None], "values": (v * vs[..., None, None]).transpose(2, 3), "key_scales": ks,
            "value_scales": vs}
