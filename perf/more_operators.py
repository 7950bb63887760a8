"""The operators of a decoding step around a cache in 4 bits, as cases that can be timed and checked.

  plan     dav2_hip_cache_plan: page table, starts, lengths, positions and slots of a step from its requests
  store    dav2_hip_cache_store_i4: new keys and values into a paged cache of 4-bit codes, one scale per token and head
  attend   dav2_hip_attention_cache_i4: attention over such a cache, single tokens and prompts
  norm     dav2_hip_add_rms_norm: a residual's addition, the root-mean-square norm, rows in 8 bits
  sample   dav2_hip_sample: the next token from temperature, min-p, top-k, top-p and a given random number

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
        # a decoding step of a batch of 48: most sequences get a token, some none, some end
        dict(name="plan_step", kind="plan", sequences=48, max_new=1, max_length=4096, page_size=16, short=False),
        # many prompts at once, more than there are pages for
        dict(name="plan_prompts", kind="plan", sequences=1024, max_new=1024, max_length=2048, page_size=32, short=True),
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
        # three drafted tokens and one more of 16 sequences, a width that is no power of two
        dict(name="attend_draft", kind="attend", sequences=16, max_query=4, max_length=5003, heads=24, kv_heads=6,
             head_dim=96, page_size=48, causal=True, dtype="f16"),
        # the last quarter of two prompts
        dict(name="attend_prompt_chunk", kind="attend", sequences=2, max_query=2048, max_length=8192, heads=32,
             kv_heads=8, head_dim=128, page_size=64, causal=True, dtype="f16"),
        # one token between two layers of an encoder's width: the latency of a call
        dict(name="norm_token", kind="norm", rows=1, columns=1024, residual=True, codes=True, dtype="f32"),
        # a long prompt, its rows for an int8 product
        dict(name="norm_prompt", kind="norm", rows=8191, columns=4096, residual=True, codes=True, dtype="bf16"),
        # four answers, every filter
        dict(name="sample_step", kind="sample", rows=4, vocabulary=32000, filters="all", dtype="f32"),
        # a full batch over a large vocabulary
        dict(name="sample_batch", kind="sample", rows=256, vocabulary=100003, filters="top_p", dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["plan", "store", "attend", "attend", "norm", "sample"])
        case = dict(kind=kind)
        if kind != "plan":
            case["dtype"] = rng.choice(list(DTYPES))
        if kind == "plan":
            new = rng.choice([1, 1, _log_int(rng, 2, 4096)])
            case.update(sequences=_log_int(rng, 1, 4096 if new < 64 else 1024), max_new=new,
                        max_length=new + _log_int(rng, 1, 16384), page_size=rng.choice([16, 32, 48, 64, 128, 256]),
                        short=rng.random() < 0.3)
        elif kind == "store":
            new = rng.choice([1, 1, _log_int(rng, 2, 2048)])
            case.update(sequences=_log_int(rng, 1, 64), max_new=new, max_length=new + _log_int(rng, 1, 256),
                        kv_heads=_log_int(rng, 1, 16), head_dim=rng.choice([64, 80, 96, 128]),
                        page_size=rng.choice([16, 32, 48, 64, 128]))
        elif kind == "attend":
            queries = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 2048)])
            kv = _log_int(rng, 1, 16)
            case.update(sequences=_log_int(rng, 1, 48 if queries < 9 else 4), max_query=queries,
                        max_length=queries + _log_int(rng, 1, 32768 if queries < 9 else 8192), kv_heads=kv,
                        heads=kv * rng.choice([1, 2, 4, 5, 8]), head_dim=rng.choice([64, 80, 96, 128]),
                        page_size=rng.choice([16, 32, 48, 64, 128]), causal=rng.random() < 0.7)
        elif kind == "norm":
            case.update(rows=_log_int(rng, 1, 16384), columns=_log_int(rng, 64, 16384), residual=rng.random() < 0.8,
                        codes=rng.random() < 0.6)
        else:
            case.update(rows=_log_int(rng, 1, 256), vocabulary=_log_int(rng, 1000, 200000),
                        filters=rng.choice(["all", "top_p", "top_k", "none"]))
        if _cost(case) <= most and _plain_floats(case) <= 3e9:
            return case


def _plain_floats(case):
    """Values that the plain form holds at a time."""
    if case["kind"] == "attend":
        return (case["sequences"] * case["max_length"] * (case["heads"] * case["max_query"] +
                                                          2 * case["kv_heads"] * case["head_dim"]))
    if case["kind"] == "norm":
        return 10 * case["rows"] * case["columns"]
    if case["kind"] == "sample":
        return 20 * case["rows"] * case["vocabulary"]
    return 0


def _cost(case):
    w = work(case)
    # the products of 32-bit tensors are several of 16 bits
    return w["flops"] * (4.0 if case.get("dtype") == "f32" else 1.0) + 100.0 * w["bytes"]


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


def _requests(case, seed):
    """What a step's sequences hold and get (-1: they end)."""
    r = random.Random("%d %d" % (case["sequences"], seed))
    held, added = [], []
    for i in range(case["sequences"]):
        n = max(1, round(case["max_new"] * (r.uniform(0.1, 1.0) if i else 1.0)))
        kind = r.random() if i else 1.0
        added.append(-1 if kind < 0.1 else 0 if kind < 0.2 else n)
        held.append(r.randint(0, case["max_length"] - n))
    return held, added


def _plan_tokens(case):
    """Rows that a step is laid out for: of every sequence's largest share."""
    return case["sequences"] * case["max_new"]


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table(case):
    """A page table over shuffled pages: [sequences][most pages of one], and how many pages there are."""
    most = -(-case["max_length"] // case["page_size"])
    count = case["sequences"] * most
    order = torch.randperm(count, generator=torch.Generator().manual_seed(count + case["page_size"]))
    return order.to(torch.int32).view(case["sequences"], most).cuda(), count


def _quantized(x):
    """Codes -7 .. 7 of x [..][features] with one scale for its last axis, and the scales."""
    s = torch.clamp_min(x.abs().amax(dim=-1) / 7.0, 1e-8)
    return torch.round(x / s[..., None]).to(torch.int8), s


def _packed(codes):
    """Pairs of neighbours of the last axis in a byte each, the first one in the low four bits, as code + 8."""
    c = (codes + 8).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _unpacked(b):
    return torch.stack([b & 15, b >> 4], dim=-1).flatten(-2).to(torch.int8) - 8


def _chunked(values):
    """Codes [..][page_size][head_dim] as a cache holds its values: [..][page_size / 16][head_dim][16]."""
    return values.unflatten(-2, (-1, 16)).transpose(-1, -2)


def _random_cache(case, pages, g):
    """Keys and values of a decoder, quantized: some features of the keys are large, values differ from token to token."""
    h, p, d = case["kv_heads"], case["page_size"], case["head_dim"]
    wide = 1.0 + 3.0 * (torch.rand((h, 1, d), generator=g, device="cuda") < 0.05)
    keys = torch.empty((pages, h, p, d // 2), dtype=torch.uint8, device="cuda")
    values = torch.empty((pages, h, p // 16, d, 8), dtype=torch.uint8, device="cuda")
    ks, vs = (torch.empty((pages, h, p), device="cuda") for _ in range(2))
    step = max(1, int(2 ** 26 // (h * p * d)))
    for a in range(0, pages, step):
        n = min(step, pages - a)
        c, ks[a:a + n] = _quantized(torch.randn((n, h, p, d), generator=g, device="cuda") * wide)
        keys[a:a + n] = _packed(c)
        v = torch.randn((n, h, p, d), generator=g, device="cuda")
        v *= 0.25 + torch.rand((n, h, p, 1), generator=g, device="cuda")
        c, vs[a:a + n] = _quantized(v)
        values[a:a + n] = _packed(_chunked(c))
    return keys, values, ks, vs


def prepare(case, seed):
    g = _generator(seed)
    kind, state = case["kind"], {"case": case}
    dtype = DTYPES.get(case.get("dtype"))

    def normal(*shape, scale=1.0):
        return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)

    if kind == "plan":
        _prepare_plan(case, seed, state)
    elif kind in ("store", "attend"):
        total, new = _sizes(case)
        table, pages = _table(case)
        keys, values, ks, vs = _random_cache(case, pages, g)
        starts = [sum(new[:i]) for i in range(len(new) + 1)]
        state.update(keys=keys, values=values, key_scales=ks, value_scales=vs, table=table, starts=_int32(starts),
                     lengths=_int32(total))
        n, h, d = starts[-1], case["kv_heads"], case["head_dim"]
        if kind == "store":
            state.update(new_keys=normal(n, h, d, scale=1.1), new_values=normal(n, h, d, scale=0.6))
        else:
            state.update(q=normal(n, case["heads"], d),
                         out=torch.zeros((n, case["heads"], d), dtype=dtype, device="cuda"))
    elif kind == "norm":
        n, c = case["rows"], case["columns"]
        state.update(x=normal(n, c, scale=0.7), residual=normal(n, c, scale=2.0) if case["residual"] else None,
                     weight=1.0 + 0.2 * torch.randn(c, generator=g, device="cuda"),
                     sum=torch.empty((n, c), dtype=dtype, device="cuda"),
                     out=torch.empty((n, c), dtype=dtype, device="cuda"), scales=torch.empty(n, device="cuda"),
                     codes=torch.empty((n, -(-c // 64) * 64), dtype=torch.int8, device="cuda"))
    else:
        n, v, which = case["rows"], case["vocabulary"], case["filters"]
        logits = normal(n, v, scale=2.5)
        logits[:, ::97] -= 20.0  # tokens that hardly ever come
        r = torch.rand((5, n), generator=g, device="cuda")
        all_of = which == "all"
        # rows 0, 8, .. of a step with every filter take the largest logit
        temperature = 0.6 + 0.8 * r[0]
        temperature[0 if all_of else n::8] = 0.0
        state.update(logits=logits, temperature=temperature, uniform=r[1],
                     top_k=(1 + 120 * r[2]).to(torch.int32) if which in ("all", "top_k") else None,
                     top_p=0.7 + 0.29 * r[3] if which in ("all", "top_p") else None,
                     min_p=0.08 * r[4] if all_of else None, tokens=torch.empty(n, dtype=torch.int32, device="cuda"),
                     probabilities=torch.empty(n, device="cuda"))
    return state


def _prepare_plan(case, seed, state):
    held, added = _requests(case, seed)
    p, n = case["page_size"], case["sequences"]
    most = -(-case["max_length"] // p)
    r = random.Random(seed)
    count = 2 * n * most
    order = torch.randperm(count, generator=torch.Generator().manual_seed(seed & 0x7FFFFFFF)).to(torch.int32)
    owned = [-(-h // p) for h in held]
    need = sum(-(-(h + a) // p) - o for h, a, o in zip(held, added, owned) if a > 0)
    # the entries after a sequence's pages are what earlier steps left there
    table = torch.randint(0, count, (n, most), generator=torch.Generator().manual_seed(seed & 0x7FFFFFFF),
                          dtype=torch.int32)
    at = 0
    for i, o in enumerate(owned):
        table[i, :o] = order[at:at + o]
        at += o
    free = count - at if not case["short"] else max(1, need * 3 // 4)
    first = r.randrange(count)
    ring = torch.full((count,), -1, dtype=torch.int32)
    where = (first + torch.arange(free)) % count
    ring[where] = order[at:at + free]
    # one value more in each for what the plain form writes nowhere
    flat = torch.cat([table.flatten(), torch.zeros(1, dtype=torch.int32)]).cuda()
    ring = torch.cat([ring, torch.zeros(1, dtype=torch.int32)]).cuda()
    t = _plan_tokens(case)
    state.update(held=_int32(held), added=_int32(added), flat=flat, table=flat[:n * most].view(n, most), ring=ring,
                 free_state=_int32([first, free]), pages=count, tokens=t,
                 held_out=torch.empty(n, dtype=torch.int32, device="cuda"), free_out=_int32([0, 0]),
                 starts=torch.empty(n + 1, dtype=torch.int32, device="cuda"),
                 lengths=torch.empty(n, dtype=torch.int32, device="cuda"),
                 positions=torch.empty(t, dtype=torch.int32, device="cuda"),
                 owners=torch.empty(t, dtype=torch.int32, device="cuda"),
                 slots=torch.empty(t, dtype=torch.int64, device="cuda"))


# ---- the operators in elementary operations -----------------------------------------


def _planned(state):
    """The step's plan, in whole numbers of 64 bits; pages come from the front of a ring and go back to its end."""
    case = state["case"]
    p, n, t, pages = case["page_size"], case["sequences"], state["tokens"], state["pages"]
    most = state["table"].shape[1]
    held, added = state["held"].long(), state["added"].long()
    first, count = state["free_state"].long().unbind()
    new = added.clamp_min(0)
    ends = new.cumsum(0)
    owned = (held + p - 1) // p
    fits = (added >= 0) & (held + new <= most * p) & (ends <= t)
    need = torch.where(fits, (held + new + p - 1) // p - owned, 0)
    taken = need.cumsum(0)
    served = fits & ((need == 0) | (taken <= count))
    # the rows
    row = torch.arange(t, device="cuda")
    s = torch.searchsorted(ends, row, right=True)
    real = s < n
    s = s.clamp_max(n - 1)
    position = held[s] + row - (ends - new)[s]
    place = position // p
    fresh = place >= owned[s]
    front = (first + (taken - need)[s] + place - owned[s]) % pages
    entry = (s * most + place).clamp_max(n * most - 1)
    page = torch.where(fresh, state["ring"][front.clamp_min(0)].long(), state["flat"][entry].long())
    known = real & served[s] & (page >= 0) & (page < pages)
    writes = real & served[s] & fresh & (position % p == 0)
    state["flat"][torch.where(writes, entry, n * most)] = page.int()
    # what ended sequences give back
    column = torch.arange(most, device="cuda")
    given = (added < 0)[:, None] & (column < owned[:, None])
    order = given.flatten().cumsum(0) - 1
    back = torch.where(given.flatten() & (order < pages - count), (first + count + order) % pages, pages)
    state["ring"][back] = state["flat"][:n * most]
    used = (need * served).sum()
    released = torch.minimum(given.sum(), pages - count)
    return {"table": state["table"], "ring": state["ring"][:pages],
            "free": torch.stack([(first + used) % pages, count - used + released]).int(),
            "held": torch.where(added < 0, 0, torch.where(served, held + new, held)).int(),
            "lengths": torch.where(served, held + new, 0).int(),
            "starts": torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), ends]).clamp_max(t).int(),
            "positions": torch.where(real, position, 0).int(), "owners": torch.where(real, s, -1).int(),
            "slots": torch.where(known, page * p + position % p, -1)}


def _stored(state):
    """The cache with the new tokens in it, in place: every page that gets one is put together anew."""
    case = state["case"]
    p = case["page_size"]
    starts, lengths = state["starts"].long(), state["lengths"].long()
    first = (lengths - starts.diff())[:, None]  # the first new token's position
    touched = (case["max_new"] + p - 2) // p + 1
    # past a sequence's last page: that page again
    place = torch.minimum(first // p + torch.arange(touched, device="cuda"), (lengths[:, None] - 1) // p)
    page = state["table"].long().gather(1, place)  # [sequences][touched]
    pos = place[..., None] * p + torch.arange(p, device="cuda")
    fresh = ((pos >= first[..., None]) & (pos < lengths[:, None, None]))[:, :, None, :]
    row = (starts[:-1, None, None] + pos - first[..., None]).clamp(0, state["new_keys"].shape[0] - 1)
    for name, scales in (("keys", "key_scales"), ("values", "value_scales")):
        x = state["new_" + name].float()
        s = torch.clamp_min((x.abs().amax(dim=-1).double() / 7.0).float(), 1e-8)
        c = torch.round((x.double() / s.double()[..., None]).float()).to(torch.int8)
        c, s = c[row].transpose(2, 3), s[row].transpose(2, 3)  # [sequences][touched][heads][page_size](..)
        held = _unpacked(state[name][page])
        mask = fresh[..., None]
        if name == "values":
            c = _chunked(c)
            mask = _chunked(mask)
        state[name][page] = _packed(torch.where(mask, c, held))
        state[scales][page] = torch.where(fresh, s, state[scales][page])


def _cache_values(state):
    """What the cache stands for."""
    return {"keys": _unpacked(state["keys"]) * state["key_scales"][..., None],
            "values": _unpacked(state["values"]) * state["value_scales"].unflatten(2, (-1, 1, 16)),
            "key_scales": state["key_scales"], "value_scales": state["value_scales"]}


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
    k = _unpacked(state["keys"][table]).float() * state["key_scales"][table][..., None]
    k = k.permute(0, 2, 1, 3, 4).reshape(b, h, span, d)
    v = _unpacked(state["values"][table]) * state["value_scales"][table].unflatten(3, (-1, 1, 16))
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(b, h, span, d)
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


def _normed(state):
    """The sum is rounded to the tensors' type before its norm. A row's factor is formed in 64 bits and rounded to 32:
    a code next to a border then does not go by the order of the sum."""
    case = state["case"]
    h = state["x"]
    if case["residual"]:
        h = (h.float() + state["residual"].float()).to(h.dtype)
    x = h.float()
    factor = (1.0 / torch.sqrt(x.double().square().mean(dim=-1, keepdim=True) + EPSILON)).float()
    y = x * factor * state["weight"]
    out = {"normed": y.to(h.dtype)}
    if case["residual"]:
        out["sum"] = h
    if case["codes"]:
        s = torch.clamp_min((y.abs().amax(dim=-1).double() / 127.0).float(), 1e-8)
        c = torch.round((y.double() / s.double()[:, None]).float()).to(torch.int8)
        out.update(codes=c * s[:, None], scales=s)
    return out


def _sampled(state):
    """Tokens in order of their logits, ties by index; the weights of a prefix of them are kept, in 64 bits as a
    random number next to a border decides."""
    v = state["case"]["vocabulary"]
    logits, index = torch.sort(state["logits"].float(), dim=-1, descending=True, stable=True)
    rank = torch.arange(v, device="cuda")
    t = state["temperature"].double()[:, None]
    e = torch.exp((logits.double() - logits[:, :1].double()) / torch.where(t > 0, t, torch.ones_like(t)))
    keep = (t > 0) | (rank == 0)
    if state["min_p"] is not None:
        keep = keep & (e >= state["min_p"].double()[:, None])
    if state["top_k"] is not None:
        keep = keep & (rank < state["top_k"][:, None])
    e = e * keep
    sums = e.cumsum(dim=-1)
    if state["top_p"] is not None:
        before = torch.cat([torch.zeros_like(sums[:, :1]), sums[:, :-1]], dim=-1)
        e = e * (before < state["top_p"].double()[:, None] * sums[:, -1:])
        sums = e.cumsum(dim=-1)
    total = sums[:, -1:]
    at = (sums <= state["uniform"].double()[:, None] * total).sum(dim=-1, keepdim=True)
    at = torch.minimum(at, (e > 0).sum(dim=-1, keepdim=True) - 1)
    return {"tokens": index.gather(1, at)[:, 0].int(), "probabilities": (e.gather(1, at) / total)[:, 0].float()}


def _plain(state):
    kind = state["case"]["kind"]
    if kind == "store":
        _stored(state)
        return _cache_values(state)
    return {"plan": _planned, "attend": _attended, "norm": _normed, "sample": _sampled}[kind](state)


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
    kind, code = case["kind"], CODES.get(case.get("dtype"))
    if kind == "plan":
        args = pkg.CachePlanArgs(
            held=_at(state["held"]), added=_at(state["added"]), page_table=_at(state["table"]),
            free_pages=_at(state["ring"]), free_state=_at(state["free_state"]), held_out=_at(state["held_out"]),
            free_state_out=_at(state["free_out"]), starts=_at(state["starts"]), lengths=_at(state["lengths"]),
            positions=_at(state["positions"]), owners=_at(state["owners"]), slots=_at(state["slots"]),
            sequences=case["sequences"], table_pages=state["table"].shape[1], tokens=state["tokens"],
            pages=state["pages"], page_size=case["page_size"])
        _scratch(state, args, lib.dav2_hip_cache_plan_scratch_bytes(ctypes.byref(args)))
        return lib.dav2_hip_cache_plan, args
    if kind == "norm":
        x, r = state["x"], state["residual"]
        c = case["columns"]
        args = pkg.AddRmsNormArgs(
            input=_at(x), residual=_at(r), weight=_at(state["weight"]), sum=_at(state["sum"]) if r is not None else None,
            output=_at(state["out"]), codes=_at(state["codes"]) if case["codes"] else None,
            scales=_at(state["scales"]) if case["codes"] else None, input_stride=c, residual_stride=c, sum_stride=c,
            output_stride=c, code_stride=state["codes"].stride(0), rows=case["rows"], columns=c, dtype=code,
            epsilon=EPSILON)
        return lib.dav2_hip_add_rms_norm, args
    if kind == "sample":
        args = pkg.SampleArgs(
            logits=_at(state["logits"]), logit_stride=case["vocabulary"], temperature=_at(state["temperature"]),
            top_k=_at(state["top_k"]), top_p=_at(state["top_p"]), min_p=_at(state["min_p"]),
            uniform=_at(state["uniform"]), tokens=_at(state["tokens"]), probabilities=_at(state["probabilities"]),
            rows=case["rows"], vocabulary=case["vocabulary"], dtype=code)
        _scratch(state, args, lib.dav2_hip_sample_scratch_bytes(ctypes.byref(args)))
        return lib.dav2_hip_sample, args
    cache = pkg.CacheI4(keys=_at(state["keys"]), values=_at(state["values"]), key_scales=_at(state["key_scales"]),
                        value_scales=_at(state["value_scales"]), pages=state["key_scales"].shape[0],
                        kv_heads=case["kv_heads"], page_size=case["page_size"], head_dim=case["head_dim"])
    shared = dict(cache=cache, page_table=_at(state["table"]), starts=_at(state["starts"]),
                  lengths=_at(state["lengths"]), sequences=case["sequences"], table_pages=state["table"].shape[1],
                  dtype=code)
    if kind == "store":
        x = state["new_keys"]
        args = pkg.CacheStoreI4Args(keys=_at(x), values=_at(state["new_values"]), key_stride=x.stride(0),
                                    value_stride=x.stride(0), tokens=x.shape[0], max_new=case["max_new"], **shared)
        return lib.dav2_hip_cache_store_i4, args
    q = state["q"]
    args = pkg.AttentionCacheI4Args(query=_at(q), output=_at(state["out"]), query_stride=q.stride(0),
                                    output_stride=q.stride(0), tokens=q.shape[0], heads=case["heads"],
                                    max_query=case["max_query"], max_length=case["max_length"],
                                    causal=int(case["causal"]), scale=1.0 / math.sqrt(case["head_dim"]), **shared)
    _scratch(state, args, lib.dav2_hip_attention_cache_i4_scratch_bytes(ctypes.byref(args)))
    return lib.dav2_hip_attention_cache_i4, args


def _own(state):
    if "call" not in state:
        state["call"] = _arguments(state)
    entry, args = state["call"]
    case = state["case"]
    kind = case["kind"]
    status = entry(ctypes.byref(args), torch.cuda.current_stream().cuda_stream)
    if status:
        raise RuntimeError("%s: status %d" % (kind, status))
    if kind == "plan":
        return {"table": state["table"], "ring": state["ring"][:state["pages"]], "free": state["free_out"],
                "held": state["held_out"], **{x: state[x] for x in ("lengths", "starts", "positions", "owners", "slots")}}
    if kind == "store":
        return _cache_values(state)
    if kind == "attend":
        return state["out"]
    if kind == "sample":
        return {"tokens": state["tokens"], "probabilities": state["probabilities"]}
    out = {"normed": state["out"]}
    if case["residual"]:
        out["sum"] = state["sum"]
    if case["codes"]:
        out.update(codes=state["codes"][:, :case["columns"]] * state["scales"][:, None], scales=state["scales"])
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without -------------------------------------------------------


def work(case):
    kind, e = case["kind"], 4.0 if case.get("dtype") == "f32" else 2.0
    if kind == "plan":
        held, added = _requests(case, 0)
        p = case["page_size"]
        rows = _plan_tokens(case)
        moved = sum(-(-(h + a) // p) - -(-h // p) if a > 0 else -(-h // p) if a < 0 else 0 for h, a in zip(held, added))
        # what a sequence has and gets; of a row its position, sequence and slot; pages from or to the ring
        return {"bytes": 20.0 * case["sequences"] + 16.0 * rows + 8.0 * moved, "flops": 4.0 * rows}
    if kind == "norm":
        n = float(case["rows"]) * case["columns"]
        coded = (1.0 + 1.0 + 4.0) if case["codes"] else 0.0  # the codes, and the values that they stand for
        return {"bytes": n * (e * (4.0 if case["residual"] else 2.0) + coded) + 4.0 * case["columns"], "flops": 6.0 * n}
    if kind == "sample":
        n = float(case["rows"]) * case["vocabulary"]
        return {"bytes": n * e + 28.0 * case["rows"], "flops": 20.0 * n}
    total, new = _sizes(case)
    if kind == "store":
        rows = sum(new) * case["kv_heads"] * case["head_dim"]
        span = -(-case["max_length"] // case["page_size"]) * case["page_size"] * case["sequences"]
        cache = span * case["kv_heads"] * case["head_dim"]
        # the new rows, their codes, and the values that the whole cache stands for
        return {"bytes": 2.0 * rows * (e + 0.5) + 2.0 * cache * (0.5 + 4.0), "flops": 4.0 * rows + 2.0 * cache}
    pairs = sum(sum(t - n + 1 + i for i in range(n)) if case["causal"] else t * n for t, n in zip(total, new))
    return {"bytes": 2.0 * case["kv_heads"] * sum(total) * (0.5 * case["head_dim"] + 4.0) +
            2.0 * e * sum(new) * case["heads"] * case["head_dim"],
            "flops": 4.0 * case["heads"] * case["head_dim"] * pairs}


# ---- the same in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    """What `run` returns, from the definitions, in whole numbers or in 64 bits."""
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "plan":
        return _plan_one_by_one(case, state)
    if kind == "norm":
        return _norm64(case, state)
    if kind == "sample":
        return _sample64(case, state)
    if kind == "store":
        return _store64(case, state)
    d = case["head_dim"]
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    total, new = _sizes(case)
    at = 0
    for b, (t, n) in enumerate(zip(total, new)):
        pages = state["table"][b, :-(-t // case["page_size"])].long()
        for h in range(case["kv_heads"]):
            k, v = _nibbles64(state["keys"][pages, h]), _nibbles64(state["values"][pages, h])
            k = (k * state["key_scales"][pages, h].double()[..., None]).reshape(-1, d)[:t]
            v = v.transpose(2, 3).reshape(-1, d) * state["value_scales"][pages, h].double().reshape(-1, 1)
            for j in range(group):
                q = state["q"][at:at + n, h * group + j].double() / math.sqrt(d)
                s = q @ k.T
                if case["causal"]:
                    s = s + torch.full((n, t), -math.inf, dtype=torch.float64, device="cuda").triu(t - n + 1)
                out[at:at + n, h * group + j] = torch.softmax(s, dim=-1) @ v[:t]
        at += n
    return out


def _plan_one_by_one(case, state):
    """The plan of a step, sequence by sequence and page by page."""
    p, pages, t = case["page_size"], state["pages"], state["tokens"]
    table, ring = state["table"].tolist(), state["ring"][:pages].tolist()
    held, added = state["held"].tolist(), state["added"].tolist()
    first, count = state["free_state"].tolist()
    most = len(table[0])
    left, asked, back = count, 0, []
    out = {"held": [], "lengths": [], "starts": [0], "positions": [], "owners": [], "slots": []}
    for s, (h, a) in enumerate(zip(held, added)):
        n, own_pages = max(a, 0), -(-h // p)
        end = out["starts"][-1] + n
        length = h + n if a >= 0 and h + n <= most * p and end <= t else 0
        if length:
            need = -(-length // p) - own_pages
            asked += need
            if need and asked > count:
                length = 0
            else:
                for i in range(need):
                    table[s][own_pages + i] = ring[(first + count - left) % pages]
                    left -= 1
        if a < 0:
            back += table[s][:own_pages]
        out["held"].append(0 if a < 0 else length if length else h)
        out["lengths"].append(length)
        out["starts"].append(end)
        out["positions"] += range(h, h + n)
        out["owners"] += [s] * n
        out["slots"] += [table[s][x // p] * p + x % p if length else -1 for x in range(h, h + n)]
    back = back[:pages - count]
    for i, page in enumerate(back):
        ring[(first + count + i) % pages] = page
    padding = t - len(out["positions"])
    out["positions"] += [0] * padding
    out["owners"] += [-1] * padding
    out["slots"] += [-1] * padding
    out.update(table=table, ring=ring, free=[(first + count - left) % pages, left + len(back)])
    return {x: torch.tensor(y, dtype=torch.int64 if x == "slots" else torch.int32, device="cuda")
            for x, y in out.items()}


def _nibbles64(b):
    """Numbers of a cache's bytes: the low half first, each less 8."""
    low = torch.remainder(b.double(), 16.0)
    return torch.stack([low, (b.double() - low) / 16.0], dim=-1).flatten(-2) - 8.0


def _norm64(case, state):
    """In 64 bits, with the roundings that the definition has: the sum to its type, a row's factor, each of the two
    products, a row's scale and a quotient to 32 bits."""
    def fp32(x):
        return x.float().double()

    h = state["x"].double()
    if case["residual"]:
        h = fp32(h + state["residual"].double()).to(state["x"].dtype).double()
    factor = fp32((torch.linalg.vector_norm(h, dim=1).square() / case["columns"] + EPSILON).pow(-0.5))
    y = fp32(fp32(torch.mul(h, factor.view(-1, 1))) * state["weight"].double())
    out = {"normed": y}
    if case["residual"]:
        out["sum"] = h
    if case["codes"]:
        s = torch.maximum(fp32(torch.linalg.vector_norm(y, ord=math.inf, dim=1) / 127.0),
                          torch.tensor(1e-8, device="cuda").double())
        out.update(codes=torch.round(fp32(y / s.view(-1, 1))) * s.view(-1, 1), scales=s)
    return out


def _sample64(case, state):
    """Row by row: how many tokens are kept, then where the random number falls."""
    tokens, probabilities = [], []
    for i in range(case["rows"]):
        x = state["logits"][i].double()
        t = float(state["temperature"][i])
        order = torch.argsort(x, descending=True, stable=True)
        kept = case["vocabulary"] if t > 0 else 1
        w = torch.softmax(x / (t if t > 0 else 1.0), dim=0)[order]
        if state["min_p"] is not None:
            kept = min(kept, max(1, int((w >= w[0] * float(state["min_p"][i])).sum())))
        if state["top_k"] is not None:
            kept = min(kept, int(state["top_k"][i]))
        w = w[:kept] / w[:kept].sum()
        if state["top_p"] is not None:
            ends = w.cumsum(0)
            kept = int(torch.searchsorted(ends, float(state["top_p"][i]) * ends[-1])) + 1
            w = w[:kept] / w[:kept].sum()
        at = int(torch.searchsorted(w.cumsum(0), float(state["uniform"][i]), right=True))
        at = min(at, w.numel() - 1)
        tokens.append(int(order[at]))
        probabilities.append(float(w[at]))
    return {"tokens": _int32(tokens), "probabilities": torch.tensor(probabilities, dtype=torch.float64, device="cuda")}


def _store64(case, state):
    """Sequence by sequence in 64 bits; a scale and a quotient are rounded to 32 bits before the code is."""
    p = case["page_size"]
    total, new = _sizes(case)
    out = {}
    row, at = 0, []
    for b, (t, n) in enumerate(zip(total, new)):
        pos = torch.arange(t - n, t, device="cuda")
        at.append(torch.stack([state["table"][b].long()[pos // p], pos % p]))
        row += n
    page, slot = torch.cat(at, dim=1)
    for name, scales in (("keys", "key_scales"), ("values", "value_scales")):
        codes, s = _nibbles64(state[name]), state[scales].double()
        x = state["new_" + name].double()
        mine = torch.linalg.vector_norm(x, ord=math.inf, dim=2) / 7.0
        mine = torch.maximum(mine.float(), torch.tensor(1e-8, device="cuda")).double()
        s[page, :, slot] = mine
        c = torch.round((x / mine[..., None]).float().double())
        if name == "keys":
            codes[page, :, slot] = c
            out[name] = codes * s[..., None]
        else:
            codes[page, :, slot // 16, :, slot % 16] = c
            out[name] = codes * s.view(*s.shape[:2], -1, 1, 16)
        out[scales] = s
    return out
