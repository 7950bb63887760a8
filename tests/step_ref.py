"""The operators of a decoding step (plan of a paged cache, the 4-bit cache,
residual addition with RMS norm, sampling) from their definitions, on the CPU
or in float64."""

from __future__ import annotations

import math

import numpy as np
import torch

import decoder_ref as ref


# ---- the 4-bit cache ----------------------------------------------------------------


def pack(codes):
    """Codes [..][2 n] as bytes [..][n]: the first of a pair in the low half, as code + 8."""
    c = (codes + 8).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def unpack(b):
    return torch.stack([b & 15, b >> 4], dim=-1).flatten(-2).to(torch.int8) - 8


def key_codes(keys):
    """[pages][heads][page][dim / 2] bytes -> codes [pages][heads][page][dim]."""
    return unpack(keys)


def value_codes(values):
    """[pages][heads][page / 16][dim][8] bytes -> codes [pages][heads][page][dim]."""
    return unpack(values).transpose(-1, -2).flatten(-3, -2)


def pack_values(codes):
    """Codes [pages][heads][page][dim] as the cache holds values."""
    return pack(codes.unflatten(-2, (-1, 16)).transpose(-1, -2).contiguous())


def quantized(x):
    """x float32 [..][dim]: codes and scales, each quotient rounded to fp32."""
    s = torch.clamp_min((x.abs().amax(-1).double() / 7.0).float(), 1e-8)
    return torch.round((x.double() / s.double()[..., None]).float()).clamp(-7, 7).to(torch.int8), s


def store(keys, values, key_scales, value_scales, new_keys, new_values, table, starts, lengths):
    """cache_store_i4 on CPU copies: the new cache."""
    ks, vs = key_scales.clone().cpu(), value_scales.clone().cpu()
    kc, vc = key_codes(keys.cpu()), value_codes(values.cpu())
    page_size, pages, tokens = ks.shape[2], ks.shape[0], new_keys.shape[0]
    table, starts, lengths = table.cpu().tolist(), starts.cpu().tolist(), lengths.cpu().tolist()
    new_kc, new_ks = quantized(new_keys.float().cpu())
    new_vc, new_vs = quantized(new_values.float().cpu())
    for s, total in enumerate(lengths):
        begin = min(max(starts[s], 0), tokens)
        end = min(max(starts[s + 1], begin), tokens)
        total = max(total, 0)
        for r in range(begin, end):
            pos = total - (end - begin) + (r - begin)
            if pos < 0 or pos >= len(table[s]) * page_size:
                continue
            page, slot = table[s][pos // page_size], pos % page_size
            if 0 <= page < pages:
                kc[page, :, slot], ks[page, :, slot] = new_kc[r], new_ks[r]
                vc[page, :, slot], vs[page, :, slot] = new_vc[r], new_vs[r]
    return [pack(kc), pack_values(vc), ks, vs]


def attend(q, cache, table, starts, lengths, causal, scale, dtype):
    """Float64 attention over a 4-bit cache, and how far a kernel may be off: as decoder_ref.attend."""
    keys, values, ks, vs = cache
    kc, vc = key_codes(keys), value_codes(values)
    heads, d = q.shape[1], q.shape[2]
    pages, kv_heads, page_size = ks.shape
    group = heads // kv_heads
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    step = 2.0 ** -21 if dtype == "f32" else 2.0 ** -11
    starts, lengths, table = starts.tolist(), lengths.tolist(), table.cpu()
    for s, total in enumerate(lengths):
        begin = min(max(starts[s], 0), q.shape[0])
        end = min(max(starts[s + 1], begin), q.shape[0])
        n, total = end - begin, max(total, 0)
        if n == 0:
            continue
        span = min(total, table.shape[1] * page_size)
        entry = table[s, :-(-span // page_size)].long()
        good = (entry >= 0) & (entry < pages)
        entry = torch.where(good, entry, torch.zeros_like(entry)).to(q.device)
        exists = good.to(q.device).repeat_interleave(page_size)[:span]
        t = torch.arange(span, device=q.device)
        limit = total - n + 1 + torch.arange(n, device=q.device) if causal else torch.full((n,), total, device=q.device)
        visible = (t < limit[:, None]) & exists
        for h in range(kv_heads):
            k = (kc[entry, h].double() * ks[entry, h].double()[..., None]).reshape(-1, d)[:span]
            v = (vc[entry, h].double() * vs[entry, h].double()[..., None]).reshape(-1, d)[:span]
            for j in range(h * group, (h + 1) * group):
                out[begin:end, j], bound[begin:end, j] = ref.attend_rows(q[begin:end, j].double(), k, v, visible, scale,
                                                                         dtype, step)
    return out, bound


# ---- the plan ---------------------------------------------------------------------------


def plan(held, added, table, ring, state, tokens, page_size):
    """cache_plan one sequence after the other, on lists: every output, and the new table and ring."""
    pages, most = len(ring), len(table[0])
    table, ring = [list(r) for r in table], list(ring)
    first, count = min(max(state[0], 0), pages - 1), min(max(state[1], 0), pages)
    out = {"held_out": [], "lengths": [], "starts": [0], "positions": [], "owners": [], "slots": []}
    rows = asked = taken = 0
    back = []
    for s, (h, a) in enumerate(zip(held, added)):
        h = max(h, 0)
        n = max(a, 0)
        rows += n
        owned = -(-h // page_size)
        length = 0
        if a >= 0 and h + n <= most * page_size and rows <= tokens:
            need = -(-(h + n) // page_size) - owned
            asked += need
            if need == 0 or asked <= count:
                length = h + n
                for i in range(need):
                    table[s][owned + i] = ring[(first + taken + i) % pages]
                taken += need
                served = True
            else:
                served = False
        else:
            served = False
        if a < 0:
            back += table[s][:min(owned, most)]
        out["held_out"].append(0 if a < 0 else length if served else h)
        out["lengths"].append(length)
        for i in range(n):
            if len(out["positions"]) == tokens:
                break
            p = h + i
            page = table[s][p // page_size] if served else -1
            out["positions"].append(p)
            out["owners"].append(s)
            out["slots"].append(page * page_size + p % page_size if 0 <= page < pages else -1)
        out["starts"].append(min(rows, tokens))
    back = back[:pages - count]
    for i, page in enumerate(back):
        ring[(first + count + i) % pages] = page
    spare = tokens - len(out["positions"])
    out["positions"] += [0] * spare
    out["owners"] += [-1] * spare
    out["slots"] += [-1] * spare
    out.update(table=table, ring=ring, state_out=[(first + taken) % pages, count - taken + len(back)])
    return out


# ---- the norm ------------------------------------------------------------------------------


def add_rms_norm(x, residual, weight, epsilon):
    """On the CPU: the sum in x's type, y in fp32, scales and codes. Bit for bit what the definition says."""
    x = x.cpu()
    h = x if residual is None else (x.float() + residual.cpu().float()).to(x.dtype)
    f = h.float()
    factor = (1.0 / torch.sqrt(f.double().square().mean(-1, keepdim=True) + np.float32(epsilon).item())).float()
    y = f * factor
    if weight is not None:
        y = y * weight.cpu()
    s = torch.clamp_min((y.abs().amax(-1).double() / 127.0).float(), 1e-8)
    codes = torch.round((y.double() / s.double()[:, None]).float()).clamp(-127, 127)
    return h, y, s, codes.nan_to_num(0.0).to(torch.int8)


# ---- sampling --------------------------------------------------------------------------------


def sample(logits, temperature, top_k, top_p, min_p, uniform):
    """One row in float64 (numpy): the token and its probability. The parameters as numbers."""
    l = np.asarray(logits, dtype=np.float64).copy()
    l[np.isnan(l)] = -np.inf
    order = np.argsort(-l, kind="stable")
    l = l[order]
    top = l[0]
    if top == -np.inf:
        return -1, 0.0
    greedy = not temperature > 0
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        e = np.where(l == top, 1.0, np.exp((l - top) / (1.0 if greedy else float(temperature))))
    e[l == -np.inf] = 0.0
    if top == np.inf:
        e = (l == top).astype(np.float64)
    kept = 1 if greedy else top_k if 0 < top_k < len(l) else len(l)
    e[kept:] = 0.0
    if 0 < min_p <= 1:
        e[e < np.float64(np.float32(min_p))] = 0.0
    if top_p < 1:
        ends = np.cumsum(e)
        before = np.concatenate([[0.0], ends[:-1]])
        last = before < np.float64(np.float32(max(top_p, 0.0))) * ends[-1]
        last[0] = True
        e[~last] = 0.0
    ends = np.cumsum(e)
    u = 0.0 if math.isnan(uniform) else min(max(uniform, 0.0), float(np.nextafter(np.float32(1), np.float32(0))))
    at = min(int(np.searchsorted(ends, u * ends[-1], side="right")), int(np.nonzero(e)[0][-1]))
    return int(order[at]), float(e[at] / ends[-1])
