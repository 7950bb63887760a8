"""The decoder operators from their definitions in float64 (torch, on the
tensors' own device), with the bounds that the tests hold the kernels to."""

from __future__ import annotations

import math

import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype: str) -> float:
    return torch.finfo(DTYPES[dtype]).eps / 2


def floor_of(dtype: str) -> float:
    """Half the distance of the smallest numbers of a type."""
    f = torch.finfo(DTYPES[dtype])
    return f.tiny * f.eps / 2


def frequencies(rotary_dim: int, base: float = 10000.0, device="cuda"):
    i = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
    return base ** (-2.0 * i / rotary_dim)


def rotary(x, positions, freq, rotary_dim, layout, amplitude=1.0):
    """x float64 [tokens][heads][head_dim]: the rotated heads, and |a| + |b| of every feature's pair."""
    t = positions.double()[:, None, None] * freq
    cos, sin = torch.cos(t) * amplitude, torch.sin(t) * amplitude
    y, size = x.clone(), x.abs()
    if layout == "halves":
        first, second = slice(0, rotary_dim // 2), slice(rotary_dim // 2, rotary_dim)
    else:
        first, second = slice(0, rotary_dim, 2), slice(1, rotary_dim, 2)
    a, b = x[..., first], x[..., second]
    y[..., first] = a * cos - b * sin
    y[..., second] = b * cos + a * sin
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(amplitude)
    return y, size


def norm(x, weight, kind, epsilon):
    """x float64: the normed heads, and a bound of every intermediate value."""
    c = x - x.mean(-1, keepdim=True) if kind == "layer" else x
    factor = 1.0 / torch.sqrt(c.square().mean(-1, keepdim=True) + epsilon)
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if weight is None else weight.double()
    most = 2.0 * x.abs().amax(-1, keepdim=True) * factor * w.abs().max()
    return c * factor * w, most


def quantized_pages(x):
    """Codes and scales of x [..][a][b] float, one scale for the last two axes."""
    s = torch.clamp_min((x.abs().amax(dim=(-2, -1)).double() / 127.0).float(), 1e-8)
    return torch.round((x.double() / s.double()[..., None, None]).float()).clamp(-127, 127).to(torch.int8), s


def store(keys, values, key_scales, value_scales, new_keys, new_values, table, starts, lengths):
    """cache_store on copies (lists and CPU tensors inside): the new cache.
    keys [pages][heads][page][dim], values [pages][heads][dim][page]."""
    out = [t.clone().cpu() for t in (keys, values, key_scales, value_scales)]
    page_size = keys.shape[2]
    floor = torch.tensor(1e-8, dtype=torch.float32)
    table, starts, lengths = table.cpu().tolist(), starts.cpu().tolist(), lengths.cpu().tolist()
    news = [new_keys.float().cpu(), new_values.float().cpu()]
    tokens = news[0].shape[0]
    for s, total in enumerate(lengths):
        begin = min(max(starts[s], 0), tokens)
        end = min(max(starts[s + 1], begin), tokens)
        total = max(total, 0)
        where = {}  # page -> (slots, rows)
        for r in range(begin, end):
            pos = total - (end - begin) + (r - begin)
            if pos < 0 or pos >= len(table[s]) * page_size:
                continue
            page = table[s][pos // page_size]
            if 0 <= page < keys.shape[0]:
                slots, rows = where.setdefault(page, ([], []))
                slots.append(pos % page_size)
                rows.append(r)
        for page, (slots, rows) in where.items():
            for side in range(2):
                codes = out[side][page] if side == 0 else out[side][page].transpose(1, 2)  # [heads][page][dim]
                x = news[side][rows].transpose(0, 1)  # [heads][n][dim]
                old = out[2 + side][page].clone()
                now = torch.maximum((x.abs().amax(dim=(1, 2)).double() / 127).float(), floor)
                if slots[0] > 0:
                    now = torch.maximum(now, old)
                    held = (codes[:, :slots[0]].double() * old.double()[:, None, None]).float()
                    again = torch.round((held.double() / now.double()[:, None, None]).float())
                    codes[:, :slots[0]] = again.to(torch.int8)
                codes[:, slots] = torch.round((x.double() / now.double()[:, None, None]).float()).to(torch.int8)
                out[2 + side][page] = now
    return out


def attend_rows(q, k, v, visible, scale, dtype, weight_step):
    """One head in float64: q [n][d], k and v [t][d], visible bool [n][t].
    The result and how far a kernel may be off.

    Scores are fp32 sums of d products (at most d + 4 roundings of at most
    sum |q k|) and the argument of the exponential is rounded once more; that
    changes a weight by a factor of at most 1 + 2 ds. A weight is rounded by
    weight_step, or by 2^-25 of the largest one; their sums with the values
    and the division are fp32: n + d roundings would bound them, of which
    blocks of 32 and more are summed apart, so 64 + n / 16 are counted."""
    if k.shape[0] == 0:
        z = torch.zeros_like(q)
        return z, z + floor_of(dtype)
    k = torch.where(visible.any(0)[:, None], k, torch.zeros_like(k))
    v = torch.where(visible.any(0)[:, None], v, torch.zeros_like(v))
    s = (q @ k.T) * scale
    ds = (q.abs() @ k.abs().T) * abs(scale) * (q.shape[1] + 4) * U + s.abs() * 4 * U
    s = s.masked_fill(~visible, -math.inf)
    most = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(most == -math.inf, torch.zeros_like(most), most))
    total = p.sum(-1, keepdim=True)
    total = torch.where(total == 0, torch.ones_like(total), total)
    p = p / total
    o, size = p @ v, p @ v.abs()
    ds = torch.where(visible, ds, torch.zeros_like(ds)).amax(-1, keepdim=True)
    n = k.shape[0]
    bound = size * (weight_step + 2 * ds + (64 + n / 16) * U) + o.abs() * half_step(dtype) + floor_of(dtype)
    return o, bound + n * 2.0 ** -25 * v.abs().max() / total


def attend(q, cache, table, starts, lengths, causal, scale, dtype):
    """Float64 attention over a cache: q [tokens][heads][d]. Rows of no sequence are NaN."""
    keys, values, ks, vs = cache
    heads, d = q.shape[1], q.shape[2]
    kv_heads, page_size, pages = keys.shape[1], keys.shape[2], keys.shape[0]
    group = heads // kv_heads
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    # weights are binary16, two of them in the fp32 mode
    step = 2.0 ** -21 if dtype == "f32" else 2.0 ** -11
    starts, lengths, table = starts.tolist(), lengths.tolist(), table.cpu()
    for s, total in enumerate(lengths):
        begin = min(max(starts[s], 0), q.shape[0])
        end = min(max(starts[s + 1], begin), q.shape[0])
        n, total = end - begin, max(total, 0)
        if n == 0:
            continue
        span = min(total, table.shape[1] * page_size)
        count = -(-span // page_size)
        entry = table[s, :count].long()
        good = (entry >= 0) & (entry < pages)
        entry = torch.where(good, entry, torch.zeros_like(entry)).to(q.device)
        exists = good.to(q.device).repeat_interleave(page_size)[:span]
        t = torch.arange(span, device=q.device)
        limit = total - n + 1 + torch.arange(n, device=q.device) if causal else torch.full((n,), total, device=q.device)
        visible = (t < limit[:, None]) & exists
        for h in range(heads):
            k = (keys[entry, h // group].double() * ks[entry, h // group].double()[:, None, None]).reshape(-1, d)[:span]
            v = values[entry, h // group].double() * vs[entry, h // group].double()[:, None, None]
            v = v.transpose(1, 2).reshape(-1, d)[:span]
            out[begin:end, h], bound[begin:end, h] = attend_rows(q[begin:end, h].double(), k, v, visible, scale, dtype,
                                                                 step)
    return out, bound


def cross(q, k, v, lengths, mask, scale, dtype):
    """Float64 cross attention: q [batch][n][heads][d], k, v [batch][t][kv_heads][d]."""
    group = q.shape[2] // k.shape[2]
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    # weights are rounded to the tensors' type; the fp32 mode keeps 22 bits of them at least
    step = 2.0 ** -21 if dtype == "f32" else half_step(dtype)
    for b in range(q.shape[0]):
        visible = torch.ones(k.shape[1], dtype=torch.bool, device=q.device)
        if lengths is not None:
            visible &= torch.arange(k.shape[1], device=q.device) < int(lengths[b])
        if mask is not None:
            visible &= mask[b] != 0
        for h in range(q.shape[2]):
            out[b, :, h], bound[b, :, h] = attend_rows(
                q[b, :, h].double(), k[b, :, h // group].double(), v[b, :, h // group].double(),
                visible.expand(q.shape[1], -1), scale, dtype, step)
    return out, bound


def assert_within(got, want, bound, what=""):
    got, want = got.double(), want.double()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    bad = (got - want).abs() > bound
    bad &= ~want.isnan() & (got != want)
    if bad.any():
        i = tuple(int(x) for x in bad.nonzero()[0])
        worst = ((got - want).abs() / bound.clamp_min(1e-300)).nan_to_num(0.0).max()
        raise AssertionError(f"{what}: {int(bad.sum())} values off, first at {i}: {float(got[i])} for "
                             f"{float(want[i])}, bound {float(bound[i])}; worst is {float(worst):.3g} bounds")
