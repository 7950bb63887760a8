"""Softmax weights of the decoder's attention over their whole range: keys far
below the largest, whose sum is what the output holds, and scores so large that
their rounding is larger than the exponentials' range. Against float64, with
bounds that leave a small weight no more than its own rounding."""

import math

import pytest

import decoder_ref as ref
from test_gpu_decoder import attend_args, cross_args, ints, launch, rand

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f16", "bf16"]


def want_of(q, k, v, scale, dtype, step, floor, exponent=0.0):
    """softmax(scale q k^T) v of float64 rows, and how far a kernel may be off.

    A score is an fp32 sum of d products (d + 4 roundings of at most sum |q k|;
    the kernels' other factors are exact or counted there), changed to units of
    log2 and rounded beside the exponent of a value scale (`exponent` at most).
    A weight is rounded by `step` of itself, or by `floor` of the largest one.
    Sums over n keys are of blocks of 32 and more, one after the other: 64 +
    n / 32 roundings."""
    s = (q @ k.T) * scale
    ds = (q.abs() @ k.abs().T) * abs(scale) * (q.shape[1] + 4) * ref.U + (s.abs() + exponent) * 4 * ref.U
    p = torch_exp(s)
    total = p.sum(-1, keepdim=True)
    n = k.shape[0]
    off = (p * (step + 2 * ds + (64 + n / 32) * ref.U) + floor) @ v.abs()
    # the sum of the weights is of unrounded ones
    want = (p @ v) / total
    off = off / total + want.abs() * ((p * 2 * ds).sum(-1, keepdim=True) / total + (64 + n / 32) * ref.U)
    return want, off + want.abs() * ref.half_step(dtype) + ref.floor_of(dtype)


def torch_exp(s):
    return (s - s.amax(-1, keepdim=True)).exp()


def sink_cache(torch, n, gap, at, page_size, kv, d, seed):
    """A cache of n tokens whose key `at` is ahead of all others by about `gap` for a query whose first feature is 1,
    and has values of zero; the others' scores lie close together and their values are of one sign."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = n // page_size
    keys = torch.randint(-3, 4, (pages, kv, page_size, d), generator=g, dtype=torch.int8, device="cuda")
    values = torch.randint(40, 128, (pages, kv, d, page_size), generator=g, dtype=torch.int8, device="cuda")
    keys[..., 0] = 0
    keys[at // page_size, :, at % page_size] = 0
    keys[at // page_size, :, at % page_size, 0] = 127
    values[at // page_size, :, :, at % page_size] = 0
    ks = torch.full((pages, kv), gap / 127.0, device="cuda")
    vs = 0.005 + 0.02 * torch.rand((pages, kv), generator=g, device="cuda")
    return [keys, values, ks, vs]


def sink_query(torch, tokens, heads, d, dtype, seed):
    q = rand(torch, seed, tokens, heads, d, dtype=dtype, scale=0.2)
    q[..., 0] = 1.0
    return q


# half a step of a weight, and what a small one may lose, of the largest
CACHE_STEPS = {"f32": (2.0 ** -22, 2.0 ** -47), "f16": (2.0 ** -11 + 2.0 ** -19, 2.0 ** -37),
               "bf16": (2.0 ** -11 + 2.0 ** -19, 2.0 ** -37)}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [12, 16, 18])
@pytest.mark.parametrize("queries,sequences,most", [(1, 1, 1), (1, 1, 16384), (40, 512, 127), (40, 1, 16384)])
@pytest.mark.parametrize("at", [0, 9000])
def test_cache_attention_dominant_key(gpu, pkg, lib, dtype, gap, queries, sequences, most, at):
    # rows and tiles of the cache kernels, the keys whole and split; the sequences behind the first are empty
    torch = gpu
    n, page_size, kv, d, heads = 16384, 64, 1, 64, 8
    cache = sink_cache(torch, n, gap, at, page_size, kv, d, 3)
    q = sink_query(torch, queries, heads, d, dtype, 5)
    table = torch.randperm(n // page_size, device="cuda").to(torch.int32)
    table = table.expand(sequences, -1).contiguous()
    # the sink stays at position `at`
    where = (table[0] == at // page_size).nonzero()[0, 0]
    table[:, where], table[:, at // page_size] = table[:, at // page_size].clone(), at // page_size
    starts, lengths = ints(torch, [0] + [queries] * sequences), ints(torch, [n] + [0] * (sequences - 1))
    out = torch.full(q.shape, math.nan, dtype=q.dtype, device="cuda")
    a, keep = attend_args(torch, pkg, lib, cache, q, out, table, starts, lengths, False, dtype, 1.0, max_length=most)
    launch(torch, lib, "dav2_hip_attention_cache_i8", a)
    entry = table[0].long()
    k = (cache[0][entry, 0].double() * cache[2][entry, 0].double()[:, None, None]).reshape(n, d)
    v = (cache[1][entry, 0].double() * cache[3][entry, 0].double()[:, None, None]).transpose(1, 2).reshape(n, d)
    torch.cuda.synchronize()
    step, floor = CACHE_STEPS[dtype]
    for h in range(heads):
        want, bound = want_of(q[:, h].double(), k, v, 1.0, dtype, step, floor, exponent=8.0)
        ref.assert_within(out[:, h], want, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries,sequences,most", [(1, 1, 1), (1, 1, 16384), (40, 512, 127), (40, 1, 16384)])
def test_cache_attention_pages_with_a_scale_of_zero(gpu, pkg, lib, dtype, queries, sequences, most):
    # half of a long context in pages whose values are zeros by their scale: the sum of the weights stays finite
    torch = gpu
    n, page_size, d, heads = 16384, 64, 64, 8
    cache = sink_cache(torch, n, 4, 100, page_size, 1, d, 3)
    cache[3][:128] = 0.0
    q = sink_query(torch, queries, heads, d, dtype, 5)
    starts, lengths = ints(torch, [0] + [queries] * sequences), ints(torch, [n] + [0] * (sequences - 1))
    for table in (torch.arange(256, device="cuda"), torch.arange(256, device="cuda").flip(0)):
        table = table.to(torch.int32).expand(sequences, -1).contiguous()
        out = torch.full(q.shape, math.nan, dtype=q.dtype, device="cuda")
        a, keep = attend_args(torch, pkg, lib, cache, q, out, table, starts, lengths, False, dtype, 1.0, max_length=most)
        launch(torch, lib, "dav2_hip_attention_cache_i8", a)
        k = (cache[0][:, 0].double() * cache[2][:, 0].double()[:, None, None]).reshape(n, d)
        v = (cache[1][:, 0].double() * cache[3][:, 0].double()[:, None, None]).transpose(1, 2).reshape(n, d)
        torch.cuda.synchronize()
        step, floor = CACHE_STEPS[dtype]
        for h in range(heads):
            # a scale of 2^-80, of 1e-24 of the others, stands for zero; its logarithm is rounded to 2^-18
            want, bound = want_of(q[:, h].double(), k, v, 1.0, dtype, step + 2.0 ** -18, floor, exponent=80.0)
            ref.assert_within(out[:, h], want, bound + 127 * 2.0 ** -80)


def mean_of_largest(s, v):
    """The values of the keys with the largest score, in equal parts: what is left where scores lie 10^3 and more apart."""
    most = (s == s.amax(-1, keepdim=True)).double()
    return (most / most.sum(-1, keepdim=True)) @ v


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("queries,sequences,most", [(1, 1, 1), (1, 1, 2 ** 22), (40, 512, 127), (40, 1, 2 ** 22)])
def test_cache_attention_scores_past_2_to_30(gpu, pkg, lib, dtype, sign, queries, sequences, most):
    # scores of one feature, multiples of 2^24 and more: their rounding in fp32 is larger than what an exponential
    # bears; ties, which are exact as the pages share a scale, are halved
    torch = gpu
    n, page_size, d, heads = 640, 32, 64, 8
    g = torch.Generator(device="cuda").manual_seed(3)
    pages = n // page_size
    keys = torch.zeros((pages, 1, page_size, d), dtype=torch.int8, device="cuda")
    keys[..., 0] = sign * torch.randint(2, 127, (pages, 1, page_size), generator=g, device="cuda").to(torch.int8)
    same = torch.tensor([3, 70, 300, 639], device="cuda")
    keys.view(n, d)[same, 0] = 127 if sign > 0 else -1  # the largest, several times
    values = torch.randint(-127, 128, (pages, 1, d, page_size), generator=g, dtype=torch.int8, device="cuda")
    ks = torch.full((pages, 1), 0.7310585786 * 2.0 ** 12, device="cuda")
    vs = torch.full((pages, 1), 0.0123, device="cuda")
    q = torch.zeros((queries, heads, d), dtype=ref.DTYPES[dtype], device="cuda")
    q[..., 0] = (2.0 ** 15 - 2.0 ** 7 * torch.arange(heads, device="cuda")).to(q.dtype)
    table = torch.arange(pages, device="cuda", dtype=torch.int32).expand(sequences, -1).contiguous()
    starts, lengths = ints(torch, [0] + [queries] * sequences), ints(torch, [n] + [0] * (sequences - 1))
    out = torch.full(q.shape, math.nan, dtype=q.dtype, device="cuda")
    a, keep = attend_args(torch, pkg, lib, [keys, values, ks, vs], q, out, table, starts, lengths, False, dtype, 1.0,
                          max_length=most)
    launch(torch, lib, "dav2_hip_attention_cache_i8", a)
    k, v = keys.view(n, d).double(), values.transpose(2, 3).reshape(n, d).double() * vs[0].double()
    torch.cuda.synchronize()
    for h in range(heads):
        want = mean_of_largest(q[:, h].double() @ k.T, v)
        bound = want.abs() * (ref.half_step(dtype) + 2.0 ** -10) + v.abs().max() * 2.0 ** -20
        ref.assert_within(out[:, h], want, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [12, 16, 18])
@pytest.mark.parametrize("batch,queries,kv", [(1, 1, 1), (1, 70, 1), (256, 70, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_cross_attention_dominant_key(gpu, pkg, lib, dtype, gap, batch, queries, kv, d):
    # one batch's keys for all: 512 planes are not split
    torch = gpu
    n, heads, at = 16384, 2, 5000
    q = sink_query(torch, batch * queries, heads, d, dtype, 5).view(batch, queries, heads, d)
    k = rand(torch, 6, 1, n, kv, d, dtype=dtype, scale=0.2)
    k[..., 0] = 0
    k[:, at] = 0
    k[:, at, :, 0] = gap
    v = rand(torch, 7, 1, n, kv, d, dtype=dtype).abs() + 0.5
    v[:, at] = 0
    out = torch.full(q.shape, math.nan, dtype=q.dtype, device="cuda")
    a, keep = cross_args(torch, pkg, lib, q, k.expand(batch, -1, -1, -1), v.expand(batch, -1, -1, -1), out, None, None,
                         dtype, 1.0)
    launch(torch, lib, "dav2_hip_cross_attention", a)
    torch.cuda.synchronize()
    step, floor = {"f32": (2.0 ** -24, 0.0), "f16": (2.0 ** -11, 2.0 ** -37), "bf16": (2.0 ** -8, 0.0)}[dtype]
    for b in (0, batch - 1):
        for h in range(heads):
            head = h * kv // heads
            want, bound = want_of(q[b, :, h].double(), k[0, :, head].double(), v[0, :, head].double(), 1.0, dtype, step,
                                  floor)
            ref.assert_within(out[b, :, h], want, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("batch,queries,masked", [(1, 1, False), (3, 70, False), (64, 70, False), (2, 300, True)])
@pytest.mark.parametrize("d", [64, 128])
def test_cross_attention_scores_past_2_to_30(gpu, pkg, lib, dtype, sign, batch, queries, masked, d):
    # as over the cache: multiples of 2^30
    torch = gpu
    n, heads = 700, 8
    g = torch.Generator(device="cuda").manual_seed(3)
    k = torch.zeros((batch, n, heads, d), device="cuda")
    k[..., 0] = sign * torch.randint(2, 127, (batch, n, heads), generator=g, device="cuda") * 2.0 ** 15 / 128
    same = torch.tensor([3, 70, 300, 699], device="cuda")
    k[:, same, :, 0] = (127 if sign > 0 else -1) * 2.0 ** 15 / 128  # the largest, several times
    k = k.to(ref.DTYPES[dtype])
    k[..., 1:4] = k[..., :1]
    v = rand(torch, 7, batch, n, heads, d, dtype=dtype)
    q = torch.zeros((batch, queries, heads, d), dtype=k.dtype, device="cuda")
    q[..., :4] = (2.0 ** 15 - 2.0 ** 8 * torch.arange(heads, device="cuda"))[:, None].to(k.dtype)
    mask = torch.ones((batch, n), dtype=torch.uint8, device="cuda") if masked else None
    if masked:
        mask[:, 70] = mask[:, 300:400] = 0
    out = torch.full(q.shape, math.nan, dtype=q.dtype, device="cuda")
    a, keep = cross_args(torch, pkg, lib, q, k, v, out, None, mask, dtype, 1.0)
    launch(torch, lib, "dav2_hip_cross_attention", a)
    torch.cuda.synchronize()
    for b in range(batch):
        for h in range(heads):
            s = q[b, :, h].double() @ k[b, :, h].double().T
            if masked:
                s = s.masked_fill(mask[b] == 0, -math.inf)
            want = mean_of_largest(s, v[b, :, h].double())
            bound = want.abs() * (ref.half_step(dtype) + 2.0 ** -8) + v[b, :, h].abs().max().double() * 2.0 ** -20
            ref.assert_within(out[b, :, h], want, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length", [1, 2, 9, 68, 1580])
@pytest.mark.parametrize("d", [64, 128])
def test_cache_attention_of_single_tokens_rounds_once(gpu, pkg, lib, dtype, length, d):
    # few rows: weights of 22 bits and more for every type, so that the output's own rounding is what is left
    torch = gpu
    page_size, heads = 32, 16
    pages = -(-length // page_size)
    g = torch.Generator(device="cuda").manual_seed(length + d)
    keys = torch.randint(-127, 128, (pages, 2, page_size, d), generator=g, dtype=torch.int8, device="cuda")
    values = torch.randint(-127, 128, (pages, 2, d, page_size), generator=g, dtype=torch.int8, device="cuda")
    ks, vs = (0.005 + 0.02 * torch.rand((pages, 2), generator=g, device="cuda") for _ in range(2))
    table = torch.arange(pages, device="cuda", dtype=torch.int32)[None]
    q = rand(torch, 8, 2, heads, d, dtype=dtype)
    out = torch.full_like(q, math.nan)
    a, keep = attend_args(torch, pkg, lib, [keys, values, ks, vs], q, out, table, ints(torch, [0, 2]),
                          ints(torch, [length]), False, dtype, 0.125)
    launch(torch, lib, "dav2_hip_attention_cache_i8", a)
    torch.cuda.synchronize()
    for h in range(heads):
        k = (keys[:, h // 8].double() * ks[:, h // 8].double()[:, None, None]).reshape(-1, d)[:length]
        v = (values[:, h // 8].double() * vs[:, h // 8].double()[:, None, None]).transpose(1, 2).reshape(-1, d)[:length]
        want, bound = want_of(q[:, h].double(), k, v, 0.125, dtype, 2.0 ** -22, 2.0 ** -47, exponent=8.0)
        ref.assert_within(out[:, h], want, bound)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("queries", [1, 70])
def test_cross_attention_scale_of_zero(gpu, pkg, lib, dtype, queries):
    # the mean of the values, however large the products are; what is not finite stays so
    torch = gpu
    q, k, v = (rand(torch, i, 2, n, 2, 64, dtype=dtype) for i, n in ((1, queries), (2, 333), (3, 333)))
    q, k = q * 1e18, k * 1e18
    q[1, 0, 1, 5] = math.nan
    out = torch.zeros_like(q)
    a, keep = cross_args(torch, pkg, lib, q, k, v, out, None, None, dtype, 0.0)
    launch(torch, lib, "dav2_hip_cross_attention", a)
    torch.cuda.synchronize()
    want = v.double().mean(1, keepdim=True).expand(q.shape).clone()
    want[1, 0, 1] = math.nan
    size = v.double().abs().mean(1, keepdim=True)
    # weights of one are exact; sums of 333 values in fp32
    ref.assert_within(out, want, size * 333 * ref.U + want.abs() * ref.half_step(dtype))
