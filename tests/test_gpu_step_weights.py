"""Softmax weights of attention over the 4-bit cache over their whole range: keys
far below the largest, whose sum is what the output holds, value scales of zero,
and scores so large that their rounding is larger than the exponentials' range."""

import math

import pytest

import decoder_ref as ref
import step_ref
from test_gpu_decoder_weights import CACHE_STEPS, mean_of_largest, sink_query, want_of
from test_gpu_step import attend_args, ints, launch, rand

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f16", "bf16"]
# rows and tiles of the kernels, the keys whole and split; the sequences behind the first are empty
WAYS = [(1, 1, 1), (1, 1, 16384), (40, 512, 127), (40, 1, 16384)]


def sink_cache(torch, n, gap, at, page_size, d, seed):
    """A cache of n tokens whose key `at` is ahead of all others by about `gap` for a query whose first feature is 1,
    and has values of zero; the others' scores lie close together and their values are of one sign."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = n // page_size
    keys = torch.randint(-3, 4, (pages, 1, page_size, d), generator=g, dtype=torch.int8, device="cuda")
    values = torch.randint(2, 8, (pages, 1, page_size, d), generator=g, dtype=torch.int8, device="cuda")
    ks = torch.full((pages, 1, page_size), gap / 127.0, device="cuda")
    vs = 0.05 + 0.2 * torch.rand((pages, 1, page_size), generator=g, device="cuda")
    keys[..., 0] = 0
    page, slot = at // page_size, at % page_size
    keys[page, :, slot] = 0
    keys[page, :, slot, 0] = 7
    ks[page, :, slot] = gap / 7.0
    values[page, :, slot] = 0
    return [step_ref.pack(keys), step_ref.pack_values(values), ks, vs], keys, values


def rows_of(x, scales, entry):
    d = x.shape[-1]
    return (x[entry, 0].double() * scales[entry, 0].double()[..., None]).reshape(-1, d)


def attend(torch, pkg, lib, cache, q, table, n, queries, sequences, most, dtype, scale=1.0):
    starts, lengths = ints(torch, [0] + [queries] * sequences), ints(torch, [n] + [0] * (sequences - 1))
    out = torch.full(q.shape, math.nan, dtype=q.dtype, device="cuda")
    a, keep = attend_args(torch, pkg, lib, cache, q, out, table.expand(sequences, -1).contiguous(), starts, lengths, False,
                          dtype, scale, max_length=most)
    launch(torch, lib, "dav2_hip_attention_cache_i4", a)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [12, 16, 18])
@pytest.mark.parametrize("queries,sequences,most", WAYS)
@pytest.mark.parametrize("at", [0, 9000])
def test_dominant_key(gpu, pkg, lib, dtype, gap, queries, sequences, most, at):
    torch = gpu
    n, page_size, d, heads = 16384, 64, 64, 8
    cache, keys, values = sink_cache(torch, n, gap, at, page_size, d, 3)
    q = sink_query(torch, queries, heads, d, dtype, 5)
    table = torch.randperm(n // page_size, device="cuda").to(torch.int32)
    # the sink stays at position `at`
    where = (table == at // page_size).nonzero()[0, 0]
    table[where], table[at // page_size] = table[at // page_size].clone(), at // page_size
    out = attend(torch, pkg, lib, cache, q, table, n, queries, sequences, most, dtype)
    k, v = rows_of(keys, cache[2], table.long()), rows_of(values, cache[3], table.long())
    step, floor = CACHE_STEPS[dtype]
    for h in range(heads):
        want, bound = want_of(q[:, h].double(), k, v, 1.0, dtype, step, floor, exponent=8.0)
        ref.assert_within(out[:, h], want, bound)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries,sequences,most", WAYS)
def test_scales_of_zero(gpu, pkg, lib, dtype, queries, sequences, most):
    # every other token of a long context has values that are zeros by their scale: the sum of the weights stays finite
    torch = gpu
    n, page_size, d, heads = 16384, 64, 64, 8
    cache, keys, values = sink_cache(torch, n, 4, 100, page_size, d, 3)
    cache[3][..., ::2] = 0.0
    cache[3][50:100] = 0.0
    q = sink_query(torch, queries, heads, d, dtype, 5)
    table = torch.arange(256, device="cuda").to(torch.int32)
    out = attend(torch, pkg, lib, cache, q, table, n, queries, sequences, most, dtype)
    k, v = rows_of(keys, cache[2], table.long()), rows_of(values, cache[3], table.long())
    step, floor = CACHE_STEPS[dtype]
    for h in range(heads):
        # a scale of 2^-80, of 1e-23 of the others, stands for zero; its logarithm is rounded to 2^-18
        want, bound = want_of(q[:, h].double(), k, v, 1.0, dtype, step + 2.0 ** -18, floor, exponent=80.0)
        ref.assert_within(out[:, h], want, bound + 8 * 2.0 ** -80)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("queries,sequences,most", [(1, 1, 1), (1, 1, 2 ** 22), (40, 512, 127), (40, 1, 2 ** 22)])
def test_scores_past_2_to_30(gpu, pkg, lib, dtype, sign, queries, sequences, most):
    # scores of one feature, multiples of 2^24 and more: their rounding in fp32 is larger than what an exponential
    # bears; ties, which are exact as the tokens share their scales, are halved
    torch = gpu
    n, page_size, d, heads = 640, 32, 64, 8
    g = torch.Generator(device="cuda").manual_seed(3)
    pages = n // page_size
    keys = torch.zeros((pages, 1, page_size, d), dtype=torch.int8, device="cuda")
    keys[..., 0] = torch.randint(-7, 8, (pages, 1, page_size), generator=g, dtype=torch.int8, device="cuda")
    values = torch.randint(-7, 8, (pages, 1, page_size, d), generator=g, dtype=torch.int8, device="cuda")
    ks, vs = (torch.full((pages, 1, page_size), x, device="cuda") for x in (1.0, 0.25))
    cache = [step_ref.pack(keys), step_ref.pack_values(values), ks, vs]
    q = torch.zeros((queries, heads, d), dtype=ref.DTYPES[dtype], device="cuda")
    q[..., 0] = 1.0
    scale = sign * 2.0 ** 28
    table = torch.arange(pages, device="cuda").to(torch.int32)
    out = attend(torch, pkg, lib, cache, q, table, n, queries, sequences, most, dtype, scale)
    k, v = rows_of(keys, ks, table.long()), rows_of(values, vs, table.long())
    for h in range(heads):
        want = mean_of_largest((q[:, h].double() @ k.T) * scale, v)
        # equal weights: the sums of n products, the quotient, the output's rounding
        bound = v.abs().max() * (64 + n / 32) * ref.U + want.abs() * ref.half_step(dtype) + ref.floor_of(dtype)
        ref.assert_within(out[:, h], want, bound + 0 * want)


@pytest.mark.parametrize("dtype,queries", [("f32", 1), ("f16", 1), ("bf16", 1), ("f32", 32), ("f16", 32), ("f32", 40),
                                           ("f16", 40)])
@pytest.mark.parametrize("sequences,most", [(4, 2 ** 22), (128, 255)])
@pytest.mark.parametrize("length", [40, 68, 1580])
@pytest.mark.parametrize("d", [48, 64, 96, 128])
def test_outputs_round_once(gpu, pkg, lib, dtype, queries, sequences, most, length, d):
    # weights of 20 bits, so that the output's own rounding is what is left: rows and tiles of both heights,
    # the keys whole and split, scales of values far apart
    torch = gpu
    page_size, heads, kv = 32, 16, 2
    pages = -(-length // page_size)
    g = torch.Generator(device="cuda").manual_seed(length + d)
    keys, values = (torch.randint(-8, 8, (pages, kv, page_size, d), generator=g, dtype=torch.int8, device="cuda")
                    for _ in range(2))
    ks, vs = (0.02 + 0.2 * torch.rand((pages, kv, page_size), generator=g, device="cuda") for _ in range(2))
    vs *= 2.0 ** -torch.randint(0, 8, vs.shape, generator=g, device="cuda")
    cache = [step_ref.pack(keys), step_ref.pack_values(values), ks, vs]
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    q = rand(torch, 8, queries, heads, d, dtype=dtype)
    out = attend(torch, pkg, lib, cache, q, table, length, queries, sequences, most, dtype, 0.02)
    for h in range(heads):
        k, v = ((c[table.long(), h // 8].double() * s[table.long(), h // 8].double()[..., None]).reshape(-1, d)[:length]
                for c, s in ((keys, ks), (values, vs)))
        # a weight's two parts, 2^-22 of it, and its exponent with a scale's logarithm, 2^-20 at most, which is in
        # the sum of the weights too
        want, bound = want_of(q[:, h].double(), k, v, 0.02, dtype, 2.0 ** -22 + 2.0 ** -20, 2.0 ** -37, exponent=8.0)
        ref.assert_within(out[:, h], want, bound + want.abs() * 2.0 ** -20)
