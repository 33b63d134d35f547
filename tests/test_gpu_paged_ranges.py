"""The paged attention at the ends of its numeric ranges, on a B200: weights far
below the largest, large scores, maxima that keep growing, against the definition
in 64 bits."""
import importlib
import math

import pytest
import torch

from test_gpu_paged import BF16, DEV, F16, F32, Step, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    return importlib.import_module("index-tts-25-metal_b200.paged")


def one_key_ahead(paged, dtype, n, fresh, dim, requests, lead, top, value):
    """Attention over n keys of equal scores but for key `top`, which is `lead` nats ahead and has the value `value`
    where the others have 1.  Returns the output and, per row, what it should be."""
    bs = 128
    blocks = (n + bs - 1) // bs
    k = torch.zeros(blocks * bs, 1, dim, dtype=dtype, device=DEV)
    v = torch.ones_like(k)
    k[top, 0, 0], v[top] = lead, value
    q = torch.zeros(fresh * requests, 1, dim, dtype=dtype, device=DEV)
    q[:, 0, 0] = 1.0
    table = torch.arange(blocks, dtype=torch.int32, device=DEV).expand(requests, blocks).contiguous()
    out = paged.attention(q, k.view(blocks, bs, 1, dim), v.view(blocks, bs, 1, dim), table, ints([n] * requests),
                          ints([fresh * b for b in range(requests + 1)]), fresh, scale=1.0)
    others = torch.arange(n - fresh, n, dtype=torch.float64, device=DEV)  # equal keys that a row sees
    tail = others * math.exp(-float(k[top, 0, 0]))
    return out.double().view(requests, fresh, dim), ((value + tail) / (1 + tail))[None, :, None]


@pytest.mark.parametrize("fresh,dim,requests", [(1, 128, 300), (1, 64, 150), (2, 128, 150), (8, 64, 150), (16, 128, 150),
                                                (300, 128, 160), (129, 64, 160)])
@pytest.mark.parametrize("value", [0.0, 1.0])
def test_attention_fp32_sums_over_many_keys(paged, value, fresh, dim, requests):
    """Items of 2^19 keys in one CTA, one key so far ahead that each other one is below half a step of a sum that holds
    it.  For the sums above and below the line: 2^8 additions of units at a stretch and 2^6 of stretches (2^-16 and
    2^-18), 2^-18 within a unit of up to 64 keys (24 accumulations of the tensor core, not to the nearest, 2^-23 each,
    and less on the CUDA cores); the exponent, up to 2^5 in size, 2^-24 of it from each of two roundings and 2^-22 from
    the exponential itself: 2^-17."""
    n = 2 ** 19 + 77
    for lead in (17.2, 17.35):
        for top in (0, n - fresh):
            got, want = one_key_ahead(paged, F32, n, fresh, dim, requests, lead, top, value)
            tol = want * (2 * (2.0 ** -16 + 2.0 ** -18 + 2.0 ** -18) + 2.0 ** -17 + 2.0 ** -24)
            assert bool(((got - want).abs() <= tol).all()), float((got / want - 1).abs().max())


# Weights: half a step of the type where the products take them rounded, and of fp16, whose steps end, half of the
# last (2^-25 of the largest weight's 2^11) for every key.  Half a step for the output.  Sums over at most 2^14 keys at
# a stretch: 2^-13 and 2^-18 (see test_attention_long_sums).  The exponent, up to 2^5 in size: 2^-24 of it from each
# of two roundings, and 2^-22 from the exponential itself: 2^-17 in all.
def allowed(dtype, n, want):
    last = n * 2.0 ** -36 if dtype is F16 else 0.0
    return want * (torch.finfo(dtype).eps + 2.0 ** -13 + 2.0 ** -18 + 2.0 ** -17) + last


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("fresh,dim,requests", [(1, 128, 1), (1, 64, 150), (8, 128, 300), (300, 128, 2), (300, 64, 160)])
@pytest.mark.parametrize("n", [131089, 2 ** 19 + 77])
def test_attention_small_weights_stay_in_the_mean(paged, n, fresh, dim, requests, dtype):
    """Values that are all 1 have the mean 1, however far one key's score is ahead."""
    for lead in (17.2, 17.35):
        for top in (0, n - fresh):
            got, want = one_key_ahead(paged, dtype, n, fresh, dim, requests, lead, top, 1.0)
            assert float((got - want).abs().max()) <= float(allowed(dtype, n, want).max())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("fresh,dim", [(1, 64), (1, 128), (16, 128), (40, 64), (300, 128)])
@pytest.mark.parametrize("lead", [12, 14, 15, 16, 17, 18])
def test_attention_small_weights_beside_a_key_without_value(paged, lead, fresh, dim, dtype):
    """The key that is ahead has a value of 0, so the others' weights are all there is."""
    n = 100_003
    for top in (0, 4321, n - fresh):
        got, want = one_key_ahead(paged, dtype, n, fresh, dim, 1, float(lead), top, 0.0)
        assert bool(((got - want).abs() <= allowed(dtype, n, want)).all()), float((got / want - 1).abs().max())


def check_large_scores(s, out, scale):
    """As Step.check, with the exponents' errors by their size: of |s| log2(e), three roundings of the scale's product
    (to both ends of a difference), one each of the maximum and its lift, two of the difference and of a rescaling:
    12 2^-24 |s| of a weight, and that above and below the line.  fp16 weights end as in allowed()."""
    u, half = 2.0 ** -24, 0.0 if s.dtype is F32 else torch.finfo(s.dtype).eps / 2
    group = s.heads // s.kv
    for b, n in enumerate(s.lens_h):
        rows = slice(s.start[b], s.start[b + 1])
        f = rows.stop - rows.start
        seen = torch.arange(n, device=DEV)[None, :] <= (n - f + torch.arange(f, device=DEV))[:, None]
        for h in range(s.heads):
            q, k, v = s.q[rows, h].double(), s.k[b][:, h // group].double(), s.v[b][:, h // group].double()
            x = (q @ k.T * scale).masked_fill(~seen, -torch.inf)
            p = torch.softmax(x, -1)
            want, a = p @ v, p @ v.abs()
            products = (q.abs() @ k.abs().T * abs(scale)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            largest = x.masked_fill(~seen, 0.0).abs().amax(-1, keepdim=True)
            rel = half + 2 * (s.dim + 2) * u * products + 24 * u * largest + 2 * n * u + 2.0 ** -20
            tol = torch.finfo(s.dtype).eps / 2 * want.abs() + a * rel * 1.01
            if s.dtype is F16:
                tol = tol + n * 2.0 ** -36 * v.abs().max()
            err = (out[rows, h].double() - want).abs()
            assert bool((err <= tol).all()), (b, h, float((err / tol).max()))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("fresh", [1, 4, 8, 33, 200])
@pytest.mark.parametrize("scale,qscale", [(3.0, 4.0), (-3.0, 4.0), (0.5, 30.0)])
def test_attention_scores_of_hundreds(paged, scale, qscale, fresh, dim, dtype):
    s = Step([(fresh, 200), (fresh, 1900)], 4, 2, dim, bs=64, dtype=dtype, qscale=qscale)
    check_large_scores(s, s.run(paged, scale=scale), scale)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("fresh,dim", [(1, 128), (3, 64), (8, 64), (40, 64), (300, 128), (300, 64)])
@pytest.mark.parametrize("step", [1, 3, 4, 5, 7, 8, 9, 15, -4, -9])
def test_attention_maxima_that_grow(paged, step, fresh, dim, dtype):
    """Scores that rise (or fall) by `step` octaves from each 64 keys to the next: below, at and above the growth that
    the tile kernels let pass before they rescale."""
    s = Step([(fresh, 1000)], 4, 2, dim, bs=32, dtype=dtype, qscale=0.3)
    s.q[:, :, 0] = 1.0
    n = s.lens_h[0]
    rise = (step * (torch.arange(n, device=DEV) // 64)).to(dtype)
    s.k[0][:, :, 0] = rise[:, None]
    for j in range((n + 31) // 32):
        s.kc[s.table[0, j].item(), :min(32, n - 32 * j)] = s.k[0][32 * j:min(n, 32 * j + 32)]
    scale = math.log(2.0)
    check_large_scores(s, s.run(paged, scale=scale), scale)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("fresh,dim,requests", [(1, 128, 300), (1, 64, 170), (4, 64, 170), (8, 128, 150), (16, 128, 150),
                                                (40, 64, 149), (130, 128, 150), (300, 64, 80)])
def test_attention_long_items(paged, fresh, dim, requests, dtype):
    """Items whose sums meet several times within a share and across shares: random keys that all requests have in
    common, blocks among them that the table does not name.  Each of the stretches' sums is an fp32 one, and a
    tensor-core sum of up to 2^14 keys is off by 2^-13 of it at most (fp32: 2^-18, a unit of 64 keys)."""
    n, bs, u = 40_077, 64, 2.0 ** -24
    g = torch.Generator(device=DEV).manual_seed(fresh + dim)
    blocks = (n + bs - 1) // bs
    k = torch.randn(blocks * bs, 1, dim, generator=g, device=DEV).to(dtype)
    v = torch.randn(blocks * bs, 1, dim, generator=g, device=DEV).to(dtype)
    q = (torch.randn(fresh * requests, 1, dim, generator=g, device=DEV) * 2).to(dtype)
    row = torch.arange(blocks, dtype=torch.int32, device=DEV)
    row[3], row[300], row[555] = -1, blocks, 1 << 30
    table = row.expand(requests, blocks).contiguous()
    out = paged.attention(q, k.view(blocks, bs, 1, dim), v.view(blocks, bs, 1, dim), table, ints([n] * requests),
                          ints([fresh * b for b in range(requests + 1)]), fresh)
    j = torch.arange(n, device=DEV)
    named = (j // bs != 3) & (j // bs != 300) & (j // bs != 555)
    seen = (j[None, :] <= (n - fresh + torch.arange(fresh, device=DEV))[:, None]) & named
    kd, vd, half = k[:n, 0].double(), v[:n, 0].double(), 0.0 if dtype is F32 else torch.finfo(dtype).eps / 2
    for b in [*range(0, requests, 9), requests - 2, requests - 1]:
        rows = slice(b * fresh, (b + 1) * fresh)
        x = (q[rows, 0].double() @ kd.T * dim ** -0.5).masked_fill(~seen, -torch.inf)
        p = torch.softmax(x, -1)
        want, a = p @ vd, p @ vd.abs()
        size = (q[rows, 0].double().abs() @ kd.abs().T).amax(-1, keepdim=True) * dim ** -0.5
        sums = 2.0 ** -18 if dtype is F32 else 2.0 ** -13
        rel = half + 2 * (dim + 2) * u * size + 2.0 ** -20 + 2 * (sums + 2.0 ** -16 + 2.0 ** -20)
        tol = torch.finfo(dtype).eps / 2 * want.abs() + a * rel * 1.01
        if dtype is F16:
            tol = tol + n * 2.0 ** -36 * vd.abs().max()
        err = (out[rows, 0].double() - want).abs()
        assert bool((err <= tol).all()), (b, float((err / tol).max()))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("group", [16, 17, 64, 100, 127, 128])
def test_attention_wide_groups(paged, group, dtype):
    """Up to 128 query heads a key head: a token fills a tile, or does not divide it."""
    s = Step([(1, 0), (1, 200), (3, 130), (5, -2), (0, 7), (40, 90)], 2 * group, 2, 64, bs=32, dtype=dtype, pad=2)
    s.check(s.run(paged))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("max_fresh", [2, 40])
def test_attention_most_requests(paged, max_fresh, dim, dtype):
    s = Step([(i % 3, i % 7) for i in range(8192)], 1, 1, dim, bs=16, dtype=dtype, pad=1)
    out = s.run(paged, max_fresh=max_fresh)
    want = []
    for b in range(8192):
        f, n = s.fresh[b], s.lens_h[b]
        if f:
            x = s.q[s.start[b]:s.start[b + 1], 0].double() @ s.k[b][:, 0].double().T * dim ** -0.5
            x = x.masked_fill(torch.ones_like(x, dtype=torch.bool).triu(n - f + 1), -torch.inf)
            want.append(torch.softmax(x, -1) @ s.v[b][:, 0].double())
    want, top = torch.cat(want), float(max(v.abs().max() for v in s.v if v.numel()))
    # half a step each for weights and output; scores of up to 2^5: their products' roundings and the exponent, 2^-14
    eps = 0.0 if dtype is F32 else torch.finfo(dtype).eps
    assert float((out[:len(want), 0].double() - want).abs().max()) <= top * (eps + 2.0 ** -14)
    assert bool((out[len(want):] == 5).all())
