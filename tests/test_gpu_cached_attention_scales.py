"""Values of any size that a cache can hold: value scales from fp32's smallest
number to far above 1, alone, side by side in a tile, and along the cache.

The tolerance is ``formula``'s with two changes that come from the range.

Weights below fp16's normal range.  A row's weights are held relative to its
largest product of weight and value scale, M, at 2^6 or more, and rounded to
fp16: off by 2^-25 there at most, which in an output is 2^-31 M times the code.
``formula`` has the scales near one another and takes |v| for M |code|.

Scores and log2 of a value scale (150 at most in size) are added in fp32 and
taken apart again for the sum of weights: 2^-23 (150 + |s| log2 e) in the
exponent each time, at most four times, so a weight is off by the factor
2^(that) - 1.
"""
import math

import pytest
import torch

from gsq_b200.runtime import QuantizedKVCache
from gsq_b200.runtime.kernels import cached_attention, kv_append, kv_read
from test_gpu_cached_attention import DEV, check, filled, formula, i32, queries, visible

pytestmark = pytest.mark.gpu


def wide_formula(q, cache, see, gate=None):
    """(out, bound): ``formula`` with the bounds that hold for any value scales."""
    want, bound = formula(q, cache, see, gate)
    b, n, heads, d = q.shape
    g = heads // cache.heads
    for i in range(b):
        for h in range(cache.heads):
            any_row = see[i].any(0)
            clean = lambda t: torch.where(any_row.view(-1, *[1] * (t.dim() - 1)), t, torch.zeros_like(t))  # noqa: E731
            ks, vs = clean(cache.k_scale[i, h].double()), clean(cache.v_scale[i, h].double())
            kc, vc = clean(cache.k[i, h].double()), clean(cache.v[i, h].double())
            s = torch.einsum("ngd,ld->ngl", q[i, :, h * g:(h + 1) * g].double(), kc * ks[:, None]) / math.sqrt(d)
            s = s.masked_fill(~see[i][:, None, :], -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0)
            m = (p * vs).amax(-1, keepdim=True)
            small = 2.0 ** -31 * m * torch.einsum("nl,ld->nd", see[i].double(), vc.abs())[:, None, :]
            top = s.masked_fill(~see[i][:, None, :], 0).abs().amax(-1, keepdim=True)
            apart = torch.expm1(4 * math.log(2) * 2.0 ** -23 * (150 + 1.45 * top))
            more = small + apart * torch.einsum("ngl,ld->ngd", p, (vc * vs[:, None]).abs())
            if gate is not None:
                more = more * torch.sigmoid(gate[i, :, h * g:(h + 1) * g].double())
            bound[i, :, h * g:(h + 1) * g] += more
    return want, bound


# few rows: clusters, tiles split evenly; units of 16 rows; row blocks whole and in parts
SHAPES = [(1, 6, 400), (2, 5, 9000), (12, 6, 400), (50, 6, 700), (40, 8, 8300)]


def compare(cache, n, group, cap, seed, see=None, gate=None):
    q = queries(1, n, cache.heads * group, cache.dim, torch.bfloat16, seed)
    see = visible(1, n, cap, [cap - n], None, None) if see is None else see
    if gate:
        gate = torch.randn(q.shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)
    want, bound = wide_formula(q, cache, see, gate)
    check(cached_attention(q, cache, i32(cap - n), gate=gate), want, bound)
    return want


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("n,group,cap", SHAPES)
@pytest.mark.parametrize("power", [-140, -130, -126, -115, -105, -70, 70, 110])
def test_all_values_of_one_size(n, group, cap, power, fmt):
    cache = filled(1, 1, cap, 128, fmt, 61)
    cache.v_scale.copy_(torch.exp2(power + torch.rand(cache.v_scale.shape, device=DEV,
                                                      generator=torch.Generator(device=DEV).manual_seed(62))))
    want = compare(cache, n, group, cap, 63, gate=None)
    assert power < -120 or float(want.abs().amax()) > 2.0 ** power  # the outputs do not vanish in the bound


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("n,group,cap", SHAPES)
@pytest.mark.parametrize("low,high", [(-148, 0), (0, -148), (-100, 118), (118, -100), (-60, 20), (20, -60), (-146, 60),
                                      (50, 110)])
def test_sizes_along_the_cache(n, group, cap, low, high, dim):
    """Rising: a row's last positions decide; falling: its first. The sum of weights has all of them alike."""
    cache = filled(1, 2, cap, dim, "int8", 64)
    cache.v_scale.copy_(torch.exp2(torch.linspace(low, high, cap, device=DEV)).expand_as(cache.v_scale))
    cache.v_scale[0, 0, 5::37] = 0
    compare(cache, n, group, cap, 65, gate=True)


@pytest.mark.parametrize("n,group,cap", SHAPES)
@pytest.mark.parametrize("power", [-130, -60, 0, 90])
@pytest.mark.parametrize("share", [2, 1])
def test_scales_of_zero_over_any_codes(n, group, cap, power, share):
    """Every other vector's scale is 0, or all are: zero vectors, whatever their codes are."""
    cache = filled(1, 1, cap, 128, "int8", 76)
    cache.v_scale.fill_(2.0 ** power)
    cache.v_scale[..., ::share] = 0
    want = compare(cache, n, group, cap, 77)
    assert share == 2 or not want.any()


@pytest.mark.parametrize("n,group,cap", SHAPES)
@pytest.mark.parametrize("every", [2, 64, 96, 300])
def test_small_and_large_side_by_side(n, group, cap, every):
    """All but every so many of a cache's vectors 2^-90 as large, in a tile and in tiles of their own."""
    cache = filled(1, 1, cap, 128, "fp8", 66)
    at = torch.arange(cap, device=DEV)
    small = (at % every != 0) if every <= 2 else (at // (every // 2)) % 2 == 0
    cache.v_scale[..., small] *= 2.0 ** -90
    compare(cache, n, group, cap, 67)


@pytest.mark.parametrize("n,group,cap", SHAPES)
@pytest.mark.parametrize("low,high", [(-130, 60), (-10, 60), (50, 115), (56, 100)])
def test_any_size_anywhere(n, group, cap, low, high):
    cache = filled(1, 1, cap, 128, "fp8", 78)
    g = torch.Generator(device=DEV).manual_seed(79)
    cache.v_scale.copy_(torch.exp2(low + (high - low) * torch.rand(cache.v_scale.shape, generator=g, device=DEV)))
    compare(cache, n, group, cap, 80)


@pytest.mark.parametrize("n,group", [(7, 2), (60, 6)])
def test_rows_that_see_only_the_small_ones(n, group):
    """A tree's tokens with values of their own size each, and a first token before the larger text: rows of one block
    with outputs from 2^-120 to 1."""
    cap = 64 + n
    cache = filled(1, 1, cap, 128, "int8", 68)
    cache.v_scale[..., :64] *= 2.0 ** -120
    cache.v_scale[..., 64:] = torch.exp2(torch.linspace(-110, 0, n, device=DEV))
    words = torch.zeros(n, (n + 31) // 32, dtype=torch.int64)
    see = torch.zeros(1, n, cap, dtype=torch.bool, device=DEV)
    see[..., :64] = True
    for i in range(n):  # each sees itself alone, after the text
        words[i, i // 32] |= 1 << i % 32
        see[0, i, 64 + i] = True
    tree = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32).to(DEV)
    q = queries(1, n, group, 128, torch.bfloat16, 69)
    want, bound = wide_formula(q, cache, see)
    check(cached_attention(q, cache, i32(64), tree=tree), want, bound)


@pytest.mark.parametrize("n,group,cap", SHAPES)
def test_a_large_or_lost_vector_that_a_row_does_not_see(n, group, cap):
    """A vector of NaN and one of 2^100 at the last position, among small ones: the rows before are as without them."""
    if n == 1:
        cap += 1  # the row does not see the last position
    cache = filled(1, 1, cap, 128, "int8", 70)
    cache.v_scale.fill_(2.0 ** -105)
    q = queries(1, n, group, 128, torch.bfloat16, 71)
    start = cap - max(n, 2)
    see = visible(1, n, cap, [start], None, None)
    want, bound = wide_formula(q, cache, see)
    seen = ~see[0, :, -1]
    for scale in (2.0 ** 100, float("nan")):
        cache.v_scale[..., -1] = scale
        got = cached_attention(q, cache, i32(start))[:, seen]
        assert ((got.double() - want[:, seen]).abs() <= bound[:, seen]).all()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("n,group", [(1, 6), (60, 6)])
def test_tiny_vectors_from_the_inputs_on(n, group, fmt):
    """Written, read back and attended to: bf16 vectors of 2^-112."""
    cap, dim = 200, 256
    cache = QuantizedKVCache.empty(1, 1, cap, dim, fmt, DEV)
    g = torch.Generator(device=DEV).manual_seed(72)
    k, v = (torch.randn(1, cap, 1, dim, generator=g, device=DEV) for _ in range(2))
    kv_append(cache, k.bfloat16(), (v * 2.0 ** -112).bfloat16(), i32(0))
    read = kv_read(cache, i32(0), cap, dtype=torch.float32)[1]
    assert float((read * 2.0 ** 112 - v).norm() / v.norm()) < 0.05  # the codes hold them
    compare(cache, n, group, cap, 73)


@pytest.mark.parametrize("n,group,cap", SHAPES)
@pytest.mark.parametrize("power", [-130, -60, 10, 50])
@pytest.mark.parametrize("big", [2.0 ** 24, 1e30])
def test_scores_so_large_that_a_scale_is_lost_beside_them(n, group, cap, power, big):
    """Rows whose scores reach 2^30 and more: fp32 has no place for log2 of a scale beside them. Such a row attends to the
    position of its largest score, whose products may differ from fp64's in the last places of fp32, so only the size of its
    output is asked for: that of a stored vector. The other rows are held to the bound. (Scales above 2^57 beside such scores
    are outside of what the entry point promises.)"""
    cache = filled(1, 1, cap, 128, "int8", 74)
    cache.v_scale.fill_(2.0 ** power)
    q = queries(1, n, group, 128, torch.bfloat16, 75)
    rows = q.view(-1, 128)
    large = torch.zeros(n * group, dtype=torch.bool, device=DEV)
    large[2::7] = True
    rows[large] *= big
    want, bound = wide_formula(q, cache, visible(1, n, cap, [cap - n], None, None))
    got = cached_attention(q, cache, i32(cap - n))
    assert torch.isfinite(got.float()).all()
    got, want, bound = (t.view(-1, 128).double() for t in (got, want, bound))
    assert ((got - want).abs() <= bound)[~large].all()
    top = got[large].abs().amax(-1) * 2.0 ** -power
    # codes of a vector reach 127; a mean of vectors of equal score has codes of order 10 at least
    assert (top <= 127 * 1.01).all() and (top >= 5).all()


@pytest.mark.parametrize("n,group,cap", SHAPES)
def test_a_zero_vector_beside_a_large_one_that_a_row_does_not_see(n, group, cap):
    if n == 1:
        cap += 1
    cache = filled(1, 1, cap, 128, "int8", 81)
    cache.v_scale.fill_(2.0 ** -10)
    cache.v_scale[..., -3] = 0
    cache.v_scale[..., -1] = 2.0 ** 30
    q = queries(1, n, group, 128, torch.bfloat16, 82)
    start = cap - max(n, 2)
    want, bound = wide_formula(q, cache, visible(1, n, cap, [start], None, None))
    check(cached_attention(q, cache, i32(start)), want, bound)
