"""Attention over the quantised cache (gsq_cached_attention) against the
formula in 64 bits, on the codes and scales as they are stored.

The bound on every output follows from the roundings that are made.  With
weights p = softmax, A = sum p |v| of the row:
  - the output rounds once:                  eps/2 |out|
  - a weight rounds to fp16 before p v:      2^-11 A
  - a score is a D-term fp32 dot, off by at most
    d = (D + 4) 2^-24 scale max_p sum|q||k|; a weight and the weights' sum
    each carry e^d:                          (e^(2d) - 1) A
  - the exponential and the gate (2 ulp each, 2^-21 with the scaling in
    base 2 of scores up to 2^6):             2^-15 |s|max / 64 A, taken as 2^-14 A
  - fp32 sums over L positions:              (L + 64) 2^-24 2 A
  - weights below fp16's normal range are off by 2^-25 of the largest
    weight times 2^-6 or less:               2^-31 sum |v|
"""
import math

import pytest
import torch

from gsq_b200 import _lib
from gsq_b200.runtime import QuantizedKVCache
from gsq_b200.runtime.kernels import cached_attention, kv_append, tree_mask

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def filled(batch, heads, cap, dim, fmt, seed, used=None):
    """A cache of random vectors; past ``used[b]`` positions its bytes are NaN codes (e4m3) under NaN scales."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    cache = QuantizedKVCache.empty(batch, heads, cap, dim, fmt, DEV)
    k = torch.randn(batch, cap, heads, dim, generator=g, device=DEV)
    v = torch.randn(batch, cap, heads, dim, generator=g, device=DEV)
    v *= torch.exp(torch.randn(batch, cap, heads, 1, generator=g, device=DEV))
    kv_append(cache, k, v, i32(0))
    for b, u in enumerate(used if used is not None else []):
        for t in (cache.k, cache.v):
            t.view(torch.uint8)[b, :, u:] = 0x7F
        cache.k_scale[b, :, u:] = float("nan")
        cache.v_scale[b, :, u:] = float("nan")
    return cache


def visible(batch, n, cap, start, counts, sees):
    """[batch, n, cap]: the positions each row sees.  sees: [batch, n, n] truth values of a tree, or None."""
    pos = torch.arange(cap, device=DEV)
    out = torch.zeros(batch, n, cap, dtype=torch.bool, device=DEV)
    for b in range(batch):
        c = n if counts is None else counts[b]
        for i in range(min(c, n)):
            if sees is None:
                out[b, i] = pos <= start[b] + i
            else:
                out[b, i] = pos < start[b]
                for j in range(c):
                    if sees[b][i][j] and 0 <= start[b] + j < cap:
                        out[b, i, start[b] + j] = True
    return out


def formula(q, cache, see, gate=None, scale=None):
    """(out, bound) in float64 for rows seeing ``see`` [batch, n, cap]."""
    b, n, heads, d = q.shape
    g = heads // cache.heads
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(out)
    eps = torch.finfo(q.dtype).eps
    for i in range(b):
        for h in range(cache.heads):
            k = cache.k[i, h].double() * cache.k_scale[i, h, :, None].double()
            v = cache.v[i, h].double() * cache.v_scale[i, h, :, None].double()
            any_row = see[i].any(0)
            k, v = (torch.where(any_row[:, None], t, torch.zeros_like(t)) for t in (k, v))
            x = q[i, :, h * g:(h + 1) * g].double()
            s = torch.einsum("ngd,ld->ngl", x, k) * scale
            size = torch.einsum("ngd,ld->ngl", x.abs(), k.abs()) * abs(scale)
            hide = ~see[i][:, None, :]
            s = s.masked_fill(hide, -math.inf)
            m = s.amax(-1, keepdim=True)
            w = torch.exp(s - torch.where(m > -math.inf, m, torch.zeros_like(m)))
            p = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
            o = torch.einsum("ngl,ld->ngd", p, v)
            a = torch.einsum("ngl,ld->ngd", p, v.abs())
            dd = (d + 4) * 2.0 ** -24 * size.masked_fill(hide, 0).amax(-1, keepdim=True)
            e = 2.0 ** -11 + torch.expm1(2 * dd) + 2.0 ** -14 + (see.shape[2] + 64) * 2.0 ** -23
            tiny = 2.0 ** -31 * torch.einsum("ngl,ld->ngd", (~hide).double().expand_as(s), v.abs())
            if gate is not None:
                f = torch.sigmoid(gate[i, :, h * g:(h + 1) * g].double())
                o, a, tiny = o * f, a * f, tiny * f
            out[i, :, h * g:(h + 1) * g] = o
            bound[i, :, h * g:(h + 1) * g] = (1.01 * eps / 2 * o.abs() + e * a + tiny
                                              + torch.finfo(q.dtype).smallest_normal * eps)
    return out, bound


def check(got, want, bound):
    assert torch.isfinite(got.float()).all()
    off = (got.double() - want).abs()
    worst = float((off / bound).max())
    assert worst <= 1, f"{worst:.3g} of the bound, off by {float(off.max()):.3g}"
    torch.cuda.synchronize()
    assert _lib.device_status(torch.device(DEV)) == 0


def queries(b, n, heads, d, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (2 * torch.randn(b, n, heads, d, generator=g, device=DEV)).to(dtype)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("kv,group", [(1, 1), (4, 6), (2, 8), (3, 5), (1, 16), (2, 24)])
def test_single_tokens_of_a_ragged_batch(fmt, dtype, dim, kv, group):
    """Lengths from one token to a few hundred; 16, 128 and odd numbers around them; NaN behind every end."""
    start = [0, 1, 14, 15, 16, 127, 128, 200, 383, 399]
    b, cap = len(start), 400
    cache = filled(b, kv, cap, dim, fmt, 3, [s + 1 for s in start])
    q = queries(b, 1, kv * group, dim, dtype, 4)
    want, bound = formula(q, cache, visible(b, 1, cap, start, None, None))
    check(cached_attention(q, cache, i32(*start)), want, bound)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("n,group", [(2, 1), (2, 6), (3, 2), (5, 6), (17, 6), (40, 8), (130, 3), (257, 1)])
def test_chunks_are_causal(fmt, dim, n, group):
    start = [0, 5, 300]
    cap, kv = 300 + n, 2
    cache = filled(3, kv, cap, dim, fmt, 5, [s + n for s in start])
    q = queries(3, n, kv * group, dim, torch.float16, 6)
    want, bound = formula(q, cache, visible(3, n, cap, start, None, None))
    check(cached_attention(q, cache, i32(*start)), want, bound)


def random_tree(n, seed):
    g = torch.Generator().manual_seed(seed)
    return [-1] + [int(torch.randint(-1 if i < 4 else 0, i, (1,), generator=g)) for i in range(1, n)]


def ancestors(parents):
    n = len(parents)
    sees = [[False] * n for _ in range(n)]
    for i, p in enumerate(parents):
        j = i
        while j >= 0:
            sees[i][j] = True
            j = parents[j]
    return sees


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("n,group", [(1, 6), (2, 8), (7, 1), (8, 6), (31, 4), (33, 6), (64, 2), (100, 8)])
def test_trees_see_their_ancestors(dtype, dim, n, group):
    start = [0, 11, 500]
    cap, kv = 500 + n, 2
    cache = filled(3, kv, cap, dim, "fp8", 7, [s + n for s in start])
    parents = [random_tree(n, 10 + b) for b in range(3)]
    q = queries(3, n, kv * group, dim, dtype, 8)
    gate = torch.randn(q.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    see = visible(3, n, cap, start, None, [ancestors(p) for p in parents])
    want, bound = formula(q, cache, see, gate)
    check(cached_attention(q, cache, i32(*start), tree=tree_mask(parents, DEV), gate=gate), want, bound)
    shared = tree_mask(parents[0], DEV)  # one tree for all
    see = visible(3, n, cap, start, None, [ancestors(parents[0])] * 3)
    want, bound = formula(q, cache, see)
    check(cached_attention(q, cache, i32(*start), tree=shared), want, bound)


@pytest.mark.parametrize("n", [1, 5, 40])
def test_a_chain_is_the_causal_chunk(n):
    cache = filled(2, 2, 200, 256, "int8", 9)
    q = queries(2, n, 12, 256, torch.float16, 10)
    a = cached_attention(q, cache, i32(17, 90))
    b = cached_attention(q, cache, i32(17, 90), tree=tree_mask(list(range(-1, n - 1)), DEV))
    # the same weights over the same positions: sums that may be split elsewhere, then one rounding
    assert ((a - b).abs().float() <= 2.0 ** -9 * a.abs().float().amax()).all()


@pytest.mark.parametrize("n,group", [(3, 2), (9, 6), (40, 4)])
@pytest.mark.parametrize("with_tree", [False, True])
def test_rows_that_see_nothing_and_padding_are_zero(n, group, with_tree):
    start, counts = [0, 50, 0, 7], [n, 0, n - 1, 1]
    cap = 50 + n
    used = [s + c for s, c in zip(start, counts)]
    cache = filled(4, 2, cap, 128, "fp8", 11, used)
    q = queries(4, n, 2 * group, 128, torch.bfloat16, 12)
    sees = None
    tree = None
    if with_tree:  # row 1 has no bit at all; every row has bits past the counts
        sees = [[[j <= i or j >= n - 1 for j in range(n)] for i in range(n)] for _ in range(4)]
        for s in sees:
            s[1] = [False] * n
        words = torch.zeros(4, n, (n + 31) // 32, dtype=torch.int64)
        for b in range(4):
            for i in range(n):
                for j in range(n):
                    words[b, i, j // 32] |= int(sees[b][i][j]) << (j % 32)
        tree = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32).to(DEV)
    see = visible(4, n, cap, start, counts, sees)
    want, bound = formula(q, cache, see)
    got = cached_attention(q, cache, i32(*start), counts=i32(*counts), tree=tree)
    check(got, want, bound)
    empty = ~see.any(-1)
    assert empty[1].all() and not got[empty].any()
    if with_tree:
        assert empty[0, 1]


def test_positions_outside_the_cache():
    """Negative starts and starts at or past the end: only positions inside count."""
    n, cap = 6, 40
    cache = filled(4, 2, cap, 128, "int8", 13)
    q = queries(4, n, 4, 128, torch.float16, 14)
    start = [-3, -50, 36, 1000]
    see = visible(4, n, cap, start, None, None)
    want, bound = formula(q, cache, see)
    check(cached_attention(q, cache, i32(*start)), want, bound)
    parents = list(range(-1, n - 1))
    see = visible(4, n, cap, start, None, [ancestors(parents)] * 4)
    want, bound = formula(q, cache, see)
    check(cached_attention(q, cache, i32(*start), tree=tree_mask(parents, DEV)), want, bound)


@pytest.mark.parametrize("n", [1, 7, 40])
def test_non_finite_vectors_stay_in_the_rows_that_see_them(n):
    cap, at = 150, 100
    cache = filled(1, 2, cap, 128, "int8", 15)
    bad = torch.randn(1, 1, 2, 128, device=DEV)
    bad[0, 0, 1, 3] = float("inf")  # head 1 only
    kv_append(cache, torch.randn(1, 1, 2, 128, device=DEV), bad, i32(at))
    q = queries(1, n, 4, 128, torch.float16, 16)
    got = cached_attention(q, cache, i32(at - n // 2))
    see = torch.arange(n, device=DEV) + at - n // 2 >= at
    assert torch.isfinite(got[:, :, :2]).all()
    assert torch.isnan(got[0, see, 2:]).all() and torch.isfinite(got[0, ~see, 2:]).all()


@pytest.mark.parametrize("n,group", [(1, 6), (12, 6)])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_extreme_scales_and_scores(n, group, fmt):
    """Values of very different size along the cache, zero vectors, scores large enough that one position takes all,
    and queries near both ends of the types."""
    cap, d = 700, 128
    cache = filled(1, 1, cap, d, fmt, 17)
    cache.v_scale *= torch.exp2(torch.linspace(-12, 12, cap, device=DEV))
    cache.v_scale[0, 0, 5::50] = 0
    cache.k_scale[0, 0, 7::90] = 0
    for factor, dtype in ((30.0, torch.float16), (1e-3, torch.float16), (1e30, torch.bfloat16), (1e-30, torch.bfloat16)):
        q = (queries(1, n, group, d, torch.float32, 18) * factor).to(dtype)
        scale = None if factor < 100 and factor > 1e-9 else 1.0 / factor / math.sqrt(d)
        see = visible(1, n, cap, [cap - n], None, None)
        want, bound = formula(q, cache, see, None, scale)
        check(cached_attention(q, cache, i32(cap - n), scale=scale), want, bound)


def test_views_of_a_joined_projection():
    """q and gate interleaved per head in one row, as the model's projection leaves them; an odd offset; a given out."""
    b, n, heads, d = 2, 3, 6, 128
    cache = filled(b, 2, 64, d, "int8", 19)
    x = torch.randn(b, n, heads, 2, d, device=DEV)
    gate = x[..., 1, :]
    q16 = x.to(torch.float16)[..., 0, :]
    want = cached_attention(q16.contiguous(), cache, i32(10, 20), gate=gate.contiguous())
    assert torch.equal(cached_attention(q16, cache, i32(10, 20), gate=gate), want)
    flat = torch.zeros(b * n * heads * d + 3, dtype=torch.float16, device=DEV)
    odd = flat[3:].view(b, n, heads, d).copy_(q16)
    out = torch.empty_like(want)
    assert cached_attention(odd, cache, i32(10, 20), gate=gate, out=out) is out
    assert torch.equal(out, want)
    turned = q16.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)
    assert torch.equal(cached_attention(turned, cache, i32(10, 20), gate=gate), want)


@pytest.mark.parametrize("n,heads,dim,length", [(1, 12, 256, 70001), (20, 12, 256, 20011), (1, 6, 128, 9000)])
def test_long_contexts_are_split(n, heads, dim, length):
    cache = filled(1, 2, length, dim, "int8", 20)
    q = queries(1, n, heads, dim, torch.bfloat16, 21)
    want, bound = formula(q, cache, visible(1, n, length, [length - n], None, None))
    first = cached_attention(q, cache, i32(length - n))
    check(first, want, bound)
    assert torch.equal(cached_attention(q, cache, i32(length - n)), first)  # the same sums in the same order


def test_far_positions_pass_32_bits():
    cap, d = 5_000_000, 256  # head 1 starts at 1.28e9 codes, its end passes 2^31
    cache = QuantizedKVCache.empty(1, 2, cap, d, "int8", DEV)
    k = torch.randn(1, 300, 2, d, device=DEV)
    kv_append(cache, k, k + 1, i32(cap - 300))
    q = queries(1, 1, 4, d, torch.float16, 22)
    got = cached_attention(q, cache, i32(cap - 1))
    # all positions before have zero keys and values: their scores are 0 and they add nothing
    s = torch.einsum("ghd,lhd->hgl", q[0, 0].double().view(2, 2, d).transpose(0, 1),
                     cache.k[0, :, -300:].double().mul(cache.k_scale[0, :, -300:, None]).transpose(0, 1)) / 16
    w = torch.exp(s)
    v = cache.v[0, :, -300:].double() * cache.v_scale[0, :, -300:, None]
    o = torch.einsum("hgl,hld->hgd", w, v) / (w.sum(-1, keepdim=True) + cap - 300)
    a = torch.einsum("hgl,hld->hgd", w, v.abs()) / (w.sum(-1, keepdim=True) + cap - 300)
    off = (got[0, 0].double().view(2, 2, d) - o).abs()
    # one split and one order of sums per 128 or so positions: L 2^-24 for the sum of five million weights is the bound
    assert (off <= 2.0 ** -11 * o.abs() + (2.0 ** -11 + 2.0 ** -13 + cap * 2.0 ** -24) * a + 2.0 ** -24).all()


@pytest.mark.parametrize("n", [1, 30])
def test_captured_and_on_another_stream(n):
    """A captured call replays at the device's position; two graphs and an eager call do not share scratch."""
    cap, heads = 3000, 12
    cache = filled(2, 2, cap, 256, "int8", 23)
    q = queries(2, n, heads, 256, torch.float16, 24)
    pos = i32(100)
    cached_attention(q, cache, pos)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cached_attention(q, cache, pos))
        graphs.append(g)
    side = torch.cuda.Stream()
    for p in (0, 700, cap - n):
        pos.fill_(p)
        want = cached_attention(q, cache, i32(p))
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
            other = cached_attention(q, cache, pos)
        torch.cuda.synchronize()
        for got in (*outs, other):
            assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,fmt", [(128, "fp8"), (256, "int8")])
@pytest.mark.parametrize("n,group", [(1, 6), (2, 6), (1, 16), (8, 1), (3, 7)])
@pytest.mark.parametrize("with_tree", [False, True])
def test_long_caches_of_ragged_batches(dtype, dim, fmt, n, group, with_tree):
    """Caches past 8192 positions are split over the GPU at any tile: with padding, starts outside, a gate, few heads."""
    start, counts, cap = [0, 8192, -2, 137, 9000, 5000], [n, n, n, max(n - 1, 0), n, 0], 8205
    b, kv = len(start), 2
    used = [min(max(s + c, 0), cap) for s, c in zip(start, counts)]
    cache = filled(b, kv, cap, dim, fmt, 31, used)
    q = queries(b, n, kv * group, dim, dtype, 32)
    gate = torch.randn(q.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    parents = random_tree(n, 3)
    see = visible(b, n, cap, start, counts, [ancestors(parents)] * b if with_tree else None)
    want, bound = formula(q, cache, see, gate)
    got = cached_attention(q, cache, i32(*start), counts=i32(*counts), gate=gate,
                           tree=tree_mask(parents, DEV) if with_tree else None)
    check(got, want, bound)
    assert not got[~see.any(-1)].any()


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("batch,kv", [(1, 1), (3, 7), (10, 4), (37, 2), (75, 4), (2, 150)])
@pytest.mark.parametrize("n", [1, 9])
def test_any_number_of_sequences_and_heads(dim, batch, kv, n):
    """From one head of one sequence to more of them than CTAs run at once; lengths differ along the batch."""
    cap = 300
    start = [(37 * b) % (cap - n) for b in range(batch)]
    cache = filled(batch, kv, cap, dim, "int8", 33, [s + n for s in start])
    q = queries(batch, n, kv, dim, torch.float16, 34)
    want, bound = formula(q, cache, visible(batch, n, cap, start, None, None))
    check(cached_attention(q, cache, i32(*start)), want, bound)


@pytest.mark.parametrize("cap", [8192, 8193])
@pytest.mark.parametrize("n", [1, 3])
def test_both_ways_to_split_a_cache(cap, n):
    cache = filled(2, 2, cap, 256, "fp8", 35)
    q = queries(2, n, 12, 256, torch.float16, 36)
    start = [cap - n, 4000]
    want, bound = formula(q, cache, visible(2, n, cap, start, None, None))
    check(cached_attention(q, cache, i32(*start)), want, bound)


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("cap", [130, 9000])
def test_starts_at_the_ends_of_int32(n, cap):
    cache = filled(4, 1, cap, 128, "int8", 37)
    q = queries(4, n, 2, 128, torch.float16, 38)
    start = [2 ** 31 - 1, -2 ** 31, 2 ** 30, -1]
    want, bound = formula(q, cache, visible(4, n, cap, start, None, None))
    check(cached_attention(q, cache, i32(*start)), want, bound)


def test_a_shared_start_and_counts_past_the_rows():
    cache = filled(3, 2, 90, 128, "fp8", 39)
    for n in (2, 20):
        q = queries(3, n, 4, 128, torch.float16, 40)
        want, bound = formula(q, cache, visible(3, n, 90, [33] * 3, [n, n, 0], None))
        check(cached_attention(q, cache, i32(33), counts=i32(n, n + 7, -5)), want, bound)


def test_tree_mask_words():
    assert tree_mask([-1, 0, 0, 1, -1], "cpu").flatten().tolist() == [1, 3, 5, 11, 16]
    w = tree_mask(torch.arange(-1, 39), "cpu")
    assert w.shape == (40, 2) and w[39].tolist() == [-1, 255] and w[31].tolist() == [-1, 0]
    assert tree_mask([[-1, 0], [-1, -1]], "cpu").shape == (2, 2, 1)
    for bad in ([0], [-1, 1], [-1, -2]):
        with pytest.raises(ValueError):
            tree_mask(bad, "cpu")


def test_refusals():
    c = QuantizedKVCache.empty(2, 2, 16, 128, "int8", DEV)
    q = torch.zeros(2, 3, 4, 128, dtype=torch.float16, device=DEV)
    s = i32(0, 0)
    for bad in (q[:1], q[..., :64], q[:, :, :3], q[0]):
        with pytest.raises(ValueError):
            cached_attention(bad, c, s)
    with pytest.raises(TypeError):
        cached_attention(q.float(), c, s)
    with pytest.raises(TypeError):
        cached_attention(q, c, s.long())
    with pytest.raises(RuntimeError):
        cached_attention(q.cpu(), c, s)
    with pytest.raises(ValueError):
        cached_attention(q, c, i32(0, 0, 0))
    with pytest.raises(ValueError):
        cached_attention(q, c, s, counts=i32(1))
    with pytest.raises(TypeError):
        cached_attention(q, c, s, tree=torch.zeros(3, 1, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError):
        cached_attention(q, c, s, tree=torch.zeros(3, 2, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        cached_attention(torch.zeros(2, 1025, 2, 128, dtype=torch.float16, device=DEV), c, s,
                         tree=torch.zeros(1025, 33, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        cached_attention(q, c, s, gate=q)
    with pytest.raises(ValueError):
        cached_attention(q, c, s, out=torch.empty(2, 3, 4, 128, device=DEV))
    assert cached_attention(q[:, :0], c, s).shape == (2, 0, 4, 128)
