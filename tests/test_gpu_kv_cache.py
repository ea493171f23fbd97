"""Quantised key/value cache: writing (gsq_kv_append) and reading back
(gsq_kv_read) against the format's definition, in torch on the host (IEEE fp32
divisions) and as distances from the inputs.

A code is the nearest of x / scale, so a value read back in fp32 is off by at
most half a step: int8 scale / 2; e4m3 2^-4 of |x|, or half of its smallest
step, 2^-10 * scale.  The quotient's and the product's fp32 roundings (2^-24 of
up to 448 steps each) are far below 2^-10 of a step: the factor 1.001.
"""
import pytest
import torch

from gsq_b200 import _lib
from gsq_b200.runtime import QuantizedKVCache
from gsq_b200.runtime.kernels import kv_append, kv_read

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
MAX = {"int8": 127.0, "fp8": 448.0}


def quantise(x, fmt):
    """Codes and scales of host vectors, from the definition in fp32."""
    x = x.float()
    scale = x.abs().amax(-1) * (torch.ones(()) / torch.tensor(MAX[fmt]))
    y = x / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    return (y.round().to(torch.int8) if fmt == "int8" else y.to(torch.float8_e4m3fn)), scale


def rand(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(2 * torch.randn(shape[:-1] + (1,), generator=g))
    return x.to(dtype)


def status():
    torch.cuda.synchronize()
    return _lib.device_status(torch.device(DEV))


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("batch,heads,tokens", [(1, 1, 1), (1, 4, 1), (3, 5, 7), (2, 3, 130)])
def test_append_and_read_back(fmt, dtype, dim, batch, heads, tokens):
    cap = tokens + 9
    cache = QuantizedKVCache.empty(batch, heads, cap, dim, fmt, DEV)
    k, v = (rand((batch, tokens, heads, dim), dtype, s) for s in (1, 2))
    k[0, 0, 0] = 0  # a zero vector
    start = torch.arange(batch, dtype=torch.int32) * 3 % 10
    kv_append(cache, k.to(DEV), v.to(DEV), start.to(DEV))
    got = kv_read(cache, start.to(DEV), tokens, dtype=torch.float32)
    for x, codes, scales, read in ((k, cache.k, cache.k_scale, got[0]), (v, cache.v, cache.v_scale, got[1])):
        want, scale = quantise(x, fmt)
        codes, scales, read = codes.cpu(), scales.cpu(), read.cpu()
        for b in range(batch):
            at = slice(int(start[b]), int(start[b]) + tokens)
            assert torch.equal(codes[b, :, at].transpose(0, 1).contiguous().view(torch.uint8),
                               want[b].contiguous().view(torch.uint8))
            assert torch.equal(scales[b, :, at].T, scale[b])
            untouched = torch.ones(cap, dtype=torch.bool)
            untouched[at] = False
            assert not codes[b].view(torch.uint8)[:, untouched].any() and not scales[b][:, untouched].any()
        assert torch.equal(read, want.float() * scale[..., None])
        s, x = scale[..., None].double(), x.double()
        half = 0.5 * s if fmt == "int8" else torch.maximum(2.0 ** -4 * x.abs(), 2.0 ** -10 * s)
        assert ((read.double() - x).abs() <= 1.001 * half).all()
        for out in (torch.float16, torch.bfloat16):  # one rounding of the fp32 value
            low = kv_read(cache, start.to(DEV), tokens, dtype=out)[0 if x.data_ptr() == k.data_ptr() else 1]
            assert low.dtype == out
    low = kv_read(cache, start.to(DEV), tokens, dtype=torch.bfloat16)
    assert torch.equal(low[0], got[0].to(torch.bfloat16)) and torch.equal(low[1], got[1].to(torch.bfloat16))
    assert status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_unaligned_inputs(dtype):
    """Keys and values as views of one joined projection, at an odd offset, transposed, and expanded over the batch."""
    b, t, h, d = 2, 5, 3, 128
    x = rand((b, t, 1 + 2 * h * d), dtype, 5).to(DEV)
    k, v = x[..., 1:1 + h * d].unflatten(-1, (h, d)), x[..., 1 + h * d:].unflatten(-1, (h, d))
    tk = rand((h, t, b, d), dtype, 6).to(DEV).permute(2, 1, 0, 3)
    one = rand((1, t, h, d), dtype, 7).to(DEV).expand(b, -1, -1, -1)
    for kk, vv in ((k, v), (tk, one), (k.transpose(-1, -2).contiguous().transpose(-1, -2), v)):
        a, c = (QuantizedKVCache.empty(b, h, t, d, "int8", DEV) for _ in range(2))
        kv_append(a, kk, vv, i32(0))
        kv_append(c, kk.contiguous(), vv.contiguous(), i32(0, 0))
        assert torch.equal(a.k, c.k) and torch.equal(a.v, c.v)
        assert torch.equal(a.k_scale, c.k_scale) and torch.equal(a.v_scale, c.v_scale)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_counts_and_positions_outside(fmt):
    b, t, h, d, cap = 4, 6, 2, 128, 8
    k, v = (rand((b, t, h, d), torch.float16, s).to(DEV) for s in (1, 2))
    cache = QuantizedKVCache.empty(b, h, cap, d, fmt, DEV)
    kv_append(cache, k, v, i32(0, 2, 7, -2), i32(0, 6, 1, 0))
    assert status() == 0
    written = cache.k_scale[:, 0].cpu() > 0
    assert written.sum(1).tolist() == [0, 6, 1, 0]
    got = kv_read(cache, i32(0, 2, 7, -2), t, counts=i32(0, 6, 1, 0), dtype=torch.float32)
    want, scale = quantise(k.cpu(), fmt)
    want = want.float() * scale[..., None]
    want[0], want[2, 1:], want[3] = 0, 0, 0
    assert torch.equal(got[0].cpu(), want)
    # past either end: skipped, and reported; the neighbours stay as they were
    kv_append(cache, k, v, i32(0, 0, 6, -3))
    assert status() == 3 and status() == 0
    assert (cache.k_scale[2, 0].cpu() > 0).tolist() == [False] * 6 + [True] * 2
    assert (cache.k_scale[3, 0].cpu() > 0).tolist() == [True] * 3 + [False] * 5
    got = kv_read(cache, i32(0, 0, 6, -3), t, dtype=torch.float16)[0]
    assert not got[2, 2:].any() and not got[3, :3].any() and got[3, 3:].any()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_values_at_the_edges(fmt):
    """Zeros, subnormals, the types' largest values, Inf and NaN."""
    d = 128
    rows = torch.zeros(8, d)
    rows[1] = 1e-44  # a scale that underflows to 0: reads back as 0
    rows[2, 0], rows[2, 1] = 2.7e-43, -1.4e-43  # a subnormal scale, one or two units
    rows[3, ::2] = torch.finfo(torch.float32).max
    rows[4, 5] = float("inf")
    rows[5, 7], rows[5, 8] = float("nan"), 3.0
    rows[6, 0], rows[6, 1:3] = -MAX[fmt], torch.tensor([0.5, 1.5])  # scale 1: ties to even (int8)
    rows[7] = torch.linspace(-1, 1, d)
    cache = QuantizedKVCache.empty(1, 1, 8, d, fmt, DEV)
    x = rows[None, :, None].to(DEV)
    kv_append(cache, x, x, i32(0))
    got = kv_read(cache, i32(0), 8, dtype=torch.float32)[0][0, :, 0].cpu()
    scale = cache.k_scale[0, 0].cpu()
    assert not got[:2].any() and scale[0] == 0 and scale[1] == 0
    assert torch.isfinite(got[[2, 3, 6, 7]]).all()
    # 2.7e-43 is 193 of the smallest subnormal u: 193 / 127 rounds to 1 u (codes up to 127), 193 / 448 to 0
    if fmt == "int8":
        assert scale[2] > 0 and ((got[2] - rows[2]).abs() <= 127 * 1.5e-45 * 1.5).all()
    else:
        assert scale[2] == 0 and not got[2].any()
    assert torch.isnan(got[4]).all() and torch.isnan(got[5]).all()
    assert scale[6] == 1 and got[6, 0] == -MAX[fmt]
    if fmt == "int8":
        assert got[6, 1:3].tolist() == [0.0, 2.0]
    assert status() == 0


def test_far_positions_pass_32_bits():
    """Codes past 2^31 bytes of a long cache."""
    heads, cap, d = 2, 5_000_000, 256
    cache = QuantizedKVCache.empty(1, heads, cap, d, "int8", DEV)
    k, v = (rand((1, 3, heads, d), torch.float16, s) for s in (1, 2))
    kv_append(cache, k.to(DEV), v.to(DEV), i32(cap - 3))
    got = kv_read(cache, i32(cap - 3), 3, dtype=torch.float32)
    for x, r in zip((k, v), got):
        c, s = quantise(x, "int8")
        assert torch.equal(r.cpu(), c.float() * s[..., None])
    assert int((cache.k_scale > 0).sum()) == 6
    assert status() == 0


def test_captured_append_follows_the_position():
    b, h, d = 3, 2, 128
    cache = QuantizedKVCache.empty(b, h, 16, d, "fp8", DEV)
    k, v = (rand((b, 1, h, d), torch.float32, s).to(DEV) for s in (1, 2))
    pos = i32(4)
    kv_append(cache, k, v, pos)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pos.add_(1)
        kv_append(cache, k, v, pos)
        read = kv_read(cache, pos, 1, dtype=torch.float32)
    for step in range(3):
        k.copy_(rand((b, 1, h, d), torch.float32, 10 + step))
        g.replay()
        c, s = quantise(k.cpu(), "fp8")
        assert torch.equal(read[0].cpu(), c.float() * s[..., None])
    assert (cache.k_scale[:, 0].cpu() > 0).sum(1).tolist() == [4] * 3


def test_refusals():
    c = QuantizedKVCache.empty(2, 3, 8, 128, "int8", DEV)
    x = torch.zeros(2, 4, 3, 128, device=DEV)
    with pytest.raises(NotImplementedError):
        QuantizedKVCache.empty(1, 1, 8, 128, "int4", DEV)
    with pytest.raises(ValueError):
        QuantizedKVCache.empty(1, 1, 8, 64, "int8", DEV)
    with pytest.raises(TypeError):
        QuantizedKVCache(x, x, x[..., 0], x[..., 0])
    with pytest.raises(ValueError):
        QuantizedKVCache(c.k[:, :, ::2], c.v[:, :, ::2], c.k_scale[:, :, ::2], c.v_scale[:, :, ::2])
    with pytest.raises(ValueError):
        QuantizedKVCache(c.k, c.v, c.k_scale, c.v_scale[:, :2])
    with pytest.raises(RuntimeError):
        QuantizedKVCache(c.k.cpu(), c.v.cpu(), c.k_scale.cpu(), c.v_scale.cpu())
    for bad in (x[:1], x[:, :, :2], torch.zeros(2, 4, 3, 64, device=DEV)):
        with pytest.raises(ValueError):
            kv_append(c, bad, bad, i32(0))
    with pytest.raises(TypeError):
        kv_append(c, x.double(), x.double(), i32(0))
    with pytest.raises(TypeError):
        kv_append(c, x, x.half(), i32(0))
    with pytest.raises(TypeError):
        kv_append(c, x, x, i32(0).long())
    with pytest.raises(ValueError):
        kv_append(c, x, x, i32(0, 0, 0))
    with pytest.raises(ValueError):
        kv_append(c, x, x, i32(0, 0), i32(1))
    with pytest.raises(RuntimeError):
        kv_append(c, x, x, i32(0).cpu())
    with pytest.raises(TypeError):
        kv_read(c, i32(0), 2, dtype=torch.int8)
    with pytest.raises(ValueError):
        kv_read(c, i32(0), -1)
    kv_append(c, x[:, :0], x[:, :0], i32(0))  # nothing to do
    assert kv_read(c, i32(0), 0)[0].shape == (2, 0, 3, 128)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("size", [1.0, 1e-3, 300.0, 1e30, 1e37, 1e-17, 1e-30])
def test_codes_are_the_divisions(fmt, dtype, size):
    """Every code of many vectors is the nearest of the fp32 quotient, bit for bit, zeros' signs included; short types
    make many ties (a value half as large as the vector's largest is one of int8)."""
    if dtype == torch.float16 and not 1e-3 <= size <= 300:
        pytest.skip("outside fp16")
    g = torch.Generator().manual_seed(41)
    x = (torch.randn(1, 3000, 2, 256, generator=g) * size).to(dtype)
    x[0, ::7, 0, 5] = -0.0
    x[0, ::5, 1, 9] = 0.0
    x[0, ::3, 0, 7] = x[0, ::3, 0].abs().amax(-1) / 2
    x[0, ::4, 1, 8] = -x[0, ::4, 1].abs().amax(-1) / 4
    cache = QuantizedKVCache.empty(1, 2, 3000, 256, fmt, "cuda:0")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda:0")
    kv_append(cache, x.to("cuda:0"), (-x).to("cuda:0"), zero)
    m = 127.0 if fmt == "int8" else 448.0
    for v, codes, scales in ((x, cache.k, cache.k_scale), (-x, cache.v, cache.v_scale)):
        f = v.float().transpose(1, 2)
        scale = f.abs().amax(-1) * torch.tensor(1 / m, dtype=torch.float32)
        q = f / scale[..., None]
        want = q.round().to(torch.int8) if fmt == "int8" else q.clamp(-448, 448).to(torch.float8_e4m3fn)
        assert torch.equal(scales.cpu(), scale)
        assert torch.equal(codes.cpu().view(torch.int8), want.view(torch.int8))
