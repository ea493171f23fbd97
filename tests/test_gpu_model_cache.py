"""The model harness with an 8-bit key/value cache (``kv_format``), a prompt
that goes on from a later position (``extend``), and controlled logits, against
the plain fp32 restatement of the model and against the harness itself.

Tolerances: logits of the fp32-cache model are held to TOL (rel-L2). An 8-bit
cache adds its own error to the keys and values of one layer of four: int8 at
most half a step of max|x| / 127, and with a 256-wide vector's max|x| below 4.5
of its rms (Gaussian) that is 4.5 / 254 / sqrt(3) = 1.0 % of the vector; e4m3
2^-4 / sqrt(3) = 3.6 %. Values enter the layer's output linearly and weights move
by about as much, so twice these bound what the layer's output moves.
"""
import pytest
import torch

from gsq_b200 import _lib
from gsq_b200.models import build_qwen35
from gsq_b200.runtime import QuantizedKVCache, TokenHistory
from gsq_b200.runtime.kernels import kv_read
from test_gpu_model import CFG, TOL, Reference, rel, setup  # noqa: F401

pytestmark = pytest.mark.gpu
EXTRA = {"int8": 2 * 0.010, "fp8": 2 * 0.036}


def prompt(n, dev, seed=5):
    return torch.randint(0, CFG.vocab_size, (n,), generator=torch.Generator().manual_seed(seed)).to(torch.int32).to(dev)


def fine(dev):
    torch.cuda.synchronize()
    assert _lib.device_status(dev) == 0


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("T", [3, 12, 70])  # few rows a head; row blocks of one and of several tiles
def test_prefill_and_decode_match_reference(setup, fmt, T):  # noqa: F811
    dev, w = setup
    model = build_qwen35(w, CFG, dev, max_len=96, kv_format=fmt)
    ref = Reference(w, CFG, dev)
    ids = prompt(T, dev)
    for t in ids.tolist():
        want = ref.step(t)
    assert rel(model.prefill(ids), want) <= TOL + EXTRA[fmt]
    for t in prompt(4, dev, 6).tolist():
        e = rel(model.decode_step(t)[0], ref.step(t))
        assert e <= TOL + EXTRA[fmt], e
    fine(dev)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("parts", [(9, 14), (1, 22), (20, 3), (8, 8, 7)])
def test_extend_goes_on_where_the_prompt_ended(setup, fmt, parts):  # noqa: F811
    """A prompt in parts gives the whole prompt's logits and cache: the attention is the same sums over the same codes;
    the projections of 2 to 7 rows round their activations differently from longer ones, within TOL."""
    dev, w = setup
    ids = prompt(sum(parts), dev)
    whole, piecewise = (build_qwen35(w, CFG, dev, max_len=64, kv_format=fmt) for _ in range(2))
    want = whole.prefill(ids)
    at = 0
    for i, n in enumerate(parts):
        got = (piecewise.prefill if i == 0 else piecewise.extend)(ids[at:at + n])
        at += n
    assert piecewise.n_pos == whole.n_pos == len(ids) and int(piecewise.pos) == len(ids)
    assert rel(got, want) <= TOL + EXTRA[fmt]
    start = torch.zeros(1, dtype=torch.int32, device=dev)
    for a, b in zip(whole.layers, piecewise.layers):
        if not a["linear"]:
            for x, y in zip(*(kv_read(m["kv"][1], start, len(ids), dtype=torch.float32) for m in (a, b))):
                assert rel(y, x) <= TOL + EXTRA[fmt]
    # decode, then a next turn
    one = whole.decode_step(7).clone()
    two = piecewise.decode_step(7)
    assert rel(two, one) <= TOL + EXTRA[fmt]
    more = prompt(11, dev, 8)
    assert rel(piecewise.extend(more), whole.extend(more)) <= TOL + EXTRA[fmt]
    fine(dev)


def test_batched_and_captured_decode(setup):  # noqa: F811
    dev, w = setup
    B = 3
    model = build_qwen35(w, CFG, dev, max_len=64, max_batch=5, kv_format="int8")
    one = build_qwen35(w, CFG, dev, max_len=64, kv_format="int8")
    ids = prompt(7, dev)
    toks = [(17 * b + 5) % CFG.vocab_size for b in range(B)]

    def start():
        model.prefill(ids)
        model.fork(B)
        return model.decode_step(toks).clone()

    first = start()
    eager = [model.decode_step().clone() for _ in range(4)]
    for b in range(B):
        one.prefill(ids)
        assert rel(first[b], one.decode_step(toks[b])[0]) <= TOL
    start()
    model.capture_decode()
    for i in range(4):
        model.replay_decode(1)
        assert torch.equal(model.graph_logits, eager[i])
    assert model.n_pos == 7 + 5
    fine(dev)


def test_the_fp32_cache_is_unchanged_by_default(setup):  # noqa: F811
    dev, w = setup
    model = build_qwen35(w, CFG, dev, max_len=32)
    model.prefill(prompt(5, dev))
    with pytest.raises(NotImplementedError):
        model.extend(prompt(3, dev))
    assert all("k_cache" in L and "kv" not in L for L in model.layers if not L["linear"])
    with pytest.raises(NotImplementedError):
        build_qwen35(w, CFG, dev, max_len=32, kv_format="int3")


def test_extend_refusals(setup):  # noqa: F811
    dev, w = setup
    model = build_qwen35(w, CFG, dev, max_len=16, max_batch=2, kv_format="fp8")
    model.prefill(prompt(10, dev))
    with pytest.raises(ValueError):
        model.extend(prompt(7, dev))
    with pytest.raises(ValueError):
        model.extend(prompt(0, dev))
    model.extend(prompt(4, dev))
    model.fork(2)
    with pytest.raises(ValueError):
        model.extend(prompt(1, dev))
    model.decode_step()
    model.decode_step()
    with pytest.raises(ValueError):
        model.decode_step()
    fine(dev)


def test_control_of_the_logits(setup):  # noqa: F811
    """Greedy decoding within a mask, without repeats under a heavy frequency penalty, eagerly and captured; the history
    is the prompt and the chosen tokens."""
    dev, w = setup
    B, steps = 2, 6
    model = build_qwen35(w, CFG, dev, max_len=64, max_batch=B, kv_format="int8")
    ids = prompt(6, dev)
    plain = model.prefill(ids).clone()
    allowed_tokens = torch.arange(0, CFG.vocab_size, 3)
    bits = torch.zeros(CFG.vocab_size, dtype=torch.int64)
    bits[allowed_tokens] = 1
    words = (bits.view(-1, 32) << torch.arange(32)).sum(-1)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32).to(dev)
    h = TokenHistory.empty(B, CFG.vocab_size, dev)
    model.control_logits(history=h, frequency=torch.full((B,), 1e4, device=dev), allowed=words)

    def run(captured):
        logits = model.prefill(ids)
        assert torch.equal(logits.cpu()[allowed_tokens], plain.cpu()[allowed_tokens])
        model.fork(B)
        chosen = [model.cur_id.clone()]
        for i in range(steps):
            if captured and i == 1:
                model.capture_decode()
            if captured and i >= 1:
                model.replay_decode(1)
            else:
                model.decode_step()
            chosen.append(model.cur_id.clone())
        return torch.stack(chosen).cpu()

    a = run(False)
    assert (a % 3 == 0).all()
    assert all(len(set(a[:, b].tolist())) == steps + 1 for b in range(B))
    counts = torch.zeros(B, CFG.vocab_size, dtype=torch.int32)
    for b in range(B):
        counts[b, a[:, b].long()] = 1
    assert torch.equal(h.counts.cpu(), counts)
    seen = counts > 0
    seen[:, ids.cpu().long()] = True
    got = (h.seen.cpu()[:, :, None] >> torch.arange(32)) & 1 > 0
    assert torch.equal(got.reshape(B, -1)[:, :CFG.vocab_size], seen)
    assert torch.equal(run(True), a)
    model.control_logits()
    assert torch.equal(model.prefill(ids), plain) and int(model.cur_id[0]) == int(plain.argmax())
    with pytest.raises(ValueError):
        model.control_logits(history=TokenHistory.empty(1, CFG.vocab_size, dev))
    fine(dev)


def test_the_three_together_outside_the_model():
    """Write, attend, adjust, in a loop as a decoder makes them, with the state carried along: against the plain sums on
    the cache's own values."""
    from gsq_b200.runtime.kernels import adjust_logits, cached_attention, kv_append
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(1)
    b, heads, kv, d, vocab, steps = 3, 6, 2, 128, 1000, 5
    cache = QuantizedKVCache.empty(b, kv, steps + 40, d, "fp8", dev)
    h = TokenHistory.empty(b, vocab, dev)
    head = torch.randn(heads * d, vocab, generator=g, device=dev) / 28
    start = torch.tensor([0, 7, 33], dtype=torch.int32, device=dev)
    kv_append(cache, *(torch.randn(b, 40, kv, d, generator=g, device=dev) for _ in range(2)),
              torch.zeros(1, dtype=torch.int32, device=dev))
    pen = torch.full((b,), 2.0, device=dev)
    picked = []
    for _ in range(steps):
        k, v = (torch.randn(b, 1, kv, d, generator=g, device=dev, dtype=torch.float32) for _ in range(2))
        q = torch.randn(b, 1, heads, d, generator=g, device=dev).to(torch.bfloat16)
        kv_append(cache, k, v, start)
        out = cached_attention(q, cache, start)
        for i in range(b):
            n = int(start[i]) + 1
            kk, vv = ((c[i, :, :n].double() * s[i, :, :n, None].double()).repeat_interleave(heads // kv, 0)
                      for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
            p = torch.softmax((kk @ q[i, 0].double()[..., None])[..., 0] / d ** 0.5, -1)
            want = (p[..., None] * vv).sum(1)
            # bf16 output 2^-9, fp16 weights 2^-11 of the sum of absolute values, fp32 sums below that
            bound = 2.0 ** -8 * want.abs() + 2.0 ** -10 * (p[..., None] * vv.abs()).sum(1) + 1e-6
            assert ((out[i, 0].double() - want).abs() <= bound).all()
        logits = out.reshape(b, -1).float() @ head
        adjusted, token = adjust_logits(logits, history=h, frequency=pen, presence=pen, record=True)
        counts = torch.zeros(b, vocab, device=dev)
        for t in picked:
            counts[torch.arange(b, device=dev), t.long()] += 1
        want = logits - pen[:, None] * counts
        want = want - pen[:, None] * (counts > 0)
        assert torch.equal(adjusted, want) and torch.equal(token, want.argmax(-1).int())
        picked.append(token)
        start += 1
    fine(dev)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("rot", [0, 64, 256])
@pytest.mark.parametrize("b, t, nq, nkv, pad", [(1, 1, 1, 1, 0), (3, 1, 6, 2, 0), (1, 5, 3, 3, 7), (2, 3, 7, 1, 1)])
def test_the_step_from_projection_to_cache(fmt, rot, b, t, nq, nkv, pad):
    """gsq_qkv_append against its formula in 64 bits. Beyond the half steps of fp16 and of the codes: an angle is p times
    a power whose exponent (up to 17 in units of e) is rounded to fp32, so it is off by p times 2^-19 at most, and norm
    and rotation by a few 2^-24 of the pair's length."""
    dev, hd, cap, eps, theta = torch.device("cuda:0"), 256, 128, 1e-6, 1e7
    g = torch.Generator(device=dev).manual_seed(b * 100 + nq)
    wide = torch.randn(b * t, 512 * (nq + nkv) + pad, generator=g, device=dev) * 3
    qkv = wide[:, :512 * (nq + nkv)]
    qw, kw = (1 + 0.2 * torch.randn(hd, generator=g, device=dev) for _ in range(2))
    start = torch.tensor([0, 60, 97][:b], dtype=torch.int32, device=dev)
    kv = QuantizedKVCache.empty(b, nkv, cap, hd, fmt, dev)
    q = torch.empty(b, t, nq, hd, dtype=torch.float16, device=dev)
    _lib.check(_lib.load().gsq_qkv_append(
        qkv.data_ptr(), qkv.stride(0), b, t, nq, nkv, qw.data_ptr(), kw.data_ptr(), eps, rot, theta, start.data_ptr(),
        1, q.data_ptr(), kv.fmt, *kv.pointers, cap, _lib.stream_ptr(dev)))
    x = qkv.double().view(b, t, -1)
    pos = start.double()[:, None] + torch.arange(t, device=dev).double()

    def rotated(x, w):
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
        if rot == 0:
            return x, x.abs()
        inv = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
        ang = (pos[..., None] * inv)[:, :, None]
        x1, x2 = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([x1 * ang.cos() - x2 * ang.sin(), x2 * ang.cos() + x1 * ang.sin(), x[..., rot:]], -1)
        pair = torch.sqrt(x1 ** 2 + x2 ** 2)
        return y, torch.cat([pair, pair, x[..., rot:].abs()], -1)

    off = (pos * 2.0 ** -19 + 2.0 ** -20)[..., None, None]
    want, size = rotated(x[..., :512 * nq].view(b, t, nq, 512)[..., :hd], qw)
    assert ((q.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -25 + 2 * off * size).all()
    keys = x[..., 512 * nq:512 * nq + hd * nkv].view(b, t, nkv, hd)
    vals = x[..., 512 * nq + hd * nkv:].view(b, t, nkv, hd)
    exact = (vals, torch.zeros_like(vals))
    for codes, scales, (want, size) in ((kv.k, kv.k_scale, rotated(keys, kw)), (kv.v, kv.v_scale, exact)):
        for i in range(b):
            p = int(start[i])
            c, s = codes[i, :, p:p + t].double(), scales[i, :, p:p + t, None].double()
            got, w, z = (c * s).transpose(0, 1), want[i], 2 * off[i] * size[i]
            s = s.transpose(0, 1)
            # a code's half step, of the quotient's own rounding to fp32 as well
            step = s * 0.5 if fmt == "int8" else torch.maximum(2.0 ** -4 * w.abs(), s * 2.0 ** -10)
            assert ((got - w).abs() <= step * (1 + 2.0 ** -10) + w.abs() * 2.0 ** -22 + z * 1.1).all()
            rest = torch.ones(cap, dtype=torch.bool, device=dev)
            rest[p:p + t] = False
            assert not scales[i][:, rest].any() and not codes[i].view(torch.int8)[:, rest].any()
    fine(dev)


def test_refusals_of_the_step_from_projection_to_cache():
    dev = torch.device("cuda:0")
    kv = QuantizedKVCache.empty(1, 1, 8, 256, "int8", dev)
    buf = torch.zeros(1, 1024, device=dev)
    pos = torch.zeros(1, dtype=torch.int32, device=dev)
    q = torch.zeros(1, 1, 1, 256, dtype=torch.float16, device=dev)

    def call(stride=1024, tokens=1, rot=64, fmt=0, q_ptr=q.data_ptr(), nq=1, start=pos.data_ptr()):
        return _lib.load().gsq_qkv_append(buf.data_ptr(), stride, 1, tokens, nq, 1, buf.data_ptr(), buf.data_ptr(), 1e-6,
                                          rot, 1e4, start, 0, q_ptr, fmt, *kv.pointers, 8, _lib.stream_ptr(dev))

    assert call() == 0 and call(tokens=0) == 0
    for bad in (dict(stride=1023), dict(tokens=65536), dict(tokens=-1), dict(rot=3), dict(rot=258), dict(fmt=2),
                dict(q_ptr=q.data_ptr() + 2), dict(nq=0), dict(start=0), dict(q_ptr=0)):
        assert call(**bad) != 0, bad
    # a position outside the cache is not written and reported
    pos.fill_(8)
    kv.k_scale.fill_(7)
    assert call() == 0
    torch.cuda.synchronize()
    assert (kv.k_scale == 7).all()
    assert _lib.load().gsq_device_status(_lib.stream_ptr(dev)) == 3
    assert _lib.load().gsq_device_status(_lib.stream_ptr(dev)) == 0
