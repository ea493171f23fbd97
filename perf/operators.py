"""Cases for the operators of one decoding step with a quantised key/value cache.

Three kinds of case, by the field ``op``:

``cache``   new keys and values of B sequences are quantised into the cache (8-bit
            codes and one fp32 scale per token and head) and the written positions
            are read back;
``attend``  queries of the newest tokens of each sequence against its cached keys
            and values: single tokens (n = 1), chunks of a prompt (causal), and trees
            of drafted tokens (each sees the cached text and its own ancestors);
``logits``  repetition, frequency and presence penalties, biases and a grammar's
            mask on the rows of logits, and the token of the highest result.

Formats of the cache.  For one token's vector x of one head, with a = max|x| and
m = 127 (int8) or 448 (fp8, e4m3): scale = a / m in fp32 (0 for a zero vector),
code = round to nearest even of x / scale, value = code * scale.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

MAXIMA = {"int8": 127.0, "fp8": 448.0}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
EPS = {"fp32": 4, "fp16": 2, "bf16": 2}  # bytes of a value


def listed():
    return [
        # One new token of one sequence: the call of every decoding step, where only latency counts.
        dict(name="cache: one token", op="cache", fmt="int8", dtype="fp32", batch=1, tokens=1, kv=4, dim=256, cap=2304),
        # A batch of prompts entering the cache, an odd number of tokens each.
        dict(name="cache: prompts", op="cache", fmt="fp8", dtype="bf16", batch=8, tokens=1999, kv=4, dim=256, cap=2304),
        # Decoding of one sequence in the default cache length of the model harness.
        dict(name="attend: one sequence", op="attend", fmt="int8", dtype="fp16", batch=1, n=1, heads=24, kv=4, dim=256,
             length=2301, spread=0, mask="causal", gate=True),
        # Decoding of a ragged batch (the benchmark's batch 64), gated as in the model.
        dict(name="attend: batch of 64", op="attend", fmt="int8", dtype="fp16", batch=64, n=1, heads=24, kv=4, dim=256,
             length=2304, spread=90, mask="causal", gate=True),
        # One sequence with a long history: the long axis has to be split over the card.
        dict(name="attend: long context", op="attend", fmt="fp8", dtype="bf16", batch=1, n=1, heads=24, kv=4, dim=256,
             length=131071, spread=0, mask="causal", gate=False),
        # Many long sequences: the largest reads of a serving step.
        dict(name="attend: long batch", op="attend", fmt="int8", dtype="bf16", batch=24, n=1, heads=32, kv=4, dim=128,
             length=65536, spread=60, mask="causal", gate=False),
        # A small tree of drafted tokens (two branches or so) after an ordinary history.
        dict(name="attend: small tree", op="attend", fmt="fp8", dtype="fp16", batch=1, n=7, heads=24, kv=4, dim=256,
             length=1900, spread=0, mask="tree", gate=True),
        # Large drafted trees of several sequences, verified together.
        dict(name="attend: wide trees", op="attend", fmt="int8", dtype="bf16", batch=8, n=61, heads=24, kv=4, dim=256,
             length=8191, spread=70, mask="tree", gate=False),
        # The next turn of a conversation: a chunk of prompt on top of a long cache.
        dict(name="attend: chunk", op="attend", fmt="int8", dtype="fp16", batch=1, n=777, heads=24, kv=4, dim=256,
             length=24001, spread=0, mask="causal", gate=True),
        # The LM head's row of one sequence with penalties only.
        dict(name="logits: one row", op="logits", dtype="fp32", rows=1, vocab=248320, used=700, biases=0, grammar=False),
        # A batch with everything on: penalties, biases, grammar masks.
        dict(name="logits: batch of 64", op="logits", dtype="fp32", rows=64, vocab=248320, used=2000, biases=100, grammar=True),
        # A small odd vocabulary in bf16: rows that start at unaligned addresses, many ties.
        dict(name="logits: odd vocabulary", op="logits", dtype="bf16", rows=5, vocab=50257, used=300, biases=17, grammar=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same ranges: any of the three kinds, sizes over their logarithm."""
    op = rng.choice(["cache", "attend", "attend", "attend", "logits"])
    dtype = rng.choice(["fp16", "bf16", "fp32"] if op != "attend" else ["fp16", "bf16"])
    if op == "logits":
        rows = _log(rng, 1, 64)
        vocab = _log(rng, 1000, 248320)
        return dict(op=op, dtype=dtype, rows=rows, vocab=vocab, used=min(vocab // 2, _log(rng, 1, 4000)),
                    biases=rng.choice([0, _log(rng, 1, 300)]), grammar=rng.random() < 0.5)
    fmt, dim = rng.choice(["int8", "fp8"]), rng.choice([128, 256])
    kv = rng.choice([1, 2, 4, 8])
    if op == "cache":
        batch = _log(rng, 1, 64)
        tokens = _log(rng, 1, max(1, 16000 // batch // max(1, kv * dim // 1024)))
        return dict(op=op, fmt=fmt, dtype=dtype, batch=batch, tokens=tokens, kv=kv, dim=dim, cap=tokens + rng.randint(0, 2000))
    mask = rng.choice(["causal", "tree"])
    kind = rng.choice(["token", "chunk"]) if mask == "causal" else "tree"
    group = rng.choice([1, 2, 4, 6, 8])
    n = 1 if kind == "token" else _log(rng, 2, 96) if kind == "tree" else _log(rng, 2, 1000)
    batch = _log(rng, 1, 64 if kind == "token" else 16 if kind == "tree" else 2)
    # at most as many cached bytes as the longest listed batch reads, and as many products as the listed chunk makes
    most = min(131072, 1_000_000_000 // (batch * kv * dim * 2), 110_000_000_000 // (4 * batch * n * kv * group * dim) + n)
    length = max(n, _log(rng, max(n, 16), max(n, 16, most)))
    return dict(op=op, fmt=fmt, dtype=dtype, batch=batch, n=n, heads=kv * group, kv=kv, dim=dim, length=length,
                spread=rng.choice([0, rng.randint(1, 95)]), mask=mask, gate=rng.random() < 0.5)


# ---- what the cases stand for, shared by all sides: sizes and inputs ----

def _lengths(case):
    """Cached tokens of each sequence, the new ones included: the longest first, at least n."""
    b, top, n = case["batch"], case["length"], case["n"]
    return [max(n, top - (i * top * case["spread"]) // (100 * b)) for i in range(b)]


def _tree(n, rng):
    """Parents of a drafted tree's tokens (-1: follows the cached text), and each token's ancestors, itself included."""
    parents = [-1] + [int(rng.randint(-1 if i < 4 else 0, i)) for i in range(1, n)]
    sees = np.zeros((n, n), dtype=bool)
    for i, p in enumerate(parents):
        if p >= 0:
            sees[i] = sees[p]
        sees[i, i] = True
    return sees


def _words(bits):
    """Rows of truth values as int32 words, bit j of word w standing for column 32 w + j."""
    r, n = bits.shape
    w = (n + 31) // 32
    padded = np.zeros((r, w * 32), dtype=np.uint8)
    padded[:, :n] = bits
    return np.packbits(padded, axis=1, bitorder="little").view("<i4").reshape(r, w)


def _quantise(x, fmt):
    """Codes and scales of the rows of x (fp32, last dimension the head's)."""
    scale = x.abs().amax(-1, keepdim=True) / MAXIMA[fmt]
    y = x / torch.where(scale > 0, scale, torch.ones_like(scale))
    codes = y.round().to(torch.int8) if fmt == "int8" else y.to(torch.float8_e4m3fn)
    return codes, scale.squeeze(-1)


def _vectors(shape, g, dev, spread):
    """Keys or values: normal, a few strong channels, tokens of different size (``spread``)."""
    x = torch.randn(shape, generator=g, device=dev)
    x[..., ::37] *= 3
    if spread:
        x *= torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=g, device=dev))
    return x


def _make(case, seed):
    """The inputs of a case as plain tensors."""
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.RandomState(seed % (1 << 31))
    dt = TYPES[case["dtype"]]
    if case["op"] == "cache":
        b, t, h, d = case["batch"], case["tokens"], case["kv"], case["dim"]
        start = torch.tensor(rng.randint(0, case["cap"] - t + 1, b), dtype=torch.int32, device=dev)
        codes = torch.zeros((2, b, h, case["cap"], d), device=dev).to(CODES[case["fmt"]])
        scales = torch.zeros((2, b, h, case["cap"]), device=dev)
        return dict(k=_vectors((b, t, h, d), g, dev, False).to(dt), v=_vectors((b, t, h, d), g, dev, True).to(dt),
                    start=start, kc=codes[0], vc=codes[1], ks=scales[0], vs=scales[1])
    if case["op"] == "attend":
        b, n, h, d = case["batch"], case["n"], case["kv"], case["dim"]
        lengths = _lengths(case)
        cap = max(lengths)
        kc, vc = (torch.empty((b, h, cap, d), dtype=CODES[case["fmt"]], device=dev) for _ in range(2))
        ks, vs = (torch.empty((b, h, cap), device=dev) for _ in range(2))
        for i in range(b):
            kc[i], ks[i] = _quantise(_vectors((h, cap, d), g, dev, False), case["fmt"])
            vc[i], vs[i] = _quantise(_vectors((h, cap, d), g, dev, True), case["fmt"])
        s = dict(q=(2 * torch.randn((b, n, case["heads"], d), generator=g, device=dev)).to(dt), kc=kc, vc=vc, ks=ks, vs=vs,
                 start=torch.tensor([m - n for m in lengths], dtype=torch.int32, device=dev), tree=None, sees=None, gate=None)
        if case["mask"] == "tree":
            sees = np.stack([_tree(n, rng) for _ in range(b)])
            s["sees"] = torch.tensor(sees, device=dev)
            s["tree"] = torch.tensor(_words(sees.reshape(b * n, n)).reshape(b, n, -1), device=dev)
        if case["gate"]:
            s["gate"] = torch.randn(s["q"].shape, generator=g, device=dev)
        return s
    r, v, used, nb = case["rows"], case["vocab"], case["used"], case["biases"]
    logits = (3 * torch.randn((r, v), generator=g, device=dev)).to(dt)
    counts = torch.zeros((r, v), dtype=torch.int32, device=dev)
    seen = np.zeros((r, v), dtype=bool)
    for i in range(r):
        prompt, made = (rng.randint(0, v, max(1, used // 2)) for _ in range(2))
        seen[i, prompt] = seen[i, made] = True
        at, c = np.unique(made, return_counts=True)
        counts[i, torch.tensor(at, device=dev)] = torch.tensor(c, dtype=torch.int32, device=dev)
    s = dict(logits=logits, counts=counts, seen=torch.tensor(_words(seen), device=dev),
             repetition=1 + torch.rand(r, generator=g, device=dev), frequency=torch.rand(r, generator=g, device=dev),
             presence=torch.rand(r, generator=g, device=dev) - 0.3, bias_ids=None, bias_values=None, allowed=None)
    if nb:
        ids = np.stack([rng.permutation(v)[:nb] for _ in range(r)])
        ids[:, nb - nb // 4:] = -1  # rows with fewer biases end in padding
        s["bias_ids"] = torch.tensor(ids, dtype=torch.int32, device=dev)
        s["bias_values"] = 4 * torch.randn((r, nb), generator=g, device=dev)
    if case["grammar"]:
        s["allowed"] = torch.tensor(_words(rng.rand(r, v) < 0.2), device=dev)
    return s


def prepare(case, seed):
    s = _make(case, seed)
    s["case"] = case
    if own:
        root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "mlx-gsq-rco_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        from gsq_b200.runtime import QuantizedKVCache, TokenHistory
        if case["op"] == "logits":
            s["history"] = TokenHistory(s["seen"], s["counts"])
        else:  # the handle holds the same tensors
            s["cache"] = QuantizedKVCache(s["kc"], s["vc"], s["ks"], s["vs"])
    return s


# ---- one pass ----

def _run_own(s):
    from gsq_b200.runtime.kernels import adjust_logits, cached_attention, kv_append, kv_read
    case = s["case"]
    if case["op"] == "cache":
        kv_append(s["cache"], s["k"], s["v"], s["start"])
        return kv_read(s["cache"], s["start"], case["tokens"], dtype=TYPES[case["dtype"]])
    if case["op"] == "attend":
        return cached_attention(s["q"], s["cache"], s["start"], tree=s["tree"], gate=s["gate"])
    return adjust_logits(s["logits"], history=s["history"], repetition=s["repetition"], frequency=s["frequency"],
                         presence=s["presence"], bias_ids=s["bias_ids"], bias_values=s["bias_values"], allowed=s["allowed"])


def _unpack(words, n):
    at = torch.arange(n, device=words.device)
    return (words[..., at // 32] >> (at % 32)) & 1 > 0


def _plain_cache(s):
    case, out = s["case"], []
    b, t = s["k"].shape[:2]
    at = s["start"].long()[:, None] + torch.arange(t, device=s["k"].device)  # [B, T]
    rows = torch.arange(b, device=at.device)[:, None]
    for x, codes, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        c, f = _quantise(x.float(), case["fmt"])
        codes.transpose(1, 2).view(torch.uint8)[rows, at] = c.view(torch.uint8)
        scales.transpose(1, 2)[rows, at] = f
        read = codes.transpose(1, 2).view(torch.uint8)[rows, at].view(codes.dtype)
        out.append((read.float() * scales.transpose(1, 2)[rows, at][..., None]).to(TYPES[case["dtype"]]))
    return tuple(out)


def _sees(s, n, cap):
    """[B, n, cap]: which cached positions each new token sees."""
    pos = torch.arange(cap, device=s["q"].device)
    base = s["start"].long()  # where the new tokens begin
    if s["sees"] is None:
        return pos[None, None, :] <= (base[:, None] + torch.arange(n, device=pos.device))[:, :, None]
    off = pos[None, :] - base[:, None]  # [B, cap]
    new = torch.gather(s["sees"], 2, off.clamp(0, n - 1)[:, None, :].expand(-1, n, -1)) & (off < n)[:, None, :]
    return (off < 0)[:, None, :] | ((off >= 0)[:, None, :] & new)


def _plain_attend(s):
    b, n, heads, d = s["q"].shape
    kv, cap = s["kc"].shape[1:3]
    g = heads // kv
    q = s["q"].float().reshape(b, n, kv, g, d).permute(0, 2, 1, 3, 4).reshape(b, kv, n * g, d)
    k = s["kc"].float() * s["ks"][..., None]
    v = s["vc"].float() * s["vs"][..., None]
    sees = _sees(s, n, cap)[:, None, :, None, :].expand(b, 1, n, g, cap).reshape(b, 1, n * g, cap)
    w = (q @ k.transpose(-1, -2) / math.sqrt(d)).masked_fill_(~sees, -math.inf)
    w = torch.exp(w.sub_(w.amax(-1, keepdim=True)))
    o = (w @ v) / w.sum(-1, keepdim=True)
    o = o.reshape(b, kv, n, g, d).permute(0, 2, 1, 3, 4).reshape(b, n, heads, d)
    if s["gate"] is not None:
        o = o / (1 + torch.exp(-s["gate"]))
    return o.to(s["q"].dtype)


def _plain_logits(s):
    z = s["logits"].float()
    r, v = z.shape
    seen = _unpack(s["seen"], v)
    rep = s["repetition"][:, None]
    z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
    z = z - s["frequency"][:, None] * s["counts"].float()
    z = z - s["presence"][:, None] * (s["counts"] > 0).float()
    if s["bias_ids"] is not None:
        ids = torch.where(s["bias_ids"] >= 0, s["bias_ids"], v).long()
        z = z + torch.zeros((r, v + 1), device=z.device).scatter_add_(1, ids, s["bias_values"])[:, :v]
    if s["allowed"] is not None:
        z = torch.where(_unpack(s["allowed"], v), z, -math.inf)
    best = z.amax(-1, keepdim=True)
    at = torch.arange(v, device=z.device, dtype=torch.int32)
    return z, torch.where(z == best, at, v).amin(-1).to(torch.int32)


def run(state):
    if own:
        return _run_own(state)
    return {"cache": _plain_cache, "attend": _plain_attend, "logits": _plain_logits}[state["case"]["op"]](state)


def work(case):
    size = EPS[case["dtype"]]
    if case["op"] == "cache":
        vectors = 2 * case["batch"] * case["tokens"] * case["kv"]  # read, stored as codes and scales, read back from them, returned
        return {"bytes": vectors * (2 * size * case["dim"] + 2 * (case["dim"] + 4)), "flops": 3 * vectors * case["dim"]}
    if case["op"] == "attend":
        n, d, lengths = case["n"], case["dim"], _lengths(case)
        rows = case["batch"] * n * case["heads"] * d
        pairs = sum(n * (m - n) + (n * (n + 1) // 2 if case["mask"] == "causal" else n * min(n, 6)) for m in lengths)
        return {"bytes": sum(lengths) * case["kv"] * 2 * (d + 4) + rows * (2 * size + (4 if case["gate"] else 0)),
                "flops": 4 * pairs * case["heads"] * d}
    r, v = case["rows"], case["vocab"]
    masks = r * ((v + 31) // 32) * 4 * (2 if case["grammar"] else 1)
    return {"bytes": r * v * (size + 4) + masks + r * (case["used"] // 2 * 4 + case["biases"] * 8 + 16), "flops": 6 * r * v}


# ---- the same from the definitions, in 64 bits ----

def _e4m3(y):
    """Nearest value of the 8-bit type with four exponent and three fraction bits, ties to even (|y| <= 448)."""
    m, e = np.frexp(np.abs(y))  # y = m 2^e, m in [1/2, 1)
    step = np.ldexp(1.0, np.maximum(e - 4, -9))
    return np.sign(y) * np.rint(np.abs(y) / step) * step


def _exact_cache(case, s):
    out = []
    for x in (s["k"], s["v"]):
        x = x.float().cpu().numpy()
        scale = (np.abs(x).max(-1, keepdims=True) / np.float32(MAXIMA[case["fmt"]])).astype(np.float32)
        y = np.divide(x, scale, out=np.zeros_like(x), where=scale > 0).astype(np.float64)
        out.append((np.rint(y) if case["fmt"] == "int8" else _e4m3(y)) * scale.astype(np.float64))
    return tuple(out)


def _exact_attend(case, s):
    b, n, heads, d = s["q"].shape
    kv = s["kc"].shape[1]
    g, out = heads // kv, torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for i, m in enumerate(_lengths(case)):
        for h in range(kv):
            k = s["kc"][i, h, :m].double() * s["ks"][i, h, :m, None].double()
            v = s["vc"][i, h, :m].double() * s["vs"][i, h, :m, None].double()
            for a in range(0, n, 64):  # so many tokens at a time that their scores fit
                z = min(n, a + 64)
                hidden = torch.zeros((z - a, m), dtype=torch.bool, device=k.device)
                if s["sees"] is None:
                    last = torch.arange(m - n + a, m - n + z, device=k.device)
                    hidden = torch.arange(m, device=k.device)[None, :] > last[:, None]
                else:
                    hidden[:, m - n:] = ~s["sees"][i, a:z]
                dots = torch.einsum("ngd,ld->ngl", s["q"][i, a:z, h * g:(h + 1) * g].double(), k) / math.sqrt(d)
                dots = torch.where(hidden[:, None, :], torch.full_like(dots, -math.inf), dots)
                out[i, a:z, h * g:(h + 1) * g] = torch.einsum("ngl,ld->ngd", torch.softmax(dots, -1), v)
    return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())


def _exact_logits(case, s):
    z = s["logits"].double().cpu().numpy()
    counts, v = s["counts"].cpu().numpy().astype(np.float64), case["vocab"]
    bits = lambda t: np.unpackbits(t.cpu().numpy().view(np.uint8).reshape(z.shape[0], -1), axis=1, bitorder="little")[:, :v] > 0  # noqa: E731
    rep, freq, pres = (s[k].double().cpu().numpy()[:, None] for k in ("repetition", "frequency", "presence"))
    z = np.where(bits(s["seen"]), np.where(z > 0, z / rep, z * rep), z) - freq * counts - pres * (counts > 0)
    if s["bias_ids"] is not None:
        ids, values = s["bias_ids"].cpu().numpy(), s["bias_values"].double().cpu().numpy()
        for i, j in zip(*np.nonzero(ids >= 0)):
            z[i, ids[i, j]] += values[i, j]
    if s["allowed"] is not None:
        z = np.where(bits(s["allowed"]), z, -np.inf)
    return z, None  # near ties make the token depend on how the values round


def exact(case, seed):
    s = _make(case, seed)
    return {"cache": _exact_cache, "attend": _exact_attend, "logits": _exact_logits}[case["op"]](case, s)
