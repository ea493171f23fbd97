"""Penalties, biases and masks on logits (gsq_adjust_logits) and the token
history (gsq_record_tokens) against the formula on the host: every step is one
IEEE fp32 operation, so the values are equal and not merely close."""
import pytest
import torch

from gsq_b200.runtime import TokenHistory
from gsq_b200.runtime.kernels import adjust_logits, record_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def words(bits):
    r, v = bits.shape
    p = torch.zeros(r, (v + 31) // 32 * 32, dtype=torch.int64)
    p[:, :v] = bits.long()
    w = (p.view(r, -1, 32) << torch.arange(32)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def formula(z, seen=None, counts=None, rep=None, freq=None, pres=None, ids=None, values=None, allowed=None):
    """Host tensors, one fp32 rounding a step; the biases of one token are summed in list order first."""
    z = z.float().clone()
    r, v = z.shape
    if seen is not None:
        if rep is not None:
            z = torch.where(seen, torch.where(z > 0, z / rep[:, None], z * rep[:, None]), z)
        if freq is not None:
            z = torch.where(counts > 0, z - freq[:, None] * counts.float(), z)
        if pres is not None:
            z = torch.where(counts > 0, z - pres[:, None], z)
    if ids is not None:
        for i in range(r):
            sums = {}
            for t, b in zip(ids[i].tolist(), values[i]):
                if 0 <= t < v:
                    sums[t] = sums.get(t, torch.zeros(())) + b
            for t, b in sums.items():
                z[i, t] = z[i, t] + b
    if allowed is not None:
        z = torch.where(allowed, z, torch.full_like(z, -float("inf")))
    return z


def lowest_best(z):
    key = torch.where(torch.isnan(z), torch.full_like(z, float("inf")), z)
    key = torch.where(torch.isnan(z).any(-1, keepdim=True), torch.isnan(z).float(), key)
    return (key == key.amax(-1, keepdim=True)).int().argmax(-1).int()


def history(r, v, seed, share=0.1):
    g = torch.Generator().manual_seed(seed)
    counts = torch.randint(1, 9, (r, v), generator=g) * (torch.rand(r, v, generator=g) < share / 2)
    seen = (torch.rand(r, v, generator=g) < share) | (counts > 0)
    return seen, counts.int(), TokenHistory(words(seen).to(DEV), counts.int().to(DEV))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 31), (2, 32), (3, 33), (1, 2048), (2, 2049), (4, 5001), (3, 50257),
                                        (1, 248320)])
def test_all_steps_together(dtype, rows, vocab):
    g = torch.Generator().manual_seed(vocab)
    z = (3 * torch.randn(rows, vocab, generator=g)).to(dtype)
    seen, counts, h = history(rows, vocab, 1)
    rep, freq, pres = 1 + torch.rand(rows, generator=g), torch.rand(rows, generator=g), torch.rand(rows, generator=g) - .5
    ids = torch.randint(-1, vocab + 1, (rows, 40), generator=g).int()  # padding, repeats, past the end
    values = torch.randn(rows, 40, generator=g)
    allowed = torch.rand(rows, vocab, generator=g) < 0.3
    allowed[:, vocab // 2] = True
    d = lambda t: t.to(DEV)  # noqa: E731
    want = formula(z, seen, counts, rep, freq, pres, ids, values, allowed)
    got, nxt = adjust_logits(d(z), history=h, repetition=d(rep), frequency=d(freq), presence=d(pres), bias_ids=d(ids),
                             bias_values=d(values), allowed=d(words(allowed)))
    assert got.dtype == torch.float32 and torch.equal(got.cpu(), want)
    assert torch.equal(nxt.cpu(), lowest_best(want))
    assert torch.equal(h.counts.cpu(), counts) and torch.equal(h.seen.cpu(), words(seen))


@pytest.mark.parametrize("use", ["repetition", "frequency", "presence", "bias", "allowed", "shared mask", "nothing"])
def test_each_step_alone(use):
    rows, vocab = 3, 4100
    g = torch.Generator().manual_seed(3)
    z = torch.randn(rows, vocab, generator=g)
    seen, counts, h = history(rows, vocab, 4)
    value = torch.rand(rows, generator=g) + 0.5
    d = lambda t: t.to(DEV)  # noqa: E731
    if use in ("repetition", "frequency", "presence"):
        want = formula(z, seen, counts, **{{"repetition": "rep", "frequency": "freq", "presence": "pres"}[use]: value})
        got, nxt = adjust_logits(d(z), history=h, **{use: d(value)})
    elif use == "bias":
        ids, values = torch.randint(0, vocab, (rows, 9), generator=g).int(), torch.randn(rows, 9, generator=g)
        want = formula(z, ids=ids, values=values)
        got, nxt = adjust_logits(d(z), bias_ids=d(ids), bias_values=d(values))
    elif use == "nothing":
        want = z
        got, nxt = adjust_logits(d(z), history=h)
    else:
        allowed = torch.rand(rows if use == "allowed" else 1, vocab, generator=g) < 0.5
        want = formula(z, allowed=allowed)
        w = d(words(allowed))
        got, nxt = adjust_logits(d(z), allowed=w if use == "allowed" else w[0])
    assert torch.equal(got.cpu(), want) and torch.equal(nxt.cpu(), lowest_best(want))


def test_repeated_biases_add_up_in_list_order():
    vocab = 3000
    ids = torch.tensor([[7, 2500, 7, -1, 7, 2500, vocab, 2 ** 31 - 1, -2 ** 31]], dtype=torch.int32)
    values = torch.tensor([[1e8, 1.0, 1.0, 5.0, -1e8, 2.0, 9.0, 9.0, 9.0]])
    z = torch.zeros(1, vocab)
    got, nxt = adjust_logits(z.to(DEV), bias_ids=ids.to(DEV), bias_values=values.to(DEV))
    assert torch.equal(got.cpu(), formula(z, ids=ids, values=values))
    assert got[0, 7] == 0 and got[0, 2500] == 3 and int(nxt[0]) == 2500


def test_many_biases_of_one_token():
    ids = torch.full((2, 5000), 11, dtype=torch.int32, device=DEV)
    values = torch.full((2, 5000), 0.125, device=DEV)
    got, nxt = adjust_logits(torch.zeros(2, 20, device=DEV), bias_ids=ids, bias_values=values)
    assert got[:, 11].tolist() == [625.0, 625.0] and nxt.tolist() == [11, 11] and int((got != 0).sum()) == 2


def test_ties_and_special_values():
    inf, nan = float("inf"), float("nan")
    vocab = 5000
    rows = torch.zeros(7, vocab)
    rows[0, 4000] = rows[0, 2047] = rows[0, 2048] = 2.0
    rows[1] = -inf
    rows[2, [4999, 100]] = inf
    rows[3, 4500] = nan
    rows[3, 3] = inf
    rows[4] = -0.0
    rows[4, 77] = 0.0  # equal to -0
    rows[5] = -1
    rows[5, 2048:] = -1e-45  # the smallest subnormal
    rows[6] = torch.finfo(torch.float32).min
    got, nxt = adjust_logits(rows.to(DEV))
    assert torch.equal(torch.nan_to_num(got.cpu(), nan=7.5), torch.nan_to_num(rows, nan=7.5))
    assert nxt.tolist() == [2047, 0, 100, 4500, 0, 2048, 0]
    none = torch.zeros((vocab + 31) // 32, dtype=torch.int32, device=DEV)  # a mask that leaves nothing
    got, nxt = adjust_logits(rows.to(DEV), allowed=none)
    assert (got == -inf).all() and not nxt.any()
    # a masked NaN is masked
    some = none.clone()
    some[0] = 1 << 9
    assert adjust_logits(rows.to(DEV), allowed=some)[1].tolist() == [9] * 7 or rows[1, 9] == -inf


def test_in_place_strided_rows_and_a_wider_history():
    rows, vocab = 3, 4097
    g = torch.Generator().manual_seed(5)
    seen, counts, h = history(5, vocab, 6)
    rep = torch.tensor([1.5, 1.1, 2.0])
    wide = torch.randn(rows, vocab + 7, generator=g)
    z = wide[:, 3:3 + vocab]
    want = formula(z, seen[:3], counts[:3], rep=rep)
    got, _ = adjust_logits(wide.to(DEV)[:, 3:3 + vocab], history=h, repetition=rep.to(DEV))
    assert torch.equal(got.cpu(), want)
    x = z.contiguous().to(DEV)
    got, _ = adjust_logits(x, history=h, repetition=rep.to(DEV), out=x)
    assert got is x and torch.equal(x.cpu(), want)
    t = z.T.contiguous().to(DEV).T
    assert torch.equal(adjust_logits(t, history=h, repetition=rep.to(DEV))[0].cpu(), want)
    one = z[:1].expand(3, -1)
    got, _ = adjust_logits(one.to(DEV)[:1].expand(3, -1), history=h, repetition=rep.to(DEV))
    assert torch.equal(got.cpu(), formula(one, seen[:3], counts[:3], rep=rep))


def test_record():
    vocab = 100
    h = TokenHistory.empty(3, vocab, DEV)
    record_tokens(h, torch.tensor([[5, 99, 5, -1], [31, 32, 100, 64]], dtype=torch.int32, device=DEV), generated=False)
    assert not h.counts.any()
    record_tokens(h, torch.tensor([[5, 5, 6, -7], [0, 0, 0, 0]], dtype=torch.int32, device=DEV))
    seen = torch.zeros(3, vocab, dtype=torch.bool)
    seen[0, [5, 6, 99]] = seen[1, [0, 31, 32, 64]] = True
    counts = torch.zeros(3, vocab, dtype=torch.int32)
    counts[0, 5], counts[0, 6], counts[1, 0] = 2, 1, 4
    assert torch.equal(h.seen.cpu(), words(seen)) and torch.equal(h.counts.cpu(), counts)
    z = torch.zeros(3, vocab, device=DEV)
    z[0, 42] = z[1, 31] = z[2, 99] = 1
    _, nxt = adjust_logits(z, history=h, record=True)
    assert nxt.tolist() == [42, 31, 99]
    seen[0, 42] = seen[2, 99] = True
    counts[0, 42] += 1
    counts[1, 31] += 1
    counts[2, 99] += 1
    assert torch.equal(h.seen.cpu(), words(seen)) and torch.equal(h.counts.cpu(), counts)
    h.clear()
    assert not h.seen.any() and not h.counts.any()
    record_tokens(h, torch.zeros(3, 0, dtype=torch.int32, device=DEV))


def test_captured_steps_penalise_what_they_chose():
    """A captured step that records: each replay goes on from the history the last one left."""
    rows, vocab = 2, 6000
    z = torch.zeros(rows, vocab)
    z[:, 10], z[:, 4000], z[:, 20] = 3.0, 2.5, 2.0
    h = TokenHistory.empty(rows, vocab, DEV)
    freq = torch.ones(rows, device=DEV)
    x = z.to(DEV)
    adjust_logits(x, history=h, frequency=freq)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _, nxt = adjust_logits(x, history=h, frequency=freq, record=True)
    chosen = []
    for _ in range(5):
        g.replay()
        chosen.append(nxt.tolist()[0])
    assert chosen == [10, 4000, 10, 20, 4000]  # 3 | 2.5 | 2 (10, before 20) | 2 (20) | 1.5 (4000)


def test_refusals():
    z = torch.zeros(2, 64, device=DEV)
    h = TokenHistory.empty(2, 64, DEV)
    f = torch.ones(2, device=DEV)
    ids, vals = torch.zeros(2, 3, dtype=torch.int32, device=DEV), torch.zeros(2, 3, device=DEV)
    for bad in (dict(repetition=f), dict(record=True), dict(history=TokenHistory.empty(2, 65, DEV)),
                dict(history=TokenHistory.empty(1, 64, DEV)), dict(history=h, frequency=f[:1]),
                dict(history=h, presence=f.double()), dict(bias_ids=ids), dict(bias_ids=ids[:1], bias_values=vals[:1]),
                dict(allowed=torch.zeros(3, dtype=torch.int32, device=DEV)), dict(out=torch.zeros(2, 63, device=DEV)),
                dict(out=torch.zeros(2, 64, dtype=torch.float16, device=DEV))):
        with pytest.raises(ValueError):
            adjust_logits(z, **bad)
    for bad in (dict(bias_ids=ids.long(), bias_values=vals), dict(bias_ids=ids, bias_values=vals.half()),
                dict(allowed=torch.zeros(2, dtype=torch.int64, device=DEV))):
        with pytest.raises(TypeError):
            adjust_logits(z, **bad)
    with pytest.raises(TypeError):
        adjust_logits(z.double())
    with pytest.raises(ValueError):
        adjust_logits(z[0])
    with pytest.raises(RuntimeError):
        adjust_logits(z.cpu())
    with pytest.raises(TypeError):
        record_tokens(h, ids.long())
    with pytest.raises(ValueError):
        record_tokens(h, torch.zeros(3, 1, dtype=torch.int32, device=DEV))
    with pytest.raises(TypeError):
        TokenHistory(h.seen.long(), h.counts)
    with pytest.raises(ValueError):
        TokenHistory(h.seen[:, :1], h.counts)
    got, nxt = adjust_logits(z[:0])
    assert got.shape == (0, 64) and nxt.shape == (0,)


@pytest.mark.parametrize("rows,vocab,share", [(40, 9001, 0.05), (80, 32000, 0.5), (300, 4097, 1.0), (149, 131, 1.0),
                                              (2, 1 << 20, 0.3)])
def test_many_rows_and_dense_histories(rows, vocab, share):
    """More rows than clusters fit at once; histories up to every token; the largest vocabulary; many biases."""
    g = torch.Generator().manual_seed(rows)
    z = 3 * torch.randn(rows, vocab, generator=g)
    seen, counts, h = history(rows, vocab, 5, share)
    if share == 1.0:
        seen[:], counts[counts == 0] = True, 3
        h = TokenHistory(words(seen).to(DEV), counts.to(DEV))
    rep, freq, pres = 1 + torch.rand(rows, generator=g), torch.rand(rows, generator=g), torch.rand(rows, generator=g) - .5
    many = 700
    ids = torch.stack([torch.randperm(max(vocab, many), generator=g)[:many] for _ in range(rows)]).int()
    values = torch.randn(rows, many, generator=g)
    allowed = torch.rand(rows, vocab, generator=g) < 0.7
    allowed[:, 0] = True
    # no id comes twice: the sums are the values, and one indexed add does them all
    want = formula(z, seen, counts, rep, freq, pres)
    inside = ids < vocab
    r = torch.arange(rows)[:, None].expand_as(ids)[inside]
    want[r, ids[inside].long()] += values[inside]
    want = torch.where(allowed, want, torch.full_like(want, -float("inf")))
    d = lambda t: t.to(DEV)  # noqa: E731
    got, nxt = adjust_logits(d(z), history=h, repetition=d(rep), frequency=d(freq), presence=d(pres), bias_ids=d(ids),
                             bias_values=d(values), allowed=d(words(allowed)), record=True)
    assert torch.equal(got.cpu(), want) and torch.equal(nxt.cpu(), lowest_best(want))
    counts[torch.arange(rows), nxt.cpu().long()] += 1
    seen[torch.arange(rows), nxt.cpu().long()] = True
    assert torch.equal(h.counts.cpu(), counts) and torch.equal(h.seen.cpu(), words(seen))


def test_a_full_list_of_biases():
    vocab, many = 70000, 65536
    g = torch.Generator().manual_seed(6)
    ids = torch.randperm(vocab, generator=g)[None, :many].int()
    values = torch.randn(1, many, generator=g)
    z = torch.randn(1, vocab, generator=g)
    want = z.clone()
    want[0, ids[0].long()] += values[0]
    got, nxt = adjust_logits(z.to(DEV), bias_ids=ids.to(DEV), bias_values=values.to(DEV))
    assert torch.equal(got.cpu(), want) and int(nxt) == int(want.argmax())
