"""What the entry points of the quantised cache, its attention and the logits refuse, before any launch (host-side
checks only: the pointers are not memory)."""
import ctypes

import pytest
import torch

from gsq_b200 import _lib
from gsq_b200.runtime import QuantizedKVCache, TokenHistory
from gsq_b200.runtime.kernels import adjust_logits, tree_mask

P = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 2)
STRIDES = (ctypes.c_int64 * 3)(768, 768, 128)
F32, F16 = _lib.DTYPE_CODES[torch.float32], _lib.DTYPE_CODES[torch.float16]


def call(name, values, **changes):
    assert set(changes) <= set(values)
    return getattr(_lib.load(), name)(*{**values, **changes}.values(), None)


CACHE = dict(fmt=0, kc=P, vc=P, ks=P, vs=P)
APPEND = dict(k=P, v=P, dtype=F16, batch=1, tokens=1, heads=2, dim=128, k_strides=STRIDES, v_strides=STRIDES, start=P,
              start_stride=1, counts=None, **CACHE, cap=64)
READ = dict(**CACHE, batch=1, heads=2, cap=64, dim=128, start=P, start_stride=1, counts=None, tokens=1, k=P, v=P,
            dtype=F16)
QKV = dict(qkv=P, stride=1024, batch=1, tokens=1, nq=1, nkv=1, qw=P, kw=P, eps=1e-6, rot=64, theta=1e4, start=P,
           start_stride=0, q=P, **CACHE, cap=64)
ATTEND = dict(q=P, dtype=F16, q_strides=STRIDES, batch=1, n=1, heads=6, kv_heads=2, dim=128, **CACHE, cap=9000, start=P,
              start_stride=1, counts=None, tree=None, tree_stride=0, gate=None, gate_strides=None, scale=0.1, out=P,
              workspace=P, bytes=1 << 40)
ADJUST = dict(logits=P, dtype=F32, stride=100, rows=1, vocab=100, seen=P, counts=P, rep=None, freq=None, pres=None,
              ids=None, values=None, biases=0, allowed=None, allowed_stride=0, out=P, next=P, record=0)
RECORD = dict(tokens=P, stride=4, rows=1, n=4, vocab=100, seen=P, counts=P, generated=1)
SIZE, ARG, ALIGN, WORKSPACE = _lib.GSQ_ERR_SIZE, _lib.GSQ_ERR_ARG, _lib.GSQ_ERR_ALIGN, _lib.GSQ_ERR_WORKSPACE


@pytest.mark.parametrize("name, values", [("gsq_kv_append", APPEND), ("gsq_kv_read", READ), ("gsq_qkv_append", QKV),
                                          ("gsq_cached_attention", ATTEND)])
def test_bad_caches(name, values):
    for bad, code in ((dict(fmt=2), ARG), (dict(fmt=-1), ARG), (dict(kc=None), ARG), (dict(vs=None), ARG),
                      (dict(vc=ODD), ALIGN), (dict(cap=0), SIZE), (dict(cap=(1 << 30) + 1), SIZE),
                      (dict(batch=-1), SIZE), (dict(start=None), ARG), (dict(start=ODD), ALIGN), (dict(ks=ODD), ALIGN)):
        assert call(name, values, **bad) == code, bad
    if "dim" in values:
        for dim in (0, 64, 192, 512):
            assert call(name, values, dim=dim) == SIZE
    assert call(name, values, batch=0) == 0  # nothing to do is no error
    assert name in _lib.last_error()


def test_bad_writes_and_reads():
    for name, values in (("gsq_kv_append", APPEND), ("gsq_kv_read", READ)):
        for bad, code in ((dict(dtype=9), ARG), (dict(tokens=-1), SIZE), (dict(tokens=1 << 30), SIZE),
                          (dict(heads=0), SIZE), (dict(heads=65536), SIZE), (dict(k=None), ARG), (dict(v=None), ARG)):
            assert call(name, values, **bad) == code, (name, bad)
        assert call(name, values, tokens=0) == 0
    assert call("gsq_kv_append", APPEND, k_strides=None) == ARG
    assert call("gsq_kv_append", APPEND, k=ctypes.c_void_p((1 << 20) + 1)) == ALIGN
    assert call("gsq_kv_read", READ, v=ODD) == ALIGN
    for bad, code in ((dict(stride=1023), SIZE), (dict(tokens=65536), SIZE), (dict(rot=3), SIZE), (dict(rot=258), SIZE),
                      (dict(nq=0), SIZE), (dict(q=None), ARG), (dict(q=ODD), ALIGN), (dict(qw=None), ARG)):
        assert call("gsq_qkv_append", QKV, **bad) == code, bad


def test_bad_attention():
    for bad, code in ((dict(dtype=F32), ARG), (dict(heads=5), SIZE), (dict(heads=0), SIZE), (dict(n=-1), SIZE),
                      (dict(n=65537), SIZE), (dict(n=1025, tree=P), SIZE), (dict(q=None), ARG), (dict(out=None), ARG),
                      (dict(q=ODD), ALIGN), (dict(out=ODD), ALIGN), (dict(gate=P), ARG),
                      (dict(q_strides=(ctypes.c_int64 * 3)(768, 768, 4)), ALIGN),
                      (dict(workspace=None), WORKSPACE), (dict(bytes=1024), WORKSPACE),
                      (dict(workspace=ODD), ALIGN), (dict(tree=ODD), ALIGN), (dict(counts=ODD), ALIGN),
                      (dict(batch=60000, n=60000), SIZE)):
        assert call("gsq_cached_attention", ATTEND, **bad) == code, bad
    assert call("gsq_cached_attention", ATTEND, n=0) == 0
    size = _lib.load().gsq_cached_attention_workspace_size
    assert size(1, 1, 6, 2, 128, 8192) == 0 < size(1, 1, 6, 2, 128, 8193)
    for nothing in ((0, 1, 6, 2, 128, 64), (1, 0, 6, 2, 128, 64), (1, 1, 6, 0, 128, 64), (1, 1, 1, 2, 128, 9000),
                    (1, 1, 6, 2, 100, 9000), (1 << 40, 1, 6, 2, 128, 9000), (1, 1 << 40, 6, 2, 128, 1 << 40)):
        size(*nothing)  # any answer: gsq_cached_attention refuses these; no crash


def test_bad_logits():
    for bad, code in ((dict(dtype=9), ARG), (dict(rows=-1), SIZE), (dict(rows=65536), SIZE), (dict(vocab=0), SIZE),
                      (dict(vocab=(1 << 20) + 1), SIZE), (dict(stride=99), SIZE), (dict(biases=65537), SIZE),
                      (dict(biases=-1), SIZE), (dict(biases=3), ARG), (dict(logits=None), ARG), (dict(out=None), ARG),
                      (dict(next=None), ARG), (dict(seen=None), ARG), (dict(counts=None), ARG),
                      (dict(seen=None, counts=None, record=1), ARG), (dict(seen=None, counts=None, rep=P), ARG),
                      (dict(out=ODD), ALIGN), (dict(counts=ODD), ALIGN), (dict(allowed=ODD), ALIGN)):
        assert call("gsq_adjust_logits", ADJUST, **bad) == code, bad
    assert call("gsq_adjust_logits", ADJUST, rows=0) == 0
    for bad, code in ((dict(tokens=None), ARG), (dict(seen=None), ARG), (dict(n=-1), SIZE), (dict(vocab=0), SIZE),
                      (dict(tokens=ODD), ALIGN)):
        assert call("gsq_record_tokens", RECORD, **bad) == code, bad
    assert call("gsq_record_tokens", RECORD, n=0) == 0


def test_there_is_no_cpu_path():
    with pytest.raises(RuntimeError, match="CUDA"):
        QuantizedKVCache.empty(1, 1, 8, 128, "int8", "cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        TokenHistory.empty(1, 8, "cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        adjust_logits(torch.zeros(1, 8))
    with pytest.raises(NotImplementedError):
        QuantizedKVCache.empty(1, 1, 8, 128, "int4", "cpu")
    with pytest.raises(ValueError):
        QuantizedKVCache.empty(1, 1, 8, 64, "int8", "cpu")


def test_tree_masks_are_ancestors():
    parents = [-1, 0, 0, 1, 3, -1, 5]
    m = tree_mask(parents, "cpu")
    for i in range(len(parents)):
        path, j = set(), i
        while j >= 0:
            path.add(j)
            j = parents[j]
        assert {j for j in range(32) if int(m[i, 0]) >> j & 1} == path
    assert tree_mask([], "cpu").shape == (0, 0)
    with pytest.raises(ValueError):
        tree_mask([0], "cpu")
