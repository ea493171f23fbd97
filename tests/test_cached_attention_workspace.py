"""The scratch of an attention call stays the call's own until its launches
are queued.

Torch's allocator hands a freed block to the next tensor of the same stream,
and ctypes lets other Python threads run during a call into the library: a
workspace that is free before the call returns may become another thread's
tensor between the call's launches.
"""
import threading
import weakref

import pytest
import torch

from gsq_b200 import _lib
from gsq_b200.runtime import QuantizedKVCache
from gsq_b200.runtime.kernels import cached_attention, kv_append


def test_the_workspace_lives_until_the_call_returns(monkeypatch):
    """Without a GPU: the tensors that the call allocates, and the addresses that it passes on."""
    cache = object.__new__(QuantizedKVCache)
    cache.batch, cache.heads, cache.length, cache.dim = 1, 2, 9000, 128
    cache.fmt, cache.device, cache.pointers, cache.checked = 0, torch.device("cpu"), (0, 0, 0, 0), {}
    made, alive = {}, []
    plain = torch.Tensor.new_empty

    def new_empty(self, *args, **kwargs):
        t = plain(self, *args, **kwargs)
        made[t.data_ptr()] = weakref.ref(t)
        return t

    def launch(device, fn, *args):
        alive.extend((at, made[at]() is not None) for at in args if isinstance(at, int) and at in made)

    monkeypatch.setattr(torch.Tensor, "new_empty", new_empty)
    monkeypatch.setattr(_lib, "launch", launch)
    for n in (1, 40):  # tokens over a long cache, row blocks
        made.clear()
        alive.clear()
        q = torch.zeros(1, n, 12, 128, dtype=torch.float16)
        out = cached_attention(q, cache, torch.zeros(1, dtype=torch.int32))
        assert len(alive) == 2 and all(a for _, a in alive)  # out and the workspace
        assert out.data_ptr() in dict(alive)


@pytest.mark.gpu
def test_two_threads_on_one_stream():
    """A long cache (tiles split evenly, then joined) in one thread, a chunk (row blocks, then joined) in the other, both on
    the default stream: what each gives alone, bit for bit."""
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(1)
    calls = []
    for n, cap, dim in ((1, 20011, 256), (90, 5003, 128)):
        cache = QuantizedKVCache.empty(1, 2, cap, dim, "int8", dev)
        k, v = (torch.randn(1, cap, 2, dim, generator=g, device=dev) for _ in range(2))
        kv_append(cache, k, v, torch.zeros(1, dtype=torch.int32, device=dev))
        q = torch.randn(1, n, 12, dim, generator=g, device=dev).half()
        assert _lib.load().gsq_cached_attention_workspace_size(1, n, 12, 2, dim, cap) > 0
        calls.append((q, cache, torch.tensor([cap - n], dtype=torch.int32, device=dev)))
    want = [cached_attention(*c).clone() for c in calls]
    torch.cuda.synchronize()
    wrong, begin = [], threading.Barrier(2)

    def work(i):
        begin.wait()
        for _ in range(300):
            got = cached_attention(*calls[i])
            if not torch.equal(got, want[i]):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    torch.cuda.synchronize()
    assert _lib.device_status(dev) == 0
