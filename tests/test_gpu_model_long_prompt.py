"""A prompt of more tokens than one call of the cache's write takes (65535)."""
import pytest
import torch

from gsq_b200.models import build_qwen35
from test_gpu_model import CFG, TOL, rel, setup  # noqa: F401
from test_gpu_model_cache import EXTRA, fine, prompt

pytestmark = pytest.mark.gpu


def test_a_long_prompt_at_once_and_in_two_calls(setup):  # noqa: F811
    dev, w = setup
    n = 65535 + 40
    ids = prompt(n, dev)
    model = build_qwen35(w, CFG, dev, max_len=n + 8, kv_format="int8")
    whole = model.prefill(ids).clone()
    assert model.n_pos == n and int(model.pos) == n
    step = model.decode_step(3).clone()
    model.prefill(ids[:30000])
    halves = model.extend(ids[30000:])
    assert rel(halves, whole) <= TOL + EXTRA["int8"]
    assert rel(model.decode_step(3), step) <= TOL + EXTRA["int8"]
    fine(dev)


def test_a_long_extension(setup):  # noqa: F811
    dev, w = setup
    n = 65535 + 100
    ids = prompt(n + 9, dev)
    model = build_qwen35(w, CFG, dev, max_len=n + 9, kv_format="fp8")
    model.prefill(ids[:9])
    more = model.extend(ids[9:]).clone()
    assert model.n_pos == n + 9
    model.prefill(ids[:40009])
    assert rel(model.extend(ids[40009:]), more) <= TOL + EXTRA["fp8"]
    with pytest.raises(ValueError):
        model.extend(ids[:1])
    fine(dev)
