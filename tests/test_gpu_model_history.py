"""The token history of a model with controlled logits: the prompt, and the
tokens that were chosen and went on, however the prompt came."""
import pytest
import torch

from gsq_b200.models import build_qwen35
from gsq_b200.runtime import TokenHistory
from test_gpu_model import CFG, TOL, rel, setup  # noqa: F401
from test_gpu_model_cache import EXTRA, fine, prompt

pytestmark = pytest.mark.gpu


def controlled(w, dev, B=1, **more):
    model = build_qwen35(w, CFG, dev, max_len=96, max_batch=B, kv_format="int8")
    h = TokenHistory.empty(B, CFG.vocab_size, dev)
    model.control_logits(history=h, frequency=torch.full((B,), 1e3, device=dev),
                         repetition=torch.full((B,), 1.5, device=dev), **more)
    return model, h


def seen(h):
    return ((h.seen.cpu()[:, :, None] >> torch.arange(32)) & 1 > 0).reshape(h.rows, -1)[:, :h.vocab]


@pytest.mark.parametrize("parts", [(9, 14), (8, 8, 7)])
def test_a_prompt_in_parts_has_the_whole_ones_history(setup, parts):  # noqa: F811
    dev, w = setup
    ids = prompt(sum(parts), dev)
    (whole, a), (piecewise, b) = controlled(w, dev), controlled(w, dev)
    want = whole.prefill(ids).clone()
    at = 0
    for i, n in enumerate(parts):
        got = (piecewise.prefill if i == 0 else piecewise.extend)(ids[at:at + n])
        at += n
    assert torch.equal(a.seen, b.seen) and torch.equal(a.counts, b.counts)
    assert rel(got, want) <= TOL + EXTRA["int8"]
    only = torch.zeros(1, CFG.vocab_size, dtype=torch.bool)
    only[0, ids.cpu().long()] = True
    assert torch.equal(seen(b), only) and not b.counts.any()
    # the last part's token goes on, and counts from then on
    token = int(piecewise.cur_id[0])
    piecewise.decode_step()
    assert int(b.counts[0, token]) == 1 and int(b.counts.sum()) == 2  # and the one chosen now
    fine(dev)


def test_a_token_of_the_callers_own_takes_the_chosen_ones_place(setup):  # noqa: F811
    dev, w = setup
    B = 2
    model, h = controlled(w, dev, B)
    model.prefill(prompt(9, dev))
    model.fork(B)
    chosen = int(model.cur_id[0])
    want, counts = seen(h), torch.zeros(B, CFG.vocab_size, dtype=torch.int32)
    with pytest.raises(ValueError):
        model.decode_step([1, 2, 3])
    model.decode_step([(chosen + 1) % CFG.vocab_size, chosen])  # the second sequence is given the chosen one
    now = model.cur_id[:B].tolist()
    for b, t in ((1, chosen), (0, now[0]), (1, now[1])):
        want[b, t] = True
        counts[b, t] += 1
    assert torch.equal(seen(h), want) and torch.equal(h.counts.cpu(), counts)
    fine(dev)


@pytest.mark.parametrize("captured", [False, True])
def test_every_sequence_of_a_fork_records_the_prompts_token(setup, captured):  # noqa: F811
    """Also where the first step after the prompt is a replay."""
    dev, w = setup
    B = 3
    model, h = controlled(w, dev, B)
    ids = prompt(9, dev)

    def start():
        model.prefill(ids)
        model.fork(B)

    start()
    model.decode_step()  # sizes the workspaces
    start()
    chosen = [model.cur_id[:B].clone()]
    if captured:
        model.capture_decode()
    for _ in range(3):
        model.replay_decode(1) if captured else model.decode_step()
        chosen.append(model.cur_id[:B].clone())
    counts = torch.zeros(B, CFG.vocab_size, dtype=torch.int32)
    for b in range(B):
        for t in torch.stack(chosen)[:, b].tolist():
            counts[b, t] += 1
    assert torch.equal(h.counts.cpu(), counts)
    fine(dev)


def test_the_history_of_the_prompt_is_the_one_that_learns_its_token(setup):  # noqa: F811
    """Penalties taken away, or changed, between a prompt and the first step."""
    dev, w = setup
    for change in (dict(), "same"):
        model, h = controlled(w, dev)
        model.prefill(prompt(9, dev))
        token = int(model.cur_id[0])
        model.control_logits(**(dict(history=h, presence=torch.ones(1, device=dev)) if change == "same" else change))
        model.decode_step()
        assert int(h.counts[0, token]) >= 1
    # a prompt without a history leaves nothing to record
    model = build_qwen35(w, CFG, dev, max_len=96, kv_format="int8")
    model.prefill(prompt(9, dev))
    h = TokenHistory.empty(1, CFG.vocab_size, dev)
    model.control_logits(history=h)
    model.decode_step()
    assert int(h.counts.sum()) == 1 and int(h.counts[0, int(model.cur_id[0])]) == 1
    fine(dev)
