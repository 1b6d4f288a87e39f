"""GPU: the engine where a step fails or pages are short, over a small decoder."""
import pytest
import torch

from test_model_gpu import _small_model
from test_serving_gpu import _assert_greedy

pytestmark = pytest.mark.gpu

PROMPTS = [[5, 6, 7, 8] * 6, list(range(40, 90)), [3], [9, 9, 9, 9, 9, 9]]


def _finish(engine):
    out, raised = {}, 0
    while engine.running:
        try:
            for key, tokens in engine.step().items():
                out.setdefault(key, []).extend(tokens)
        except ZeroDivisionError:
            raised += 1
    return out, raised


def test_a_small_pool(cuda):
    """Five pages of the ten that the sequences need at once: prompts wait, and one is read again."""
    from omlx_exl3_b200.serving import PagedEngine
    model = _small_model(cuda, fuse=True, layers=1)
    engine = PagedEngine(model, num_pages=5, page_size=16, chunk=16, max_drafts=3)
    out = engine.generate(PROMPTS, 21)
    for p, o in zip(PROMPTS, out):
        assert len(o) == 21
        _assert_greedy(model, p, o)
    assert engine.cache.free_pages == 5


@pytest.mark.parametrize("when", [1, 4])
def test_a_forward_pass_that_raises(cuda, when):
    """After the pages were written: the next step feeds the same rows, and the text is a greedy one."""
    from omlx_exl3_b200.serving import PagedEngine
    model = _small_model(cuda, fuse=True, layers=1)
    engine = PagedEngine(model, num_pages=40, page_size=16, chunk=32, max_drafts=3)
    for i, p in enumerate(PROMPTS):
        engine.add(i, p, 12)
    calls, forward = [], model.forward_paged

    def once(*args, **kw):
        calls.append(1)
        logits = forward(*args, **kw)
        if len(calls) == when:
            raise ZeroDivisionError
        return logits
    model.forward_paged = once
    out, raised = _finish(engine)
    del model.forward_paged
    assert raised == 1 and engine.cache.free_pages == 40
    for i, p in enumerate(PROMPTS):
        assert len(out[i]) == 12
        _assert_greedy(model, p, out[i])


def test_nan_logits_of_one_sequence(cuda):
    """One sequence's rows are NaN from its third token on: it leaves, named, and the others' text is a greedy one."""
    from omlx_exl3_b200.serving import PagedEngine
    model = _small_model(cuda, fuse=True, layers=1)
    engine = PagedEngine(model, num_pages=40, page_size=16, chunk=512, max_drafts=0)
    for i, p in enumerate(PROMPTS):
        engine.add(i, p, 12)
    gather, steps = model.gather_logits, []

    def spoiled(local):
        logits = gather(local).clone()
        steps.append(1)
        if len(steps) == 3:
            logits[1] = float("nan")
        return logits
    model.gather_logits = spoiled
    out, _ = _finish(engine)
    del model.gather_logits
    assert list(engine.failed) == [1] and len(out[1]) == 2 and engine.cache.free_pages == 40
    for i in (0, 2, 3):
        assert len(out[i]) == 12
        _assert_greedy(model, PROMPTS[i], out[i])
