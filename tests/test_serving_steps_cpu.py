"""CPU: the engine's steps over a stand-in for the decoder, undisturbed and disturbed."""
import pytest

from omlx_exl3_b200 import serving
from omlx_exl3_b200.serving import PagedEngine
from serving_util import HistoryModel, greedy_text, on_cpu

PROMPTS = [[1, 2, 3, 1, 2, 3, 1], list(range(30, 70)), [5], [9, 9, 9, 9]]


@pytest.fixture(autouse=True)
def _cpu(monkeypatch):
    on_cpu(monkeypatch)


def _run(engine, out=None):
    """Steps until nothing runs; the tokens of each key."""
    out = {} if out is None else out
    for _ in range(2000):
        if not engine.running:
            return out
        for key, tokens in engine.step().items():
            out.setdefault(key, []).extend(tokens)
    raise AssertionError("the engine does not finish")


def _state(engine):
    return ({k: engine.cache.length(k) for k in engine._seqs}, engine.cache.free_pages,
            {k: (list(s.tokens), list(s.new)) for k, s in engine._seqs.items()})


def _mostly_right(tokens, most):
    """Drafts of the true text, some of them wrong."""
    want = greedy_text(tokens, most)
    return [t if (len(tokens) + i) % 3 else (t + 1) % 97 for i, t in enumerate(want)]


@pytest.mark.parametrize("chunk,drafts", [(512, 0), (7, 4), (1, 2)])
def test_undisturbed(chunk, drafts):
    engine = PagedEngine(HistoryModel(), 40, 16, chunk=chunk, max_drafts=drafts, propose=_mostly_right)
    assert engine.generate(PROMPTS, 13) == [greedy_text(p, 13) for p in PROMPTS]
    assert engine.cache.free_pages == 40


class Broken(Exception):
    pass


@pytest.mark.parametrize("part", ["forward", "gather", "verify", "status", "noise"])
@pytest.mark.parametrize("when", [1, 2, 4])
def test_a_step_that_raises_changes_nothing(monkeypatch, part, when):
    """Whatever fails within a step, sequences and pages are as before it, and the next steps write the undisturbed text."""
    calls = []

    def once(result):
        def f(*args, **kw):
            calls.append(1)
            if len(calls) == when:
                raise Broken
            return result(*args, **kw)
        return f
    model = HistoryModel()
    engine = PagedEngine(model, 40, 16, chunk=16, max_drafts=3, propose=_mostly_right, check_every=1)
    if part == "forward":
        model.fail = once(lambda step: None)
    elif part == "gather":
        model.gather_logits = once(lambda x: x)
    elif part == "noise":
        monkeypatch.setattr(serving.torch, "rand", once(serving.torch.rand))
    else:
        name = {"verify": "verify_drafts", "status": "check_paged_status"}[part]
        monkeypatch.setattr(serving, name, once(getattr(serving, name)))
    for i, p in enumerate(PROMPTS):
        engine.add(i, p, 13)
    out, before, raised = {}, None, 0
    while engine.running:
        before = _state(engine)
        try:
            for key, tokens in engine.step().items():
                out.setdefault(key, []).extend(tokens)
        except Broken:
            raised += 1
            assert _state(engine) == before
    assert raised == 1
    assert [out[i] for i in range(len(PROMPTS))] == [greedy_text(p, 13) for p in PROMPTS]
    assert engine.cache.free_pages == 40


@pytest.mark.parametrize("at", [0, 1, 5])
def test_a_sequence_without_probabilities_leaves_alone(at):
    """One sequence's logits become NaN after some tokens: it leaves with what it had and is named; the others' text is their own."""
    bad = PROMPTS[1]
    model = HistoryModel(spoil=lambda text: text[:len(bad)] == bad and len(text) >= len(bad) + at)
    engine = PagedEngine(model, 40, 16, chunk=16, max_drafts=3, propose=_mostly_right)
    for i, p in enumerate(PROMPTS):
        engine.add(i, p, 13)
    out = _run(engine)
    assert list(engine.failed) == [1] and "no probabilities" in engine.failed[1]
    assert out.pop(1, []) == greedy_text(bad, 13)[:at]
    assert out == {i: greedy_text(p, 13) for i, p in enumerate(PROMPTS) if i != 1}
    assert engine.cache.free_pages == 40
    engine.add(1, [4], 2)
    assert not engine.failed and _run(engine) == {1: greedy_text([4], 2)}
    with pytest.raises(RuntimeError, match="no probabilities"):
        PagedEngine(model, 40, 16).generate(PROMPTS, 13)


def test_steps_of_prompt_chunks_ask_for_no_logits():
    """Only a prompt's last row and decoded rows need logits: a step without any asks for none."""
    model = HistoryModel()
    engine = PagedEngine(model, 40, 16, chunk=8, max_drafts=0)
    assert engine.generate([PROMPTS[1]], 3) == [greedy_text(PROMPTS[1], 3)]
    assert model.fed == [8] * 5 + [1, 1] and model.asked == [0] * 4 + [1, 1, 1]


@pytest.mark.parametrize("propose", [
    lambda t, n: [97] * n, lambda t, n: greedy_text(t, n)[:1] + [-1] * (n - 1), lambda t, n: [2 ** 40], lambda t, n: greedy_text(t, n + 6),
    lambda t, n: tuple(greedy_text(t, n)),
])
def test_proposers_that_offer_too_much(propose):
    """Drafts outside the vocabulary never reach the embedding, and no more than max_drafts are fed."""
    model = HistoryModel()
    engine = PagedEngine(model, 40, 16, max_drafts=2, propose=propose)
    assert engine.generate([PROMPTS[0]], 9) == [greedy_text(PROMPTS[0], 9)]
    assert max(model.fed[1:]) <= 3


def test_add_refuses_tokens_that_the_model_does_not_have():
    engine = PagedEngine(HistoryModel(), 40, 16)
    for prompt in ([97], [1, -1, 2], [2 ** 40]):
        with pytest.raises(ValueError, match="vocabulary"):
            engine.add("x", prompt, 3)
    with pytest.raises(ValueError):
        engine.add("x", [1], 3, temperature=float("nan"))
    assert engine.running == 0 and engine.step() == {}
    engine.add("x", [96, 0], 3)
    assert _run(engine) == {"x": greedy_text([96, 0], 3)}


@pytest.mark.parametrize("kw", [dict(chunk=0), dict(chunk=-1), dict(max_drafts=-1)])
def test_engine_refuses_sizes_that_it_cannot_step_with(kw):
    with pytest.raises(ValueError):
        PagedEngine(HistoryModel(), 40, 16, **kw)


def test_generate_beside_other_sequences_is_refused():
    """It would take the others' tokens and lose them."""
    engine = PagedEngine(HistoryModel(), 40, 16)
    engine.add("mine", PROMPTS[0], 6)
    with pytest.raises(ValueError, match="running"):
        engine.generate([PROMPTS[2]], 4)
    assert _run(engine) == {"mine": greedy_text(PROMPTS[0], 6)}
    assert engine.generate([PROMPTS[2]], 4) == [greedy_text(PROMPTS[2], 4)]


def test_generate_that_raises_leaves_nothing_behind():
    """A prompt that is refused, a step that fails: the engine is empty again and the next call is a fresh one."""
    def fail(step):
        if step == 2:
            raise Broken
    model = HistoryModel(fail)
    engine = PagedEngine(model, 40, 16)
    with pytest.raises(ValueError):
        engine.generate([PROMPTS[0], []], 5)
    assert engine.running == 0 and engine.cache.free_pages == 40
    with pytest.raises(Broken):
        engine.generate(PROMPTS, 5)
    assert engine.running == 0 and engine.cache.free_pages == 40
    assert engine.generate(PROMPTS, 5) == [greedy_text(p, 5) for p in PROMPTS]


@pytest.mark.parametrize("pages", [6, 7, 8, 9, 12, 20])
@pytest.mark.parametrize("chunk,drafts", [(512, 3), (5, 0), (16, 3)])
def test_a_nearly_full_pool_finishes_everything(pages, chunk, drafts):
    """16 positions a page: each sequence alone needs up to 6 pages, all together 20. Whatever is short waits, or is read again."""
    prompts = [list(range(10 + i, 10 + i + n)) for i, n in enumerate((40, 3, 58, 20, 1))]
    engine = PagedEngine(HistoryModel(), pages, 16, chunk=chunk, max_drafts=drafts, propose=_mostly_right)
    for i, p in enumerate(prompts):
        engine.add(i, p, 35)
    assert _run(engine) == {i: greedy_text(p, 35) for i, p in enumerate(prompts)}
    assert engine.cache.free_pages == pages


def test_what_the_pool_can_never_hold_does_not_stop_the_others():
    """A prompt longer than the pool, and a sequence that outgrows it: the others finish, then MemoryError names them; cancelled,
    they are gone."""
    engine = PagedEngine(HistoryModel(), 6, 16, chunk=16, max_drafts=0)
    engine.add("long", [7] * 97, 2)
    engine.add("grows", [8] * 60, 60)
    for i, p in enumerate(PROMPTS):
        engine.add(i, p, 13)
    out = {}
    with pytest.raises(MemoryError, match="'long', 'grows'"):
        _run(engine, out)
    assert out.pop("grows") == greedy_text([8] * 60, 37)               # its 97th token needs a position for its 98th
    assert out == {i: greedy_text(p, 13) for i, p in enumerate(PROMPTS)}
    with pytest.raises(MemoryError):
        engine.step()
    engine.cancel("long")
    engine.cancel("grows")
    assert engine.running == 0 and engine.cache.free_pages == 6 and engine.step() == {}
    with pytest.raises(KeyError):
        engine.cancel("long")


def test_cancel_in_the_middle():
    engine = PagedEngine(HistoryModel(), 40, 16, chunk=16, max_drafts=2, propose=_mostly_right)
    for i, p in enumerate(PROMPTS):
        engine.add(i, p, 13)
    out = {}
    for _ in range(3):
        for key, tokens in engine.step().items():
            out.setdefault(key, []).extend(tokens)
    engine.cancel(1)
    out.pop(1, None)
    assert _run(engine, out) == {i: greedy_text(p, 13) for i, p in enumerate(PROMPTS) if i != 1}
    assert engine.cache.free_pages == 40
