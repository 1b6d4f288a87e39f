"""GPU: the decoder over a paged cache (Qwen3EXL3.forward_paged) and the engine that batches, drafts and verifies."""
import pytest
import torch

from oracle import model_oracle, oracle as O
from test_model_gpu import _small_model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("chunks", [[24], [1, 7, 16], [9, 9, 1, 1, 4]])
def test_paged_logits_match_the_oracle(cuda, chunks):
    """A prompt fed in chunks, another sequence beside it: logits as the fp32 oracle's (the bound of the dense path)."""
    model = _small_model(cuda, fuse=True)
    cache = model.make_paged_cache(64, 16)
    cache.add("a"), cache.add("b")
    prompt = (torch.arange(24) * 37 % 2048).tolist()
    at, logits = 0, []
    for n in chunks:
        batch = cache.extend([("b", 3), ("a", n)])
        toks = torch.tensor([1, 2, 3] + prompt[at:at + n], device=cuda)
        logits.append(model.forward_paged(toks, cache, batch)[3:])
        at += n
    got = torch.cat(logits).float().cpu().numpy()
    dense = model.make_cache(64)
    ck = [c.float().cpu().numpy() for c in dense.k]
    cv = [c.float().cpu().numpy() for c in dense.v]
    ref = model_oracle.forward(model, torch.tensor(prompt).numpy(), ck, cv, 0)
    assert O.kl_div(ref, got[:, :ref.shape[1]]).mean() < 1e-4


def test_paged_rows_can_be_picked(cuda):
    model = _small_model(cuda, fuse=False, layers=1)
    cache = model.make_paged_cache(16, 16)
    cache.add(0)
    batch = cache.extend([(0, 12)])
    toks = torch.arange(12, device=cuda)
    every = model.forward_paged(toks, cache, batch)
    cache.truncate(0, 0)
    batch = cache.extend([(0, 12)])
    some = model.forward_paged(toks, cache, batch, torch.tensor([11, 3], device=cuda))
    # the head's product has another row count (GEMV or GEMM): equal within its fp16 input and bf16 output rounding
    assert torch.allclose(every[[11, 3]].float(), some.float(), rtol=2e-2, atol=2e-2 * float(every.abs().max()))


def _assert_greedy(model, prompt, new):
    """Each generated token is the largest logit of the whole text fed at once, within the rounding of two paths."""
    cache = model.make_paged_cache(64, 32)
    cache.add(0)
    text = prompt + new
    batch = cache.extend([(0, len(text))])
    logits = model.forward_paged(torch.tensor(text, device=model.rope_cos.device), cache, batch).float()
    rows = logits[len(prompt) - 1:len(text) - 1]
    top = rows.max(-1).values
    got = rows.gather(1, torch.tensor(new, device=rows.device)[:, None])[:, 0]
    assert (got >= top - 3e-2 * rows.abs().amax(-1)).all()


@pytest.mark.parametrize("max_drafts,chunk", [(0, 512), (4, 512), (7, 16), (3, 5)])
def test_engine_greedy(cuda, max_drafts, chunk):
    from omlx_exl3_b200.serving import PagedEngine
    model = _small_model(cuda, fuse=True)
    prompts = [[5, 6, 7, 8] * 6, list(range(40, 90)), [3], [9, 9, 9, 9, 9, 9]]
    engine = PagedEngine(model, num_pages=40, page_size=16, chunk=chunk, max_drafts=max_drafts)
    out = engine.generate(prompts, 21)
    assert [len(o) for o in out] == [21] * 4 and engine.running == 0 and engine.cache.free_pages == 40
    for p, o in zip(prompts, out):
        _assert_greedy(model, p, o)
    if max_drafts:
        assert engine.drafted > 0 and 0 <= engine.accepted <= engine.drafted


def test_engine_takes_right_drafts_and_drops_wrong_ones(cuda):
    """A proposer that knows the greedy text gets every draft accepted, so a step yields drafts + 1 tokens; one that is
    always wrong gets none, and the text is the same."""
    from omlx_exl3_b200.serving import PagedEngine
    model = _small_model(cuda, fuse=True)
    prompt = list(range(100, 120))
    plain = PagedEngine(model, 20, 16, max_drafts=0).generate([prompt], 16)[0]
    _assert_greedy(model, prompt, plain)
    text = prompt + plain
    wrong = PagedEngine(model, 20, 16, max_drafts=3, propose=lambda t, n: [(text[len(t) + i] + 1) % 2048 for i in range(min(n, len(text) - len(t)))])
    out = wrong.generate([prompt], 16)[0]
    _assert_greedy(model, prompt, out)
    if out == plain:
        assert wrong.accepted == 0 and wrong.drafted > 0
    right = PagedEngine(model, 20, 16, max_drafts=3, propose=lambda t, n: text[len(t):len(t) + n])
    out = right.generate([prompt], 16)[0]
    _assert_greedy(model, prompt, out)
    if out == plain:
        assert right.accepted == right.drafted > 0


def test_engine_stops_samples_and_refuses(cuda):
    from omlx_exl3_b200.serving import PagedEngine
    model = _small_model(cuda, fuse=True, layers=1)
    engine = PagedEngine(model, 20, 16, seed=3)
    greedy = engine.generate([[1, 2, 3]], 8)[0]
    stopped = PagedEngine(model, 20, 16).generate([[1, 2, 3]], 8, stop=[greedy[2]])[0]
    assert stopped == greedy[:greedy.index(greedy[2]) + 1]
    a = PagedEngine(model, 20, 16, seed=5).generate([[1, 2, 3], [4, 5]], 12, temperature=1.0)
    b = PagedEngine(model, 20, 16, seed=5).generate([[1, 2, 3], [4, 5]], 12, temperature=1.0)
    c = PagedEngine(model, 20, 16, seed=6).generate([[1, 2, 3], [4, 5]], 12, temperature=1.0)
    assert a == b and a != c
    for bad in (dict(prompt=[], max_new=3), dict(prompt=[1], max_new=0), dict(prompt=[1], max_new=5000), dict(prompt=[1], max_new=2, temperature=-1.0)):
        with pytest.raises(ValueError):
            engine.add("x", **bad)
    engine.add("long", list(range(400)), 4)                            # 25 pages, of 20
    with pytest.raises(MemoryError):
        for _ in range(10):
            engine.step()


def test_no_rows_wanted_means_no_head(cuda):
    """A step of prompt chunks alone: the cache is filled, the vocabulary's projection is not run."""
    model = _small_model(cuda, fuse=False, layers=1)
    cache = model.make_paged_cache(16, 16)
    cache.add(0)
    ran = []
    hook = model.lm_head.register_forward_hook(lambda *a: ran.append(1))
    out = model.forward_paged(torch.arange(12, device=cuda), cache, cache.extend([(0, 12)]), torch.empty(0, dtype=torch.int64, device=cuda))
    assert out.shape == (0, model.lm_head.out_features) and not ran and cache.k[0].any()
    batch = cache.extend([(0, 1)])
    assert model.forward_paged(torch.tensor([12], device=cuda), cache, batch).shape[0] == 1 and ran == [1]
    hook.remove()
