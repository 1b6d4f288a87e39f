"""GPU: verification of drafted tokens against a plain form in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _plain(target, tokens, cu, u, noise, max_drafts, draft=None, temp=None):
    """(tokens, count, accept_prob) from the definition, one sequence at a time, in 64 bits."""
    S = len(cu) - 1
    out = torch.full((S, max_drafts + 1), -1, dtype=torch.long)
    count, prob = torch.zeros(S, dtype=torch.int32), torch.zeros(target.shape[0] - S, dtype=torch.float64)

    def soft(x, t):
        x = x.double()
        if x.max() == float("-inf") or torch.isnan(x).any():
            return torch.zeros_like(x)
        if t == 0:
            p = torch.zeros_like(x)
            p[(x == x.max()).nonzero()[0, 0]] = 1
            return p
        return torch.softmax((x - x.max()) / t, -1)

    for s in range(S):
        t = 1.0 if temp is None else float(temp[s])
        n, left = 0, None
        for j in range(cu[s + 1] - cu[s] - 1):
            r = cu[s] + j
            i, x = r - s, int(tokens[r - s])
            p = soft(target[r], t)
            if draft is None or t == 0:
                q = torch.zeros_like(p)
                if 0 <= x < len(p):
                    q[x] = 1
            else:
                q = soft(draft[i], t)
            px, qx = (float(p[x]), float(q[x])) if 0 <= x < len(p) else (0.0, 0.0)
            prob[i] = min(1.0, px / qx) if qx > 0 else float(px > 0)
            if left is None and n == j and j < max_drafts:
                if float(u[i]) < float(prob[i]):
                    out[s, j] = x
                    n += 1
                else:
                    left = (p - q).clamp(min=0)
                    left = left if left.max() > 0 else p
        if left is None:
            left = soft(target[cu[s] + n], t)
        race = left / noise[s].double()
        if t == 0:
            race = left
        out[s, n] = int((race == race.max()).nonzero()[0, 0]) if race.max() > 0 else -1
        count[s] = n + 1
    return out, count, prob


def _inputs(rows, n, dtype, seed, agree=0.95):
    g = torch.Generator().manual_seed(seed)
    S, R = len(rows), sum(rows)
    target = 2 * torch.randn((R, n), generator=g)
    target.scatter_add_(1, torch.randint(0, n, (R, min(n, 6)), generator=g), 6 + torch.randn((R, min(n, 6)), generator=g))
    cu = [sum(rows[:i]) for i in range(S + 1)]
    drafted = torch.ones(R, dtype=torch.bool)
    drafted[torch.tensor(cu[1:]) - 1] = False
    draft = agree * target[drafted] + 0.7 * torch.randn((R - S, n), generator=g)
    tokens = (draft - torch.empty_like(draft).exponential_(generator=g).clamp_(min=1e-20).log()).argmax(1)
    noise = torch.empty((S, n)).exponential_(generator=g).clamp_(min=1e-20)
    u = torch.rand(R - S, generator=g)
    temp = torch.tensor([0.0, 0.7, 1.0, 1.3])[torch.randint(0, 4, (S,), generator=g)]
    return target.to(dtype), tokens, cu, u, noise, draft.to(dtype), temp


def _check(cuda, target, tokens, cu, u, noise, max_drafts, draft, temp):
    from omlx_exl3_b200 import verify_drafts
    dev = lambda t: None if t is None else t.to(cuda)                  # noqa: E731
    got = verify_drafts(dev(target), dev(tokens), torch.tensor(cu, dtype=torch.int32, device=cuda), dev(u), dev(noise),
                        max_drafts, draft_logits=dev(draft), temperature=dev(temp))
    want = _plain(target, tokens, cu, u, noise, max_drafts, draft, temp)
    # p / q of two fp32 softmaxes: exponents of up to 25 units rounded at 2^-24 each, times log2(e), and the sums
    assert torch.allclose(got[2].cpu().double(), want[2], rtol=2e-5, atol=1e-12)
    assert torch.equal(got[1].cpu(), want[1])
    assert torch.equal(got[0].cpu(), want[0])
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n", [
    ([1], 1), ([1], 7), ([2], 2), ([4], 1000), ([3, 1, 8, 1, 2], 32003), ([8] * 9, 4099), ([5], 151936),
    ([2, 8, 1] * 20, 515), ([16], 10007), ([1] * 70, 333),
])
@pytest.mark.parametrize("dist", [True, False])
def test_verify_matches_plain(cuda, dtype, rows, n, dist):
    x = _inputs(rows, n, dtype, seed=sum(rows) + n)
    target, tokens, cu, u, noise, draft, temp = x
    _check(cuda, target, tokens, cu, u, noise, max(rows) - 1, draft if dist else None, temp)
    _check(cuda, target, tokens, cu, u, noise, max(rows) + 2, draft if dist else None, None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_verify_masked_logits(cuda, dtype):
    """Forbidden tokens (-inf, or the type's lowest value), rows with nothing left, drafts that are forbidden."""
    target, tokens, cu, u, noise, draft, temp = _inputs([4, 4, 4, 4, 2, 1], 700, dtype, seed=5)
    gen = torch.Generator().manual_seed(6)
    low = torch.finfo(dtype).min
    target[torch.rand(target.shape, generator=gen) < 0.5] = float("-inf")
    target[4:8][torch.rand((4, 700), generator=gen) < 0.5] = low
    target[8] = float("-inf")                                          # nothing left in a judged row
    target[14] = low                                                   # all alike: the lowest value is no -inf
    target[18] = float("-inf")                                         # the only row of the last sequence
    draft[3][torch.rand(700, generator=gen) < 0.5] = float("-inf")
    target[1, tokens[1]] = float("-inf")
    temp = torch.tensor([1.0, 0.7, 1.0, 1.0, 0.0, 1.0])
    got = _check(cuda, target, tokens, cu, u, noise, 3, draft, temp)
    assert got[0][2].tolist() == [-1] * 4 and int(got[1][2]) == 1 and int(got[0][5, 0]) == -1


@pytest.mark.parametrize("dist", [True, False])
def test_verify_extreme_temperatures(cuda, dist):
    """Temperatures whose reciprocal is no fp32 number, or nearly none: as good as greedy, as good as uniform."""
    target, tokens, cu, u, noise, draft, _ = _inputs([3, 3, 3, 3], 900, torch.float32, seed=12)
    target[1, 5:80] = draft[1, 9:100] = float("-inf")
    temp = torch.tensor([1e-39, 1e-32, 1e35, 3e38])
    _check(cuda, target, tokens, cu, u, noise, 2, draft if dist else None, temp)


def test_verify_greedy_ties_and_foreign_drafts(cuda):
    """Equal logits: the first is the greedy token. Drafted ids outside the vocabulary are never accepted."""
    n = 5000
    target = torch.zeros((6, n))
    target[:, [17, 4000]] = 3.0
    tokens = torch.tensor([17, 17, 4000, -1, n])
    cu = [0, 6]
    temp = torch.zeros(1)
    u = torch.zeros(5)
    noise = torch.rand((1, n)) + 0.1
    got = _check(cuda, target, tokens, cu, u, noise, 5, None, temp)
    assert got[0][0].tolist() == [17, 17, 17, -1, -1, -1]
    for bad in (-1, n, 2 ** 40, -2 ** 40):
        _check(cuda, target, torch.tensor([bad] * 5), cu, u, noise, 5, None, torch.ones(1))
        _check(cuda, target, torch.tensor([bad] * 5), cu, u, noise, 5, target[:5].clone(), torch.ones(1))


def test_verify_identical_models_accept_everything(cuda):
    target, tokens, cu, u, noise, _, _ = _inputs([8, 8, 3], 20000, torch.float16, seed=9)
    drafted = [r for s in range(3) for r in range(cu[s], cu[s + 1] - 1)]
    got = _check(cuda, target, tokens, cu, u * 0.999, noise, 7, target[drafted].clone(), None)
    assert got[1].tolist() == [8, 8, 3]


@pytest.mark.parametrize("off,extra", [(0, 8), (8, 24), (1, 3)])
def test_verify_strided_rows(cuda, off, extra):
    """Rows inside wider buffers, aligned and not; what lies beside them is NaN."""
    from omlx_exl3_b200 import verify_drafts
    n = 2053
    target, tokens, cu, u, noise, draft, temp = _inputs([5, 2], n, torch.bfloat16, seed=10)

    def inside(x):
        w = torch.full((x.shape[0], n + extra), float("nan"), dtype=x.dtype)
        w[:, off:off + n] = x
        return w.to(cuda)[:, off:off + n]

    got = verify_drafts(inside(target), tokens.to(cuda), torch.tensor(cu, dtype=torch.int32, device=cuda), u.to(cuda),
                        inside(noise), 4, draft_logits=inside(draft), temperature=temp.to(cuda))
    want = _plain(target, tokens, cu, u, noise, 4, draft, temp)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    assert torch.allclose(got[2].cpu().double(), want[2], rtol=2e-5, atol=1e-12)


def test_verify_follows_the_target_distribution(cuda):
    """Whatever the draft, the first token is distributed as the target's p (the rule's whole point): 60,000 sequences with
    one draft each over 8 tokens; each frequency within 5 standard deviations."""
    from omlx_exl3_b200 import verify_drafts
    S, n = 60000, 8
    g = torch.Generator(device=cuda).manual_seed(12)
    p = torch.tensor([0.3, 0.02, 0.18, 0.1, 0.05, 0.25, 0.04, 0.06], device=cuda)
    q = torch.tensor([0.05, 0.3, 0.1, 0.1, 0.2, 0.05, 0.1, 0.1], device=cuda)
    tokens = torch.multinomial(q, S, replacement=True, generator=g)
    cu = torch.arange(0, 2 * S + 1, 2, dtype=torch.int32, device=cuda)
    u = torch.rand(S, device=cuda, generator=g)
    noise = torch.empty((S, n), device=cuda).exponential_(generator=g).clamp_(min=1e-20)
    out, _, _ = verify_drafts(p.log().expand(2 * S, n).contiguous(), tokens, cu, u, noise, 1,
                              draft_logits=q.log().expand(S, n).contiguous())
    got = torch.bincount(out[:, 0], minlength=n).double().cpu() / S
    want = p.double().cpu()
    assert ((got - want).abs() <= 5 * (want * (1 - want) / S).sqrt()).all()


def test_verify_repeats_and_graph(cuda):
    from omlx_exl3_b200 import verify_drafts
    target, tokens, cu, u, noise, draft, temp = (t if isinstance(t, list) else t.to(cuda)
                                                 for t in _inputs([4, 8, 1], 30001, torch.bfloat16, seed=13))
    cu = torch.tensor(cu, dtype=torch.int32, device=cuda)
    call = lambda: verify_drafts(target, tokens, cu, u, noise, 7, draft_logits=draft, temperature=temp)   # noqa: E731
    first = call()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, call()))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for seed in range(3):
        u.copy_(torch.rand(u.shape, generator=torch.Generator().manual_seed(seed)))
        g.replay()
        want = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
