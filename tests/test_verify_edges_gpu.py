"""GPU: verification of drafted tokens where logits, noise or tables are out of the ordinary."""
import pytest
import torch

from test_verify_gpu import DTYPES, _check, _inputs

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def _verify(cuda, target, tokens, cu, u, noise, most, draft=None, temp=None):
    from omlx_exl3_b200 import verify_drafts
    dev = lambda t: None if t is None else t.to(cuda)                  # noqa: E731
    return [t.cpu() for t in verify_drafts(dev(target), dev(tokens), torch.tensor(cu, dtype=torch.int32, device=cuda), dev(u),
                                           dev(noise), most, draft_logits=dev(draft), temperature=dev(temp))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [700, 30001])
@pytest.mark.parametrize("temp", [None, 0.0, 0.7])
@pytest.mark.parametrize("dist", [True, False])
def test_rows_that_are_not_numbers_accept_nothing(cuda, dtype, n, temp, dist):
    """NaN in the whole row, at the drafted token, or somewhere else in it: no probabilities, so no draft stands."""
    target, tokens, cu, u, noise, draft, _ = _inputs([4, 4, 4, 2], n, dtype, seed=n)
    u = torch.zeros_like(u)                                            # whatever has any probability stands
    target[0] = NAN
    target[4, tokens[3]] = NAN
    target[8, (int(tokens[6]) + 1) % n] = NAN
    target[13] = NAN                                                   # the row that the last sequence's token comes from
    t = None if temp is None else torch.full((4,), temp)
    got = _check(cuda, target, tokens, cu, u, noise, 3, draft if dist else None, t)
    assert got[1].tolist()[:3] == [1, 1, 1] and got[0][:3, 0].tolist() == [-1] * 3
    assert got[2][[0, 3, 6]].tolist() == [0.0] * 3


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [41.0, 47.0, 55.0])
@pytest.mark.parametrize("seqs", [1, 40])                              # wide CTAs, and narrow ones
@pytest.mark.parametrize("n,off", [(8, 0), (1 << 12, 0), (1 << 12, 1), (1 << 15, 8)])
def test_equal_weights_go_to_the_first(cuda, dtype, value, seqs, n, off):
    """Equal logits and equal noise: all quotients are one number, so the first column wins, whichever thread, vector or
    scalar path it falls to; after a rejection the first that is not the draft (one-hot q) or that p - q leaves."""
    wide = torch.zeros((2 * seqs, n + 16), dtype=dtype, device=cuda)
    target = wide[:, off:off + n]
    noise = torch.full((seqs, n + 16), value, device=cuda)[:, off:off + n]
    cu = list(range(0, 2 * seqs + 1, 2))
    tokens, u = torch.zeros(seqs, dtype=torch.int64), torch.full((seqs,), 0.9999)
    ones = torch.arange(seqs + 1).tolist()
    out, count, _ = _verify(cuda, target[:seqs], tokens[:0], ones, u[:0], noise, 0)
    assert not out.any() and (count == 1).all()
    draft = torch.zeros((seqs, n), dtype=dtype)
    draft[:, 0] = 2.0                                                  # q is above p there and below it, alike, elsewhere
    for d in (None, draft):
        out, count, prob = _verify(cuda, target, tokens, cu, u, noise, 1, d)
        assert (prob < 0.9999).all() and (count == 1).all() and (out[:, 0] == 1).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seqs", [18, 70])                             # wide CTAs, and narrow ones
@pytest.mark.parametrize("off", [0, 3])
def test_close_races_go_by_the_rounded_quotient(cuda, dtype, seqs, off):
    """p is 2^-12 in every column, exactly, and a sequence's noise takes three neighbouring fp32 numbers, whose quotients are equal
    or one unit apart: the first column with the largest fp32 quotient wins in every layout."""
    n = 1 << 12
    g = torch.Generator().manual_seed(seqs)
    noise = 1.5 + 0.45 * torch.rand((seqs, 1), generator=g) + torch.randint(0, 3, (seqs, n), generator=g) * 2.0 ** -23
    want = 2.0 ** -12 / noise
    want = (want == want.amax(1, keepdim=True)).int().argmax(1)
    wide = torch.zeros((seqs, n + 8), device=cuda)
    wide[:, off:off + n] = noise.to(cuda)
    target = torch.zeros((seqs, n), dtype=dtype)
    out, _, _ = _verify(cuda, target, torch.zeros(0, dtype=torch.int64), list(range(seqs + 1)), torch.zeros(0), wide[:, off:off + n], 0)
    assert torch.equal(out[:, 0], want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [700, 40001])
def test_greedy_takes_infinity_as_the_largest_logit(cuda, dtype, n):
    """At T = 0 a token forced by +inf is the first maximum, alone or among others and beside -inf; a NaN in the row still means
    that it has no answer. At other temperatures inf / inf is no probability."""
    target, tokens, cu, u, noise, _, _ = _inputs([3, 2, 2, 1, 1], n, dtype, seed=n + 1)
    u = torch.full_like(u, 0.999)
    target[0, n - 1] = INF
    tokens[0] = n - 1
    target[1, [n // 2, n - 5]] = INF
    tokens[1] = n - 5                                                  # not the first maximum
    target[3] = -INF
    target[3, n // 3] = INF
    tokens[2] = n // 3
    target[4, 5] = INF
    target[5, [3, n - 2]] = INF
    target[5, n // 2] = NAN
    target[7] = INF
    target[8, 1] = INF
    temp = torch.tensor([0.0, 0.0, 0.0, 0.0, 1.0])
    tokens[3] = 3
    out, count, prob = _verify(cuda, target, tokens, cu, u, noise, 2, None, temp)
    assert prob.tolist() == [1.0, 0.0, 1.0, 0.0] and count.tolist() == [2, 2, 1, 1, 1]
    assert out[0].tolist() == [n - 1, n // 2, -1] and out[1].tolist() == [n // 3, 5, -1]
    assert out[2:, 0].tolist() == [-1, 0, -1]


@pytest.mark.parametrize("dist", [True, False])
def test_rows_that_no_table_claims(cuda, dist):
    """cu_rows past the rows, or going back: such a sequence gives count 0 and no tokens, and drafts that none judged have
    acceptance 0, not what the memory held."""
    target, tokens, _, u, noise, draft, _ = _inputs([1, 4], 300, torch.float16, seed=3)
    u = torch.zeros_like(u)
    for bad in ([0, 1, 9], [0, 1, 0], [0, 1, 1], [0, 1, -4], [0, 1, 2 ** 31 - 1]):
        for _ in range(3):                                             # memory that the outputs may be given next
            junk = [torch.full((3,), 7.0, device=cuda) for _ in range(64)]
            del junk
            out, count, prob = _verify(cuda, target, tokens, bad, u, noise, 3, draft if dist else None)
            assert count.tolist() == [1, 0] and out[1].tolist() == [-1] * 4 and out[0, 0] >= 0
            assert prob.tolist() == [0.0] * 3
