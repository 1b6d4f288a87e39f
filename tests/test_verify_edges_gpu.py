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
