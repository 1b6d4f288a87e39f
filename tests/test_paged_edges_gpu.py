"""GPU: paged-cache operators where batches or tables are out of the ordinary, against 64-bit plain forms."""
import math
import random

import pytest
import torch

from paged_util import attn_exact, attn_tolerance, make_batch

pytestmark = pytest.mark.gpu


def _attn(q, b, **kw):
    from omlx_exl3_b200 import paged_attn
    return paged_attn(q, b["kp"], b["vp"], b["table"], b["cu"], b["lens"], **kw)


def _assert_close(got, q, b, dtype):
    ref, weight = attn_exact(q.cpu(), b, 1 / math.sqrt(q.shape[2]))
    err = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got).all()
    assert (err <= attn_tolerance(ref, weight, b, dtype)).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("context", [0, 140])
def test_hundreds_of_short_prompts(cuda, hd, context):
    """Many items in a row of one tile and one step (with context: two), each ending inside its last page: the issuing warp that has
    no step in them must not lose count of the tiles that are cleaned behind a sequence's end. No wait may run out."""
    from omlx_exl3_b200 import check_paged_status
    check_paged_status(cuda)
    rng = random.Random(hd + context)
    rows = [rng.randint(7, 25) for _ in range(300)]
    lens = [r + (rng.randint(0, context) if context else 0) for r in rows]
    b = make_batch(rows, lens, 2, hd, 32, torch.float16, cuda, seed=hd)
    q = torch.randn((sum(rows), 10, hd), generator=torch.Generator().manual_seed(1)).half().to(cuda)
    first = _attn(q, b)
    for _ in range(20):
        assert torch.equal(_attn(q, b), first)
    check_paged_status(cuda)
    _assert_close(first, q, b, torch.float16)
