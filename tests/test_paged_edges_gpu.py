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


# 8 rows: going back, negative, past the rows, a first row behind the next
BAD_ROWS = [[0, 5, 3, 8], [-1, 2, 4, 8], [0, -6, 4, 8], [0, 2, 9, 8], [0, 2, 4, 9], [0, 2 ** 31 - 1, -2 ** 31, 8], [6, 2, 4, 8],
            [-2 ** 31, 0, 4, 8], [0, 1, 1, 2 ** 31 - 1]]


@pytest.mark.parametrize("cu", BAD_ROWS)
@pytest.mark.parametrize("hq,max_rows", [(2, 0), (40, 1), (40, 0)])      # few rows at a time, by what is known or said; tiles too
def test_rows_out_of_order_are_reported(cuda, cu, hq, max_rows):
    """A cu_rows that is no list of rows: zeros, the status says so, and nothing beside the output is written."""
    from omlx_exl3_b200 import check_paged_status, paged_qkv_post
    check_paged_status(cuda)
    b = make_batch([2, 2, 4], [300, 20, 140], 2, 128, 16, torch.float16, cuda, seed=4)
    good = b["cu"]
    b["cu"] = torch.tensor(cu, dtype=torch.int32, device=cuda)
    whole = torch.full((24, hq, 128), 7.0, dtype=torch.float16, device=cuda)
    queries = torch.randn((24, hq, 128), device=cuda).half()
    out = _attn(queries[8:16], b, out=whole[8:16], max_rows=max_rows)
    with pytest.raises(RuntimeError, match="outside its range"):
        check_paged_status(cuda)
    assert not out.any() and (whole[:8] == 7).all() and (whole[16:] == 7).all()
    _attn(queries[8:16], {**b, "cu": good}, max_rows=max_rows)
    check_paged_status(cuda)
    if cu == BAD_ROWS[0]:                                              # row 3's sequence would begin at row 5 and end at 3
        kp, vp = b["kp"].clone(), b["vp"].clone()
        y = torch.randn((8, 6 * 128), device=cuda).half()
        angle = torch.zeros((400, 64), device=cuda)
        paged_qkv_post(*y.split([256, 256, 256], 1), None, None, 1e-6, angle.cos(), angle.sin(), kp, vp, b["table"], b["cu"], b["lens"])
        with pytest.raises(RuntimeError, match="outside its range"):
            check_paged_status(cuda)


@pytest.mark.parametrize("seqs", [33, 400])
def test_rows_that_every_other_sequence_claims(cuda, seqs):
    """All rows again and again: the work list would be many times what its 32 bits were checked for."""
    from omlx_exl3_b200 import check_paged_status
    check_paged_status(cuda)
    rows = 600
    b = make_batch([1] * seqs, [700] * seqs, 1, 64, 64, torch.float16, cuda, fill=0.0)
    b["cu"] = torch.tensor([0 if i % 2 == 0 else rows for i in range(seqs + 1)], dtype=torch.int32, device=cuda)
    out = _attn(torch.randn((rows, 8, 64), device=cuda).half(), b)
    assert not out.any()
    with pytest.raises(RuntimeError, match="outside its range"):
        check_paged_status(cuda)


@pytest.mark.parametrize("lead,rows,more", [(2, [1, 3], 0), (1, [70, 1], 3), (5, [0, 2], 1)])
def test_rows_before_the_first_sequence_are_padding(cuda, lead, rows, more):
    from omlx_exl3_b200 import check_paged_status
    check_paged_status(cuda)
    b = make_batch(rows, [200, 90], 2, 64, 16, torch.bfloat16, cuda, seed=6)
    n = sum(rows)
    q = torch.randn((lead + n + more, 6, 64), device=cuda).bfloat16()
    out = torch.full_like(q, 7.0)
    _attn(q, {**b, "cu": b["cu"] + lead}, out=out)
    assert not out[:lead].any() and not out[lead + n:].any()
    _assert_close(out[lead:lead + n], q[lead:lead + n], b, torch.bfloat16)
    check_paged_status(cuda)
