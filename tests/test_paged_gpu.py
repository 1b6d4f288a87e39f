"""GPU: the paged-cache operators (q/k/v post step into the pages, attention over them) against 64-bit plain forms.

Everything a batch does not hold (spare pages, the slots behind a sequence's end) is NaN in these tests."""
import math

import pytest
import torch

from paged_util import UNIT, attn_exact, attn_tolerance, make_batch, norm_rope_exact

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def _attn(q, b, **kw):
    from omlx_exl3_b200 import paged_attn
    return paged_attn(q, b["kp"], b["vp"], b["table"], b["cu"], b["lens"], **kw)


def _check_attn(got, q, b, dtype, scale=None):
    scale = scale or 1 / math.sqrt(q.shape[2])
    ref, weight = attn_exact(q.cpu(), b, scale)
    tol = attn_tolerance(ref, weight, b, dtype)
    err = (got.cpu().double() - ref).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"{float((err / tol).max()):.2f} of the bound at {int((err / tol).argmax())}"


# rows of each sequence, its length once they are appended
BATCHES = {
    "one-token": ([1], [1]),
    "one-row-127": ([1], [127]),
    "one-row-128": ([1], [128]),
    "one-row-129": ([1], [129]),
    "one-row-long": ([1], [4097]),
    "decode-ragged": ([1] * 7, [1, 2, 16, 17, 255, 256, 1000]),
    "verify": ([4, 1, 8, 3], [4, 300, 129, 515]),
    "chunk-exact": ([128], [128]),
    "chunk-from-zero": ([200], [200]),
    "chunk-over-context": ([130], [130 + 777]),
    "mixed": ([1, 257, 1, 64, 31], [901, 257, 1, 64 + 128, 31 + 5]),
    "many": ([1] * 40 + [5] * 5, [i * 13 + 1 for i in range(40)] + [500, 5, 6, 128, 133]),
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", BATCHES)
def test_attn_batches(cuda, name, dtype):
    rows, lens = BATCHES[name]
    b = make_batch(rows, lens, 2, 128, 16, dtype, cuda, seed=len(name))
    q = (1.5 * torch.randn((sum(rows), 10, 128), generator=torch.Generator().manual_seed(1))).to(dtype).to(cuda)
    _check_attn(_attn(q, b), q, b, dtype)


@pytest.mark.parametrize("hq,hkv,hd,ps", [
    (40, 8, 128, 64), (8, 8, 128, 32), (7, 1, 128, 128), (16, 1, 128, 256), (64, 1, 128, 16), (128, 1, 64, 16),
    (4, 4, 64, 16), (10, 2, 64, 512), (24, 8, 64, 64), (100, 1, 128, 32),
])
def test_attn_layouts(cuda, hq, hkv, hd, ps):
    rows, lens = [1, 70, 5, 2], [260, 70, 133, 2]
    dtype = torch.bfloat16 if (hq + ps) % 3 == 0 else torch.float16
    b = make_batch(rows, lens, hkv, hd, ps, dtype, cuda, seed=hq)
    q = torch.randn((sum(rows), hq, hd), generator=torch.Generator().manual_seed(2)).to(dtype).to(cuda)
    _check_attn(_attn(q, b), q, b, dtype)


@pytest.mark.parametrize("hd", [64, 128])
def test_attn_padding_rows_and_empty_sequences(cuda, hd):
    """A sequence with more rows than positions: the rows before position 0 give zeros. Sequences without rows, and
    without positions, between others."""
    rows, lens = [5, 0, 1, 300, 0, 2], [2, 40, 0, 290, 0, 130]
    b = make_batch(rows, lens, 2, hd, 32, torch.float16, cuda, seed=3)
    q = torch.randn((sum(rows), 6, hd), generator=torch.Generator().manual_seed(3)).half().to(cuda)
    out = _attn(q, b)
    assert not out[:3].any() and not out[5].any() and not out[6:16].any()
    _check_attn(out, q, b, torch.float16)
    none = make_batch([0, 0], [3, 4], 2, hd, 32, torch.float16, cuda)
    assert _attn(q[:0], none).shape == (0, 6, hd)


@pytest.mark.parametrize("rows,lens", [([1, 2], [40, 130]), ([200, 1, 0], [300, 77, 0]), ([0], [16])])
@pytest.mark.parametrize("hd", [64, 128])
def test_rows_behind_the_last_sequence_are_padding(cuda, rows, lens, hd):
    """A call of more rows than the sequences have (a captured graph's width): zeros for them, nothing appended, and the
    others as in a call without them."""
    from omlx_exl3_b200 import check_paged_status, paged_qkv_post
    n, more, hq, hkv = sum(rows), 5, 4, 2
    b = make_batch(rows, lens, hkv, hd, 16, torch.float16, cuda, seed=40, spare=1)
    q = torch.randn((n + more, hq, hd), generator=torch.Generator().manual_seed(41)).half().to(cuda)
    out = torch.full_like(q, 7.0)
    assert _attn(q, b, out=out) is out
    assert torch.equal(out[:n], _attn(q[:n], b)) and not out[n:].any()
    y = torch.randn((n + more, (hq + 2 * hkv) * hd), device=cuda).half()
    cos, sin = (t.to(cuda) for t in _rope_tables(512, hd // 2))
    split = [hq * hd, hkv * hd, hkv * hd]
    pages = [(b["kp"].clone(), b["vp"].clone()) for _ in range(2)]
    outs = [paged_qkv_post(*x.split(split, 1), None, None, 1e-6, cos, sin, *p, b["table"], b["cu"], b["lens"])
            for x, p in zip((y, y[:n]), pages)]
    assert torch.equal(outs[0][:n], outs[1]) and not outs[0][n:].any()
    for x, z in zip(*pages):
        assert torch.equal(x.view(torch.int16), z.view(torch.int16))
    check_paged_status(cuda)


def test_attn_sharp_and_growing_scores(cuda):
    """Scores of +-60 whose maximum moves along the cache: the running maximum has to follow it."""
    dtype = torch.float16
    rows, lens = [3, 150], [900, 700]
    b = make_batch(rows, lens, 1, 128, 16, dtype, cuda, seed=4)
    for s in range(2):                                      # keys grow with the position
        ramp = torch.linspace(0.05, 3, lens[s])[:, None, None]
        b["k"][s] = (b["k"][s].float() * ramp).to(dtype)
        for p in range(lens[s]):
            b["kp"][b["table"][s, p // 16], :, p % 16] = b["k"][s][p].to(cuda)
    q = (2 * torch.randn((153, 4, 128), generator=torch.Generator().manual_seed(5))).to(dtype).to(cuda)
    got = _attn(q, b)
    ref, weight = attn_exact(q.cpu(), b, 1 / math.sqrt(128))
    # scores up to 2 * 3 * 128^.5 * 4 = 270 units: their fp32 error grows in proportion (128 rounded sums of that size)
    tol = attn_tolerance(ref, weight, b, dtype) + 4e-4 * weight
    assert ((got.cpu().double() - ref).abs() <= tol).all()


def test_attn_equal_keys_give_the_mean(cuda):
    """All scores alike: the output is the mean of the values, over every split of the positions."""
    rows, lens = [1], [5000]
    b = make_batch(rows, lens, 1, 128, 64, torch.float16, cuda, seed=5)
    b["kp"][~torch.isnan(b["kp"])] = 0.5
    b["k"][0] = torch.full_like(b["k"][0], 0.5)
    q = torch.ones((1, 5, 128), dtype=torch.float16, device=cuda)
    _check_attn(_attn(q, b), q, b, torch.float16)


def test_attn_strided_and_misaligned_queries(cuda):
    rows, lens = [3, 66], [50, 200]
    b = make_batch(rows, lens, 2, 128, 16, torch.float16, cuda, seed=6)
    wide = torch.randn((69, 14 * 128 + 8), generator=torch.Generator().manual_seed(6)).half().to(cuda)
    views = [wide[:, :1280].unflatten(1, (10, 128)), wide[:, 8:1288].unflatten(1, (10, 128)),
             wide[:, 3:1283].unflatten(1, (10, 128)), wide[:, :1280].unflatten(1, (128, 10)).transpose(1, 2)]
    for q in views:
        assert torch.equal(_attn(q, b), _attn(q.contiguous(), b))
        _check_attn(_attn(q, b), q, b, torch.float16)


def test_attn_scale_out_and_repeat(cuda):
    rows, lens = [1, 40, 9], [3000, 1500, 9]
    b = make_batch(rows, lens, 2, 128, 16, torch.bfloat16, cuda, seed=7)
    q = torch.randn((50, 10, 128), generator=torch.Generator().manual_seed(7)).bfloat16().to(cuda)
    out = torch.full_like(q, float("nan"))
    assert _attn(q, b, scale=0.25, out=out) is out
    _check_attn(out, q, b, torch.bfloat16, scale=0.25)
    for _ in range(5):                                      # the same bits each time
        assert torch.equal(_attn(q, b, scale=0.25), out)


@pytest.mark.parametrize("max_rows", [1, 4, 30, 1000])
def test_attn_most_rows_changes_no_result(cuda, max_rows):
    """Known, unknown or wrong: every row is computed, within the bound."""
    rows, lens = [30, 1, 4], [700, 260, 9]
    b = make_batch(rows, lens, 2, 128, 16, torch.float16, cuda, seed=40)
    q = torch.randn((35, 10, 128), generator=torch.Generator().manual_seed(40)).half().to(cuda)
    _check_attn(_attn(q, b, max_rows=max_rows), q, b, torch.float16)


def test_attn_streams_do_not_share_scratch(cuda):
    """Calls on several streams at once, each against its own result alone."""
    sets = []
    for i in range(4):
        b = make_batch([1, 1, 2], [2000 + i, 700, 64], 2, 128, 16, torch.float16, cuda, seed=20 + i)
        q = torch.randn((4, 10, 128), generator=torch.Generator().manual_seed(i)).half().to(cuda)
        sets.append((q, b, _attn(q, b)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    outs = []
    for _ in range(10):
        for st, (q, b, _) in zip(streams, sets):
            with torch.cuda.stream(st):
                outs.append(_attn(q, b))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, sets[i % 4][2])


def test_attn_in_a_graph_follows_the_tables(cuda):
    """Captured once, replayed after the tables, the pages and the queries changed; beside eager calls."""
    b1 = make_batch([1, 1, 1], [900, 33, 0], 2, 128, 16, torch.float16, cuda, seed=30, spare=10)
    b2 = make_batch([1, 1, 1], [40, 800, 90], 2, 128, 16, torch.float16, cuda, seed=31, spare=10)
    q1 = torch.randn((3, 10, 128), device=cuda).half()
    q2 = torch.randn((3, 10, 128), device=cuda).half()
    num, cols = max(x["kp"].shape[0] for x in (b1, b2)), max(x["table"].shape[1] for x in (b1, b2))

    def padded(b):
        kp = torch.zeros((num, *b["kp"].shape[1:]), dtype=torch.float16, device=cuda)
        vp, tb = kp.clone(), torch.full((3, cols), -1, dtype=torch.int32, device=cuda)
        kp[:len(b["kp"])], vp[:len(b["vp"])], tb[:, :b["table"].shape[1]] = b["kp"], b["vp"], b["table"]
        return {"kp": kp, "vp": vp, "table": tb, "cu": b["cu"].clone(), "lens": b["lens"].clone()}

    live, p1, p2 = padded(b1), padded(b1), padded(b2)
    q = q1.clone()
    want = [_attn(q1, p1), _attn(q2, p2)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = _attn(q, live)
    for i, (p, qq) in enumerate([(p1, q1), (p2, q2), (p1, q1)]):
        for k in live:
            live[k].copy_(p[k])
        q.copy_(qq)
        g.replay()
        beside = _attn(qq, p)
        torch.cuda.synchronize()
        assert torch.equal(out, want[i % 2]) and torch.equal(beside, want[i % 2])


def test_attn_pool_past_32_bit_offsets(cuda):
    """Pages whose first element lies past 2^31 elements in the pool."""
    hkv, ps, hd = 8, 256, 128
    num = (1 << 31) // (hkv * ps * hd) + 6
    kp = torch.empty((num, hkv, ps, hd), dtype=torch.bfloat16, device=cuda)
    vp = torch.empty_like(kp)
    b = make_batch([1, 140], [300, 500], hkv, hd, ps, torch.bfloat16, cuda, seed=8, spare=0)
    n = b["kp"].shape[0]
    kp[-n:], vp[-n:] = b["kp"], b["vp"]
    b["kp"], b["vp"] = kp, vp
    b["table"] = torch.where(b["table"] >= 0, b["table"] + (num - n), b["table"])
    q = torch.randn((141, 8, hd), generator=torch.Generator().manual_seed(8)).bfloat16().to(cuda)
    _check_attn(_attn(q, b), q, b, torch.bfloat16)


def test_attn_pages_outside_the_pool_are_reported(cuda):
    """A page the pool does not have is left out, and the status says so; the other sequences are not touched by it."""
    from omlx_exl3_b200 import check_paged_status
    check_paged_status(cuda)
    b = make_batch([1, 1], [100, 60], 2, 128, 16, torch.float16, cuda, seed=9)
    q = torch.randn((2, 4, 128), device=cuda).half()
    want = _attn(q, b)
    check_paged_status(cuda)
    for bad in (b["kp"].shape[0], -1, 2 ** 31 - 1, -2 ** 31):
        t = b["table"].clone()
        t[0, 2] = bad
        got = _attn(q, {**b, "table": t})
        assert torch.isfinite(got).all() and torch.equal(got[1], want[1])
        with pytest.raises(RuntimeError, match="outside its range"):
            check_paged_status(cuda)
    check_paged_status(cuda)
    long = {**b, "lens": b["lens"] + torch.tensor([1000, 0], dtype=torch.int32, device=cuda)}      # past the table's columns
    got = _attn(q, long)
    assert torch.equal(got[1], want[1])
    with pytest.raises(RuntimeError, match="outside its range"):
        check_paged_status(cuda)


# ------------------------------------------------------------------------------ q/k/v post step

def _rope_tables(n, half):
    inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return torch.cos(a).float(), torch.sin(a).float()


@pytest.mark.parametrize("src", DTYPES)
@pytest.mark.parametrize("cache", DTYPES)
@pytest.mark.parametrize("hq,hkv,hd,ps,rot,norm", [
    (40, 8, 128, 64, 128, True), (5, 1, 128, 16, 64, True), (12, 12, 64, 16, 64, False), (3, 1, 64, 32, 16, True),
    (64, 2, 128, 128, 32, False),
])
@pytest.mark.parametrize("layout", ["fused", "odd", "apart"])
def test_qkv_post(cuda, src, cache, hq, hkv, hd, ps, rot, norm, layout):
    from omlx_exl3_b200 import paged_qkv_post
    rows, lens = [1, 37, 3, 2, 0, 1], [1, 37 + 15, 600, 1, 8, 0]       # the fourth's first row and the last's are padding
    b = make_batch(rows, lens, hkv, hd, ps, cache, cuda, seed=hq, fill=7.0)
    n, nq, nk = sum(rows), hq * hd, hkv * hd
    g = torch.Generator().manual_seed(hq + rot)
    off = {"fused": 0, "odd": 3, "apart": 0}[layout]
    y = (2 * torch.randn((n, nq + 2 * nk + off), generator=g)).to(src).to(cuda)[:, off:]
    q, k, v = y.split([nq, nk, nk], dim=1)
    if layout == "apart":
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    wq = (1 + 0.2 * torch.randn(hd, generator=g)).to(src).to(cuda) if norm else None
    wk = (1 + 0.2 * torch.randn(hd, generator=g)).to(src).to(cuda) if norm else None
    cos, sin = _rope_tables(700, rot // 2)
    kp, vp = b["kp"].clone(), b["vp"].clone()
    out = paged_qkv_post(q, k, v, wq, wk, 1e-6, cos.to(cuda), sin.to(cuda), kp, vp, b["table"], b["cu"], b["lens"])
    assert out.dtype == cache and out.shape == (n, hq, hd)

    cpu = lambda t: None if t is None else t.cpu()                     # noqa: E731
    seq = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows))
    pos = torch.tensor([lens[s] - rows[s] + i for s in range(len(rows)) for i in range(rows[s])])
    live = pos >= 0
    at = pos.clamp(min=0)
    rq = norm_rope_exact(q.cpu().reshape(n, hq, hd), cpu(wq), 1e-6, cos, sin, at)
    rk = norm_rope_exact(k.cpu().reshape(n, hkv, hd), cpu(wk), 1e-6, cos, sin, at)
    rv = v.cpu().reshape(n, hkv, hd).double()
    rq[~live] = 0
    u = UNIT[cache]

    def close(got, ref, size):
        # one rounding (u |y|), fp32 steps on values of `size` (a dozen of 2^-24 each), fp16's smallest spacing
        tol = u * ref.abs() + 2e-6 * size + 2.0 ** -25
        assert ((got.cpu().double() - ref).abs() <= tol).all()

    close(out, rq, float(rq.abs().max()))
    want_k, want_v = b["kp"].cpu().clone(), b["vp"].cpu().clone()
    page = b["table"].cpu()[seq, at // ps].long()
    got_k, got_v = kp.cpu()[page[live], :, at[live] % ps], vp.cpu()[page[live], :, at[live] % ps]
    close(got_k, rk[live], float(rk.abs().max()))
    assert torch.equal(got_v, rv[live].to(cache))
    want_k[page[live], :, at[live] % ps] = got_k                       # and nothing else was written
    want_v[page[live], :, at[live] % ps] = got_v
    assert torch.equal(kp.cpu(), want_k) and torch.equal(vp.cpu(), want_v)


def test_qkv_post_beside_a_rotation_of_part_of_the_head(cuda):
    """What is not rotated passes unchanged, infinities too."""
    from omlx_exl3_b200 import paged_qkv_post
    b = make_batch([1], [5], 1, 128, 16, torch.float16, cuda)
    q = torch.randn((1, 128), device=cuda).half()
    q[0, 64:] = float("inf")
    k = v = torch.randn((1, 128), device=cuda).half()
    cos, sin = _rope_tables(8, 32)
    out = paged_qkv_post(q, k, v, None, None, 1e-6, cos.to(cuda), sin.to(cuda), b["kp"], b["vp"], b["table"], b["cu"], b["lens"])
    assert torch.isinf(out[0, 0, 64:]).all() and torch.isfinite(out[0, 0, :64]).all()


def test_qkv_post_out_of_range_is_reported(cuda):
    from omlx_exl3_b200 import check_paged_status, paged_qkv_post
    check_paged_status(cuda)
    b = make_batch([2, 1], [20, 4], 1, 128, 16, torch.float16, cuda)
    y = torch.randn((3, 3 * 128), device=cuda).half()
    cos, sin = (t.to(cuda) for t in _rope_tables(19, 64))              # position 19 of the first sequence is past it
    kp, vp = torch.zeros_like(b["kp"]), torch.zeros_like(b["vp"])
    out = paged_qkv_post(*y.split(128, 1), None, None, 1e-6, cos, sin, kp, vp, b["table"], b["cu"], b["lens"])
    assert not out[1].any() and out[0].any() and out[2].any()
    assert int((vp != 0).any(-1).sum()) == 2
    with pytest.raises(RuntimeError, match="outside its range"):
        check_paged_status(cuda)
    cos, sin = (t.to(cuda) for t in _rope_tables(64, 64))
    kp.zero_(), vp.zero_()
    t = b["table"].clone()
    t[0, 1] = 99
    out = paged_qkv_post(*y.split(128, 1), None, None, 1e-6, cos, sin, kp, vp, t, b["cu"], b["lens"])
    assert out.any(-1).all() and int((vp != 0).any(-1).sum()) == 1     # only the second sequence's row was appended
    with pytest.raises(RuntimeError, match="outside its range"):
        check_paged_status(cuda)
    check_paged_status(cuda)


def test_append_then_attend_matches_one_long_prompt(cuda):
    """A prompt fed in chunks of every kind gives, row for row, what the whole prompt at once gives (the keys and values
    in the pages are the same; the outputs are equal within the bound of two roundings)."""
    from omlx_exl3_b200 import PagedKVCache, paged_attn, paged_qkv_post
    hq, hkv, hd, n = 10, 2, 128, 333
    y = torch.randn((n, (hq + 2 * hkv) * hd), generator=torch.Generator().manual_seed(11)).half().to(cuda)
    w = (1 + 0.1 * torch.randn(hd, generator=torch.Generator().manual_seed(12))).half().to(cuda)
    cos, sin = (t.to(cuda) for t in _rope_tables(400, hd // 2))

    def feed(chunks):
        cache = PagedKVCache(1, hkv, hd, 32, 16, device=cuda)
        cache.add("x"), cache.add("y")
        outs, at = [], 0
        for c in chunks:
            cache.extend([("y", 3)])                                   # another sequence takes pages in between
            b = cache.extend([("x", c)])
            q, k, v = y[at:at + c].split([hq * hd, hkv * hd, hkv * hd], 1)
            qo = paged_qkv_post(q, k, v, w, w, 1e-6, cos, sin, cache.k[0], cache.v[0], *b.tables)
            outs.append(paged_attn(qo, cache.k[0], cache.v[0], *b.tables))
            at += c
        return torch.cat(outs)

    whole, parts = feed([n]), feed([1, 1, 16, 100, 3, 128, 1, 83])
    err = (whole.float() - parts.float()).abs().max()
    assert err <= 4 * UNIT[torch.float16] * 4.5                       # |v| < 4.5: p rounded twice, the output twice


@pytest.mark.parametrize("hd,hq,hkv", [(128, 10, 2), (64, 4, 4)])
def test_steps_of_mixed_batches_in_a_graph(cuda, hd, hq, hkv):
    """Appends and attention of chunks and single tokens, step after step in one graph without a gap: each step's attention
    reads what the step before it just wrote, as when every call is waited for."""
    from omlx_exl3_b200 import check_paged_status, paged_attn, paged_qkv_post
    steps, rows = 4, [260, 1, 4, 0, 1, 33]
    lens = [[260 * (i + 1), 900 + i, 130 + 4 * i, 7, 1 + i, 2000 + 33 * i] for i in range(steps)]
    b = make_batch(rows, lens[-1], hkv, hd, 32, torch.float16, cuda, seed=50, fill=0.0)
    n = sum(rows)
    gen = torch.Generator().manual_seed(51)
    y = [torch.randn((n, (hq + 2 * hkv) * hd), generator=gen).half().to(cuda) for _ in range(steps)]
    at = [torch.tensor(x, dtype=torch.int32, device=cuda) for x in lens]
    w = (1 + 0.1 * torch.randn(hd, generator=gen)).half().to(cuda)
    cos, sin = (x.to(cuda) for x in _rope_tables(2200, hd // 2))
    first = b["kp"].clone(), b["vp"].clone()

    def run(wait):
        outs = []
        for i in range(steps):
            q = paged_qkv_post(*y[i].split([hq * hd, hkv * hd, hkv * hd], 1), w, w, 1e-6, cos, sin, b["kp"], b["vp"], b["table"],
                               b["cu"], at[i])
            if wait:
                torch.cuda.synchronize()
            outs.append(paged_attn(q, b["kp"], b["vp"], b["table"], b["cu"], at[i]))
            if wait:
                torch.cuda.synchronize()
        return outs

    def restore():
        b["kp"].copy_(first[0])
        b["vp"].copy_(first[1])

    want = run(True)
    pages = b["kp"].clone(), b["vp"].clone()
    g = torch.cuda.CUDAGraph()
    restore()
    with torch.cuda.graph(g):
        outs = run(False)
    for _ in range(5):
        restore()
        for o in outs:
            o.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, z) for x, z in zip(outs, want))
        assert torch.equal(b["kp"], pages[0]) and torch.equal(b["vp"], pages[1])
    check_paged_status(cuda)
