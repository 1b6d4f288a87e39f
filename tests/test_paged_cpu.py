"""CPU: the page pool, the batch tables, and what the paged operators and the verification refuse."""
import ctypes

import pytest
import torch


def _cache(pages=8, ps=16):
    from omlx_exl3_b200 import PagedKVCache
    return PagedKVCache(2, 2, 64, pages, ps, device="cpu")


def test_pages_grow_with_the_sequence_and_come_back():
    c = _cache()
    c.add("a"), c.add("b")
    b = c.extend([("a", 16), ("b", 1)])
    assert c.free_pages == 6 and b.rows == [16, 1] and b.lens.tolist() == [16, 1] and b.cu_rows.tolist() == [0, 16, 17]
    assert b.page_table.shape == (2, 1)
    b = c.extend([("a", 1)])
    assert c.free_pages == 5 and b.page_table.shape == (1, 2) and b.lens.tolist() == [17]
    first = b.page_table[0].tolist()
    assert len(set(first)) == 2 and all(0 <= p < 8 for p in first)
    c.truncate("a", 16)
    assert c.free_pages == 6 and c.length("a") == 16
    c.truncate("a", 0)
    assert c.free_pages == 7
    c.release("b")
    assert c.free_pages == 8
    with pytest.raises(KeyError):
        c.length("b")


def test_no_page_is_held_twice():
    c = _cache(pages=20)
    for s in range(5):
        c.add(s)
    for step in range(6):
        b = c.extend([(s, 3 + s) for s in range(5)])
        used = [p for row in b.page_table.tolist() for p in row if p >= 0]
        assert len(used) == len(set(used)) == 20 - c.free_pages
        c.truncate(step % 5, c.length(step % 5) // 2)


def test_pool_refusals_take_nothing():
    from omlx_exl3_b200 import PagedKVCache
    c = _cache(pages=2)
    c.add("a"), c.add("b")
    with pytest.raises(MemoryError):
        c.extend([("a", 17), ("b", 1)])
    assert c.free_pages == 2 and c.length("a") == 0
    for feeds in ([], [("a", 0)], [("a", -1)], [("a", 1), ("a", 1)]):
        with pytest.raises(ValueError):
            c.extend(feeds)
    with pytest.raises(KeyError):
        c.extend([("nobody", 1)])
    with pytest.raises(ValueError):
        c.add("a")
    c.extend([("a", 5)])
    for n in (-1, 6):
        with pytest.raises(ValueError):
            c.truncate("a", n)
    for ps in (0, 8, 24, -16):
        with pytest.raises(ValueError):
            PagedKVCache(1, 1, 64, 4, ps, device="cpu")


def _meta(**kw):
    """Arguments of paged_qkv_post on the meta device: shapes and types without memory."""
    t = dict(q=torch.empty(3, 512, dtype=torch.float16), k=torch.empty(3, 256, dtype=torch.float16),
             v=torch.empty(3, 256, dtype=torch.float16), q_norm_w=None, k_norm_w=None, eps=1e-6,
             cos=torch.empty(32, 64), sin=torch.empty(32, 64), k_pages=torch.empty(4, 2, 16, 128, dtype=torch.float16),
             v_pages=torch.empty(4, 2, 16, 128, dtype=torch.float16), page_table=torch.empty(1, 2, dtype=torch.int32),
             cu_rows=torch.empty(2, dtype=torch.int32), lens=torch.empty(1, dtype=torch.int32))
    t.update(kw)
    return t


def test_host_tensors_are_refused():
    from omlx_exl3_b200 import paged_attn, paged_qkv_post, verify_drafts
    a = _meta()
    with pytest.raises(ValueError, match="CUDA"):
        paged_qkv_post(**a)
    with pytest.raises(ValueError, match="CUDA"):
        paged_attn(torch.empty(3, 4, 128, dtype=torch.float16), *[a[k] for k in ("k_pages", "v_pages", "page_table", "cu_rows", "lens")])
    with pytest.raises(ValueError, match="CUDA"):
        verify_drafts(torch.empty(2, 8), torch.empty(1, dtype=torch.int64), torch.empty(2, dtype=torch.int32), torch.empty(1),
                      torch.empty(1, 8), 1)


@pytest.mark.parametrize("change", [
    {"k_pages": torch.empty(4, 2, 16, 128, dtype=torch.bfloat16)}, {"page_table": torch.empty(1, 2, dtype=torch.int64)},
    {"lens": torch.empty(1, dtype=torch.int64)}, {"cu_rows": torch.empty(2)},
    {"k_pages": torch.empty(4, 2, 16, 128), "v_pages": torch.empty(4, 2, 16, 128)},
])
def test_types_are_refused(change):
    from omlx_exl3_b200 import paged_qkv_post
    with pytest.raises(TypeError):
        paged_qkv_post(**_meta(**change))


def _desc(**kw):
    from omlx_exl3_b200._lib import PagedDesc
    d = dict(k_pages=1 << 20, v_pages=1 << 20, page_table=1 << 20, cu_rows=1 << 20, lens=1 << 20, seqs=2, rows=3, table_cols=4,
             num_pages=9, page_size=16, hkv=2, head_dim=128, dtype=0)
    d.update(kw)
    return PagedDesc(**d)


@pytest.mark.parametrize("kw,status", [
    (dict(k_pages=None), -6), (dict(v_pages=None), -6), (dict(page_table=None), -6), (dict(cu_rows=None), -6), (dict(lens=None), -6),
    (dict(seqs=0), -1), (dict(rows=-1), -1), (dict(table_cols=0), -1), (dict(num_pages=0), -1), (dict(hkv=0), -1),
    (dict(page_size=8), -1), (dict(page_size=24), -1), (dict(page_size=0), -1), (dict(table_cols=1 << 28), -1),
    (dict(head_dim=96), -1), (dict(head_dim=256), -1), (dict(dtype=2), -4), (dict(dtype=-1), -4),
    (dict(k_pages=(1 << 20) + 2), -5), (dict(lens=(1 << 20) + 1), -5),
])
def test_descriptor_refusals(kw, status):
    from omlx_exl3_b200 import _lib
    L, n = _lib.lib(), ctypes.c_size_t()
    assert L.exl3_paged_attn_workspace(_desc(**kw), 4, ctypes.byref(n)) == status
    P = 1 << 20
    assert L.exl3_paged_attn(_desc(**kw), P, 512, 4, 1.0, 0, P, P, 1 << 30, P, None) == status
    assert L.exl3_paged_qkv_post(_desc(**kw), P, P, P, 512, 256, 256, 0, 4, None, None, 1e-6, P, P, 10, 64, P, P, None) == status


def test_call_refusals():
    """Each comes before any device work."""
    from omlx_exl3_b200 import _lib
    L, n, P, d = _lib.lib(), ctypes.c_size_t(), 1 << 20, _desc()
    assert L.exl3_paged_attn_workspace(d, 4, None) == -6
    for hq in (0, 3, 2 * 129):
        assert L.exl3_paged_attn_workspace(d, hq, ctypes.byref(n)) == -1

    def attn(q=P, qs=512, hq=4, scale=1.0, most=0, out=P, ws=P, wsb=1 << 30, st=P, b=d):
        return L.exl3_paged_attn(b, q, qs, hq, scale, most, out, ws, wsb, st, None)
    assert attn(q=None) == attn(out=None) == attn(st=None) == -6
    assert attn(most=-1) == attn(qs=511) == attn(scale=0.0) == attn(scale=float("nan")) == attn(hq=5) == -1
    assert attn(q=P + 2) == attn(out=P + 8) == attn(qs=513) == -5
    assert attn(b=_desc(rows=0)) == 0                                  # nothing to do

    def post(q=P, sq=512, sk=256, t=0, hq=4, cos=P, rr=10, rh=64, st=P):
        return L.exl3_paged_qkv_post(d, q, P, P, sq, sk, 256, t, hq, None, None, 1e-6, cos, P, rr, rh, P, st, None)
    assert post(q=None) == post(cos=None) == post(st=None) == -6
    assert post(sq=511) == post(sk=255) == post(hq=3) == post(rr=0) == post(rh=0) == post(rh=12) == post(rh=72) == -1
    assert post(t=2) == -4
    assert post(q=P + 1) == post(cos=P + 4) == -5

    def verify(t=P, tl=100, d=P, dl=100, ty=0, r=5, s=2, v=100, tok=P, cu=P, u=P, e=P, el=100, m=3, out=P, c=P, p=P):
        return L.exl3_verify_drafts(t, tl, d, dl, ty, r, s, v, tok, cu, None, u, e, el, m, out, c, p, P, 1 << 30, None)
    assert verify(t=None) == verify(cu=None) == verify(e=None) == verify(out=None) == verify(c=None) == -6
    assert verify(tok=None) == verify(u=None) == verify(p=None) == -6
    assert verify(r=1) == verify(s=0) == verify(v=0) == verify(tl=99) == verify(dl=99) == verify(el=99) == verify(m=-1) == -1
    assert verify(ty=3) == -4
    assert verify(t=P + 1) == verify(tok=P + 4) == verify(e=P + 2) == -5
    assert L.exl3_verify_workspace(3, 2, 5, None) == -6 and L.exl3_verify_workspace(1, 2, 5, ctypes.byref(n)) == -1
