"""GPU: what the native calls of the paged operators refuse, before any device work: shapes, types, strides and devices."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32, I32, I64 = torch.float16, torch.bfloat16, torch.float32, torch.int32, torch.int64


def _batch(cuda):
    return dict(k_pages=torch.zeros(4, 2, 16, 128, dtype=F16, device=cuda), v_pages=torch.zeros(4, 2, 16, 128, dtype=F16, device=cuda),
                page_table=torch.zeros(2, 2, dtype=I32, device=cuda), cu_rows=torch.tensor([0, 2, 3], dtype=I32, device=cuda),
                lens=torch.tensor([5, 0], dtype=I32, device=cuda))


# of the batch's tables, for both calls
TABLES = {
    "v_pages of another type": (TypeError, lambda a: dict(v_pages=a["v_pages"].bfloat16())),
    "fp32 pages": (TypeError, lambda a: dict(k_pages=a["k_pages"].float(), v_pages=a["v_pages"].float())),
    "64-bit table": (TypeError, lambda a: dict(page_table=a["page_table"].long())),
    "64-bit rows": (TypeError, lambda a: dict(cu_rows=a["cu_rows"].long())),
    "64-bit lens": (TypeError, lambda a: dict(lens=a["lens"].long())),
    "list of lens": (TypeError, lambda a: dict(lens=[5, 0])),
    "v_pages of another shape": (ValueError, lambda a: dict(v_pages=a["v_pages"][:3])),
    "3-d pages": (ValueError, lambda a: dict(k_pages=a["k_pages"][0], v_pages=a["v_pages"][0])),
    "1-d table": (ValueError, lambda a: dict(page_table=a["page_table"][0])),
    "rows of three sequences": (ValueError, lambda a: dict(cu_rows=torch.zeros(4, dtype=I32, device=a["lens"].device))),
    "lens of one": (ValueError, lambda a: dict(lens=a["lens"][:1])),
    "no sequence": (ValueError, lambda a: dict(page_table=a["page_table"][:0], cu_rows=a["cu_rows"][:1], lens=a["lens"][:0])),
    "no column": (ValueError, lambda a: dict(page_table=a["page_table"][:, :0])),
    "strided table": (ValueError, lambda a: dict(page_table=torch.zeros(2, 4, dtype=I32, device=a["lens"].device)[:, ::2])),
    "strided lens": (ValueError, lambda a: dict(lens=torch.zeros(4, dtype=I32, device=a["lens"].device)[::2])),
    "strided rows": (ValueError, lambda a: dict(cu_rows=torch.zeros(6, dtype=I32, device=a["lens"].device)[::2])),
    "transposed pages": (ValueError, lambda a: {k: a[k].transpose(1, 2).contiguous().transpose(1, 2) for k in ("k_pages", "v_pages")}),
    "pages of 24": (ValueError, lambda a: {k: torch.zeros(4, 2, 24, 128, dtype=F16, device=a["lens"].device) for k in ("k_pages", "v_pages")}),
    "pages of 8": (ValueError, lambda a: {k: a[k][:, :, :8].contiguous() for k in ("k_pages", "v_pages")}),
    "table on the host": (ValueError, lambda a: dict(page_table=a["page_table"].cpu())),
    "lens on the host": (ValueError, lambda a: dict(lens=a["lens"].cpu())),
    "pages on the host": (ValueError, lambda a: dict(k_pages=a["k_pages"].cpu(), v_pages=a["v_pages"].cpu())),
    "v_pages on the host": (ValueError, lambda a: dict(v_pages=a["v_pages"].cpu())),
}

POST = {
    "q on the host": (ValueError, lambda a: dict(q=a["q"].cpu())),
    "3-d q": (ValueError, lambda a: dict(q=a["q"][None])),
    "q of 3 heads": (ValueError, lambda a: dict(q=a["q"][:, :384])),
    "k of other rows": (ValueError, lambda a: dict(k=a["k"][:2])),
    "v of one head": (ValueError, lambda a: dict(v=a["v"][:, :128])),
    "k of another type": (TypeError, lambda a: dict(k=a["k"].bfloat16())),
    "fp32 rows": (TypeError, lambda a: {k: a[k].float() for k in "qkv"}),
    "overlapping rows": (ValueError, lambda a: dict(q=a["q"][:1].expand(3, 512))),
    "columns apart": (ValueError, lambda a: dict(v=torch.zeros(3, 512, dtype=F16, device=a["q"].device)[:, ::2])),
    "fp16 cos": (TypeError, lambda a: dict(cos=a["cos"].half())),
    "sin of another shape": (ValueError, lambda a: dict(sin=a["sin"][:, :32])),
    "strided cos": (ValueError, lambda a: {k: torch.zeros(8, 128, device=a["q"].device)[:, ::2] for k in ("cos", "sin")}),
    "12 pairs": (ValueError, lambda a: {k: torch.zeros(8, 12, device=a["q"].device) for k in ("cos", "sin")}),
    "72 pairs": (ValueError, lambda a: {k: torch.zeros(8, 72, device=a["q"].device) for k in ("cos", "sin")}),
    "no positions": (ValueError, lambda a: {k: torch.zeros(0, 64, device=a["q"].device) for k in ("cos", "sin")}),
    "norm of another type": (TypeError, lambda a: dict(q_norm_w=torch.ones(128, device=a["q"].device))),
    "norm of another size": (ValueError, lambda a: dict(k_norm_w=torch.ones(64, dtype=F16, device=a["q"].device))),
    "norm on the host": (ValueError, lambda a: dict(k_norm_w=torch.ones(128, dtype=F16))),
    "eps of no number": (TypeError, lambda a: dict(eps="small")),
    "out of another shape": (ValueError, lambda a: dict(q_out=torch.zeros(3, 2, 128, dtype=F16, device=a["q"].device))),
    "out of another type": (ValueError, lambda a: dict(q_out=torch.zeros(3, 4, 128, dtype=BF16, device=a["q"].device))),
    "strided out": (ValueError, lambda a: dict(q_out=torch.zeros(3, 4, 256, dtype=F16, device=a["q"].device)[..., ::2])),
}

ATTN = {
    "q of another type": (TypeError, lambda a: dict(q=a["q"].bfloat16())),
    "q on the host": (ValueError, lambda a: dict(q=a["q"].cpu())),
    "2-d q": (ValueError, lambda a: dict(q=a["q"].flatten(1))),
    "q of 64": (ValueError, lambda a: dict(q=a["q"][..., :64])),
    "3 heads of 2": (ValueError, lambda a: dict(q=a["q"][:, :3])),
    "129 heads of a kv head": (ValueError, lambda a: dict(q=torch.zeros(3, 258, 128, dtype=F16, device=a["q"].device))),
    "no heads": (ValueError, lambda a: dict(q=a["q"][:, :0])),
    "scale of 0": (ValueError, lambda a: dict(scale=0.0)),
    "scale that is none": (ValueError, lambda a: dict(scale=float("nan"))),
    "endless scale": (ValueError, lambda a: dict(scale=float("inf"))),
    "scale of text": (TypeError, lambda a: dict(scale="1")),
    "max_rows below 0": (ValueError, lambda a: dict(max_rows=-1)),
    "broken max_rows": (TypeError, lambda a: dict(max_rows=1.5)),
    "out of another shape": (ValueError, lambda a: dict(out=a["q"][:2].clone())),
    "out of another type": (ValueError, lambda a: dict(out=a["q"].bfloat16())),
    "out on the host": (ValueError, lambda a: dict(out=a["q"].cpu())),
}


def _refused(call, args, case):
    error, change = case
    with pytest.raises(error):
        call(**{**args, **change(args)})
    call(**args)                                                       # and the arguments without the change are taken


@pytest.mark.parametrize("name", [*TABLES, *POST])
def test_qkv_post_refuses(cuda, name):
    from omlx_exl3_b200 import paged_qkv_post
    z = lambda *shape, t=F16: torch.zeros(shape, dtype=t, device=cuda)   # noqa: E731
    args = dict(q=z(3, 512), k=z(3, 256), v=z(3, 256), q_norm_w=None, k_norm_w=None, eps=1e-6, cos=z(8, 64, t=F32), sin=z(8, 64, t=F32),
                **_batch(cuda))
    _refused(paged_qkv_post, args, {**TABLES, **POST}[name])


@pytest.mark.parametrize("name", [*TABLES, *ATTN])
def test_attn_refuses(cuda, name):
    from omlx_exl3_b200 import paged_attn
    args = dict(q=torch.zeros(3, 4, 128, dtype=F16, device=cuda), **_batch(cuda))
    _refused(paged_attn, args, {**TABLES, **ATTN}[name])


VERIFY = {
    "integer logits": (TypeError, lambda a: dict(target_logits=a["target_logits"].int())),
    "1-d logits": (ValueError, lambda a: dict(target_logits=a["target_logits"][0])),
    "fewer rows than sequences": (ValueError, lambda a: dict(target_logits=a["target_logits"][:1])),
    "no columns": (ValueError, lambda a: dict(target_logits=a["target_logits"][:, :0])),
    "32-bit drafts": (TypeError, lambda a: dict(draft_tokens=a["draft_tokens"].int())),
    "64-bit rows": (TypeError, lambda a: dict(cu_rows=a["cu_rows"].long())),
    "64-bit u": (TypeError, lambda a: dict(u=a["u"].double())),
    "fp16 noise": (TypeError, lambda a: dict(noise=a["noise"].half())),
    "drafts of other rows": (ValueError, lambda a: dict(draft_tokens=a["draft_tokens"][:2])),
    "u of other rows": (ValueError, lambda a: dict(u=a["u"][:2])),
    "noise of one sequence": (ValueError, lambda a: dict(noise=a["noise"][:1])),
    "noise of other columns": (ValueError, lambda a: dict(noise=a["noise"][:, :39])),
    "strided u": (ValueError, lambda a: dict(u=torch.zeros(6, device=a["u"].device)[::2])),
    "columns apart": (ValueError, lambda a: dict(target_logits=torch.zeros(5, 80, device=a["u"].device)[:, ::2])),
    "overlapping noise": (ValueError, lambda a: dict(noise=a["noise"][:1].expand(2, 40))),
    "draft logits of another type": (TypeError, lambda a: dict(draft_logits=torch.zeros(3, 40, dtype=F16, device=a["u"].device))),
    "draft logits of other rows": (ValueError, lambda a: dict(draft_logits=torch.zeros(5, 40, device=a["u"].device))),
    "draft logits on the host": (ValueError, lambda a: dict(draft_logits=torch.zeros(3, 40))),
    "temperature of another type": (TypeError, lambda a: dict(temperature=torch.ones(2, dtype=F16, device=a["u"].device))),
    "temperature of other sequences": (ValueError, lambda a: dict(temperature=torch.ones(3, device=a["u"].device))),
    "temperature on the host": (ValueError, lambda a: dict(temperature=torch.ones(2))),
    "a number for temperature": (TypeError, lambda a: dict(temperature=1.0)),
    "max_drafts below 0": (ValueError, lambda a: dict(max_drafts=-1)),
    "u on the host": (ValueError, lambda a: dict(u=a["u"].cpu())),
    "logits on the host": (ValueError, lambda a: dict(target_logits=a["target_logits"].cpu())),
}


@pytest.mark.parametrize("name", VERIFY)
def test_verify_refuses(cuda, name):
    from omlx_exl3_b200 import verify_drafts
    args = dict(target_logits=torch.zeros(5, 40, device=cuda), draft_tokens=torch.zeros(3, dtype=I64, device=cuda),
                cu_rows=torch.tensor([0, 3, 5], dtype=I32, device=cuda), u=torch.zeros(3, device=cuda),
                noise=torch.ones(2, 40, device=cuda), max_drafts=2)
    _refused(verify_drafts, args, VERIFY[name])
