"""Batches over a paged cache for the tests, and the operators in 64 bits."""
import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}      # unit roundoff: half a spacing at 1


def make_batch(rows, lens, hkv, hd, ps, dtype, device, seed=0, spare=3, fill=float("nan")):
    """Pages in random order; every slot that no sequence holds (behind its end too) is `fill`. Returns a dict with the
    pages, the tables, and each sequence's dense (len, hkv, hd) keys and values."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // ps) for n in lens]
    num = sum(need) + spare
    order = torch.randperm(num, generator=g).tolist()
    kp = torch.full((num, hkv, ps, hd), fill, dtype=dtype)
    vp = torch.full((num, hkv, ps, hd), fill, dtype=dtype)
    cols = max(1, max(need))
    table = torch.full((len(rows), cols), -1, dtype=torch.int32)
    ks, vs, at = [], [], 0
    for s, n in enumerate(lens):
        n = max(n, 0)
        k = torch.randn((n, hkv, hd), generator=g).to(dtype)
        v = torch.randn((n, hkv, hd), generator=g).to(dtype)
        for c in range(need[s]):
            page = order[at]
            at += 1
            table[s, c] = page
            part = slice(c * ps, min(n, (c + 1) * ps))
            m = part.stop - part.start
            kp[page, :, :m] = k[part].transpose(0, 1)
            vp[page, :, :m] = v[part].transpose(0, 1)
        ks.append(k)
        vs.append(v)
    cu = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32)
    return {"kp": kp.to(device), "vp": vp.to(device), "table": table.to(device), "cu": cu.to(device),
            "lens": torch.tensor(lens, dtype=torch.int32).to(device), "k": ks, "v": vs, "rows": list(rows), "len": list(lens)}


def attn_exact(q, batch, scale):
    """(out, weight) in 64 bits: weight = sum_j p_j |v_j|, what rounding p to a few bits can move the output by;
    rows at negative positions are zero."""
    n, hq, hd = q.shape
    out = torch.zeros(n, hq, hd, dtype=torch.float64)
    weight = torch.zeros_like(out)
    at = 0
    for s, r in enumerate(batch["rows"]):
        k, v = batch["k"][s].double(), batch["v"][s].double()
        total = batch["len"][s]
        for i in range(r):
            pos = total - r + i
            if pos >= 0:
                g = hq // k.shape[1]
                kk = k[:pos + 1].repeat_interleave(g, dim=1)           # (pos + 1, hq, hd)
                vv = v[:pos + 1].repeat_interleave(g, dim=1)
                sc = torch.einsum("hd,thd->ht", q[at + i].double(), kk) * scale
                p = torch.softmax(sc, -1)
                out[at + i] = torch.einsum("ht,thd->hd", p, vv)
                weight[at + i] = torch.einsum("ht,thd->hd", p, vv.abs())
        at += r
    return out, weight


def attn_tolerance(out, weight, batch, dtype):
    """Elementwise bound: p rounded to the 16-bit type (u * weight; fp16 has an absolute floor of 2^-25 a position below
    2^-14), the output rounded once (u * |out|), and fp32 scores of a few units off by up to 2e-5 (64 to 128 products
    of O(1) rounded at 2^-24 each, then scaled), which moves p by that much relative, in numerator and sum."""
    u = UNIT[dtype]
    longest = max(1, max(batch["len"]))
    floor = 2.0 ** -25 * longest * 4.5 if dtype == torch.float16 else 0.0
    return u * weight + u * out.abs() + 4e-5 * weight + floor + 1e-6


def norm_rope_exact(x, w, eps, cos, sin, pos):
    """x (rows, heads, hd) -> RMSNorm and rotate-half rotation at pos (rows), in 64 bits."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    h = cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * h:]], -1)
