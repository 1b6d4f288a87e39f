"""Measured cases of the paged-serving operators: q/k/v post step into a paged cache, attention of new rows over that
cache, and verification of drafted tokens.

A batch is described by cu_rows (S + 1) and lens (S): sequence s feeds rows cu_rows[s] .. cu_rows[s + 1] - 1, and its cache
holds lens[s] positions once they are appended, so row i of it is at position lens[s] - rows[s] + i. page_table (S, P) names
the pages of each sequence in order; a page holds `page` positions of all kv heads."""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
THETA = 1000000.0


def listed():
    return [
        # one sequence decoding: the layer's q/k/v of one token; launch latency counts
        {"name": "append-decode-1", "op": "append", "seqs": 1, "rows": 1, "ctx": 4096, "spread": False, "mix": 1, "hq": 40,
         "hkv": 8, "hd": 128, "rot": 128, "page": 64, "in": "bf16", "cache": "f16", "norm": True},
        # a scheduler step of four prompts' chunks, ragged, 27B-class heads
        {"name": "append-chunks-4", "op": "append", "seqs": 4, "rows": 2048, "ctx": 2048, "spread": True, "mix": 2, "hq": 40,
         "hkv": 8, "hd": 128, "rot": 128, "page": 16, "in": "bf16", "cache": "bf16", "norm": True},
        # a decode batch at half the heads (two GPUs), half the head rotated
        {"name": "append-decode-67", "op": "append", "seqs": 67, "rows": 1, "ctx": 600, "spread": True, "mix": 3, "hq": 20,
         "hkv": 4, "hd": 128, "rot": 64, "page": 32, "in": "f16", "cache": "f16", "norm": True},
        # one sequence decoding at 4k context: latency
        {"name": "attn-decode-1", "op": "attn", "seqs": 1, "rows": 1, "ctx": 4096, "spread": False, "mix": 4, "hq": 40,
         "hkv": 8, "hd": 128, "page": 64, "cache": "f16"},
        # a decode batch with contexts of one token up to 8k: the cache's bytes count
        {"name": "attn-decode-64", "op": "attn", "seqs": 64, "rows": 1, "ctx": 8191, "spread": True, "mix": 5, "hq": 40,
         "hkv": 8, "hd": 128, "page": 16, "cache": "bf16"},
        # two long documents being decoded
        {"name": "attn-decode-long", "op": "attn", "seqs": 2, "rows": 1, "ctx": 65000, "spread": False, "mix": 6, "hq": 40,
         "hkv": 8, "hd": 128, "page": 128, "cache": "f16"},
        # verification of up to 7 drafts for a few sequences, heads of one GPU of two
        {"name": "attn-verify-9", "op": "attn", "seqs": 9, "rows": 8, "ctx": 4200, "spread": True, "mix": 7, "hq": 20,
         "hkv": 4, "hd": 128, "page": 32, "cache": "f16"},
        # chunks and single tokens of one scheduler step, small ungrouped heads
        {"name": "attn-mixed-hd64", "op": "attn", "seqs": 13, "rows": 777, "ctx": 3000, "spread": True, "mix": 8, "hq": 12,
         "hkv": 12, "hd": 64, "page": 16, "cache": "bf16"},
        # the second half of an 8k prompt in one chunk: the tensor cores count
        {"name": "attn-chunk-4096", "op": "attn", "seqs": 1, "rows": 4096, "ctx": 4096, "spread": False, "mix": 9, "hq": 40,
         "hkv": 8, "hd": 128, "page": 64, "cache": "bf16"},
        # one sequence with three drafts, the whole vocabulary
        {"name": "verify-1", "op": "verify", "seqs": 1, "drafts": 3, "spread": False, "mix": 10, "vocab": 151936,
         "logits": "bf16", "dist": True, "masked": False},
        # a batch with up to seven drafts each and a draft distribution
        {"name": "verify-64", "op": "verify", "seqs": 64, "drafts": 7, "spread": True, "mix": 11, "vocab": 151936,
         "logits": "bf16", "dist": True, "masked": False},
        # drafts from a lookup of earlier text (no distribution), an odd vocabulary with forbidden tokens
        {"name": "verify-lookup-17", "op": "verify", "seqs": 17, "drafts": 5, "spread": True, "mix": 12, "vocab": 32003,
         "logits": "f32", "dist": False, "masked": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "verify"])
    if op == "verify":
        c = {"op": op, "seqs": _log_int(rng, 1, 96), "drafts": rng.randint(1, 7), "spread": rng.random() < 0.7,
             "mix": rng.randrange(1 << 20), "vocab": _log_int(rng, 1000, 152064), "logits": rng.choice(["bf16", "f16", "f32"]),
             "dist": rng.random() < 0.7, "masked": rng.random() < 0.3}
        while work(c)["bytes"] > 190e6:
            c["seqs"] = (c["seqs"] + 1) // 2
        return c
    hkv = rng.choice([1, 2, 4, 8])
    c = {"op": op, "seqs": _log_int(rng, 1, 96), "rows": rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 4096)]),
         "ctx": _log_int(rng, 1, 66000), "spread": rng.random() < 0.7, "mix": rng.randrange(1 << 20),
         "hq": hkv * rng.choice([1, 2, 4, 5, 7, 8]), "hkv": hkv, "hd": rng.choice([64, 128, 128]),
         "page": rng.choice([16, 32, 64, 128])}
    if op == "append":
        c["ctx"] = min(c["ctx"], 8192)
        c.update({"in": rng.choice(["f16", "bf16"]), "cache": rng.choice(["f16", "bf16"]), "norm": rng.random() < 0.8})
        c["rot"] = rng.choice([c["hd"], c["hd"] // 2])
        while work(c)["bytes"] > 100e6 or c["seqs"] * (c["rows"] + c["ctx"]) * c["hkv"] * c["hd"] > 1e8:
            c["seqs"], c["rows"], c["ctx"] = (c["seqs"] + 1) // 2, (c["rows"] + 1) // 2, (c["ctx"] + 1) // 2
        return c
    c["cache"] = rng.choice(["f16", "bf16"])
    # no more than the largest listed chunk, and a batch's padded scores and keys stay within a few GB
    while (work(c)["flops"] > 5e11 or c["seqs"] * (c["rows"] + c["ctx"]) * c["hkv"] * c["hd"] > 6e8
           or c["seqs"] * c["hq"] * c["rows"] * (c["rows"] + c["ctx"]) > 1.4e9):
        c["seqs"], c["rows"], c["ctx"] = (c["seqs"] + 1) // 2, (c["rows"] + 1) // 2, (c["ctx"] + 1) // 2
    return c


def _lengths(case):
    """New rows and earlier context of each sequence, from the case alone. Spread ones go by their logarithm: a scheduler's
    batch has long and short sequences side by side; the first keeps the stated sizes."""
    rng = random.Random(case["mix"])
    if case["op"] == "verify":
        drafts = [rng.randint(0, case["drafts"]) if case["spread"] else case["drafts"] for _ in range(case["seqs"])]
        drafts[0] = case["drafts"]
        return [d + 1 for d in drafts], None
    rows = [_log_int(rng, 1, case["rows"]) if case["spread"] else case["rows"] for _ in range(case["seqs"])]
    ctx = [_log_int(rng, 1, case["ctx"] + 1) - 1 if case["spread"] else case["ctx"] for _ in range(case["seqs"])]
    rows[0], ctx[0] = case["rows"], case["ctx"]
    return rows, ctx


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rows, ctx = _lengths(case)
    S, N = len(rows), sum(rows)
    cu = torch.tensor([sum(rows[:i]) for i in range(S + 1)], dtype=torch.int32).cuda()
    if case["op"] == "verify":
        return _prepare_verify(case, gen, rows, cu)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    hq, hkv, hd, ps = case["hq"], case["hkv"], case["hd"], case["page"]
    cache = DTYPES[case["cache"]]
    total = [r + c for r, c in zip(rows, ctx)]
    need = [-(-t // ps) for t in total]
    pages = sum(need) + 3
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    host = torch.full((S, max(need)), -1, dtype=torch.long)        # -1: no page there
    at = 0
    for s, n in enumerate(need):
        host[s, :n] = torch.arange(at, at + n)
        at += n
    host = host.cuda()
    table = torch.where(host < 0, torch.full_like(order[0], -1), order[host.clamp(min=0)]).contiguous()
    lens = torch.tensor(total, dtype=torch.int32).cuda()
    st = {"case": case, "cu": cu, "lens": lens, "table": table, "max_rows": max(rows)}
    st["kp"] = normal(pages, hkv, ps, hd).to(cache)
    st["vp"] = normal(pages, hkv, ps, hd).to(cache)
    if case["op"] == "attn":
        # what lies behind a sequence's end in its last page is whatever was there before
        last = table.gather(1, ((lens.long() - 1) // ps)[:, None])[:, 0].long()
        dead = torch.arange(ps, device="cuda")[None] > ((lens.long() - 1) % ps)[:, None]
        for t in (st["kp"], st["vp"]):
            tail = t[last]
            tail.masked_fill_(dead[:, None, :, None], float("nan"))
            t[last] = tail
        st["q"] = (1.5 * normal(N, hq, hd)).to(cache)
        return st
    src = DTYPES[case["in"]]
    qkv = (2 * normal(N, (hq + 2 * hkv) * hd)).to(src)              # the fused projection's output
    st["q"], st["k"], st["v"] = qkv.split([hq * hd, hkv * hd, hkv * hd], dim=1)
    st["wq"] = (1 + 0.1 * normal(hd)).to(src) if case["norm"] else None
    st["wk"] = (1 + 0.1 * normal(hd)).to(src) if case["norm"] else None
    half = case["rot"] // 2
    inv = THETA ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    ang = torch.arange(max(total), dtype=torch.float64, device="cuda")[:, None] * inv
    st["cos"], st["sin"] = torch.cos(ang).float(), torch.sin(ang).float()
    return st


def _prepare_verify(case, gen, rows, cu):
    S, R, V = len(rows), sum(rows), case["vocab"]
    dt = DTYPES[case["logits"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def exponential(*shape):
        return torch.empty(*shape, device="cuda").exponential_(generator=gen).clamp_(min=1e-20)

    # a few likely tokens above a broad floor, and a draft model that mostly agrees
    target = 2 * normal(R, V)
    likely = torch.randint(0, V, (R, 12), device="cuda", generator=gen)
    target.scatter_add_(1, likely, 7 + 2 * normal(R, 12))
    if case["masked"]:
        target.masked_fill_(torch.rand(R, V, device="cuda", generator=gen) < 0.4, float("-inf"))
    seq = torch.repeat_interleave(torch.arange(S, device="cuda"), torch.tensor(rows).cuda())
    drafted = torch.ones(R, dtype=torch.bool, device="cuda")
    drafted[cu[1:].long() - 1] = False                              # the last row of a sequence has no draft to judge
    temp = torch.tensor([0.0, 0.7, 1.0], device="cuda")[torch.randint(0, 3, (S,), device="cuda", generator=gen)]
    temp[0] = 1.0
    draft = (0.95 * target[drafted].clamp(min=-1e4) + 0.7 * normal(R - S, V)).to(dt)
    t = temp[seq[drafted]][:, None]
    pick = torch.where(t > 0, draft.float() / t.clamp(min=1e-3) - exponential(R - S, V).log(), draft.float())
    return {"case": case, "cu": cu, "max_drafts": max(rows) - 1, "target": target.to(dt), "temp": temp,
            "tokens": pick.argmax(1), "draft": draft if case["dist"] else None, "noise": exponential(S, V),
            "u": torch.rand(R - S, device="cuda", generator=gen)}


def run(state):
    op = state["case"]["op"]
    if op == "append":
        return (_append_own if own else _append_plain)(state)
    if op == "attn":
        return (_attn_own if own else _attn_plain)(state)
    return (_verify_own if own else _verify_plain)(state)


def _append_own(st):
    from omlx_exl3_b200.paged import paged_qkv_post
    q = paged_qkv_post(st["q"], st["k"], st["v"], st["wq"], st["wk"], EPS, st["cos"], st["sin"], st["kp"], st["vp"],
                       st["table"], st["cu"], st["lens"])
    return {"q": q, "k_pages": st["kp"], "v_pages": st["vp"]}


def _attn_own(st):
    from omlx_exl3_b200.paged import paged_attn
    return paged_attn(st["q"], st["kp"], st["vp"], st["table"], st["cu"], st["lens"])


def _verify_own(st):
    from omlx_exl3_b200.speculative import verify_drafts
    tokens, count, prob = verify_drafts(st["target"], st["tokens"], st["cu"], st["u"], st["noise"], st["max_drafts"],
                                        draft_logits=st["draft"], temperature=st["temp"])
    return {"tokens": tokens, "count": count, "accept_prob": prob}


def _rows_of(st, n):
    """Sequence and position of each row."""
    rows = torch.arange(n, device="cuda")
    seq = torch.searchsorted(st["cu"][1:].long(), rows, right=True)
    pos = st["lens"].long()[seq] - st["cu"].long()[seq + 1] + rows
    return seq, pos


def _norm_rope(x, w, cos, sin):
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    h = cos.shape[-1]
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * h:]], -1)


def _append_plain(st):
    c = st["case"]
    n, hd, ps, dt = st["q"].shape[0], c["hd"], c["page"], st["kp"].dtype
    seq, pos = _rows_of(st, n)
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]
    q = _norm_rope(st["q"].float().view(n, -1, hd), st["wq"], cos, sin).to(dt)
    k = _norm_rope(st["k"].float().view(n, -1, hd), st["wk"], cos, sin).to(dt)
    page = st["table"][seq, pos // ps].long()
    st["kp"][page, :, pos % ps] = k
    st["vp"][page, :, pos % ps] = st["v"].view(n, -1, hd).to(dt)
    return {"q": q, "k_pages": st["kp"], "v_pages": st["vp"]}


def _attn_plain(st):
    c = st["case"]
    hkv, hd, g, ps = c["hkv"], c["hd"], c["hq"] // c["hkv"], c["page"]
    n, m, S = st["q"].shape[0], st["max_rows"], st["lens"].shape[0]
    seq, pos = _rows_of(st, n)
    slot = torch.arange(n, device="cuda") - st["cu"].long()[seq]
    lens = st["lens"].long()
    T = st["table"].shape[1] * ps

    def gather(pages):                                              # (S, hkv, T, hd), zero behind each sequence's end
        x = pages[st["table"].clamp(min=0).long()].transpose(1, 2).reshape(S, hkv, T, hd).float()
        return x.masked_fill_((torch.arange(T, device="cuda")[None] >= lens[:, None])[:, None, :, None], 0.0)

    q = torch.zeros(S, m, hkv, g, hd, device="cuda")
    q[seq, slot] = st["q"].float().view(n, hkv, g, hd)
    last = torch.full((S, m), -1, device="cuda", dtype=torch.long)
    last[seq, slot] = pos                                           # padding rows see nothing
    q = q.permute(0, 2, 1, 3, 4).reshape(S, hkv, m * g, hd)
    s = q @ gather(st["kp"]).transpose(2, 3)
    s.mul_(1.0 / math.sqrt(hd))
    hidden = torch.arange(T, device="cuda")[None, None] > last[:, :, None]
    s.view(S, hkv, m, g, T).masked_fill_(hidden[:, None, :, None], float("-inf"))
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    s.sub_(top).exp_()
    o = (s @ gather(st["vp"])) / s.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.view(S, hkv, m, g, hd).permute(0, 2, 1, 3, 4)[seq, slot]
    return o.reshape(n, c["hq"], hd).to(st["q"].dtype)


def _lowest_argmax(x):
    """The first column with the row's largest value."""
    col = torch.arange(x.shape[-1], device="cuda")
    return torch.where(x == x.amax(-1, keepdim=True), col, x.shape[-1]).amin(-1)


def _softmax(x, temp, greedy_at):
    """softmax(x / temp) per row, one-hot at `greedy_at` where temp is 0."""
    x = x - x.amax(-1, keepdim=True)
    e = torch.exp(x / torch.where(temp > 0, temp, torch.ones_like(temp))[:, None])
    p = e / e.sum(-1, keepdim=True)
    hot = torch.arange(x.shape[-1], device="cuda")[None] == greedy_at[:, None]
    return torch.where((temp > 0)[:, None], p, hot.float())


def _verify_plain(st):
    cu, target, tokens = st["cu"].long(), st["target"].float(), st["tokens"]
    S, R, D = cu.shape[0] - 1, target.shape[0], st["max_drafts"]
    row = torch.arange(R, device="cuda")
    seq = torch.searchsorted(cu[1:], row, right=True)
    drafted = row + 1 < cu[1:][seq]
    drow, dseq = row[drafted], seq[drafted]
    p = _softmax(target, st["temp"][seq], _lowest_argmax(target))
    hot = (torch.arange(target.shape[1], device="cuda")[None] == tokens[:, None]).float()
    q = hot if st["draft"] is None else _softmax(st["draft"].float(), st["temp"][dseq], tokens)
    pd, qd = p[drow].gather(1, tokens[:, None])[:, 0], q.gather(1, tokens[:, None])[:, 0]
    prob = torch.where(qd > 0, (pd / qd).clamp(max=1.0), (pd > 0).float())
    ok = torch.zeros(S, D + 1, dtype=torch.long, device="cuda")
    given = torch.full((S, D + 1), -1, dtype=torch.long, device="cuda")
    at = drow - cu[dseq]
    ok[dseq, at] = (st["u"] < prob).long()
    given[dseq, at] = tokens
    n = ok.cumprod(1).sum(1)
    at_row = cu[:-1] + n
    left = p[at_row]
    rejected = at_row + 1 < cu[1:]
    dcol = (at_row - torch.arange(S, device="cuda")).clamp(max=max(q.shape[0] - 1, 0))
    rest = (left - q[dcol]).clamp(min=0.0) if q.shape[0] else left
    use = rejected & (rest.amax(-1) > 0)
    race = torch.where(use[:, None], rest, left) / st["noise"]
    nxt = torch.where(race.amax(-1) > 0, _lowest_argmax(race), -1)
    col = torch.arange(D + 1, device="cuda")[None]
    out = torch.where(col < n[:, None], given, torch.where(col == n[:, None], nxt[:, None], -1))
    return {"tokens": out, "count": (n + 1).to(torch.int32), "accept_prob": prob}


def work(case):
    rows, ctx = _lengths(case)
    S, N = len(rows), sum(rows)
    if case["op"] == "verify":
        size = 4 if case["logits"] == "f32" else 2
        logits = N + (N - S if case["dist"] else 0)
        return {"bytes": logits * case["vocab"] * size + S * case["vocab"] * 4 + N * 24, "flops": 5.0 * logits * case["vocab"]}
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    if case["op"] == "append":
        return {"bytes": N * ((hq + 2 * hkv) * hd * 4 + case["rot"] * 4), "flops": 7.0 * N * (hq + hkv) * hd}
    seen = sum(r * c + r * (r + 1) // 2 for r, c in zip(rows, ctx))
    cached = sum(r + c for r, c in zip(rows, ctx))
    return {"bytes": 4 * hd * (hkv * cached + hq * N), "flops": 4.0 * hd * hq * seen}


def exact(case, seed):
    """The operators' definitions in 64 bits, one sequence (and kv head) at a time."""
    st = prepare(case, seed)
    if case["op"] == "verify":
        return _verify_exact(st)
    cu, lens, table = st["cu"].tolist(), st["lens"].tolist(), st["table"].long()
    hq, hkv, hd, ps = case["hq"], case["hkv"], case["hd"], case["page"]
    g = hq // hkv
    if case["op"] == "attn":
        out = torch.zeros(cu[-1], hq, hd, dtype=torch.float64, device="cuda")
        for s, total in enumerate(lens):
            a, b = cu[s], cu[s + 1]
            j = torch.arange(total, device="cuda")
            page = table[s, j // ps]
            i = torch.arange(a, b, device="cuda") - b + total       # each row's own position
            for h in range(hkv):
                k, v = st["kp"][page, h, j % ps].double(), st["vp"][page, h, j % ps].double()
                for r in range(0, b - a, 512):
                    q = st["q"][a + r:min(b, a + r + 512), h * g:(h + 1) * g].double()
                    x = torch.einsum("rgd,td->rgt", q, k) / hd ** 0.5
                    x = x.masked_fill(j > i[r:r + 512, None, None], float("-inf"))
                    out[a + r:min(b, a + r + 512), h * g:(h + 1) * g] = torch.einsum("rgt,td->rgd", torch.softmax(x, -1), v)
        return out
    n = cu[-1]
    kp, vp = st["kp"].double(), st["vp"].double()
    qo = torch.empty(n, hq, hd, dtype=torch.float64, device="cuda")
    half = case["rot"] // 2

    def turned(x, w, c, d):
        x = x.double()
        if w is not None:
            x = w.double() * x * (x.square().sum(-1, keepdim=True) / hd + EPS).rsqrt()
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * torch.complex(c, d)
        return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)

    for s, total in enumerate(lens):
        a, b = cu[s], cu[s + 1]
        i = torch.arange(total - (b - a), total, device="cuda")
        c, d = st["cos"][i].double()[:, None], st["sin"][i].double()[:, None]
        qo[a:b] = turned(st["q"][a:b].reshape(b - a, hq, hd), st["wq"], c, d)
        page = table[s, i // ps]
        kp[page, :, i % ps] = turned(st["k"][a:b].reshape(b - a, hkv, hd), st["wk"], c, d)
        vp[page, :, i % ps] = st["v"][a:b].reshape(b - a, hkv, hd).double()
    return {"q": qo, "k_pages": kp, "v_pages": vp}


def _verify_exact(st):
    cu, temp, tokens = st["cu"].tolist(), st["temp"].tolist(), st["tokens"].tolist()
    prob = []
    for s, t in enumerate(temp):
        for r in range(cu[s], cu[s + 1] - 1):
            i = r - s                                               # the draft that row r judges
            x = st["target"][r].double()
            if t == 0:
                first = torch.nonzero(x == x.max())[0, 0].item()
                prob.append(1.0 if first == tokens[i] else 0.0)
                continue
            p = torch.softmax(x / t, -1)[tokens[i]].item()
            q = 1.0 if st["draft"] is None else torch.softmax(st["draft"][i].double() / t, -1)[tokens[i]].item()
            prob.append(min(1.0, p / q) if q > 0 else float(p > 0))
    return {"tokens": None, "count": None, "accept_prob": torch.tensor(prob, dtype=torch.float64)}
