"""The paged K/V cache's operators as measured cases: the append of a step's rows (head norms and rotary embedding in the same pass),
the attention of new tokens over the cached pages (with the keys' accumulated attention weight where asked), and the eviction by that
weight. `run` is one pass through an operator: in elementary torch operations, or through the library where `own` is true.

Head layouts are the stacks' own (12B: 16 / 8 heads of 256, 31B-class: 32 / 16 of 128, hybrid 27B: 24 / 4 of 256 with 64 rotary
dimensions) and two with wider groups. A cache page holds `page` tokens of every key / value head."""

import math

import torch

own = False

LAYOUTS = ((16, 8, 256), (32, 16, 128), (24, 4, 256), (8, 8, 128), (32, 4, 128))
PAGES = (16, 32, 64, 128)
EPS = 1e-6


def listed():
    return [
        # one decoding step's projection rows of a full batch, 12B layout
        {"name": "append_step_64", "op": "append", "H": 16, "h": 8, "D": 256, "page": 64, "seqs": 64, "new": 1, "cached": 1500, "ragged": True, "rotary": 256},
        # a prompt pass of the 31B-class layout: 8 192 rows in four sequences
        {"name": "append_prompt_8192", "op": "append", "H": 32, "h": 16, "D": 128, "page": 64, "seqs": 4, "new": 2048, "cached": 0, "ragged": False, "rotary": 128},
        # few decoding slots on one content of the benchmark's length: launch latency counts
        {"name": "attend_step_4", "op": "attend", "H": 16, "h": 8, "D": 256, "page": 64, "seqs": 4, "new": 1, "cached": 1500, "ragged": False, "window": 0, "weights": False},
        # a full decoding batch over caches of very different lengths, 31B-class layout
        {"name": "attend_step_64_ragged", "op": "attend", "H": 32, "h": 16, "D": 128, "page": 32, "seqs": 64, "new": 1, "cached": 8191, "ragged": True, "window": 0, "weights": False},
        # one slot over a very long document, hybrid layout (six query heads per key / value head)
        {"name": "attend_step_131k", "op": "attend", "H": 24, "h": 4, "D": 256, "page": 128, "seqs": 1, "new": 1, "cached": 131071, "ragged": False, "window": 0, "weights": False},
        # 56 question branches of a content whose trunk is cached once (their tables share its pages)
        {"name": "attend_branches_56", "op": "attend", "H": 16, "h": 8, "D": 256, "page": 64, "seqs": 56, "new": 12, "cached": 2000, "ragged": False, "window": 0, "weights": False, "shared": True},
        # a chunk of a long prompt over what was read before
        {"name": "attend_chunk_2048", "op": "attend", "H": 16, "h": 8, "D": 256, "page": 64, "seqs": 1, "new": 2048, "cached": 16384, "ragged": False, "window": 0, "weights": False},
        # prompts and chunks of several contents in one call on a sliding layer, 31B-class layout
        {"name": "attend_chunks_window", "op": "attend", "H": 32, "h": 16, "D": 128, "page": 64, "seqs": 7, "new": 1501, "cached": 4001, "ragged": True, "window": 1024, "weights": False},
        # a decoding step that keeps the keys' accumulated weight
        {"name": "attend_step_weights", "op": "attend", "H": 16, "h": 8, "D": 256, "page": 64, "seqs": 16, "new": 1, "cached": 4095, "ragged": True, "window": 0, "weights": True},
        # the prompt's last chunk with the accumulated weight, from which the eviction starts
        {"name": "attend_chunk_weights", "op": "attend", "H": 32, "h": 16, "D": 128, "page": 64, "seqs": 1, "new": 1024, "cached": 7168, "ragged": False, "window": 0, "weights": True},
        # a few slots cut back to their budget
        {"name": "evict_4", "op": "evict", "H": 16, "h": 8, "D": 256, "page": 64, "seqs": 4, "cached": 2049, "ragged": False, "keep": 1024, "recent": 256},
        # long documents cut to a quarter
        {"name": "evict_16_long", "op": "evict", "H": 32, "h": 16, "D": 128, "page": 64, "seqs": 16, "cached": 16000, "ragged": True, "keep": 4096, "recent": 1024},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    H, h, D = rng.choice(LAYOUTS)
    page = rng.choice(PAGES)
    case = {"op": rng.choice(["append", "attend", "attend", "attend", "evict"]), "H": H, "h": h, "D": D, "page": page, "ragged": rng.random() < 0.7}
    if case["op"] == "append":
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, min(2048, 8192 // seqs))
        return case | {"seqs": seqs, "new": new, "cached": _log(rng, 1, 4096) - 1, "rotary": rng.choice([D, D, 64, 0])}
    if case["op"] == "evict":
        seqs = _log(rng, 1, 32)
        cached = _log(rng, 64, min(32768, 262144 // seqs))
        keep = _log(rng, 16, cached)
        return case | {"seqs": seqs, "cached": cached, "keep": keep, "recent": rng.choice([0, 1, keep // 4, keep // 2, keep])}
    kind = rng.choice(["step", "branch", "chunk"])
    case |= {"window": rng.choice([0, 0, 512, 1024]), "weights": rng.random() < 0.3}
    if kind == "step":
        seqs = _log(rng, 1, 64)
        return case | {"seqs": seqs, "new": 1, "cached": _log(rng, 1, min(131072, 262144 // seqs)) - 1}
    if kind == "branch":
        seqs = _log(rng, 1, 64)
        return case | {"seqs": seqs, "new": rng.randint(2, 48), "cached": _log(rng, 64, 4096), "shared": rng.random() < 0.5}
    seqs = _log(rng, 1, 8)
    new = _log(rng, 32, 2048 // seqs)
    return case | {"seqs": seqs, "new": new, "cached": _log(rng, 1, 16384 // seqs) - 1}


def _lengths(case):
    """(tokens cached before the call, new tokens) of every sequence: a ragged batch spreads over the lower nine tenths"""
    got = []
    for b in range(case["seqs"]):
        c, n = case["cached"], case.get("new", 0)
        if case["ragged"] and b:
            c -= (b * 2654435761 >> 7) % max(1, c * 9 // 10 + 1)
            if n > 1:
                n -= (b * 40503 >> 3) % max(1, n * 9 // 10)
        got.append((c, n))
    return got


def _cuda():
    return torch.device("cuda", torch.cuda.current_device())


def prepare(case, seed):
    dev = _cuda()
    g = torch.Generator(device=dev).manual_seed(seed)
    H, h, D, page, B = case["H"], case["h"], case["D"], case["page"], case["seqs"]
    lengths = _lengths(case)
    lens = [c + n for c, n in lengths]
    width = max(1, -(-max(lens) // page))
    whole = min(c for c, _ in lengths) // page if case.get("shared") else 0  # trunk pages that all tables begin with
    keep_pages = -(-case["keep"] // page) if case["op"] == "evict" else 0
    own_pages = [max(0, -(-x // page) - whole) for x in lens]
    total = whole + sum(own_pages) + B * keep_pages
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.zeros((B, width), dtype=torch.int32, device=dev)
    at = whole
    for b, k in enumerate(own_pages):
        table[b, :whole] = order[:whole]
        table[b, whole : whole + k] = order[at : at + k]
        at += k
    rnd = lambda *s: torch.randn(s, generator=g, device=dev, dtype=torch.bfloat16)  # noqa: E731
    st = {"case": case, "k": rnd(total, h, page, D), "v": rnd(total, h, page, D), "table": table,
          "lens": torch.tensor(lens, dtype=torch.int32, device=dev)}
    if case["op"] == "evict":
        st["new_table"] = order[at : at + B * keep_pages].view(B, keep_pages).contiguous()
        # accumulated weights: a heavy tail of much attended keys, and keys that nothing has attended to yet (exact zeros)
        w = torch.empty((B, h, width * page), device=dev).exponential_(1.0, generator=g).pow_(3.0)
        st["weights"] = w * (torch.rand(w.shape, generator=g, device=dev) > 0.05)
        return st
    cu = [0]
    for _, n in lengths:
        cu.append(cu[-1] + n)
    st["cu"] = torch.tensor(cu, dtype=torch.int32, device=dev)
    st["max_q"] = max(n for _, n in lengths)
    if case["op"] == "append":
        st["qkv"] = rnd(cu[-1], (H + 2 * h) * D) * 1.7
        st["wq"], st["wk"] = 1 + 0.1 * rnd(D), 1 + 0.1 * rnd(D)
        if case["rotary"]:
            pos = torch.cat([torch.arange(c, c + n, device=dev) for c, n in lengths]).double()
            freq = 10000.0 ** (-torch.arange(0, case["rotary"], 2, device=dev).double() / case["rotary"])
            st["cos"] = torch.cos(pos[:, None] * freq).to(torch.bfloat16)
            st["sin"] = torch.sin(pos[:, None] * freq).to(torch.bfloat16)
        return st
    # normed queries and keys; a few keys stand out, so that rows attend unevenly
    loud = 1 + 0.5 * torch.randn((total, h, page, 1), generator=g, device=dev).abs()
    st["k"] = (st["k"] * loud).to(torch.bfloat16)
    st["q"] = rnd(cu[-1], H, D)
    if case["weights"]:
        st["weights"] = torch.rand((B, h, width * page), generator=g, device=dev)
        st["weights_out"] = torch.zeros_like(st["weights"])
    return st


def run(st):
    case = st["case"]
    if own:
        from spinf_serve_b200 import ops

        if case["op"] == "append":
            q = ops.paged_append(st["qkv"], case["H"], case["h"], case["D"], st["k"], st["v"], st["table"], st["lens"], st["cu"],
                                 wq=st["wq"], wk=st["wk"], cos=st.get("cos"), sin=st.get("sin"), eps=EPS, norm_v=True)
            return {"q": q, "k": st["k"], "v": st["v"]}
        if case["op"] == "evict":
            lens, kept, weights = ops.paged_evict(st["k"], st["v"], st["table"], st["lens"], st["weights"], case["keep"], case["recent"],
                                                  st["new_table"])
            return {"k": st["k"], "v": st["v"], "lens": lens, "kept": kept, "weights": weights}
        out = ops.paged_attention(st["q"], st["k"], st["v"], st["table"], st["lens"], st["cu"], st["max_q"], case["D"] ** -0.5,
                                  window=case["window"] or None, weights=st.get("weights"), weights_out=st.get("weights_out"))
        return {"out": out, "weights": st["weights_out"]} if case["weights"] else {"out": out}
    return {"append": _append, "attend": _attend, "evict": _evict}[case["op"]](st)


def _row_places(st, n):
    """sequence, index within it and cache slot of every new row"""
    rows = torch.arange(n, device=st["cu"].device)
    b = torch.searchsorted(st["cu"][1:].contiguous(), rows, right=True)
    i = rows - st["cu"][b]
    new = st["cu"][1:] - st["cu"][:-1]
    return b, i, (st["lens"] - new)[b] + i


def _rms(x, w=None):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return y if w is None else y * w


def _rotate(x, cos, sin):
    if cos is None:
        return x
    r = cos.shape[1]
    a, b, rest = x[..., :r], x[..., r : 2 * r], x[..., 2 * r :]
    c, s = cos.float()[:, None], sin.float()[:, None]
    return torch.cat([a * c - b * s, b * c + a * s, rest], -1)


def _append(st):
    case = st["case"]
    H, h, D, page = case["H"], case["h"], case["D"], case["page"]
    n = st["qkv"].shape[0]
    x = st["qkv"].float().view(n, H + 2 * h, D)
    q = _rotate(_rms(x[:, :H], st["wq"].float()), st.get("cos"), st.get("sin")).to(torch.bfloat16)
    k = _rotate(_rms(x[:, H : H + h], st["wk"].float()), st.get("cos"), st.get("sin")).to(torch.bfloat16)
    v = _rms(x[:, H + h :]).to(torch.bfloat16)
    b, _, slot = _row_places(st, n)
    pg = st["table"][b, slot // page].long()
    st["k"][pg, :, slot % page] = k
    st["v"][pg, :, slot % page] = v
    return {"q": q, "k": st["k"], "v": st["v"]}


def _attend(st):
    case = st["case"]
    H, h, D, page, B = case["H"], case["h"], case["D"], case["page"], case["seqs"]
    n, Q, G = st["q"].shape[0], st["max_q"], H // h
    b, i, _ = _row_places(st, n)
    new = st["cu"][1:] - st["cu"][:-1]
    L = st["table"].shape[1] * page
    kk = st["k"][st["table"].long()].permute(0, 2, 1, 3, 4).reshape(B, h, L, D).float()
    vv = st["v"][st["table"].long()].permute(0, 2, 1, 3, 4).reshape(B, h, L, D).float()
    qq = torch.zeros((B, Q, H, D), device=kk.device)
    qq[b, i] = st["q"].float()
    qq = qq.view(B, Q, h, G, D).permute(0, 2, 3, 1, 4).reshape(B, h, G * Q, D)
    s = (torch.matmul(qq, kk.transpose(2, 3)) * D**-0.5).view(B, h, G, Q, L)
    row = torch.arange(Q, device=kk.device)
    slot = (st["lens"] - new)[:, None] + row
    j = torch.arange(L, device=kk.device)
    seen = (j <= slot[..., None]) & (row[:, None] < new[:, None, None])
    if case["window"]:
        seen &= j > slot[..., None] - case["window"]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    p = p / total.clamp_min(1e-30)
    out = torch.matmul(p.view(B, h, G * Q, L), vv).view(B, h, G, Q, D).permute(0, 3, 1, 2, 4).reshape(B, Q, H, D)
    res = {"out": out[b, i].to(torch.bfloat16)}
    if case["weights"]:
        w = st["weights"] + p.sum((2, 3))
        res["weights"] = st["weights_out"].copy_(torch.where((j < st["lens"][:, None])[:, None], w, st["weights_out"]))
    return res


def _evict(st):
    case = st["case"]
    h, D, page, B, keep = case["h"], case["D"], case["page"], case["seqs"], case["keep"]
    L = st["weights"].shape[-1]
    j = torch.arange(L, device=st["k"].device)
    lens = st["lens"].long()[:, None, None]
    key = st["weights"].masked_fill(j >= lens - case["recent"], math.inf).masked_fill(j >= lens, -math.inf)
    first = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]  # ties: the lowest slot first
    if first.shape[-1] < keep:
        first = torch.nn.functional.pad(first, (0, keep - first.shape[-1]), value=L)
    valid = torch.arange(keep, device=j.device) < lens
    kept = torch.sort(first.masked_fill(~valid, L), dim=-1).values
    src = kept.clamp_max(L - 1)
    pg = torch.gather(st["table"].long()[:, None].expand(B, h, -1), 2, src // page)
    heads = torch.arange(h, device=j.device)[None, :, None].expand_as(src)
    out = torch.arange(keep, device=j.device)
    dst = st["new_table"].long()[:, None, out // page].expand(B, h, keep)
    off = (out % page).expand_as(dst)
    at = valid.expand_as(dst)
    for name in ("k", "v"):
        st[name][dst[at], heads[at], off[at]] = st[name][pg[at], heads[at], (src % page)[at]]
    weights = torch.gather(st["weights"], 2, src).masked_fill(~at, 0.0)
    return {"k": st["k"], "v": st["v"], "lens": lens[:, 0, 0].clamp_max(keep).to(torch.int32), "kept": kept.masked_fill(~at, -1).to(torch.int32),
            "weights": weights}


def work(case):
    H, h, D, page = case["H"], case["h"], case["D"], case["page"]
    lengths = _lengths(case)
    n = sum(x for _, x in lengths)
    if case["op"] == "append":  # the projection rows read once, q and the two pages' rows written once, the rotary tables read once
        return {"bytes": n * ((H + 2 * h) * D * 4 + 2 * case["rotary"]), "flops": n * (H + 2 * h) * D * 6}
    if case["op"] == "evict":  # every weight read once, the kept rows of K and V read and written once
        kept = sum(min(c, case["keep"]) for c, _ in lengths)
        return {"bytes": sum(c for c, _ in lengths) * h * 4 + kept * h * (8 * D + 12), "flops": 0}
    keys, pairs = 0, 0
    whole = min(c for c, _ in lengths) // page * page if case.get("shared") else 0
    for c, x in lengths:
        first = max(0, c + 1 - case["window"]) if case["window"] else 0
        keys += max(0, c + x - max(first, whole))
        pairs += sum(min(s + 1, case["window"] or s + 1) for s in range(c, c + x))
    keys += whole
    weight = sum(c + x for c, x in lengths) * h * 8 if case["weights"] else 0
    return {"bytes": keys * h * D * 4 + n * H * D * 4 + weight, "flops": pairs * H * D * 4}


def exact(case, seed):
    """the definitions in 64 bits, one sequence and key / value head at a time"""
    st = prepare(case, seed)
    H, h, D, page = case["H"], case["h"], case["D"], case["page"]
    lengths = _lengths(case)
    dev = st["k"].device
    slots = lambda b, a, e: (st["table"][b].long()[torch.arange(a, e, device=dev) // page], torch.arange(a, e, device=dev) % page)  # noqa: E731
    if case["op"] == "append":
        x = st["qkv"].double().view(-1, H + 2 * h, D)
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + EPS)
        x[:, :H] *= st["wq"].double()
        x[:, H : H + h] *= st["wk"].double()
        r = case["rotary"] // 2
        if r:
            turn = torch.complex(st["cos"].double(), st["sin"].double())[:, None]
            z = torch.complex(x[:, : H + h, :r], x[:, : H + h, r : 2 * r]) * turn
            x[:, : H + h, :r], x[:, : H + h, r : 2 * r] = z.real, z.imag
        k, v, at = st["k"].double(), st["v"].double(), 0
        for b, (c, m) in enumerate(lengths):
            pg, off = slots(b, c, c + m)
            k[pg, :, off], v[pg, :, off] = x[at : at + m, H : H + h], x[at : at + m, H + h :]
            at += m
        return {"q": x[:, :H], "k": k, "v": v}
    if case["op"] == "evict":
        weights = torch.zeros((case["seqs"], h, case["keep"]), dtype=torch.float64, device=dev)
        for b, (c, _) in enumerate(lengths):
            m = max(0, c - case["recent"])
            for g in range(h):
                w = st["weights"][b, g, :c].double()
                if c <= case["keep"]:
                    weights[b, g, :c] = w
                    continue
                quota = case["keep"] - min(case["recent"], c)
                chosen = torch.ones(c, dtype=torch.bool, device=dev)
                chosen[:m] = False
                if quota:
                    edge = torch.topk(w[:m], quota).values[-1]
                    chosen[:m] = w[:m] > edge
                    same = (w[:m] == edge).nonzero()[:, 0]
                    chosen[same[: quota - int(chosen[:m].sum())]] = True
                weights[b, g] = w[chosen]
        return {"k": None, "v": None, "lens": None, "kept": None, "weights": weights}
    out = torch.zeros((st["q"].shape[0], H, D), dtype=torch.float64, device=dev)
    weights = st["weights_out"].double() if case["weights"] else None
    at = 0
    for b, (c, m) in enumerate(lengths):
        pg, off = slots(b, 0, c + m)
        lag = torch.arange(c, c + m, device=dev)[:, None] - torch.arange(c + m, device=dev)
        hidden = (lag < 0) | (lag >= case["window"]) if case["window"] else lag < 0
        for g in range(h):
            heads = slice(g * (H // h), (g + 1) * (H // h))
            k, v = st["k"][pg, g, off].double(), st["v"][pg, g, off].double()
            s = torch.einsum("ihd,jd->hij", st["q"][at : at + m, heads].double(), k) / math.sqrt(D)
            p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            out[at : at + m, heads] = torch.einsum("hij,jd->ihd", p, v)
            if weights is not None:
                weights[b, g, : c + m] = st["weights"][b, g, : c + m].double() + p.sum((0, 1))
        at += m
    return {"out": out, "weights": weights} if weights is not None else {"out": out}
