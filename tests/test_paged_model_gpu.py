"""The paged cache in use: the operators one after the other against the definitions in 64 bits, and a stack that reads a content once,
answers questions that come later and goes on after an eviction, against its own packed forward."""

import numpy as np
import pytest
import torch

from oracle import attention as OA
from oracle import gemma as OG
from oracle import paged as OP
from spinf_serve_b200 import ops
from spinf_serve_b200 import packer as P
from spinf_serve_b200.paged import PagedReader
from spinf_serve_b200.scorer import forward_one

pytestmark = pytest.mark.gpu


def test_append_attend_evict_and_on(dev):
    """two prompts read in chunks with the slots' weights kept, cut back, then four single tokens: after every call the attention equals
    the definition over the slots that are there, and the eviction keeps the slots its own weights choose"""
    H, h, D, page, keep, recent = 8, 4, 128, 32, 100, 24
    g = torch.Generator().manual_seed(1)
    k = torch.zeros((40, h, page, D), dtype=torch.bfloat16, device=dev)
    v = torch.zeros_like(k)
    order = torch.randperm(40, generator=g).to(torch.int32)
    table, new_table = order[:16].view(2, 8).to(dev), order[16:24].view(2, 4).to(dev)
    lens, w = [0, 0], torch.zeros((2, h, 256), device=dev)
    wq, wk = (1 + 0.1 * torch.randn(D, generator=g).to(dev).to(torch.bfloat16) for _ in range(2))
    inv = (10000.0 ** (-torch.arange(0, D, 2).float() / D)).to(dev)
    pos = [0, 0]

    def call(table, counts):
        n = sum(counts)
        qkv = torch.randn((n, (H + 2 * h) * D), generator=g).to(torch.bfloat16).to(dev)
        where = torch.cat([torch.arange(p, p + c) for p, c in zip(pos, counts)]).to(torch.int32).to(dev)
        cos, sin = ops.rope_table(where, inv)
        for b, c in enumerate(counts):
            lens[b] += c
            pos[b] += c
        on = torch.tensor(lens, dtype=torch.int32, device=dev)
        cu = torch.tensor([0, counts[0], n], dtype=torch.int32, device=dev)
        before = w.clone()
        q = ops.paged_append(qkv, H, h, D, k, v, table, on, cu, wq=wq, wk=wk, cos=cos, sin=sin, norm_v=True)
        out = ops.paged_attention(q, k, v, table, on, cu, max(counts), D**-0.5, weights=w)
        want, weights, mag, big = OP.attention(q.cpu(), k.cpu(), v.cpu(), table.cpu(), lens, cu.cpu(), D**-0.5)
        # the result's rounding and p's (half a step of bf16 each), and fp32 sums of D products and up to 256 slots
        rel = torch.expm1(2 * (D + 8) * 2.0**-24 * big) + 320 * 2.0**-24 + 2.0**-21
        assert ((out.double().cpu() - want).abs() <= 2.0**-8 * want.abs() + (2.0**-8 * 1.01 + rel[..., None]) * mag * 1.01).all()
        for b in range(2):
            ref = before[b, :, : lens[b]].double().cpu() + weights[b]
            assert ((w[b, :, : lens[b]].double().cpu() - ref).abs() <= (float(rel.max()) + 2.0**-20) * ref + 1e-30).all()
        return on

    for counts in ((90, 3), (70, 60), (1, 81), (40, 1)):
        on = call(table, counts)
    slots = [[OP.evict(w[b, x, : lens[b]].cpu(), lens[b], keep, recent) for x in range(h)] for b in range(2)]
    before = [OP.gather(k.cpu(), table[b].cpu(), lens[b]) for b in range(2)]
    on, kept, w_new = ops.paged_evict(k, v, table, on, w, keep, recent, new_table)
    for b in range(2):
        after = OP.gather(k.cpu(), new_table[b].cpu(), keep)
        for x in range(h):
            assert kept[b, x].tolist() == slots[b][x] and torch.equal(after[x], before[b][x][slots[b][x]])
            assert torch.equal(w_new[b, x], w[b, x, slots[b][x]])
    lens[:] = on.tolist()
    w[:, :, :keep], w[:, :, keep:] = w_new, 0.0
    for _ in range(4):
        call(new_table, (1, 1))


def _cfg():
    return dict(layers=3, hidden=512, heads=4, kv_heads=2, head_dim=128, ffn=1024, vocab=4096, window=64, pattern=3)


def _stack(dev, scheme):
    from spinf_serve_b200.gemma_stack import GemmaConfig, GemmaStack, GemmaWeights

    ocfg = OG.GemmaConfig(**_cfg())
    W = OG.init_weights(ocfg, seed=6)
    Q = OG.quantize(W, scheme)
    weights = GemmaWeights.from_bf16(GemmaConfig(**_cfg()), W, dev, scheme="bf16") if scheme == "bf16" else GemmaWeights.from_quantized(GemmaConfig(**_cfg()), W, Q, dev)
    return ocfg, W, Q, GemmaStack(weights)


def _packed(trunk, branches):
    prompts = [trunk + b for b in branches]
    pk = P.Packer(4096, 8192, align=True)
    (b,) = list(pk.push(0, P.build_grouped_tree(prompts, [P.ReadPlan.build([[7], [8]]) for _ in prompts]))) + list(pk.flush())
    return b


@pytest.mark.parametrize("scheme", ["bf16", "fp8row"])
def test_questions_that_come_later(dev, scheme):
    """a content read in chunks, then questions on forks of it, against one packed forward of content and questions"""
    ocfg, W, Q, stack = _stack(dev, scheme)
    rng = np.random.default_rng(2)
    trunk = rng.integers(5, 4096, 333).tolist()
    branches = [[20 + j] + rng.integers(5, 4096, int(rng.integers(2, 20))).tolist() for j in range(9)]
    b = _packed(trunk, branches)
    packed = forward_one(stack, b, dev, rows=True).float()  # the read rows: the branches' ends, in the batch's order
    reader = PagedReader(stack, n_pages=64, page=32, chunk=100)
    seq = reader.read(trunk)
    free = len(reader.cache.free)
    got = reader.ask(seq, branches)
    assert len(reader.cache.free) == free and seq.length == 333  # the forks are gone, the content is as it was
    # the oracle's own distance under one legitimate rounding change is the yardstick (P rounded to bf16 before P V)
    exact = OA.tree_attention
    plain = OG.forward(ocfg, W, Q, b.ids, b.art, b.end, b.pos, scheme=scheme)
    try:
        OA.tree_attention = lambda *a, **kw: exact(*a, **{**kw, "round_p": True})
        moved = OG.forward(ocfg, W, Q, b.ids, b.art, b.end, b.pos, scheme=scheme)
    finally:
        OA.tree_attention = exact
    ends = torch.as_tensor(np.asarray(b.sel), dtype=torch.int64)
    yard = float((moved[ends].float() - plain[ends].float()).norm() / plain[ends].float().norm())
    # every branch's row in the packed batch: the one that is nearest is its own (the rows are far apart)
    for j in range(len(branches)):
        d = (packed - got[j].float()).norm(dim=1) / got[j].float().norm()
        assert float(d.min()) < 3 * yard + 2e-3, f"branch {j}: {float(d.min())} from the packed forward, yardstick {yard}"
    assert len({int((packed - got[j].float()).norm(dim=1).argmin()) for j in range(len(branches))}) == len(branches)
    # each question alone gives the same bits (bf16 linears: rows do not depend on their neighbours; nor does the attention)
    if scheme == "bf16":
        for j in (0, 4, 8):
            assert torch.equal(reader.ask(seq, [branches[j]])[0], got[j])


def test_reading_with_weights_evicting_and_going_on(dev):
    _, _, _, stack = _stack(dev, "bf16")
    rng = np.random.default_rng(3)
    ids = rng.integers(5, 4096, 500).tolist()
    reader = PagedReader(stack, n_pages=80, page=16, chunk=128)
    seq, plain = reader.read(ids, weigh=True), reader.read(ids)
    assert torch.equal(reader.ask(seq, [[9, 8]]), reader.ask(plain, [[9, 8]]))  # keeping the weights changes nothing else
    # every row's weights sum to one per head: the full-attention layer's slots hold two heads' worth of 500 rows
    full = [i for i in range(3) if stack.cfg.layer_types[i] == "full_attention"]
    assert full == [2] and abs(float(seq.weights[2, 0, :500].sum()) - 1000.0) < 0.5
    with pytest.raises(RuntimeError, match="window"):
        reader.evict(seq, 40, 8)
    assert reader.evict(seq, 600, 100) is None
    before = seq.weights[2].clone()
    kept = reader.evict(seq, 128, 64)
    assert seq.length == 128 and seq.position == 500 and len(seq.pages) == 8
    for x in range(2):
        assert kept[2][x].tolist() == OP.evict(before[x, :500].cpu(), 500, 128, 64)
        assert kept[0][x].tolist() == list(range(372, 500))  # a sliding layer keeps the last slots
    out = reader.ask(seq, [[9, 8], [7]])
    assert torch.isfinite(out.float()).all()
    # the sliding layers see what they saw: with every layer sliding nothing changes
    reader.forward([seq], [[5]])
    assert seq.length == 129 and seq.position == 501
    for s in (seq, plain):
        reader.cache.close(s)
    assert sorted(reader.cache.free) == list(range(80))
    with pytest.raises(RuntimeError, match="out of pages"):
        reader.read(rng.integers(5, 4096, 3000).tolist())


def test_many_questions_on_a_long_content(dev, monkeypatch):
    """enough branches on enough content that the full-attention layers read it once for all of them: the same answers but for roundings (p
    to bf16 against another reference, once each way, and the output's: three times half a step of 2^-8 at most, relative)"""
    _, _, _, stack = _stack(dev, "bf16")
    rng = np.random.default_rng(8)
    reader = PagedReader(stack, n_pages=200, page=32)
    seq = reader.read(rng.integers(5, 4096, 2210).tolist())
    branches = [rng.integers(5, 4096, int(rng.integers(1, 12))).tolist() for _ in range(70)]
    seen = []
    attend = ops.paged_attention
    monkeypatch.setattr(ops, "paged_attention", lambda *a, **kw: (seen.append(kw["shared"]), attend(*a, **kw))[1])
    got = reader.ask(seq, branches)
    assert seen == [True] * 3
    monkeypatch.setattr(ops, "SHARE_BYTES", 1 << 40)
    apart = reader.ask(seq, branches)
    assert seen == [True] * 3 + [False] * 3
    off = ((got.double() - apart.double()).norm(dim=1) / apart.double().norm(dim=1)).max()
    assert 0 < off < 3 * 2.0**-8
