"""GPU parity of the paged K/V cache's operators (append, attention, eviction) against their definitions in 64 bits, with every slot
that no row sees filled with NaN; streams, captured graphs, batch invariance and far offsets."""

import math

import pytest
import torch

from oracle import paged as OP
from spinf_serve_b200 import _lib, ops

pytestmark = pytest.mark.gpu

BF = 2.0**-8  # half a step of bf16, relative


class Call:
    """one call's tensors: NaN everywhere in the pools but in the sequences' slots; pages handed out in random order"""

    def __init__(self, dev, H, h, D, page, seqs, seed=0, token_major=False, spare=3, extra_rows=0, shared_tokens=0, loud=0.5):
        g = torch.Generator().manual_seed(seed)
        self.H, self.h, self.D, self.page, self.dev = H, h, D, page, dev
        self.lens, news = [L for L, _ in seqs], [n for _, n in seqs]
        B = len(seqs)
        shared = shared_tokens // page
        need = [max(0, -(-L // page) - shared) for L in self.lens]
        self.n_pages = sum(need) + shared + spare
        order = torch.randperm(self.n_pages, generator=g).to(torch.int32)
        width = max(1, max(-(-L // page) for L in self.lens))
        self.table = torch.full((B, width), -7, dtype=torch.int32)  # entries behind a sequence's pages are never used
        at = shared
        for b in range(B):
            self.table[b, :shared] = order[:shared]
            self.table[b, shared : shared + need[b]] = order[at : at + need[b]]
            at += need[b]
        self.free = order[at:]
        shape = (self.n_pages, page, h, D) if token_major else (self.n_pages, h, page, D)
        k, v = (torch.full(shape, math.nan, dtype=torch.bfloat16) for _ in range(2))
        if token_major:
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        for b in range(B):
            for s in range(self.lens[b]):
                pg = int(self.table[b, s // page])
                if math.isnan(float(k[pg, 0, s % page, 0])):
                    size = 1 + loud * torch.randn((h, 1), generator=g).abs()
                    k[pg, :, s % page] = (torch.randn((h, D), generator=g) * size).to(torch.bfloat16)
                    v[pg, :, s % page] = torch.randn((h, D), generator=g).to(torch.bfloat16)
        self.k, self.v = k, v
        cu = [0]
        for n in news:
            cu.append(cu[-1] + n)
        self.cu, self.n = torch.tensor(cu, dtype=torch.int32), cu[-1] + extra_rows
        self.max_q = max(news)
        self.q = torch.randn((self.n, H, D), generator=g).to(torch.bfloat16)
        self.gen = g
        self.lens_t = torch.tensor(self.lens, dtype=torch.int32)
        self.on = {x: getattr(self, x).to(dev) for x in ("table", "cu", "q", "lens_t")}
        keep_layout = lambda t: t.transpose(1, 2).contiguous().to(dev).transpose(1, 2) if token_major else t.to(dev)  # noqa: E731
        self.on["k"], self.on["v"] = keep_layout(k), keep_layout(v)

    def attend(self, window=None, **kw):
        o = self.on
        return ops.paged_attention(o["q"], o["k"], o["v"], o["table"], o["lens_t"], o["cu"], self.max_q, self.D**-0.5, window=window, **kw)

    def expect(self, window=None):
        return OP.attention(self.q, self.k, self.v, self.table, self.lens, self.cu, self.D**-0.5, window)


def score_noise(c, big, longest):
    """relative error of a p from fp32 sums: scores of D products each (two sides of the softmax), then a sum over the keys"""
    return torch.expm1(2 * (c.D + 8) * 2.0**-24 * big) + (longest + 64) * 2.0**-24 + 2.0**-21


def check_out(c, got, want, mag, big):
    rows = int(c.cu[-1])
    got, want = got[:rows].double().cpu(), want[:rows]
    rel = score_noise(c, big[:rows], max(c.lens))[..., None]
    # the result's rounding, p's rounding to bf16 (each at most half a step), and the fp32 sums
    tol = BF * want.abs() + (BF * (1 + BF) + rel) * mag[:rows] * (1 + BF) + 1e-30
    off = (got - want).abs() / tol
    assert not torch.isnan(got).any()
    assert off.max() <= 1.0, f"{float(off.max())} of the tolerance at {off.argmax()}"


LAYOUTS = [(16, 8, 256), (4, 2, 128), (6, 1, 256), (3, 3, 128), (8, 1, 128)]
MIXES = [
    [(1, 1)],
    [(0, 0), (5, 5), (1, 1), (0, 0)],
    [(127, 1), (128, 1), (129, 1), (255, 2), (16, 1)],
    [(700, 3), (33, 33), (64, 0), (1000, 1)],
    [(300, 40), (300, 17), (45, 45)],
    [(2, 5), (0, 3), (40, 41)],  # more rows than cached tokens: the first rows see nothing
]


@pytest.mark.parametrize("mix", range(len(MIXES)))
@pytest.mark.parametrize("H,h,D", LAYOUTS)
def test_attention_against_the_definition(dev, H, h, D, mix):
    page = (16, 32, 64, 128, 256)[(mix + H) % 5]
    c = Call(dev, H, h, D, page, MIXES[mix], seed=mix * 100 + H, token_major=mix % 2 == 1, extra_rows=2)
    out = torch.full((c.n, H, D), 7.0, dtype=torch.bfloat16, device=dev)
    got = c.attend(out=out)
    assert got.data_ptr() == out.data_ptr()
    want, _, mag, big = c.expect()
    check_out(c, got, want, mag, big)
    assert (got[int(c.cu[-1]) :] == 7.0).all()  # rows behind the last sequence
    for b, (L, n) in enumerate(MIXES[mix]):  # rows that see nothing
        for i in range(max(0, n - L)):
            assert (got[int(c.cu[b]) + i] == 0).all()


@pytest.mark.parametrize("window", [1, 7, 64, 200])
@pytest.mark.parametrize("H,h,D", LAYOUTS[:2])
def test_attention_with_a_window(dev, H, h, D, window):
    c = Call(dev, H, h, D, 32, [(900, 2), (150, 100), (64, 64), (1, 1), (513, 35), (30, 36)], seed=window)
    want, _, mag, big = c.expect(window)
    check_out(c, c.attend(window), want, mag, big)


@pytest.mark.parametrize("window", [None, 100])
@pytest.mark.parametrize("H,h,D", LAYOUTS)
def test_attention_keeps_the_slots_weights(dev, H, h, D, window):
    seqs = [(400, 1), (130, 20), (77, 77), (50, 0), (3, 5), (257, 6)]
    c = Call(dev, H, h, D, 64, seqs, seed=H + D, spare=0)
    _, weights, _, big = c.expect(window)
    cap = 513
    old = torch.rand((len(seqs), h, cap), generator=c.gen)
    w_in = old.to(dev)
    w_out = torch.full((len(seqs), h, cap), -3.0, device=dev)
    c.attend(window, weights=w_in, weights_out=w_out, decay=0.5)
    assert (w_in.cpu() == old).all()
    rel = float(score_noise(c, big, 400).max()) + 2.0**-21
    for b, (L, _) in enumerate(seqs):
        want = 0.5 * old[b, :, :L].double() + weights[b]
        assert ((w_out[b, :, :L].double().cpu() - want).abs() <= rel * want + 1e-30).all()
        assert (w_out[b, :, L:] == -3.0).all()
    # in place, and with decay 0 (the old values are not read)
    w2 = torch.full_like(w_in, math.nan)
    c.attend(window, weights=w2, decay=0.0)
    for b, (L, _) in enumerate(seqs):
        assert ((w2[b, :, :L].double().cpu() - weights[b]).abs() <= rel * weights[b] + 1e-30).all()
        assert torch.isnan(w2[b, :, L:]).all()


@pytest.mark.parametrize("shared", [0, 256])
def test_a_sequence_alone_equals_itself_in_a_batch(dev, shared):
    seqs = [(600, 12), (300, 1), (2000, 1), (600, 300), (331, 5), (420, 100)]
    c = Call(dev, 4, 2, 128, 64, seqs, seed=3, shared_tokens=shared)
    w = torch.zeros((len(seqs), 2, c.table.shape[1] * 64), device=dev)
    every = c.attend(weights=w)
    for b in range(len(seqs)):
        r0, r1 = int(c.cu[b]), int(c.cu[b + 1])
        w1 = torch.zeros_like(w[:1])
        cu = torch.tensor([0, r1 - r0], dtype=torch.int32, device=dev)
        one = ops.paged_attention(c.on["q"][r0:r1], c.on["k"], c.on["v"], c.on["table"][b : b + 1], c.on["lens_t"][b : b + 1], cu, r1 - r0, 128**-0.5, weights=w1)
        assert torch.equal(one, every[r0:r1]) and torch.equal(w1[0], w[b])


def test_attention_long_cache_and_many_rows(dev):
    """sizes of the splits' and row tiles' other side: a cache of many tiles per split, a chunk of many row tiles"""
    for H, h, D, seqs in ((12, 2, 256, [(9000, 1), (5000, 70)]), (4, 4, 128, [(3000, 1100), (20000, 1)])):
        c = Call(dev, H, h, D, 128, seqs, seed=D)
        want, _, mag, big = c.expect()
        check_out(c, c.attend(), want, mag, big)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("H,h,D", [(16, 8, 256), (8, 4, 128), (6, 1, 256), (3, 3, 128), (8, 1, 128)])
@pytest.mark.parametrize("window", [None, 150])
def test_chunks_against_the_definition(dev, H, h, D, page, window):
    """sequences of the chunk kernel: whole and cut items, pages that end inside a tile, a prompt from the start, a batch with single
    tokens in between, more rows than cached tokens"""
    for seqs in ([(130, 130)], [(700, 161), (1, 1), (259, 259), (520, 20), (0, 0), (150, 200)]):
        c = Call(dev, H, h, D, page, seqs, seed=page + H, token_major=page == 32)
        want, _, mag, big = c.expect(window)
        got = c.attend(window)
        check_out(c, got, want, mag, big)
        for b, (L, n) in enumerate(seqs):
            assert (got[int(c.cu[b]) : int(c.cu[b]) + max(0, n - L)] == 0).all()
            if n:
                cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
                o, rows = c.on, slice(int(c.cu[b]), int(c.cu[b]) + n)
                one = ops.paged_attention(o["q"][rows], o["k"], o["v"], o["table"][b : b + 1], o["lens_t"][b : b + 1], cu, n, D**-0.5, window=window)
                assert torch.equal(one, got[rows])


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("H,h,D", [(16, 8, 256), (8, 4, 128), (6, 1, 256), (3, 3, 128), (8, 1, 128)])
@pytest.mark.parametrize("window", [None, 150])
def test_chunks_keep_the_slots_weights(dev, H, h, D, page, window):
    seqs = [(700, 161), (259, 259), (9, 2), (520, 140), (150, 200), (90, 0)]
    c = Call(dev, H, h, D, page, seqs, seed=page + H, spare=0)
    want, weights, mag, big = c.expect(window)
    w = torch.rand((len(seqs), h, 704), generator=c.gen)
    on = w.to(dev)
    check_out(c, c.attend(window, weights=on, max_len=700), want, mag, big)
    rel = float(score_noise(c, big, 700).max()) + 2.0**-20  # (the slots' sums run over up to 1 600 rows)
    for b, (L, _) in enumerate(seqs):
        ref = w[b, :, :L].double() + weights[b]
        assert ((on[b, :, :L].double().cpu() - ref).abs() <= rel * ref + 1600 * 2.0**-24 * ref).all()
        assert torch.equal(on[b, :, L:].cpu(), w[b, :, L:])


@pytest.mark.parametrize("H,h,D,page", [(32, 16, 256, 16), (32, 16, 128, 128), (96, 16, 256, 64), (64, 16, 128, 32), (16, 16, 256, 128)])
def test_long_items_of_a_step(dev, H, h, D, page):
    """many stages per work item: the ring goes round dozens of times, with warps that have no keys in some stages"""
    L, B = 30011, 2
    width = -(-L // page)
    g = torch.Generator(device=dev).manual_seed(H + D)
    k, v = (torch.randn((B * width, h, page, D), generator=g, device=dev, dtype=torch.bfloat16) for _ in range(2))
    q = torch.randn((B, H, D), generator=g, device=dev, dtype=torch.bfloat16)
    table = torch.randperm(B * width, generator=g, device=dev).to(torch.int32).view(B, width)
    lens = torch.tensor([L, L - 700], dtype=torch.int32, device=dev)
    cu = torch.arange(B + 1, dtype=torch.int32, device=dev)
    run = lambda: ops.paged_attention(q, k, v, table, lens, cu, 1, D**-0.5)  # noqa: E731
    first = run()
    for _ in range(20):
        assert torch.equal(run(), first)
    for b in range(B):
        n = int(lens[b])
        kk = k[table[b].long()].transpose(0, 1).reshape(h, -1, D)[:, :n].double()
        vv = v[table[b].long()].transpose(0, 1).reshape(h, -1, D)[:, :n].double()
        qq = q[b].double().view(h, H // h, D)
        p = torch.softmax(qq @ kk.transpose(1, 2) * D**-0.5, -1)
        want, mag = p @ vv, p @ vv.abs()
        rel = math.expm1(2 * (D + 8) * 2.0**-24 * float((qq.abs() @ kk.abs().transpose(1, 2)).max()) * D**-0.5) + (n + 64) * 2.0**-24
        tol = BF * want.abs() + (BF * (1 + BF) + rel) * mag * (1 + BF)
        assert ((first[b].double().view_as(want) - want).abs() <= tol).all()


@pytest.mark.parametrize("max_q", [3, 14, 200])
@pytest.mark.parametrize("nq", [0, 1, 3])
def test_one_sequence_with_a_loose_row_limit(dev, max_q, nq):
    """a sequence alone goes to the kernel its row limit asks for, whatever its rows: padded batches, also without rows at all"""
    c = Call(dev, 8, 4, 128, 64, [(300, nq)], seed=max_q + nq, extra_rows=max_q - nq)
    out = torch.full((c.n, 8, 128), 7.0, dtype=torch.bfloat16, device=dev)
    old = torch.rand((1, 4, 320), generator=c.gen)
    w = old.to(dev)
    o = c.on
    ops.paged_attention(o["q"], o["k"], o["v"], o["table"], o["lens_t"], o["cu"], max_q, 128**-0.5, weights=w, decay=0.25, out=out)
    want, weights, mag, big = c.expect()
    if nq:
        check_out(c, out, want, mag, big)
    assert (out[nq:] == 7.0).all()
    ref = 0.25 * old[0, :, :300].double() + weights[0]
    rel = (float(score_noise(c, big, 300).max()) if nq else 0.0) + 2.0**-20
    assert ((w[0, :, :300].double().cpu() - ref).abs() <= rel * ref).all() and torch.equal(w[0, :, 300:].cpu(), old[0, :, 300:])


def test_attention_views_streams_and_a_graph(dev):
    c = Call(dev, 8, 2, 128, 64, [(300, 3), (129, 1)], seed=5)
    want, _, mag, big = c.expect()
    wide = torch.randn((c.n, 8 * 128 + 320), dtype=torch.bfloat16, device=dev)  # q inside wider projection rows
    wide[:, : 8 * 128] = c.on["q"].view(c.n, -1)
    q = wide[:, : 8 * 128].view(c.n, 8, 128)
    wide_out = torch.full((c.n, 8 * 128 + 64), 5.0, dtype=torch.bfloat16, device=dev)
    out = wide_out[:, : 8 * 128].view(c.n, 8, 128)
    o = c.on
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.paged_attention(q, o["k"], o["v"], o["table"], o["lens_t"], o["cu"], 3, 128**-0.5, out=out)
    torch.cuda.current_stream().wait_stream(side)
    check_out(c, out, want, mag, big)
    assert (wide_out[:, 8 * 128 :] == 5.0).all()
    # two calls at once on two streams, each with a workspace of its own
    plain = c.attend()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for st in (s1, s2) * 4:
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got.append(c.attend())
    torch.cuda.synchronize()
    assert all(torch.equal(x, plain) for x in got)
    # a captured call, replayed after the lengths have moved
    lens = o["lens_t"].clone()
    call = lambda: ops.paged_attention(o["q"], o["k"], o["v"], o["table"], lens, o["cu"], 3, 128**-0.5)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = call()
    graph.replay()
    assert torch.equal(res, plain)
    lens -= torch.tensor([40, 2], dtype=torch.int32, device=dev)
    graph.replay()
    c.lens = [260, 127]
    want, _, mag, big = c.expect()
    check_out(c, res, want, mag, big)


def test_far_offsets(dev):
    """pools of more than 2^31 elements: pages at their far end"""
    h, page, D = 8, 128, 256
    n_pages = 2**31 // (h * page * D) + 40
    k = torch.empty((n_pages, h, page, D), dtype=torch.bfloat16, device=dev)
    v = torch.empty_like(k)
    c = Call(dev, 16, h, D, page, [(700, 2), (200, 30)], seed=11)
    far = n_pages - c.n_pages
    k[far:], v[far:] = c.on["k"], c.on["v"]
    o = c.on
    table = torch.where(o["table"] >= 0, o["table"] + far, o["table"])
    got = ops.paged_attention(o["q"], k, v, table, o["lens_t"], o["cu"], c.max_q, D**-0.5)
    assert torch.equal(got, c.attend())
    # append and eviction there
    qkv = torch.randn((32, 32 * D), dtype=torch.bfloat16, device=dev)
    ops.paged_append(qkv, 16, h, D, k, v, table, o["lens_t"], o["cu"])
    s = 699
    assert torch.equal(k[int(table[0, s // page]), :, s % page], qkv[1, 16 * D : 24 * D].view(h, D))
    new_table = torch.tensor([[0, 1], [2, n_pages - 1 - int(o["table"].max())]], dtype=torch.int32, device=dev)
    lens, kept, _ = ops.paged_evict(k, v, table, o["lens_t"], None, 150, 150, new_table)
    assert lens.tolist() == [150, 150] and kept[0, 0, 0] == 550
    assert torch.equal(k[int(new_table[0, 1]), :, 149 - page], qkv[1, 16 * D : 24 * D].view(h, D))


@pytest.mark.parametrize("H,h,D", LAYOUTS)
@pytest.mark.parametrize("rot,norms,norm_v,plus1,page", [(1, True, True, False, 64), (64, True, False, True, 16), (96, False, False, False, 128), (0, True, True, False, 32), (0, False, False, False, 64), (0, False, True, False, 256)])
def test_append_against_the_definition(dev, H, h, D, rot, norms, norm_v, plus1, page):
    rot = D if rot == 1 else rot
    seqs = [(37, 5), (1, 1), (9, 0), (300, 130), (64, 64)]
    c = Call(dev, H, h, D, page, seqs, seed=H + rot, token_major=H % 3 == 0, extra_rows=3)
    g = c.gen
    wide = (torch.randn((c.n, (H + 2 * h) * D + 24), generator=g) * 2).to(torch.bfloat16)
    qkv = wide[:, : (H + 2 * h) * D]
    wq, wk = ((0.2 * torch.randn(D, generator=g) + (0 if plus1 else 1)).to(torch.bfloat16) for _ in range(2)) if norms else (None, None)
    cos, sin = ((torch.cos if i else torch.sin)(torch.rand((c.n, rot // 2), generator=g) * 7).to(torch.bfloat16) for i in range(2)) if rot else (None, None)
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    o = c.on
    k0, v0 = o["k"].clone(), o["v"].clone()
    q = ops.paged_append(wide.to(dev)[:, : (H + 2 * h) * D], H, h, D, o["k"], o["v"], o["table"], o["lens_t"], o["cu"], wq=to(wq), wk=to(wk), cos=to(cos), sin=to(sin), plus1=plus1, norm_v=norm_v)
    wq64, wk64, wv64, qs, ks = OP.append(qkv, H, h, D, wq, wk, cos, sin, 1e-6, plus1, norm_v)
    near = lambda a, b, size: ((a.double().cpu() - b).abs() <= BF * b.abs() + 2.0**-19 * size).all()  # noqa: E731
    assert near(q, wq64, qs)
    for b, (L, n) in enumerate(seqs):
        for i in range(n):
            s, r = L - n + i, int(c.cu[b]) + i
            pg = int(c.table[b, s // page])
            assert near(o["k"][pg, :, s % page], wk64[r], ks[r]) and near(o["v"][pg, :, s % page], wv64[r], wv64[r].abs())
            k0[pg, :, s % page], v0[pg, :, s % page] = o["k"][pg, :, s % page], o["v"][pg, :, s % page]
    same = lambda a, b: torch.equal(a.view(torch.int16), b.view(torch.int16))  # noqa: E731
    assert same(k0.contiguous(), o["k"].contiguous()) and same(v0.contiguous(), o["v"].contiguous())  # nothing else was written


@pytest.mark.parametrize("keep,recent", [(64, 16), (100, 0), (33, 33), (1, 0), (500, 499)])
@pytest.mark.parametrize("D,page", [(128, 16), (256, 64), (128, 256)])
def test_evict_against_the_definition(dev, D, page, keep, recent):
    h = 3
    seqs = [(400, 0), (64, 0), (0, 0), (1, 0), (101, 0), (1333, 0)]
    per = -(-keep // page)
    c = Call(dev, h, h, D, page, seqs, seed=keep, spare=per * len(seqs), token_major=D == 256)
    g = c.gen
    w = torch.rand((len(seqs), h, 1400), generator=g) ** 4
    w[:, 0, ::3] = 0.0                      # ties at zero
    w[:, 1] = (w[:, 1] * 8).round() / 8     # ties everywhere
    w[0, 2, 5:50] = math.nan
    w[0, 2, 60:70] = math.inf
    w[5, 2] = -w[5, 2]
    w[5, 0, 7] = -0.0
    new_table = c.free[: per * len(seqs)].view(len(seqs), per).to(dev)
    o = c.on
    k0, v0 = o["k"].clone(), o["v"].clone()
    lens, kept, wo = ops.paged_evict(o["k"], o["v"], o["table"], o["lens_t"], w.to(dev), keep, recent, new_table)
    assert lens.tolist() == [min(L, keep) for L, _ in seqs]
    for b, (L, _) in enumerate(seqs):
        for head in range(h):
            want = OP.evict(w[b, head, :L], L, keep, recent)
            m = len(want)
            assert kept[b, head, :m].tolist() == want and (kept[b, head, m:] == -1).all()
            assert torch.equal(wo[b, head, :m].cpu().nan_to_num(7.0), w[b, head, want].nan_to_num(7.0)) and (wo[b, head, m:] == 0).all()
            for pages, before in ((o["k"], k0), (o["v"], v0)):
                new = OP.gather(pages.cpu()[:, head : head + 1], new_table[b].cpu(), m)[0]
                old = OP.gather(before.cpu()[:, head : head + 1], c.table[b], L)[0]
                assert torch.equal(new, old[want])
    used = torch.unique(new_table).tolist()
    others = torch.tensor([x for x in range(c.n_pages) if x not in used], device=dev)
    assert torch.equal(o["k"][others].view(torch.int16), k0[others].view(torch.int16))


def test_evict_long_rows(dev):
    """rows of many segments per warp, against a sort"""
    B, h, L, keep, recent = 2, 4, 70001, 5000, 100
    k = torch.randn((2 * 1100 + 2 * 79, h, 64, 128), dtype=torch.bfloat16, device=dev)
    v = torch.randn_like(k)
    table = torch.randperm(2 * 1100, device=dev).to(torch.int32).view(2, 1100)
    new_table = (2200 + torch.arange(2 * 79, device=dev)).to(torch.int32).view(2, 79)
    w = torch.rand((B, h, 1100 * 64), device=dev).mul(2000).round()  # many ties
    lens = torch.tensor([L, L - 13], dtype=torch.int32, device=dev)
    _, kept, _ = ops.paged_evict(k, v, table, lens, w, keep, recent, new_table)
    for b in range(B):
        m = int(lens[b]) - recent
        for g in range(h):
            first = torch.sort(w[b, g, :m], descending=True, stable=True).indices[: keep - recent].sort().values
            assert torch.equal(kept[b, g, : keep - recent].long(), first)


def test_out_of_range_entries_are_reported_not_followed(dev):
    """a page index outside the pool, a length above max_len: the kernels' own checks skip the access and set the status word"""
    c = Call(dev, 4, 2, 128, 64, [(200, 2), (100, 1)], seed=1)
    o = c.on
    good = c.attend()
    _lib.last_status()
    for bad in (c.n_pages, -1, 2**30):
        table = o["table"].clone()
        table[1, 0] = bad
        got = ops.paged_attention(o["q"], o["k"], o["v"], table, o["lens_t"], o["cu"], 2, 128**-0.5)
        assert _lib.last_status(raise_on_error=False) == 5
        assert torch.equal(got[:2], good[:2])
    lens = o["lens_t"].clone()
    lens[1] = 70000
    got = ops.paged_attention(o["q"], o["k"], o["v"], o["table"], lens, o["cu"], 2, 128**-0.5)
    assert _lib.last_status(raise_on_error=False) == 5
    assert torch.equal(got[:2], good[:2])
    qkv = torch.zeros((3, 8 * 128), dtype=torch.bfloat16, device=dev)
    table = o["table"].clone()
    table[0] = c.n_pages
    ops.paged_append(qkv, 4, 2, 128, o["k"], o["v"], table, o["lens_t"], o["cu"])
    assert _lib.last_status(raise_on_error=False) == 5
    ops.paged_evict(o["k"], o["v"], table, o["lens_t"], None, 64, 64, c.free[:2].view(2, 1).to(dev))
    assert _lib.last_status(raise_on_error=False) == 5


def test_a_captured_chain(dev):
    """append, attention with weights and eviction in one graph, replayed on new rows: as the calls one by one"""
    H, h, D, page = 8, 4, 128, 32
    c = Call(dev, H, h, D, page, [(200, 70), (300, 3), (150, 0)], seed=21, spare=12)
    o = c.on
    new_table = c.free[:9].view(3, 3).to(dev)
    g = torch.Generator().manual_seed(0)
    rows = [torch.randn((c.n, (H + 2 * h) * D), generator=g).to(torch.bfloat16).to(dev) for _ in range(3)]
    w0 = torch.rand((3, h, 320), generator=g).to(dev)
    qkv, w, k, v = rows[0].clone(), w0.clone(), o["k"].clone(), o["v"].clone()

    def chain():
        q = ops.paged_append(qkv, H, h, D, k, v, o["table"], o["lens_t"], o["cu"], norm_v=True)
        out = ops.paged_attention(q, k, v, o["table"], o["lens_t"], o["cu"], 70, D**-0.5, weights=w)
        return (out,) + ops.paged_evict(k, v, o["table"], o["lens_t"], w, 90, 30, new_table)

    want = []
    for r in rows:
        qkv.copy_(r)
        w.copy_(w0)
        want.append([x.clone() for x in chain()] + [k.clone(), v.clone()])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = chain()
    for r, x in zip(rows, want):
        qkv.copy_(r)
        w.copy_(w0)
        graph.replay()
        for a, b in zip(list(res) + [k, v], x):
            assert torch.equal(a.view(torch.int16) if a.dtype is torch.bfloat16 else a, b.view(torch.int16) if b.dtype is torch.bfloat16 else b)


def test_as_many_sequences_as_a_call_takes(dev):
    B, H, h, D, page = 1024, 4, 2, 128, 16
    g = torch.Generator(device=dev).manual_seed(4)
    lens = torch.randint(1, 60, (B,), generator=g, device=dev).to(torch.int32)
    n_new = torch.minimum(lens, torch.randint(0, 4, (B,), generator=g, device=dev).to(torch.int32))
    n_new[500] = lens[500] = 40  # one chunk among the steps
    cu = torch.zeros(B + 1, dtype=torch.int32, device=dev)
    cu[1:] = n_new.cumsum(0)
    table = torch.randperm(4 * B, generator=g, device=dev).to(torch.int32).view(B, 4)
    both = torch.randn((4 * B, 2, h, page, D), generator=g, device=dev, dtype=torch.bfloat16)  # K and V side by side in one tensor
    k, v = both[:, 0], both[:, 1]
    q = torch.randn((int(cu[-1]), H, D), generator=g, device=dev, dtype=torch.bfloat16)
    out = ops.paged_attention(q, k, v, table, lens, cu, 40, D**-0.5)
    for b in (0, 1, 17, 499, 500, 501, 1023):
        r0, r1, L = int(cu[b]), int(cu[b + 1]), int(lens[b])
        want, _, mag, big = OP.attention(q[r0:r1].cpu(), k.cpu(), v.cpu(), table[b : b + 1].cpu(), [L], [0, r1 - r0], D**-0.5)
        rel = torch.expm1(2 * (D + 8) * 2.0**-24 * big) + 128 * 2.0**-24 + 2.0**-21
        assert ((out[r0:r1].double().cpu() - want).abs() <= BF * want.abs() + (BF * 1.01 + rel[..., None]) * mag * 1.01 + 1e-30).all()
    with pytest.raises(_lib.SpinfError, match="maximum"):
        z = torch.zeros(1025, dtype=torch.int32, device=dev)
        ops.paged_attention(q, k, v, torch.zeros((1025, 4), dtype=torch.int32, device=dev), z, torch.zeros(1026, dtype=torch.int32, device=dev), 1, 1.0)
    with pytest.raises(_lib.SpinfError, match="must not be q"):
        ops.paged_attention(q, k, v, table, lens, cu, 40, D**-0.5, out=q)


def test_windows_that_hold_everything_are_none(dev):
    """also those whose sum with a slot would leave 32 bits; with more rows than cached tokens, and with weights"""
    for seqs in ([(300, 70), (20, 25), (260, 3)], [(40, 90)]):
        c = Call(dev, 8, 2, 128, 16, seqs, seed=33)
        w = torch.zeros((len(seqs), 2, 512), device=dev)
        want, want_w = c.attend(weights=w, weights_out=torch.zeros_like(w)), torch.zeros_like(w)
        c.attend(weights=w, weights_out=want_w)
        for window in (c.table.shape[1] * 16, 2**30, 2**31 - 1, 2**32 + 5):
            got_w = torch.zeros_like(w)
            got = c.attend(window=window, weights=w, weights_out=got_w)
            assert torch.equal(got, want) and torch.equal(got_w, want_w)


def test_weights_of_an_empty_cache(dev):
    c = Call(dev, 4, 2, 128, 16, [(20, 4)], seed=3)
    o, w = c.on, torch.ones((1, 2, 32), device=dev)
    out = ops.paged_attention(o["q"], o["k"], o["v"], o["table"], torch.zeros_like(o["lens_t"]), o["cu"], 4, 1.0, weights=w, max_len=0)
    assert (out == 0).all() and (w == 1).all()
    # rows of q that belong to no sequence (as many as a chunk has): the weights only decay
    c = Call(dev, 4, 2, 128, 16, [(20, 0)], seed=3, extra_rows=90)
    o = c.on
    w = torch.ones((1, 2, 32), device=dev)
    out = torch.full((90, 4, 128), 7.0, dtype=torch.bfloat16, device=dev)
    ops.paged_attention(o["q"], o["k"], o["v"], o["table"], o["lens_t"], o["cu"], 90, 1.0, weights=w, decay=0.5, out=out)
    assert (out == 7.0).all() and (w[..., :20] == 0.5).all() and (w[..., 20:] == 1).all()


def test_append_of_rows_that_belong_to_no_sequence(dev):
    H, h, D, page = 4, 2, 128, 16
    c = Call(dev, H, h, D, page, [(20, 4), (9, 9)], seed=5)
    o = c.on
    cu = o["cu"] + 2  # two rows ahead of the first sequence, three behind the last
    n = c.n + 5
    qkv = torch.randn((n, (H + 2 * h) * D), device=dev).to(torch.bfloat16)
    w = torch.ones(D, dtype=torch.bfloat16, device=dev)
    before = o["k"].clone()
    q = ops.paged_append(qkv, H, h, D, o["k"], o["v"], o["table"], o["lens_t"], cu, wq=w, wk=w)
    assert _lib.last_status(raise_on_error=False) == 0
    x = qkv[:, : H * D].double().view(n, H, D)
    want_q = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    assert ((q.double() - want_q).abs() <= (BF + 2.0**-19) * want_q.abs()).all()
    moved = (before.view(torch.int16) != o["k"].view(torch.int16)).any(-1).any(1)  # [pages, slots]
    want = torch.zeros_like(moved)
    for b, (L, k) in enumerate([(20, 4), (9, 9)]):
        for s in range(L - k, L):
            want[int(c.table[b, s // page]), s % page] = True
    assert torch.equal(moved, want)


class Fronts(Call):
    """sequences in groups (common tokens, [(length, new rows) ..]) whose tables begin with the same pages, others between the groups"""

    def __init__(self, dev, H, h, D, page, groups, between=(), seed=0):
        g = torch.Generator(device=dev).manual_seed(seed)
        seqs, self.first = [], []
        for i, (_, members) in enumerate(groups):
            self.first.append(len(seqs))
            seqs += members
            seqs += between[i : i + 1]
        self.H, self.h, self.D, self.page, self.dev = H, h, D, page, dev
        self.lens, news = [x for x, _ in seqs], [n for _, n in seqs]
        pages = [-(-x // page) for x in self.lens]
        start = torch.tensor([0] + pages).cumsum(0)
        order = torch.randperm(int(start[-1]) + 2, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        self.table = torch.full((len(seqs), max(pages)), -7, dtype=torch.int32)
        for b, n in enumerate(pages):
            self.table[b, :n] = order[int(start[b]) : int(start[b]) + n]
        for b0, (common, members) in zip(self.first, groups):
            self.table[b0 : b0 + len(members), : common // page] = self.table[b0, : common // page]
        used = self.table[self.table >= 0].unique()
        place = torch.full((len(order),), -7, dtype=torch.int32)
        place[used.long()] = torch.randperm(len(used), generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        self.table = torch.where(self.table >= 0, place[self.table.clamp_min(0).long()], self.table)
        self.on = {"k": torch.randn((len(used), h, page, D), generator=g, device=dev).to(torch.bfloat16)}
        self.on["v"] = torch.randn((len(used), h, page, D), generator=g, device=dev).to(torch.bfloat16)
        for b, x in enumerate(self.lens):
            if x % page:
                for pool in (self.on["k"], self.on["v"]):
                    pool[int(self.table[b, x // page]), :, x % page :] = math.nan
        self.cu = torch.tensor([0] + news).cumsum(0).to(torch.int32)
        self.n, self.max_q = int(self.cu[-1]) + 1, max(news)
        self.q = torch.randn((self.n, H, D), generator=g, device=dev).to(torch.bfloat16).cpu()
        self.lens_t = torch.tensor(self.lens, dtype=torch.int32)
        self.on |= {x: getattr(self, x).to(dev) for x in ("table", "cu", "q", "lens_t")}
        self.k, self.v = self.on["k"].cpu(), self.on["v"].cpu()

    def rows(self, x, b, k=1):
        return x[int(self.cu[b]) : int(self.cu[b + k])]

    def check(self, got, seqs):
        for b in seqs:
            cu = torch.tensor([0, int(self.cu[b + 1] - self.cu[b])])
            want, _, mag, big = OP.attention(self.rows(self.q, b), self.k, self.v, self.table[b : b + 1], self.lens[b : b + 1], cu, self.D**-0.5)
            rel = score_noise(self, big, max(self.lens))[..., None]
            tol = BF * want.abs() + (BF * (1 + BF) + rel) * mag * (1 + BF) + 1e-30
            off = ((self.rows(got, b).double().cpu() - want).abs() / tol).max()
            assert off <= 1.0, f"sequence {b}: {float(off)} of the tolerance"


def _worth(seqs, h, D):
    """the shortest front, in tokens, that a group of so many sequences reads together"""
    return max(1024, -(-(2**27) // ((seqs - 1) * h * D * 4 * 128)) * 128)


@pytest.mark.parametrize("H,h,D,page", [(16, 8, 256, 64), (32, 4, 128, 16), (24, 4, 256, 32), (8, 8, 128, 128), (32, 16, 128, 256)])
def test_common_fronts_are_read_once(dev, H, h, D, page):
    few = max(1, 32 // (H // h))  # rows of a sequence that is no chunk
    fa, fb = _worth(9, h, D), _worth(20, h, D)
    pad = lambda x: -(-x // page) * page  # noqa: E731
    a = [(pad(fa) + 1 + few + 37 * i, 1 + (3 * i) % few) for i in range(9)]
    b = [(pad(fb) + few + 5 * (i % 7), few) for i in range(20)]
    c = Fronts(dev, H, h, D, page, [(pad(fa), a), (pad(fb), b)], between=[(400, 70), (900, 1)], seed=H + D)
    a0, b0 = c.first
    out = torch.full((c.n, H, D), 7.0, dtype=torch.bfloat16, device=dev)
    got, apart = c.attend(shared=True, out=out), c.attend(shared=False)
    assert (got[-1:] == 7.0).all()
    c.check(got, [0, 4, 8, 9, b0, b0 + 11, b0 + 19])
    assert not torch.equal(c.rows(got, a0, 9), c.rows(apart, a0, 9)) and not torch.equal(c.rows(got, b0, 20), c.rows(apart, b0, 20))  # it did look
    for i in (9, 30):  # the others' bits stay
        assert torch.equal(c.rows(got, i), c.rows(apart, i))
    assert torch.equal(c.attend(shared=True)[:-1], got[:-1])
    # a group's results do not depend on what else is in the call
    o = c.on
    alone = ops.paged_attention(c.rows(o["q"], b0, 20).clone(), o["k"], o["v"], o["table"][b0 : b0 + 20], o["lens_t"][b0 : b0 + 20], o["cu"][b0 : b0 + 21] - o["cu"][b0],
                                few, D**-0.5, shared=True)
    assert torch.equal(alone, c.rows(got, b0, 20))


def test_fronts_that_do_not_make_a_group(dev):
    """too little in common, a chunk or a sequence without new rows among them, a window, weights: the same bits as without looking"""
    H, h, D, page = 16, 8, 256, 64
    f = _worth(9, h, D)
    one = (f + 20, 2)
    little = [(f - 128 + 70, 3)] * 9
    broken = [one] * 4 + [(f + 150, 100)] + [one] * 4 + [(f + 20, 0)] + [one] * 3
    c = Fronts(dev, H, h, D, page, [(f - 128, little), (f, broken)], seed=2)
    assert torch.equal(c.attend(shared=True)[:-1], c.attend(shared=False)[:-1])
    c = Fronts(dev, H, h, D, page, [(f, [one] * 9)], seed=3)
    assert not torch.equal(c.attend(shared=True)[:-1], c.attend(shared=False)[:-1])
    assert torch.equal(c.attend(window=300, shared=True)[:-1], c.attend(window=300, shared=False)[:-1])
    w = torch.zeros((9, h, f + 128), device=dev)
    assert torch.equal(c.attend(weights=w.clone(), shared=True)[:-1], c.attend(weights=w.clone(), shared=False)[:-1])


def test_fronts_within_fronts(dev):
    """nine sequences with a long common front, then eleven that share only its first part with them; rows right behind the front; a page
    index that lies outside the pool in the part that is read together"""
    H, h, D, page = 16, 8, 256, 64
    f = _worth(9, h, D)
    c = Fronts(dev, H, h, D, page, [(1088, [(3 * f + 2, 2)] * 9 + [(1088 + 1 + 3 * i, 1) for i in range(11)])], seed=4)
    c.table[:9, : 3 * f // page] = c.table[0, : 3 * f // page]
    c.on["table"] = c.table.to(dev)
    got = c.attend(shared=True)
    c.check(got, [0, 8, 9, 19])
    assert not torch.equal(c.rows(got, 0, 9), c.rows(c.attend(shared=False), 0, 9))
    assert _lib.last_status(raise_on_error=False) == 0
    c.on["table"][:9, 5] = 10**6
    c.attend(shared=True)
    assert _lib.last_status(raise_on_error=False) == 5


def test_many_fronts_and_a_graph(dev):
    """more groups than the workspace has room for (the last ones stay apart); two calls in one graph, each with a workspace of its own"""
    H, h, D, page = 8, 8, 128, 64
    f = _worth(9, h, D)
    c = Fronts(dev, H, h, D, page, [(f, [(f + 9 + i, 2) for i in range(9)]) for _ in range(12)], seed=1)
    got, apart = c.attend(shared=True), c.attend(shared=False)
    same = [torch.equal(c.rows(got, b, 9), c.rows(apart, b, 9)) for b in c.first]
    assert not any(same[:9]) and all(same[-1:])
    c.check(got, [0, 80, 107])
    assert torch.equal(c.attend()[:-1], got[:-1])  # (a pool of less than an eighth of these sequences' pages: it looks by itself)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one, two = c.attend(shared=True), c.attend(shared=True)
    for _ in range(2):
        one.zero_(), two.zero_()
        graph.replay()
        assert torch.equal(one[:-1], got[:-1]) and torch.equal(two[:-1], got[:-1])


def test_known_layouts(dev):
    """calls whose layout has been seen are made without the checks' way round: other layouts in between, addresses that do not fit, a
    workspace that is too small, and out = q are noticed all the same"""
    H, h, D, page = 4, 2, 128, 16
    c = Call(dev, H, h, D, page, [(300, 2), (40, 1)], seed=6)
    o = c.on
    want = c.attend()
    wide = torch.zeros((c.n, H * D + 64), dtype=torch.bfloat16, device=dev)
    wide[:, : H * D] = o["q"].view(c.n, -1)
    views = [o["q"], wide[:, : H * D].view(c.n, H, D), o["q"].clone()]
    kept = [o["k"], o["k"].transpose(1, 2).contiguous().transpose(1, 2)]
    for _ in range(3):
        for q in views:
            for k in kept:
                for ws in (None, torch.empty(16, dtype=torch.uint8, device=dev), torch.empty(1 << 22, dtype=torch.uint8, device=dev)):
                    got = ops.paged_attention(q, k, o["v"], o["table"], o["lens_t"], o["cu"], 2, D**-0.5, workspace=ws)
                    assert torch.equal(got, want)
    out = torch.empty_like(want)
    assert ops.paged_attention(o["q"], o["k"], o["v"], o["table"], o["lens_t"], o["cu"], 2, D**-0.5, out=out) is not None and torch.equal(out, want)
    with pytest.raises(_lib.SpinfError, match="must not be q"):
        ops.paged_attention(o["q"], o["k"], o["v"], o["table"], o["lens_t"], o["cu"], 2, D**-0.5, out=o["q"])
    odd = torch.zeros(c.n * H * D + 8, dtype=torch.bfloat16, device=dev)[1 : 1 + c.n * H * D].view(c.n, H, D)  # the layout of q at an address that does not fit
    with pytest.raises(_lib.SpinfError, match="bad argument"):
        ops.paged_attention(odd, o["k"], o["v"], o["table"], o["lens_t"], o["cu"], 2, D**-0.5)
    with pytest.raises(_lib.SpinfError, match="bad argument"):
        ops.paged_attention(o["q"], o["k"], o["v"], o["table"], o["lens_t"], o["cu"], 2, -1.0)
    with pytest.raises(_lib.SpinfError, match="different devices|CUDA"):
        ops.paged_attention(o["q"], o["k"], o["v"], c.table, o["lens_t"], o["cu"], 2, D**-0.5)
    qkv = torch.randn((c.n, 8 * D), device=dev).to(torch.bfloat16)
    for _ in range(2):
        q = ops.paged_append(qkv, H, h, D, o["k"], o["v"], o["table"], o["lens_t"], o["cu"])
        assert q.data_ptr() == qkv.data_ptr() and torch.equal(q, qkv[:, : H * D].view(c.n, H, D))
    with pytest.raises(_lib.SpinfError, match="same memory"):
        ops.paged_append(qkv, H, h, D, o["k"], o["k"], o["table"], o["lens_t"], o["cu"])
    new_table = c.free[:2].view(2, 1).to(dev)
    first = ops.paged_evict(o["k"], o["v"], o["table"], o["lens_t"], None, 16, 16, new_table)
    again = ops.paged_evict(o["k"], o["v"], o["table"], o["lens_t"], None, 16, 16, new_table)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1]) and first[2] is again[2] is None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        fresh = o["q"] * 1.0
        got = ops.paged_attention(fresh, o["k"], o["v"], o["table"], o["lens_t"], o["cu"], 2, D**-0.5)
    side.synchronize()
    assert torch.equal(got, c.attend())


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("window", [None, 150])
@pytest.mark.parametrize("H,h,D", [(16, 8, 256), (8, 4, 128), (6, 1, 256), (8, 1, 128)])
def test_weights_of_a_chunk_beside_rows_that_are_not_finite(dev, H, h, D, window, bad):
    """rows of q that belong to no sequence, or to a neighbour, take no part in a chunk's weights, whatever they hold; a row of the chunk
    itself reaches the slots that it sees and no others"""
    seqs = [(700, 161), (300, 75), (520, 141), (9, 2), (333, 70)]
    c = Call(dev, H, h, D, 64, seqs, seed=H + D, spare=0, extra_rows=70)
    cap = 704
    old, w = torch.rand((len(seqs), h, cap), generator=c.gen).to(dev), torch.empty((len(seqs), h, cap), device=dev)
    run = lambda: c.attend(window, weights=old, weights_out=w.zero_())  # noqa: E731
    out = run()
    clean = w.clone()
    q, cu = c.on["q"], c.cu.tolist()
    q[cu[-1] :] = bad
    q[cu[1] : cu[2]] = bad  # all of the second sequence
    got = run()
    for b in (0, 2, 3, 4):
        assert torch.equal(w[b], clean[b]), f"sequence {b}"
        assert torch.equal(got[cu[b] : cu[b + 1]], out[cu[b] : cu[b + 1]])
    # one row in the middle of the third: what it sees, and nothing else
    at = 97
    slot = 520 - 141 + at
    q[cu[2] + at] = bad
    got = run()
    lo = max(0, slot - window + 1) if window else 0
    assert torch.isnan(w[2, :, lo : slot + 1]).all()
    assert torch.equal(w[2, :, :lo], clean[2, :, :lo]) and torch.equal(w[2, :, slot + 1 :], clean[2, :, slot + 1 :])
    keep = [i for i in range(cu[2], cu[3]) if i != cu[2] + at]
    assert torch.equal(got[keep], out[keep])
    assert torch.equal(w[0], clean[0]) and torch.equal(w[4], clean[4])


def test_a_workspace_with_gaps_is_refused_in_a_known_layout(dev):
    c = Call(dev, 4, 2, 128, 16, [(300, 2), (40, 1)], seed=6)
    room = torch.empty(1 << 22, dtype=torch.uint8, device=dev)
    want = c.attend(workspace=room)
    assert torch.equal(c.attend(workspace=room.view(2, -1)), want)
    for ws in (room[:1].expand(1 << 22), room.view(-1, 2)[:, 0]):
        with pytest.raises(_lib.SpinfError, match="contiguous"):
            c.attend(workspace=ws)
    assert torch.equal(c.attend(), want)


def test_append_of_no_sequences_makes_q(dev):
    """q has all n rows, also where none of them is a sequence's"""
    H, h, D, page = 4, 2, 128, 16
    c = Call(dev, H, h, D, page, [(20, 4)], seed=5)
    qkv = torch.randn((9, (H + 2 * h) * D), generator=c.gen).to(torch.bfloat16).to(dev)
    w = (1 + 0.1 * torch.randn(D, generator=c.gen)).to(torch.bfloat16).to(dev)
    k, v = c.on["k"].clone(), c.on["v"].clone()
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    for width in (0, 3):
        held = torch.full((9, H, D), 7.0, dtype=torch.bfloat16, device=dev)  # where the allocator finds room for q again
        del held
        q = ops.paged_append(qkv, H, h, D, c.on["k"], c.on["v"], torch.zeros((0, width), dtype=torch.int32, device=dev), none, torch.zeros(1, dtype=torch.int32, device=dev), wq=w, wk=w)
        want = OP.append(qkv.cpu(), H, h, D, w.cpu(), w.cpu())[0]
        assert ((q.double().cpu() - want).abs() <= (BF + 2.0**-19) * want.abs()).all()
    assert torch.equal(k.view(torch.int16), c.on["k"].view(torch.int16)) and torch.equal(v.view(torch.int16), c.on["v"].view(torch.int16))


@pytest.mark.parametrize("bad", [-1, 2**30])
@pytest.mark.parametrize("H,h,D,page", [(16, 8, 256, 64), (8, 4, 128, 16), (6, 1, 256, 128), (32, 4, 128, 32)])
def test_a_page_outside_the_pool_counts_as_zeros(dev, H, h, D, page, bad):
    """in every kernel, and not as whatever another sequence's keys have left behind; the call is reported"""
    seqs = [(700, 1), (700, 3), (700, 130), (520, 1)]
    c = Call(dev, H, h, D, page, seqs, seed=H, spare=1)
    o, w = c.on, torch.zeros((4, h, 768), device=dev)
    zero = int(c.free[0])
    o["k"][zero], o["v"][zero] = 0.0, 0.0
    got = {}
    for entry in (zero, bad):
        table = o["table"].clone()
        for b in range(3):
            table[b, 2], table[b, (700 - 1) // page] = entry, entry
        got[entry] = []
        for weights in (None, w):
            for window in (None, 300):
                into = None if weights is None else torch.zeros_like(w)
                got[entry] += [ops.paged_attention(o["q"], o["k"], o["v"], table, o["lens_t"], o["cu"], 130, D**-0.5, window=window, weights=weights, weights_out=into), into]
        assert _lib.last_status(raise_on_error=False) == (0 if entry == zero else 5)
    for x, y in zip(got[zero], got[bad]):
        assert x is y is None or torch.equal(x, y)


@pytest.mark.parametrize("H,h,D", [(16, 8, 256), (8, 1, 128)])
@pytest.mark.parametrize("n", [1, 3, 90])
def test_a_row_whose_scores_are_all_minus_infinity_weighs_nothing(dev, H, h, D, n):
    """as a row that sees nothing: 0, and no weight for any slot"""
    c = Call(dev, H, h, D, 32, [(300, n)], seed=n)
    o = c.on
    o["k"][..., 0] = o["k"][..., 0].abs()  # (behind the sequence they stay NaN)
    q = o["q"]
    q[n - 1] = 0.0
    q[n - 1, :, 0] = -math.inf
    w = torch.zeros((1, h, 320), device=dev)
    got = c.attend(weights=w)
    assert (got[n - 1] == 0).all()
    q[n - 1] = math.nan  # the same call with that row taken out: its cu ends before it, the last slot is still there
    rest = torch.zeros_like(w)
    if n > 1:
        cu, lens = torch.tensor([0, n - 1], dtype=torch.int32, device=dev), o["lens_t"] - 1
        ops.paged_attention(q, o["k"], o["v"], o["table"], lens, cu, c.max_q, D**-0.5, weights=rest)
    assert torch.equal(w[..., :300], rest[..., :300])


@pytest.mark.parametrize("window", [None, 1000])
@pytest.mark.parametrize("H,h,D", [(16, 8, 256), (32, 16, 128)])
def test_more_sequences_than_one_launch_holds(dev, H, h, D, window):
    """chunks, branches, steps and sequences without rows whose parts pass the workspace's bound: the call is made in several launches, and
    every sequence's bits are those it has alone; with weights, and asked to look for common fronts"""
    B, page, L = 400, 64, 4100
    g = torch.Generator(device=dev).manual_seed(D)
    width = -(-(L + 41) // page)
    shared = 4096 // page
    k, v = (torch.randn((shared + 2 * B, h, page, D), generator=g, device=dev, dtype=torch.bfloat16) for _ in range(2))
    table = torch.full((B, width), -1, dtype=torch.int32, device=dev)
    table[:, :shared] = torch.arange(shared, device=dev)
    own = shared + torch.arange(2 * B, device=dev).view(B, 2)
    table[:, shared:] = own[:, : width - shared].to(torch.int32)
    news = torch.tensor([(40, 33, 1, 12, 0, 40, 40, 17)[b % 8] for b in range(B)])
    lens = (4096 + news + torch.arange(B) % 5).to(torch.int32).to(dev)
    cu = torch.zeros(B + 1, dtype=torch.int32)
    cu[1:] = news.cumsum(0)
    n = int(cu[-1]) + 3
    q = torch.randn((n, H, D), generator=g, device=dev, dtype=torch.bfloat16)
    assert _lib.lib().spinf_paged_attention_workspace_bytes(n, B // 3, H, h, D, 40, width * page, 0, 0) > 1 << 29  # (the whole of it would pass the bound)
    out = torch.full((n, H, D), 7.0, dtype=torch.bfloat16, device=dev)
    on = cu.to(dev)
    ops.paged_attention(q, k, v, table, lens, on, 40, D**-0.5, window=window, out=out, shared=False)
    w, w_out = torch.rand((B, h, width * page), generator=g, device=dev), torch.full((B, h, width * page), -3.0, device=dev)
    weighed = ops.paged_attention(q, k, v, table, lens, on, 40, D**-0.5, window=window, weights=w, weights_out=w_out, decay=0.5)
    assert (out[int(cu[-1]) :] == 7.0).all()
    together = ops.paged_attention(q, k, v, table, lens, on, 40, D**-0.5, window=window, shared=True)
    for b in sorted({0, 1, 2, 3, 4, 5, 99, 100, 131, 132, 133, 134, 135, 199, 200, 201, 265, 266, 267, 268, 269, 397, 398, 399}):
        r0, r1 = int(cu[b]), int(cu[b + 1])
        cu1 = torch.tensor([0, r1 - r0], dtype=torch.int32, device=dev)
        for weights in (None, w[b : b + 1]):
            w1 = None if weights is None else torch.full_like(weights, -3.0)
            # (beside an empty neighbour, so that it takes the kernel of its own rows)
            one = ops.paged_attention(q[r0:r1], k, v, table[[b, b]], torch.stack([lens[b], lens[b] * 0]), torch.cat([cu1, cu1[1:]]), 40, D**-0.5, window=window, shared=False,
                                      weights=None if weights is None else weights.repeat(2, 1, 1), weights_out=None if weights is None else (w2 := w1.repeat(2, 1, 1)), decay=0.5)
            assert torch.equal(one, (out if weights is None else weighed)[r0:r1]), b
            if weights is not None:
                assert torch.equal(w2[0], w_out[b]), b
        off = (together[r0:r1].double() - out[r0:r1].double()).abs()
        assert r0 == r1 or off.max() <= 3 * BF * float(v.abs().max()), b  # (the same sums in another order, p rounded against another maximum)
    assert torch.equal(together[: int(cu[-1])], out[: int(cu[-1])]) == (window is not None)


def test_a_group_that_finds_no_room_stays_apart(dev):
    """what the documentation says of `shared`: a group alone is read together, behind others that have taken the room it is not; either way
    it is right, and the call repeats itself"""
    H, h, D, page = 8, 8, 128, 64
    f = _worth(9, h, D)
    c = Fronts(dev, H, h, D, page, [(f, [(f + 9 + i, 2) for i in range(9)]) for _ in range(12)], seed=2)
    got, apart, o = c.attend(shared=True), c.attend(shared=False), c.on
    for b0, in_call in ((c.first[0], got), (c.first[-1], None)):
        alone = ops.paged_attention(c.rows(o["q"], b0, 9).clone(), o["k"], o["v"], o["table"][b0 : b0 + 9], o["lens_t"][b0 : b0 + 9], o["cu"][b0 : b0 + 10] - o["cu"][b0], 2,
                                    D**-0.5, shared=True)
        assert not torch.equal(alone, c.rows(apart, b0, 9))
        assert torch.equal(alone, c.rows(got, b0, 9)) == (in_call is not None)
    assert torch.equal(c.rows(got, c.first[-1], 9), c.rows(apart, c.first[-1], 9))
    c.check(got, [0, 99, 107])
    assert torch.equal(c.attend(shared=True)[:-1], got[:-1])


def test_launches_are_counted(dev):
    """COUNTS["launches"] against the kernels that the profiler sees"""
    from torch.profiler import ProfilerActivity, profile

    def kernels(f):
        f()
        torch.cuda.synchronize()
        before = ops.COUNTS["launches"]
        with profile(activities=[ProfilerActivity.CUDA]) as prof:
            f()
            torch.cuda.synchronize()
        return ops.COUNTS["launches"] - before, sum(e.count for e in prof.key_averages() if "paged_" in e.key)

    H, h, D, page = 16, 8, 256, 64
    one, chunk, mixed = (Call(dev, H, h, D, page, x, seed=1) for x in ([(70, 1)], [(700, 200)], [(300, 1), (200, 12), (400, 100)]))
    f = _worth(9, h, D)
    fronts = Fronts(dev, H, h, D, page, [(f, [(f + 20, 2)] * 9)], seed=3)
    seen = []
    for call in (lambda: one.attend(), lambda: chunk.attend(), lambda: mixed.attend(), lambda: mixed.attend(weights=torch.zeros((3, h, 448), device=dev)),
                 lambda: chunk.attend(weights=torch.zeros((1, h, 704), device=dev)), lambda: fronts.attend(shared=True)):
        got, want = kernels(call)
        if want == 0:
            pytest.skip("the profiler sees no kernels here")
        assert got == want
        seen.append(got)
    assert len(set(seen)) > 3, seen
    c = Call(dev, H, h, D, page, [(300, 2)], seed=2, spare=4)
    o = c.on
    qkv = torch.randn((2, (H + 2 * h) * D), device=dev).to(torch.bfloat16)
    new = c.free[:2].view(1, 2).to(dev)
    for call in (lambda: ops.paged_append(qkv, H, h, D, o["k"], o["v"], o["table"], o["lens_t"], o["cu"]),
                 lambda: ops.paged_append(qkv[:0], H, h, D, o["k"], o["v"], o["table"], o["lens_t"], o["cu"] * 0),
                 lambda: ops.paged_evict(o["k"], o["v"], o["table"], o["lens_t"], None, 100, 100, new)):
        got, want = kernels(call)
        assert got == want


def _levels(kind, n, g):
    """score level of every slot, in nats: what a row's maximum does as its tiles go by"""
    s = torch.arange(n) / n
    if kind == "rising":
        return -85 + 170 * s
    if kind == "falling":
        return 85 - 170 * s
    if kind == "steps":  # a level of its own for every 64 slots: up by more than the threshold, down, up by less
        return ((torch.rand((n + 63) // 64, generator=g) - 0.5) * 170).repeat_interleave(64)[:n]
    return torch.where(torch.arange(n) % 190 == 100, 60.0 * s, -60.0 + 0 * s)  # peaks


@pytest.mark.parametrize("kind", ["normed", "rising", "falling", "steps", "peaks"])
@pytest.mark.parametrize("window", [None, 300])
@pytest.mark.parametrize("H,h,D", [(16, 8, 256), (8, 4, 128), (6, 1, 256), (8, 1, 128)])
def test_scores_that_spread_widely(dev, H, h, D, window, kind):
    """heads of unit mean square attended to with scale 1, as the stacks do, and levels that move a row's reference maximum up, by much and by
    little, from tile to tile, part to part and half to half: outputs and weights of every kernel against the definition"""
    seqs = [(900, 161), (700, 1), (650, 3), (1200, 40), (333, 333), (520, 12)]
    c = Call(dev, H, h, D, 64, seqs, seed=D + H, spare=0)
    g, e = c.gen, torch.where(torch.rand(D, generator=c.gen) < 0.5, -1.0, 1.0)
    k, q = torch.full(c.k.shape, math.nan), None
    for b, L in enumerate(c.lens):
        s = torch.arange(L)
        if kind == "normed":
            rows = torch.randn((L, h, D), generator=g)
            rows = rows / rows.pow(2).mean(-1, keepdim=True).sqrt()
        else:
            rows = e * _levels(kind, L, g)[:, None, None] / D + 0.02 * torch.randn((L, h, D), generator=g)
        k[c.table[b].long()[s // 64], :, s % 64] = rows
    if kind == "normed":
        q = torch.randn((c.n, H, D), generator=g)
        q = q / q.pow(2).mean(-1, keepdim=True).sqrt()
    else:
        q = e * torch.tensor([1.0, 0.75, 0.5, 0.125])[torch.randint(0, 4, (c.n, H, 1), generator=g)]
    c.k, c.q = k.to(torch.bfloat16), q.to(torch.bfloat16)
    c.on["k"], c.on["q"] = c.k.to(dev), c.q.to(dev)
    o, w = c.on, torch.zeros((len(seqs), h, 1216), device=dev)
    want, weights, mag, big = OP.attention(c.q, c.k, c.v, c.table, c.lens, c.cu, 1.0, window)
    check_out(c, ops.paged_attention(o["q"], o["k"], o["v"], o["table"], o["lens_t"], o["cu"], c.max_q, 1.0, window=window), want, mag, big)
    check_out(c, ops.paged_attention(o["q"], o["k"], o["v"], o["table"], o["lens_t"], o["cu"], c.max_q, 1.0, window=window, weights=w, max_len=1200), want, mag, big)
    rel = float(score_noise(c, big, 1200).max()) + 2.0**-20 + 1600 * 2.0**-24
    for b, (L, n) in enumerate(seqs):
        ref = weights[b]
        assert ((w[b, :, :L].double().cpu() - ref).abs() <= rel * ref + 2.0**-126 * max(1, n) * H).all(), b  # (a p below the normal numbers is 0)
        if n > 40:  # alone: an item in several parts, or none
            cu = torch.tensor([0, n], dtype=torch.int32, device=dev)
            rows = slice(int(c.cu[b]), int(c.cu[b]) + n)
            one = ops.paged_attention(o["q"][rows], o["k"], o["v"], o["table"][b : b + 1], o["lens_t"][b : b + 1], cu, n, 1.0, window=window)
            tol = BF * want[rows].abs() + (BF * (1 + BF) + score_noise(c, big[rows], 1200)[..., None]) * mag[rows] * (1 + BF) + 1e-30
            assert ((one.double().cpu() - want[rows]).abs() <= tol).all(), b


@pytest.mark.parametrize("H,h,D,page", [(16, 8, 256, 64), (32, 16, 128, 64)])
def test_common_fronts_of_scores_that_spread_widely(dev, H, h, D, page):
    f = _worth(20, h, D)
    c = Fronts(dev, H, h, D, page, [(f, [(f + 12 + 9 * i, 12) for i in range(20)])], seed=D)
    c.q *= 16  # (exact)
    c.on["q"] *= 16
    got = c.attend(shared=True)
    assert not torch.equal(got[:-1], c.attend(shared=False)[:-1])
    c.check(got, [0, 7, 19])


def test_the_workspace_asked_for_is_enough_under_a_window(dev):
    """at the C entry point, asked to look for common fronts too: the query knows no window, and the call no fronts under one"""
    import ctypes

    B, n_new, max_len, page, D = 256, 13, 1 << 20, 256, 256
    g = torch.Generator(device=dev).manual_seed(3)
    k, v = (torch.randn((B, 1, page, D), generator=g, device=dev, dtype=torch.bfloat16) for _ in range(2))
    table = torch.zeros((B, max_len // page), dtype=torch.int32, device=dev)
    table[:, 0] = torch.arange(B, device=dev)
    lens = torch.full((B,), 200, dtype=torch.int32, device=dev)
    cu = (torch.arange(B + 1, device=dev) * n_new).to(torch.int32)
    q = torch.randn((B * n_new, 1, D), generator=g, device=dev, dtype=torch.bfloat16)
    lib, out = _lib.lib(), torch.zeros_like(q)
    need = lib.spinf_paged_attention_workspace_bytes(B * n_new, B, 1, 1, D, 40, max_len, 0, 1)
    room = torch.empty(need, dtype=torch.uint8, device=dev)
    st = (ctypes.c_int64 * 3)(*k.stride()[:3])
    for window in (0, 100, 1 << 19):
        assert lib.spinf_paged_attention(q.data_ptr(), D, B * n_new, 1, 1, D, k.data_ptr(), v.data_ptr(), B, page, st, st, table.data_ptr(), table.stride(0), lens.data_ptr(),
                                         cu.data_ptr(), B, 40, max_len, window, 1, D**-0.5, None, None, None, 1.0, out.data_ptr(), D, room.data_ptr(), need, _lib.raw_stream(0)) == 0
        want = ops.paged_attention(q, k, v, table[:, :1].contiguous(), lens, cu, 40, D**-0.5, window=window or None, shared=False)
        assert torch.equal(out, want)
