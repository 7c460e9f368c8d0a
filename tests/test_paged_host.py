"""The paged cache without a GPU: the book-keeping of pages, and what the operators refuse before any CUDA work."""

import ctypes

import pytest
import torch

from spinf_serve_b200 import _lib, ops
from spinf_serve_b200.paged import PagedCache


def _cache(n=12, page=16):
    return PagedCache(2, 3, 128, n, page, device="cpu")


def test_pages_are_shared_copied_and_returned():
    c = _cache()
    a = c.open()
    st = c.grow([a], [40])
    assert len(a.pages) == 3 and a.length == a.position == 40 and st.table.tolist() == [a.pages] and st.lens.tolist() == [40] and st.cu.tolist() == [0, 40]
    assert st.pos.tolist() == list(range(40)) and (st.max_q, st.max_len) == (40, 40)
    c.k[:, a.pages[2]], c.v[:, a.pages[2]] = 5.0, 6.0
    b = c.fork(a)
    assert b.pages[:2] == a.pages[:2] and b.pages[2] != a.pages[2]  # the begun page is copied
    assert (c.k[:, b.pages[2]] == 5.0).all() and (c.v[:, b.pages[2]] == 6.0).all()
    assert [c.refs[p] for p in a.pages] == [2, 2, 1]
    st = c.grow([a, b], [0, 9])
    assert a.length == 40 and b.length == 49 and len(b.pages) == 4 and st.table.shape == (2, 4) and st.cu.tolist() == [0, 0, 9] and st.pos.tolist() == list(range(40, 49))
    c.close(a)
    assert c.refs[b.pages[0]] == 1 and len(c.free) == 12 - 4
    c.close(b)
    assert sorted(c.free) == list(range(12)) and b.pages == []


def test_a_fork_of_whole_pages_shares_them_all():
    c = _cache()
    a = c.open()
    c.grow([a], [32])
    b = c.fork(a)
    assert b.pages == a.pages
    c.grow([b], [1])
    assert len(b.pages) == 3 and len(a.pages) == 2


def test_running_out_of_pages_changes_nothing():
    c = _cache(4)
    a, b = c.open(), c.open()
    c.grow([a], [20])
    with pytest.raises(RuntimeError, match="out of pages"):
        c.grow([a, b], [30, 17])
    assert a.length == 20 and len(a.pages) == 2 and b.pages == [] and len(c.free) == 2
    c.grow([a, b], [12, 17])
    assert len(c.free) == 0


def test_refused_steps():
    c = _cache()
    a = c.open()
    for seqs, counts in (([a], [1, 2]), ([], []), ([a], [-1]), ([a, a], [1, 1])):
        with pytest.raises(RuntimeError):
            c.grow(seqs, counts)
    c.grow([a], [30])
    for keep, recent in ((0, 0), (5, 6), (5, -1)):
        with pytest.raises(RuntimeError):
            c.evict(a, keep, recent, [False, False])
    with pytest.raises(RuntimeError, match="weights"):
        c.evict(a, 5, 2, [True, False])
    assert c.evict(a, 30, 4, [True, True]) is None and a.length == 30
    for args in ((2, 3, 128, 4, 24), (2, 3, 64, 4, 16), (2, 3, 128, 0, 16), (2, 3, 128, 4, 512)):
        with pytest.raises(RuntimeError):
            PagedCache(*args, device="cpu")


def _call(**kw):
    """a well-formed attention call but for the device"""
    a = dict(q=torch.zeros((5, 4, 128), dtype=torch.bfloat16), k_pages=torch.zeros((6, 2, 16, 128), dtype=torch.bfloat16),
             v_pages=torch.zeros((6, 2, 16, 128), dtype=torch.bfloat16), table=torch.zeros((2, 3), dtype=torch.int32),
             lens=torch.tensor([20, 30], dtype=torch.int32), cu=torch.tensor([0, 2, 5], dtype=torch.int32), max_q=3, scale=0.1)
    return ops.paged_attention(**{**a, **kw})


@pytest.mark.parametrize("kw,what", [
    ({}, "CUDA"),
    ({"q": torch.zeros((5, 4, 128))}, "bf16"),
    ({"q": torch.zeros((5, 3, 128), dtype=torch.bfloat16)}, "evenly"),
    ({"q": torch.zeros((5, 128, 4), dtype=torch.bfloat16).transpose(1, 2)}, "without gaps"),
    ({"k_pages": torch.zeros((6, 2, 24, 128), dtype=torch.bfloat16), "v_pages": torch.zeros((6, 2, 24, 128), dtype=torch.bfloat16)}, "pages hold"),
    ({"v_pages": torch.zeros((6, 2, 32, 128), dtype=torch.bfloat16)}, "agree"),
    ({"k_pages": torch.zeros((6, 2, 16, 132), dtype=torch.bfloat16)[..., :128]}, "multiples of 8"),
    ({"table": torch.zeros((2, 3), dtype=torch.int64)}, "int32"),
    ({"table": torch.zeros((3, 3), dtype=torch.int32)}, "page table"),
    ({"table": torch.zeros((3, 2), dtype=torch.int32).t()}, "page table"),
    ({"cu": torch.tensor([0, 5], dtype=torch.int32)}, "cu"),
    ({"lens": torch.zeros(4, dtype=torch.int32)[::2]}, "contiguous"),
    ({"max_len": 49}, "max_len"),
    ({"max_q": -1}, "max_q"),
    ({"window": 0}, "window"),
    ({"weights": torch.zeros((2, 2, 40))}, "weights"),
    ({"weights": torch.zeros((2, 2, 48), dtype=torch.float64)}, "weights"),
    ({"weights_out": torch.zeros((2, 2, 48))}, "comes with"),
    ({"out": torch.zeros((5, 4, 128))}, "out"),
])
def test_attention_refusals(kw, what):
    with pytest.raises(_lib.SpinfError, match=what):
        _call(**kw)


def _append(**kw):
    a = dict(qkv=torch.zeros((5, 8 * 128), dtype=torch.bfloat16), H=4, Hkv=2, D=128, k_pages=torch.zeros((6, 2, 16, 128), dtype=torch.bfloat16),
             v_pages=torch.zeros((6, 2, 16, 128), dtype=torch.bfloat16), table=torch.zeros((2, 3), dtype=torch.int32),
             lens=torch.tensor([20, 30], dtype=torch.int32), cu=torch.tensor([0, 2, 5], dtype=torch.int32))
    return ops.paged_append(**{**a, **kw})


@pytest.mark.parametrize("kw,what", [
    ({}, "CUDA"),
    ({"H": 5}, "fit"),
    ({"qkv": torch.zeros((5, 8 * 128))}, "fit"),
    ({"wq": torch.zeros(128, dtype=torch.bfloat16)}, "together"),
    ({"wq": torch.zeros(64, dtype=torch.bfloat16), "wk": torch.zeros(64, dtype=torch.bfloat16)}, "wq and wk"),
    ({"cos": torch.zeros((5, 20), dtype=torch.bfloat16), "sin": torch.zeros((5, 20), dtype=torch.bfloat16)}, "multiple of 16"),
    ({"cos": torch.zeros((4, 64), dtype=torch.bfloat16), "sin": torch.zeros((4, 64), dtype=torch.bfloat16)}, "cos and sin"),
    ({"cos": torch.zeros((5, 64), dtype=torch.bfloat16), "sin": torch.zeros((5, 32), dtype=torch.bfloat16)}, "cos and sin"),
])
def test_append_refusals(kw, what):
    with pytest.raises(_lib.SpinfError, match=what):
        _append(**kw)


def _evict(**kw):
    a = dict(k_pages=torch.zeros((6, 2, 16, 128), dtype=torch.bfloat16), v_pages=torch.zeros((6, 2, 16, 128), dtype=torch.bfloat16),
             table=torch.zeros((2, 3), dtype=torch.int32), lens=torch.tensor([20, 30], dtype=torch.int32), weights=torch.zeros((2, 2, 48)), keep=16, recent=4,
             new_table=torch.zeros((2, 1), dtype=torch.int32))
    return ops.paged_evict(**{**a, **kw})


@pytest.mark.parametrize("kw,what", [
    ({}, "CUDA"),
    ({"keep": 0}, "keep"), ({"keep": 17}, "keep"), ({"recent": 17}, "recent"), ({"recent": -1}, "recent"),
    ({"weights": torch.zeros((2, 3, 48))}, "weights"),
    ({"weights": torch.zeros((2, 2, 40)), "max_len": 41}, "max_len"),
    ({"new_table": torch.zeros((1, 1), dtype=torch.int32)}, "page table"),
])
def test_evict_refusals(kw, what):
    with pytest.raises(_lib.SpinfError, match=what):
        _evict(**kw)


def test_the_c_entry_points_refuse_on_the_host():
    lib = _lib.lib()
    p, N = ctypes.c_void_p(256), None
    st = (ctypes.c_int64 * 3)(4096, 2048, 128)
    odd = (ctypes.c_int64 * 3)(4096, 2048, 130)

    def attn(n=2, H=4, h=2, D=128, page=16, q=p, table=p, width=4, B=1, max_q=2, max_len=64, window=0, scale=1.0, w_in=N, w_out=N, strides=N, decay=1.0, ws=N, ws_bytes=0, k=st):
        return lib.spinf_paged_attention(q, H * D, n, H, h, D, p, p, 8, page, k, st, table, width, p, p, B, max_q, max_len, window, 0, scale, w_in, w_out, strides, decay, p, H * D, ws, ws_bytes, N)

    assert attn(B=0) == 0 and attn(n=0, q=N) == 0  # nothing to do
    for bad in (dict(q=N), dict(table=N), dict(H=3), dict(D=64), dict(page=24), dict(page=8), dict(max_len=65), dict(max_q=-1), dict(window=-1), dict(scale=0.0),
                dict(w_out=p), dict(w_out=p, strides=(ctypes.c_int64 * 4)(), decay=1.0), dict(width=64, max_len=1024)):  # (the last: splits need a workspace)
        assert attn(**bad) == -1, bad
    assert attn(B=2000) == -4
    assert lib.spinf_paged_attention_workspace_bytes(4, 2000, 4, 2, 128, 1, 64, 0, 0) == -4
    assert lib.spinf_paged_attention_workspace_bytes(4, 2, 4, 3, 128, 1, 64, 0, 0) == -1
    need = [lib.spinf_paged_attention_workspace_bytes(64, 64, 16, 8, 256, 1, n, w, 0) for n, w in ((100, 0), (8192, 0), (8192, 1))]
    assert need[0] == 0 and 0 < need[1] < need[2]

    def append(n=2, H=4, h=2, D=128, pitch=1024, page=16, wq=N, wk=N, cos=N, sin=N, rot=0, q=N, width=4, k=st, B=1, qkv=p):
        return lib.spinf_paged_append(qkv, pitch, n, H, h, D, wq, wk, cos, sin, rot, 1e-6, 0, 0, q, p, p, 8, page, k, st, p, width, width, p, p, B, N)

    assert append(n=0, qkv=N) == 0 and append(B=0) == 0
    for bad in (dict(qkv=N), dict(D=64), dict(pitch=1000), dict(page=20), dict(wq=p), dict(cos=p, sin=p), dict(cos=p, sin=p, rot=24, q=p), dict(cos=p, sin=p, rot=256, q=p),
                dict(wq=p, wk=p), dict(width=0), dict(k=odd)):
        assert append(**bad) == -1, bad
    assert append(B=1025) == -4

    def evict(keep=16, recent=4, w=p, w_out=p, new_pitch=1, max_len=64, D=128, page=16, k=st, B=1, kept=p):
        return lib.spinf_paged_evict(p, p, 8, page, 2, D, k, st, p, 4, p, B, max_len, w, 128, 64, keep, recent, p, new_pitch, p, kept, w_out, N)

    assert evict(B=0) == 0
    for bad in (dict(keep=0), dict(keep=17), dict(recent=17), dict(recent=-1), dict(w=N), dict(w=N, w_out=N), dict(w_out=N), dict(max_len=65), dict(D=64), dict(page=48), dict(k=odd), dict(kept=N)):
        assert evict(**bad) == -1, bad


def test_written_layouts_that_share_places_are_refused():
    one = torch.zeros((1, 2, 16, 128), dtype=torch.bfloat16).expand(6, -1, -1, -1)
    half = torch.as_strided(torch.zeros(6 * 4096, dtype=torch.bfloat16), (6, 2, 16, 128), (2048, 2048, 128, 1))
    for pool in (one, half):
        with pytest.raises(_lib.SpinfError, match="share places"):
            _append(k_pages=pool)
        with pytest.raises(_lib.SpinfError, match="share places"):
            _evict(v_pages=pool)
        with pytest.raises(_lib.SpinfError, match="CUDA"):  # reading them is fine
            _call(k_pages=pool)
    w = torch.zeros((2, 1, 48)).expand(-1, 2, -1)
    with pytest.raises(_lib.SpinfError, match="share places"):
        _call(weights=w)
    with pytest.raises(_lib.SpinfError, match="CUDA"):
        _call(weights=w, weights_out=torch.zeros((2, 2, 48)))
    with pytest.raises(_lib.SpinfError, match="CUDA"):  # K and V side by side in one tensor, token-major weights' rows apart
        both = torch.zeros((6, 2, 2, 16, 128), dtype=torch.bfloat16)
        _append(k_pages=both[:, 0], v_pages=both[:, 1])


def test_the_front_that_sequences_have_in_common():
    c = _cache(24)
    a = c.open()
    c.grow([a], [40])
    forks = [c.fork(a) for _ in range(3)]
    assert c.common_front(forks) == 32 and c.common_front([a]) == 48 and c.common_front([a, c.open()]) == 0
    c.grow(forks, [9, 1, 30])
    assert c.common_front(forks) == 32
    b = c.open()
    c.grow([b], [20])
    assert c.common_front(forks + [b]) == 0


def test_workspace_of_a_call_that_looks_for_fronts():
    need = lambda B, n, max_q, max_len, w, shared: _lib.lib().spinf_paged_attention_workspace_bytes(n, B, 16, 8, 256, max_q, max_len, w, shared)  # noqa: E731
    assert need(56, 672, 12, 2048, 0, 1) > need(56, 672, 12, 2048, 0, 0) > 0
    for args in ((56, 672, 12, 2048, 1), (1, 12, 12, 65536, 0), (2, 24, 12, 2048, 0), (56, 672, 12, 256, 0)):  # weights, one sequence, too little to save
        assert need(*args, 1) == need(*args, 0)


def test_the_common_front_of_the_first_pages():
    c = _cache(24)
    a = c.open()
    c.grow([a], [80])
    forks = [c.fork(a) for _ in range(3)]
    assert [c.common_front(forks, n) for n in (None, 0, 2, 9)] == [80, 0, 32, 80]


def test_the_short_way_wants_the_right_arguments():
    bind = _lib.paged_bind()
    x = torch.zeros((5, 8 * 128), dtype=torch.bfloat16)
    for f in (bind.append, bind.attention, bind.evict, bind.learn):
        with pytest.raises(TypeError):
            f(x)
    with pytest.raises(TypeError):
        bind.learn(0, (x,), (1,))
    assert bind.append(*[x] * 10, 4, 2, 128, 1e-6, False, False) is None  # not on a CUDA device: left to the checks
    assert bind.evict(*[None] * 6, 16, 16, None) is None and bind.evict(*["x"] * 6, 16, 16, None) is None


def _back(seq, n):
    """what a failed forward does: the sequence stays where it was, the pages that grow gave it are kept"""
    seq.length -= n
    seq.position -= n


def test_pages_kept_from_a_failed_forward_serve_their_own_sequence_only():
    c = _cache(8)
    a, b = c.open(), c.open()
    c.grow([a], [64])
    _back(a, 64)
    st = c.grow([a, b], [1, 40])
    assert a.length == 1 and b.length == 40 and len(a.pages) == 4 and len(b.pages) == 3 and len(c.free) == 1
    assert st.table[1, :3].tolist() == b.pages and not set(a.pages) & set(b.pages)
    c.close(a)
    c.close(b)
    assert sorted(c.free) == list(range(8))


def test_a_step_that_cannot_be_built_changes_nothing():
    c = _cache(8)
    a, b = c.open(), c.open()
    c.grow([a], [20])
    c.device = "no such device"  # the tables cannot be made there
    with pytest.raises(RuntimeError):
        c.grow([a, b], [30, 17])
    assert (a.length, a.position, len(a.pages), b.length, b.pages, len(c.free)) == (20, 20, 2, 0, [], 6)


class _Stack:
    """a stack that calls the reader's attention for every layer but computes nothing: `fail` raises in the layer of that number"""

    hybrid, n_layers = False, 2
    fail = None

    def __init__(self):
        from types import SimpleNamespace

        self.cfg = SimpleNamespace(kv_heads=3, head_dim=128, heads=3, window=4, layer_types=["sliding_attention", "full_attention"])
        self.w = SimpleNamespace(embed=torch.zeros(1))

    def forward(self, sc, b, inputs, masks, rows=None, attend=None):
        n = inputs["ids"].numel()
        for i, kind in enumerate(self.cfg.layer_types):
            if i == self.fail:
                raise ValueError("out of memory")
            attend.project(i, kind, torch.zeros((n, 9 * 128), dtype=torch.bfloat16), None, None, None, None, 1e-6)
        out = torch.zeros((1, n, 4))
        return out if rows is None else out[0][rows]


@pytest.fixture
def reader(monkeypatch):
    """a PagedReader without a GPU: the operators stand in (weights: one more for every slot)"""
    from spinf_serve_b200.paged import PagedReader

    def attend(q, k, v, table, lens, cu, max_q, scale, weights=None, weights_out=None, **kw):
        if weights is not None:
            n = int(lens[0])
            (weights if weights_out is None else weights_out)[:, :, :n] = weights[:, :, :n] + 1.0
        return q

    def evict(k, v, table, lens, weights, keep, recent, new_table, max_len=None):
        n, h = int(lens[0]), k.shape[1]
        if evict.fail:
            evict.fail -= 1
            if not evict.fail:
                raise _lib.SpinfError("paged_evict: refused")
        if weights is None:
            kept = torch.arange(n - keep, n).expand(h, -1)[None]
            return None, kept, None
        kept = torch.stack([torch.cat([weights[0, x, : n - recent].sort(descending=True, stable=True).indices[: keep - recent].sort().values, torch.arange(n - recent, n)]) for x in range(h)])[None]
        return None, kept, torch.gather(weights, 2, kept)

    evict.fail = 0
    monkeypatch.setattr(ops, "paged_append", lambda qkv, H, h, D, *a, **kw: qkv[:, : H * D].view(-1, H, D))
    monkeypatch.setattr(ops, "paged_attention", attend)
    monkeypatch.setattr(ops, "paged_evict", evict)
    r = PagedReader(_Stack(), n_pages=12, page=16, chunk=32)
    r.evict_op = evict
    return r


def test_a_reading_that_fails_gives_its_pages_back(reader):
    with pytest.raises(RuntimeError, match="out of pages"):
        reader.read(list(range(200)))
    assert sorted(reader.cache.free) == list(range(12)) and reader.cache.refs == [0] * 12
    reader.stack.fail = 1
    with pytest.raises(ValueError):
        reader.read(list(range(20)))
    assert len(reader.cache.free) == 12
    reader.stack.fail = None
    seq = reader.read(list(range(100)))
    assert seq.length == 100 and len(reader.cache.free) == 5


def test_an_eviction_that_fails_changes_nothing(reader):
    seq = reader.read(list(range(90)), weigh=True)
    pages, weights, free = list(seq.pages), seq.weights.clone(), list(reader.cache.free)
    for layer in (1, 2):
        reader.evict_op.fail = layer
        with pytest.raises(_lib.SpinfError):
            reader.evict(seq, 40, 8)
        assert seq.pages == pages and seq.length == seq.position == 90 and torch.equal(seq.weights, weights)
        assert sorted(reader.cache.free) == sorted(free)
    kept = reader.evict(seq, 40, 8)
    assert seq.length == 40 and len(seq.pages) == 3 and len(reader.cache.free) == 9
    assert torch.equal(seq.weights[1, :, :40], torch.gather(weights[1], 1, kept[1]))


def test_a_weight_layer_behind_one_that_failed_is_not_half_moved(reader):
    """both layers by weight: the second's failure leaves the first's weights as they were"""
    reader.stack.cfg.layer_types = ["full_attention", "full_attention"]
    seq = reader.read(list(range(90)), weigh=True)
    seq.weights[:, :, :90] = torch.randperm(90).float()
    weights = seq.weights.clone()
    reader.evict_op.fail = 2
    with pytest.raises(_lib.SpinfError):
        reader.evict(seq, 40, 8)
    assert torch.equal(seq.weights, weights) and len(reader.cache.free) == 6


def test_weights_are_those_of_the_tokens_that_are_there(reader):
    """weigh, evict, read on without and with weights: no slot has what an evicted token had in its place. (Rows that are read without
    weights add none; their slots begin at zero like any others)"""
    seq = reader.read(list(range(90)), weigh=True)
    assert (seq.weights[1, :, :90] >= 1.0).all() and (seq.weights[1, :, 90:] == 0).all()
    reader.evict(seq, 40, 8)
    assert (seq.weights[1, :, :40] >= 1.0).all()
    reader.forward([seq], [[1] * 20])
    assert (seq.weights[1, :, :40] >= 1.0).all() and (seq.weights[1, :, 40:60] == 0).all()
    reader.forward([seq], [[1] * 20], weigh=True)
    assert (seq.weights[1, :, 40:80] == 1.0).all()
    kept = reader.evict(seq, 30, 25)
    assert all(x < 40 for x in kept[1][:, :5].flatten().tolist())  # the old tokens have the larger weights


def test_growing_without_weights_past_their_room(reader):
    seq = reader.read([1] * 20, weigh=True)
    seq.weights = seq.weights[:, :, :32].clone()  # (as if the cache had been that short)
    reader.forward([seq], [[1] * 60])
    assert seq.weights.shape[2] >= 80 and (seq.weights[1, :, :20] == 1).all() and (seq.weights[1, :, 20:80] == 0).all()
    reader.evict(seq, 30, 8)
    assert seq.length == 30 and len(reader.cache.free) == 10


def test_weighing_the_last_tokens_only(reader):
    seq = reader.read([1] * 20)
    reader.forward([seq], [[1] * 4], weigh=True)
    assert (seq.weights[1, :, :24] == 1).all()
    reader.evict(seq, 10, 4)
    assert seq.length == 10


def test_a_fork_has_its_own_copy_of_the_weights(reader):
    seq = reader.read([1] * 50, weigh=True)
    before = seq.weights.clone()
    fork = reader.cache.fork(seq)
    reader.forward([fork], [[1] * 4], weigh=True)
    assert torch.equal(seq.weights, before) and torch.equal(fork.weights[1, :, :50], before[1, :, :50] + 1) and (fork.weights[1, :, 50:54] == 1).all()
    reader.evict(fork, 30, 8)
    assert torch.equal(seq.weights, before) and fork.length == 30
    plain = reader.cache.fork(reader.read([1] * 5))
    assert plain.weights is None
    reader.ask(seq, [[1], [2, 3]])
    assert torch.equal(seq.weights, before)


def test_cutting_by_place_moves_the_weights_along(reader):
    """an eviction that keeps the last slots of a weighed sequence: each slot's weight goes with it"""
    seq = reader.read([1] * 60, weigh=True)
    seq.weights[:, :, :60] = torch.arange(60.0)
    reader.cache.evict(seq, 24, 0, [False, False])
    assert (seq.weights[:, :, :24] == torch.arange(36.0, 60.0)).all() and (seq.weights[:, :, 24:] == 0).all()


def test_a_weighing_forward_that_fails_adds_nothing(reader):
    """the first layer has added its weights when the second fails: the next try counts them once"""
    reader.stack.cfg.layer_types = ["full_attention", "full_attention"]
    seq = reader.read([1] * 20, weigh=True)
    before = seq.weights.clone()
    reader.stack.fail = 1
    with pytest.raises(ValueError):
        reader.forward([seq], [[1] * 15], weigh=True)
    assert seq.length == seq.position == 20 and torch.equal(seq.weights[:, :, :20], before[:, :, :20])
    reader.stack.fail = None
    reader.forward([seq], [[1] * 15], weigh=True)
    assert (seq.weights[:, :, :20] == before[:, :, :20] + 1).all() and (seq.weights[:, :, 20:35] == 1).all() and (seq.weights[:, :, 35:] == 0).all()


def test_a_weighing_forward_that_fails_first_keeps_none(reader):
    seq = reader.cache.open()
    reader.stack.fail = 1
    with pytest.raises(ValueError):
        reader.forward([seq], [[1] * 15], weigh=True)
    assert seq.weights is None and seq.length == 0


def test_a_forward_that_fails_before_its_layers(reader):
    """token ids that are none, or weights that do not fit in: the sequences stay where they were"""
    a, b = reader.read([1] * 20), reader.read([1] * 5)
    with pytest.raises((TypeError, ValueError)):
        reader.forward([a, b], [[1, 2], ["x"]])
    assert (a.length, a.position, b.length, b.position) == (20, 20, 5, 5)

    def full(*a):
        raise MemoryError

    reader.cache._weights_room = full
    with pytest.raises(MemoryError):
        reader.forward([a], [[1, 2]], weigh=True)
    assert (a.length, a.position, a.weights) == (20, 20, None)


@pytest.mark.parametrize("ws", [torch.empty(1, dtype=torch.uint8).expand(1 << 30), torch.empty((64, 64), dtype=torch.uint8)[:, ::2], torch.empty((8, 8)).t()])
def test_a_workspace_with_gaps_is_refused(ws):
    """its number of bytes is not the room that it has"""
    with pytest.raises(_lib.SpinfError, match="contiguous"):
        _call(workspace=ws)


def _room(n, B, H, h, D, max_q, max_len, weights=0, shared=0):
    return _lib.lib().spinf_paged_attention_workspace_bytes(n, B, H, h, D, max_q, max_len, weights, shared)


@pytest.mark.parametrize("H,h,D", [(32, 16, 128), (16, 8, 256), (8, 1, 128)])
def test_a_chunk_alone_asks_for_no_scores(H, h, D):
    """its kernels compute them again: beside the parts of its items there is the rows' lse only"""
    for max_len in (4096, 131072, 1 << 20):
        assert _room(2048, 1, H, h, D, 2048, max_len, 1) - _room(2048, 1, H, h, D, 2048, max_len, 0) <= 2048 * H * 4
        assert _room(2048, 1, H, h, D, 2048, max_len, 1) <= 150 * 512 * (D * 4 + 8 + 32) + 2048 * H * 4
    assert _room(1, 1, H, h, D, 1, 4096, 1) > 4096 * H * 4  # a step keeps its scores


@pytest.mark.parametrize("H,h,D", [(16, 8, 256), (32, 16, 128), (24, 4, 256), (8, 1, 128)])
def test_the_workspace_of_many_sequences_is_bounded(H, h, D):
    """whatever the number of sequences: beside the rows' lse two gigabytes (a sequence alone may need more, where it is very long and
    its scores are kept)"""
    for B in (56, 256, 1024):
        for max_q, max_len in ((1, 4096), (12, 2012), (40, 4136), (300, 20000), (2048, 131072), (1, 1 << 20)):
            n = min(B * max_q, 1 << 20)
            for shared in (0, 1):
                assert 0 <= _room(n, B, H, h, D, max_q, max_len, 0, shared) <= 2 << 30, (B, max_q, max_len)
            if max_len < 1 << 20:
                assert 0 < _room(n, B, H, h, D, max_q, max_len, 1) <= (2 << 30) + n * H * 4 + 256
    # 56 questions of 40 tokens over 4 096: one slot of 256 rows per part, as many parts as are made
    assert _room(56 * 40, 56, 16, 8, 256, 40, 4136) < 1300 << 20


def test_the_binding_is_made_anew_for_another_torch(monkeypatch):
    """its layout follows torch's headers and the interpreter: neither the build nor the loader takes one that was made for others"""
    from spinf_serve_b200.csrc import build

    monkeypatch.setattr(build, "_stale", lambda *a: False)  # (by their times it is newer than its sources)
    assert not build.bind_stale()
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    assert build.bind_stale()
    monkeypatch.setattr(_lib, "_bind", None)
    with pytest.raises(_lib.SpinfError, match="1.0.0"):
        _lib.paged_bind()


def test_a_forward_inside_a_forward_is_refused(reader):
    """(or beside it, from another thread: the layers would find the other's tables)"""
    a, b = reader.read([1] * 20), reader.read([1] * 5)
    plain, got = reader.stack.forward, []

    def forward(*args, **kw):
        with pytest.raises(RuntimeError, match="one forward at a time"):
            reader.forward([b], [[1]])
        got.append(1)
        return plain(*args, **kw)

    reader.stack.forward = forward
    reader.forward([a], [[1, 2]])
    assert got == [1] and (a.length, b.length) == (22, 5)
    reader.stack.forward = plain
    reader.forward([b], [[1]])
    assert b.length == 6
