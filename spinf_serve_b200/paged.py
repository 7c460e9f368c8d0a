"""Reading a content once and asking about it later: a paged K/V cache for the attention layers of a stack, and the forward passes over
it. The scoring pass reads a content and all its questions in one stream and forgets both; the extraction decoder keeps padded copies
of what one pass captured. Here the keys and values stay in pages: a content is read in chunks of any length, questions that come
later run as forks that share the content's pages, a sequence goes on token by token, and a cache that has grown too long is cut back
to the slots that were attended to most (ops.paged_append, ops.paged_attention, ops.paged_evict).

The host keeps the books (which pages a sequence holds, who shares them, how far it is); tables and lengths go to the device once per
forward and serve all its layers."""

import threading
from dataclasses import dataclass, field

import torch

from spinf_serve_b200 import ops


@dataclass
class Sequence:
    """one cached sequence: its pages in slot order, cached slots, and the position of its next token (past `length` once slots were
    evicted). weights: fp32 [layers, kv heads, cap] attention weight of every slot, added up over the forwards that weigh (a slot begins at
    zero), where it is kept"""

    pages: list = field(default_factory=list)
    length: int = 0
    position: int = 0
    weights: torch.Tensor | None = None


@dataclass
class Step:
    """the device side of one forward over some sequences' new tokens"""

    table: torch.Tensor
    lens: torch.Tensor
    cu: torch.Tensor
    pos: torch.Tensor
    max_q: int
    max_len: int
    shared: bool = False  # the sequences' tables begin with so many of the same pages that reading them once pays


class PagedCache:
    """pools of pages for `layers` attention layers, [layers][pages, kv heads, page, D] for K and for V; a page index means the same
    tokens in every layer"""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, n_pages: int, page: int = 64, device="cuda:0"):
        if page < 16 or page > 256 or page & (page - 1) or head_dim not in (128, 256) or n_pages < 1:
            raise RuntimeError(f"pages hold 16, 32, 64, 128 or 256 tokens of 128 or 256 dimensions, got {n_pages} pages of {page} x {head_dim}")
        self.page, self.n_pages, self.device = page, n_pages, torch.device(device)
        self.k, self.v = (torch.empty((layers, n_pages, kv_heads, page, head_dim), dtype=torch.bfloat16, device=self.device) for _ in range(2))
        self.row_bytes = 4 * kv_heads * head_dim  # a token's K and V in one layer
        self.free = list(range(n_pages - 1, -1, -1))
        self.refs = [0] * n_pages

    def _take(self, n: int) -> list:
        if n > len(self.free):
            raise RuntimeError(f"the cache is out of pages: {n} wanted, {len(self.free)} of {self.n_pages} free")
        out = [self.free.pop() for _ in range(n)]
        for p in out:
            self.refs[p] = 1
        return out

    def _release(self, pages) -> None:
        for p in pages:
            self.refs[p] -= 1
            if self.refs[p] == 0:
                self.free.append(p)

    def _weights_room(self, weights, slots: int):
        """the weights with room for so many slots (None: new ones, all zero)"""
        if weights is not None and weights.shape[2] >= slots:
            return weights
        out = torch.zeros((self.k.shape[0], self.k.shape[2], -(-slots // 1024) * 1024), dtype=torch.float32, device=self.device)
        if weights is not None:
            out[:, :, : weights.shape[2]] = weights
        return out

    def common_front(self, seqs: list, most: int | None = None) -> int:
        """tokens of the pages that all of the sequences begin with (of their first `most` pages)"""
        n = 0
        for pages in zip(*(s.pages[:most] for s in seqs)):
            if len(set(pages)) > 1:
                break
            n += 1
        return n * self.page

    def open(self) -> Sequence:
        return Sequence()

    def close(self, seq: Sequence) -> None:
        self._release(seq.pages)
        seq.pages, seq.length, seq.position, seq.weights = [], 0, 0, None

    def fork(self, seq: Sequence, weights: bool = True) -> Sequence:
        """a sequence that goes on from where `seq` is: full pages are shared, a begun one is copied (both may go on writing), and so are the
        slots' weights where they are kept (weights=False: the fork has none)"""
        own = seq.weights.clone() if weights and seq.weights is not None else None
        whole = seq.length // self.page
        last = self._take(1) if seq.length % self.page else []
        for p in seq.pages[:whole]:
            self.refs[p] += 1
        if last:
            old = seq.pages[whole]
            for pool in (self.k, self.v):
                pool[:, last[0]].copy_(pool[:, old])
        return Sequence(seq.pages[:whole] + last, seq.length, seq.position, own)

    def grow(self, seqs: list, counts: list) -> Step:
        """room for counts[i] new tokens of seqs[i] (0: the sequence sits this one out) -> the forward's tables. The same sequence
        twice in one call is an error: its tokens would take the same slots"""
        if len(seqs) != len(counts) or not seqs or any(c < 0 for c in counts):
            raise RuntimeError("one count of new tokens per sequence, none negative")
        if len({id(s) for s in seqs}) != len(seqs):
            raise RuntimeError("a sequence can be extended once per forward")
        need = [max(0, -(-(s.length + c) // self.page) - len(s.pages)) for s, c in zip(seqs, counts)]  # (pages of a failed forward may be left)
        pages = self._take(sum(need))  # all or none
        try:
            tables, cu, pos, at = [], [0], [], 0
            for s, c, n in zip(seqs, counts, need):
                tables.append(s.pages + pages[at : at + n])
                pos += range(s.position, s.position + c)
                cu.append(cu[-1] + c)
                at += n
            width = max(1, max(len(t) for t in tables))
            lens = [s.length + c for s, c in zip(seqs, counts)]
            i32 = lambda x: torch.tensor(x, dtype=torch.int32).to(self.device)  # noqa: E731
            for s, c, t in zip(seqs, counts, tables):
                if s.weights is not None:
                    s.weights = self._weights_room(s.weights, len(t) * self.page)
                    s.weights[:, :, s.length : s.length + c] = 0.0
            step = Step(i32([t + [0] * (width - len(t)) for t in tables]), i32(lens), i32(cu), i32(pos), max(counts), max(lens))
        except BaseException:
            self._release(pages)
            raise
        for s, c, t in zip(seqs, counts, tables):  # nothing has changed up to here
            s.pages = t
            s.length += c
            s.position += c
        return step

    def evict(self, seq: Sequence, keep: int, recent: int, by_weight: list) -> list | None:
        """cuts the sequence back to `keep` slots in every layer: by accumulated weight where by_weight[layer], else the last `keep`.
        Its pages are left to whoever shares them, what stays goes to new ones -> per layer the kept old slots [kv heads, keep]
        (None: nothing to cut)"""
        if not 0 <= recent <= keep or keep < 1:
            raise RuntimeError(f"keep {keep} and recent {recent}: at least one slot, and no more recent ones than kept ones")
        if seq.length <= keep:
            return None
        if any(by_weight) and seq.weights is None:
            raise RuntimeError("the sequence was read without its slots' weights")
        pages = self._take(-(-keep // self.page))
        kept = []
        try:
            moved = None if seq.weights is None else torch.zeros_like(seq.weights)
            i32 = lambda x: torch.tensor([x], dtype=torch.int32, device=self.device)  # noqa: E731
            table, new_table, lens = i32(seq.pages), i32(pages), torch.tensor([seq.length], dtype=torch.int32, device=self.device)
            for li in range(self.k.shape[0]):
                w = seq.weights[li][None] if by_weight[li] else None
                _, slots, w_new = ops.paged_evict(self.k[li], self.v[li], table, lens, w, keep, recent, new_table, max_len=seq.length)
                if moved is not None:  # (without `w` the last slots stay, and their weights with them)
                    moved[li, :, :keep] = seq.weights[li, :, seq.length - keep : seq.length] if w is None else w_new[0]
                kept.append(slots[0])
        except BaseException:  # the old pages still hold everything
            self._release(pages)
            raise
        self._release(seq.pages)
        seq.pages, seq.length, seq.weights = pages, keep, moved
        return kept


class PagedReader:
    """forward passes of a GemmaStack over a PagedCache. `read` takes a content in, `ask` runs questions that share it, `forward` is one
    pass over new tokens of any sequences, `evict` cuts a sequence back. One call at a time, all on one stream: pages that are given back
    are taken again without waiting for kernels that other streams still run on them"""

    def __init__(self, stack, n_pages: int, page: int = 64, chunk: int = 2048):
        cfg = stack.cfg
        if getattr(stack, "hybrid", False):
            raise RuntimeError("the paged cache holds attention layers only: a hybrid stack's recurrent states are the decoder's (decode.HybridDecoder)")
        self.stack, self.chunk = stack, chunk
        self.cache = PagedCache(stack.n_layers, cfg.kv_heads, cfg.head_dim, n_pages, page, stack.w.embed.device)
        self.scaling = 1.0  # the Gemma-style layers norm q and k and attend with scaling 1
        self._step, self._weights, self._busy = None, None, threading.Lock()

    # ---- the stack's attention (GemmaStack.forward, `attend`)
    def _attend(self, i, kind, q):
        st, c, cfg = self._step, self.cache, self.stack.cfg
        sliding = kind == "sliding_attention"
        w = None if self._weights is None or sliding else self._weights[i][None]
        return ops.paged_attention(q, c.k[i], c.v[i], st.table, st.lens, st.cu, st.max_q, self.scaling, window=cfg.window if sliding else None,
                                   weights=w, max_len=st.max_len, shared=st.shared)

    def __call__(self, i, kind, q, k, v):
        """q, k, v normed and rotated, side by side in one projection's rows: k and v into the pages, then the attention"""
        c, cfg, st = self.cache, self.stack.cfg, self._step
        qkv = torch.as_strided(q, (q.shape[0], (cfg.heads + 2 * cfg.kv_heads) * cfg.head_dim), (q.stride(0), 1))
        ops.paged_append(qkv, cfg.heads, cfg.kv_heads, cfg.head_dim, c.k[i], c.v[i], st.table, st.lens, st.cu)
        return self._attend(i, kind, q)

    def project(self, i, kind, qkv, wq, wk, cos, sin, eps):
        """the same from the bare projection: head norms and rotation on the way into the pages"""
        c, cfg, st = self.cache, self.stack.cfg, self._step
        q = ops.paged_append(qkv, cfg.heads, cfg.kv_heads, cfg.head_dim, c.k[i], c.v[i], st.table, st.lens, st.cu, wq, wk, cos, sin, eps, norm_v=True)
        return self._attend(i, kind, q)

    def forward(self, seqs: list, ids: list, last: bool = True, weigh: bool = False):
        """one pass over new tokens: ids[i] (token ids) goes on from seqs[i] -> hidden states after the last norm at every sequence's
        last new token [len(seqs), hidden] (last=False: at all new tokens, sequence after sequence). weigh: the slots' attention
        weights are added up (one sequence, full-attention layers). The attention runs in calls of at most 1 024 sequences"""
        if weigh and len(seqs) != 1:
            raise RuntimeError("weights are kept for a sequence that is read alone")
        if not all(len(x) for x in ids) or len(seqs) > 1024:
            raise RuntimeError("every sequence of a forward (at most 1024) needs new tokens")
        if not self._busy.acquire(blocking=False):
            raise RuntimeError("a reader runs one forward at a time")
        try:
            return self._forward(seqs, ids, last, weigh)
        finally:
            self._busy.release()

    def _forward(self, seqs, ids, last, weigh):
        st = self.cache.grow(seqs, [len(x) for x in ids])
        weights = None
        try:
            if len(seqs) > 1:
                front = max(ops.SHARE_TOKENS, -(-ops.SHARE_BYTES // ((len(seqs) - 1) * self.cache.row_bytes)))
                st.shared = self.cache.common_front(seqs, -(-front // self.cache.page)) >= front
            if weigh:  # added up in a copy, so that a failure half way through the layers leaves none of it
                old = seqs[0].weights
                weights = old.clone() if old is not None else self.cache._weights_room(None, len(seqs[0].pages) * self.cache.page)
            self._step, self._weights = st, weights
            inputs = {"ids": torch.cat([torch.as_tensor(x, dtype=torch.int64) for x in ids]).to(self.cache.device), "pos": st.pos}
            rows = (st.cu[1:].long() - 1) if last else None
            out = self.stack.forward(None, None, inputs, None, rows=rows, attend=self)
        except BaseException:
            # the sequences stay where they were (their new pages are kept for the next try)
            for s, x in zip(seqs, ids):
                s.length -= len(x)
                s.position -= len(x)
            raise
        finally:
            self._step = self._weights = None
        if weigh:
            seqs[0].weights = weights
        return out if last else out[0]

    def read(self, ids, weigh: bool = False) -> Sequence:
        """a content's tokens into a new sequence, `chunk` at a time"""
        seq = self.cache.open()
        try:
            for at in range(0, len(ids), self.chunk):
                self.forward([seq], [ids[at : at + self.chunk]], weigh=weigh)
        except BaseException:
            self.cache.close(seq)
            raise
        return seq

    def ask(self, seq: Sequence, branches: list):
        """questions (token ids each) about a content that was read: every branch attends to the content and itself only, as in the
        scoring pass -> hidden states at the branches' last tokens [len(branches), hidden]. The sequence itself stays as it is"""
        forks = []
        try:
            for _ in branches:
                forks.append(self.cache.fork(seq, weights=False))
            return self.forward(forks, branches)
        finally:
            for f in forks:
                self.cache.close(f)

    def evict(self, seq: Sequence, keep: int, recent: int):
        """cuts the sequence back to `keep` slots: on full-attention layers the last `recent` and, of the others, those with the largest
        accumulated weight; sliding layers keep the last `keep`, which has to cover their window"""
        kinds = [self.stack.cfg.layer_types[i] for i in range(self.stack.n_layers)]
        if "sliding_attention" in kinds and keep < self.stack.cfg.window and seq.length > keep:
            raise RuntimeError(f"keep {keep} is less than the sliding layers' window {self.stack.cfg.window}")
        return self.cache.evict(seq, keep, recent, [k != "sliding_attention" for k in kinds])
