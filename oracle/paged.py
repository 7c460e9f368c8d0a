"""The paged K/V cache's operators by their definitions, in 64 bits, one sequence and one key / value head at a time. Pools are
[pages, kv heads, page, D]; a sequence's slot s is row s % page of page table[b][s // page]."""

import math

import torch


def gather(pages, table_row, n):
    """slots 0 .. n - 1 of a sequence -> [kv heads, n, D]"""
    page = pages.shape[2]
    s = torch.arange(n)
    return pages[table_row.long()[s // page], :, s % page].transpose(0, 1)


def attention(q, k_pages, v_pages, table, lens, cu, scale, window=None):
    """-> (out [n, H, D] float64 (rows behind cu[B]: NaN), scatter of the weights [B] of [kv heads, len], magnitude sum_j p_j |v_j|
    [n, H, D], largest sum_d |q_d k_d| scale of a row [n, H])"""
    n, H, D = q.shape
    h = k_pages.shape[1]
    out = torch.full((n, H, D), math.nan, dtype=torch.float64)
    mag = torch.zeros((n, H, D), dtype=torch.float64)
    big = torch.zeros((n, H), dtype=torch.float64)
    weights = []
    for b in range(len(lens)):
        r0, r1, L = int(cu[b]), int(cu[b + 1]), int(lens[b])
        w = torch.zeros((h, L), dtype=torch.float64)
        k, v = gather(k_pages, table[b], L).double(), gather(v_pages, table[b], L).double()
        slot = torch.arange(L - (r1 - r0), L)[:, None]
        j = torch.arange(L)
        seen = j <= slot
        if window:
            seen = seen & (j > slot - window)
        for hd in range(H):
            g = hd // (H // h)
            x = q[r0:r1, hd].double()
            s = x @ k[g].T * scale
            s = s.masked_fill(~seen, -math.inf)
            m = s.amax(-1, keepdim=True) if L else torch.zeros((r1 - r0, 1), dtype=torch.float64)
            e = torch.exp(s - m.clamp_min(-1e300)).masked_fill(~seen, 0.0)
            p = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
            out[r0:r1, hd] = p @ v[g]
            mag[r0:r1, hd] = p @ v[g].abs()
            if L and r1 > r0:
                big[r0:r1, hd] = (x.abs() @ k[g].abs().T * scale).amax(-1)
            w[g] += p.sum(0)
        weights.append(w)
    return out, weights, mag, big


def append(qkv, H, h, D, wq=None, wk=None, cos=None, sin=None, eps=1e-6, plus1=False, norm_v=False):
    """-> q [n, H, D], k, v [n, h, D] float64, and the size of what the rotation adds up, for tolerances"""
    n = qkv.shape[0]
    x = qkv.double().reshape(n, H + 2 * h, D)
    q, k, v = x[:, :H], x[:, H : H + h], x[:, H + h :]

    def norm(t, w):
        t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + eps)
        return t if w is None else t * ((1 + w.double()) if plus1 else w.double())

    def turn(t):
        if cos is None:
            return t, t.abs()
        r = cos.shape[1]
        a, b, rest = t[..., :r], t[..., r : 2 * r], t[..., 2 * r :]
        c, s = cos.double()[:, None], sin.double()[:, None]
        size = a.abs() + b.abs()
        return torch.cat([a * c - b * s, b * c + a * s, rest], -1), torch.cat([size, size, rest.abs()], -1)

    if wq is not None:
        q, k = norm(q, wq), norm(k, wk)
    if norm_v:
        v = norm(v, None)
    (q, qs), (k, ks) = turn(q), turn(k)
    return q, k, v, qs, ks


def evict(weights, length, keep, recent):
    """slots of one sequence and kv head that stay, ascending; weights [length]: NaN below every number, ties to the lowest slot"""
    if length <= keep:
        return list(range(length))
    m = length - recent
    key = [(-math.inf if math.isnan(float(weights[j])) else float(weights[j])) for j in range(m)]
    nan = [math.isnan(float(weights[j])) for j in range(m)]
    order = sorted(range(m), key=lambda j: (-key[j], nan[j], j))
    return sorted(order[: keep - recent]) + list(range(m, length))
