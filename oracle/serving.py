"""fp64 CPU restatements of the paged-cache operators beyond single-token decode: chunk
attention, rotary positions and page copies, from their definitions."""
from __future__ import annotations

import math

import torch


def gather(pool, pages, length):
    """K and V rows [Hkv, length, D] of a sequence, and which of them lie in the pool."""
    P, _, Hkv, page, D = pool.shape
    kv = torch.zeros((2, Hkv, length, D), dtype=torch.float64)
    ok = torch.zeros(length, dtype=torch.bool)
    for t in range(0, length, page):
        pg = int(pages[t // page])
        n = min(page, length - t)
        if 0 <= pg < P:
            kv[:, :, t:t + n] = pool[pg, :, :, :n].double()
            ok[t:t + n] = True
    return kv[0], kv[1], ok


def chunk_attention(q, q_indptr, pool, indptr, indices, last, causal=True, scale=None):
    """O [T, Hq, D], LSE [T, Hq], A = softmax |V| [T, Hq, D] and the largest |q| |k| |scale| per row
    [T, Hq] (for error bounds).  Keys that a row does not see contribute nothing at all."""
    T, Hq, D = q.shape
    page, Hkv = pool.shape[3], pool.shape[2]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    O = torch.zeros((T, Hq, D), dtype=torch.float64)
    A = torch.zeros((T, Hq, D), dtype=torch.float64)
    L = torch.full((T, Hq), -math.inf, dtype=torch.float64)
    C = torch.zeros((T, Hq), dtype=torch.float64)
    for b in range(len(last)):
        a, e = int(q_indptr[b]), int(q_indptr[b + 1])
        np_ = int(indptr[b + 1]) - int(indptr[b])
        n = (np_ - 1) * page + int(last[b]) if np_ > 0 else 0
        if e <= a or n <= 0:
            continue
        K, V, ok = gather(pool, indices[int(indptr[b]):int(indptr[b + 1])], n)
        pos = torch.arange(n - (e - a), n)
        see = ok.expand(e - a, n).clone()
        if causal:
            see &= torch.arange(n) <= pos[:, None]
        for h in range(Hq):
            k, v = K[h // G], V[h // G]
            qq = q[a:e, h].double()
            s = qq @ k.t() * scale
            s[~see] = -math.inf
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
            p[~see] = 0.0
            l = p.sum(-1, keepdim=True)
            w = torch.where(l == 0, 0.0, p / l)
            if torch.isfinite(v).all():
                O[a:e, h], A[a:e, h] = w @ v, w @ v.abs()
            else:  # a value that is not finite reaches the rows that see it, and no others
                prod = torch.where(see[:, :, None], w[:, :, None] * v[None], 0.0)
                O[a:e, h], A[a:e, h] = prod.sum(1), prod.abs().sum(1)
            L[a:e, h] = (torch.log(l) + m)[:, 0]
            norm = torch.where(see, k.norm(dim=-1), 0.0).amax(-1)
            C[a:e, h] = qq.norm(dim=-1) * norm * abs(scale)
    return O, L, A, C


def rotate(x, positions, inv_freq, interleaved=False, factor=1.0, transpose=False):
    """x [..., S, D] at positions [..., S] (broadcast), in fp64."""
    r = 2 * inv_freq.numel()
    y = x.double().clone()
    angle = positions.double()[..., None] * inv_freq
    c, s = torch.cos(angle) * factor, torch.sin(angle) * factor * (-1 if transpose else 1)
    first = slice(0, r, 2) if interleaved else slice(0, r // 2)
    second = slice(1, r, 2) if interleaved else slice(r // 2, r)
    a, b = x[..., first].double(), x[..., second].double()
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    return y


def copy_pages(pool, src, dst, num_tokens=None):
    """A copy of the pool after the page copies."""
    P, page = pool.shape[0], pool.shape[3]
    out = pool.clone()
    for i, (s, d) in enumerate(zip(src, dst)):
        n = page if num_tokens is None else min(max(int(num_tokens[i]), 0), page)
        if 0 <= s < P and 0 <= d < P and s != d:
            out[d, :, :, :n] = pool[s, :, :, :n]
    return out
