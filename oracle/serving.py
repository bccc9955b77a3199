"""fp64 CPU restatements of the paged-cache operators beyond single-token decode: chunk
attention, attention with shared prefixes, the attention that tokens draw, the choice and the move of
kept tokens, rotary positions and page copies, from their definitions."""
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


def _length(indptr, last, b, page):
    n = int(indptr[b + 1]) - int(indptr[b])
    return (n - 1) * page + int(last[b]) if n > 0 else 0


def shared_prefix_attention(q, q_indptr, pool, indptr, indices, last, group_indptr, prefix_indptr,
                            prefix_indices, prefix_last, causal=True, scale=None):
    """As chunk_attention, a sequence's keys being its group's prefix and then its own."""
    T, Hq, D = q.shape
    page, Hkv = pool.shape[3], pool.shape[2]
    G = Hq // Hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    O, A = (torch.zeros((T, Hq, D), dtype=torch.float64) for _ in range(2))
    L = torch.full((T, Hq), -math.inf, dtype=torch.float64)
    C = torch.zeros((T, Hq), dtype=torch.float64)
    for b in range(len(last)):
        a, e = int(q_indptr[b]), int(q_indptr[b + 1])
        n = e - a
        K, V, ok = gather(pool, indices[int(indptr[b]):int(indptr[b + 1])],
                          m := _length(indptr, last, b, page))
        see = ok.expand(n, m).clone()
        if causal:
            see &= torch.arange(m) <= torch.arange(m - n, m)[:, None]
        for i in range(len(prefix_last)):
            if int(group_indptr[i]) <= b < int(group_indptr[i + 1]):
                pk, pv, pok = gather(pool, prefix_indices[int(prefix_indptr[i]):int(prefix_indptr[i + 1])],
                                     _length(prefix_indptr, prefix_last, i, page))
                K, V = torch.cat((pk, K), 1), torch.cat((pv, V), 1)
                see = torch.cat((pok.expand(n, len(pok)), see), 1)
        if n <= 0 or K.shape[1] == 0:
            continue
        for h in range(Hq):
            k, v = K[h // G], V[h // G]
            qq = q[a:e, h].double()
            s = (qq @ k.t() * scale).masked_fill(~see, -math.inf)
            L[a:e, h] = torch.logsumexp(s, -1)
            w = torch.where(see, torch.softmax(s, -1), 0.0)
            w = torch.where(see.any(-1, keepdim=True), w, 0.0)
            if torch.isfinite(v).all():
                O[a:e, h], A[a:e, h] = w @ v, w @ v.abs()
            else:
                prod = torch.where(see[:, :, None], w[:, :, None] * v[None], 0.0)
                O[a:e, h], A[a:e, h] = prod.sum(1), prod.abs().sum(1)
            C[a:e, h] = qq.norm(dim=-1) * torch.where(see, k.norm(dim=-1), 0.0).amax(-1) * abs(scale)
    return O, L, A, C


def attention_weights(weights, q, q_indptr, lse, pool, indptr, indices, last, rows=None, causal=True,
                      scale=None, window=None):
    """The sums after the call, and (for error bounds) what the call adds, and its terms weighted
    by |q| |k| |scale| and by |lse|, each shaped like the sums."""
    T, Hq, D = q.shape
    page, Hkv = pool.shape[3], pool.shape[2]
    N, _, Lmax = weights.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    added, far, norm = (torch.zeros(weights.shape, dtype=torch.float64) for _ in range(3))
    for b in range(len(last)):
        row = b if rows is None else int(rows[b])
        a, e = int(q_indptr[b]), int(q_indptr[b + 1])
        m = _length(indptr, last, b, page)
        if not 0 <= row < N or e <= a or m <= 0:
            continue
        K, _, ok = gather(pool, indices[int(indptr[b]):int(indptr[b + 1])], m)
        n = e - a
        if window is not None:
            a, n = e - min(n, window), min(n, window)
        see = ok.expand(n, m).clone()
        if causal:
            see &= torch.arange(m) <= torch.arange(m - n, m)[:, None]
        top = min(m, Lmax)
        for h in range(Hq):
            k, qq, l = K[h // (Hq // Hkv)], q[a:e, h].double(), lse[a:e, h].double()[:, None]
            p = torch.exp(qq @ k.t() * scale - l)
            p = torch.where(see & (l != -math.inf), p, 0.0)
            c = qq.norm(dim=-1)[:, None] * k.norm(dim=-1) * abs(scale)
            at = (row, h // (Hq // Hkv), slice(0, top))
            added[at] += p.sum(0)[:top]
            far[at] += torch.where(p > 0, p * c, 0.0).sum(0)[:top]
            norm[at] += torch.where(p > 0, p * l.abs(), 0.0).sum(0)[:top]
    return weights.double() + added, added, far, norm


def heaviest(weights, lengths, keep, first=0, recent=0, rows=None):
    """Kept-token lists (ind [B, H, keep], nnz [B, H, 1]) by a sort on (sum, lower index)."""
    N, H, L = weights.shape
    B = len(lengths)
    ind = torch.full((B, H, keep), -1, dtype=torch.int32)
    nnz = torch.zeros((B, H, 1), dtype=torch.int32)
    for b in range(B):
        row = b if rows is None else int(rows[b])
        n = min(max(int(lengths[b]), 0), L) if 0 <= row < N else 0
        for h in range(H):
            got = list(range(n))
            if n > keep:
                w = [float(x) for x in weights[row, h, :n]]
                rank = lambda i: (not math.isnan(w[i]), 0.0 if math.isnan(w[i]) else -w[i], i)  # noqa: E731
                sure = set(range(first)) | set(range(n - recent, n))
                others = sorted((i for i in range(n) if i not in sure), key=rank)
                got = sorted(sure | set(others[: keep - first - recent]))
            ind[b, h, : len(got)] = torch.tensor(got, dtype=torch.int32)
            nnz[b, h] = len(got)
    return ind, nnz


def keep_tokens(pool, indptr, indices, last, ind, nnz, dst=None, weights=None, rows=None):
    """(pool, weights) after the kept tokens' move, from copies of both."""
    P, _, Hkv, page, _ = pool.shape
    out, w = pool.clone(), None if weights is None else weights.clone()
    dst = indices if dst is None else dst
    for b in range(len(last)):
        n, p0 = _length(indptr, last, b, page), int(indptr[b])
        row = b if rows is None else int(rows[b])
        for h in range(Hkv):
            count = min(max(int(nnz[b, h]), 0), ind.shape[2], n)
            for j in range(count):
                t = int(ind[b, h, j])
                if not j <= t < n:
                    continue
                s, d = int(indices[p0 + t // page]), int(dst[p0 + j // page])
                if 0 <= s < P and 0 <= d < P:
                    out[d, :, h, j % page] = pool[s, :, h, t % page]
                if w is not None and 0 <= row < w.shape[0] and j < w.shape[2]:
                    w[row, h, j] = weights[row, h, t] if t < w.shape[2] else 0.0
            if w is not None and 0 <= row < w.shape[0]:
                w[row, h, count:n] = 0.0
    return out, w


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
