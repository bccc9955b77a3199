"""Performance cases of the operators that keep a paged KV cache small while it is served, and the
inputs, plain form, work and exact results of each: a prefix that sequences share is read once for
all of them, and tokens that no longer draw attention are found and dropped.

A case is a dict of plain values.  Its "kind" names the call that a program makes:

  shared   flash_attention_shared_prefix_paged: new tokens of sequences that share prefixes
  weights  accumulate_attention_weights_paged: the attention that each cached token drew in a step
           is added to what it drew before
  select   select_heaviest: the tokens to keep, by those sums
  keep     keep_tokens: the kept tokens' K and V (and sums) move to the front of their sequences

Tensors are N(0, 1); pools [P, 2, Hkv, page, D] lie behind a randomly permuted page table; sums
[N, Hkv, L] have a row for each sequence, in a permuted order.  Sequence lengths follow from the
case; everything else follows from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # Two answers to one short question begin: alone on the GPU (latency).
        {"name": "shared_first_d64", "kind": "shared", "B": 2, "groups": 1, "alone": 0,
         "prefix_lo": 40, "prefix_hi": 40, "Hq": 8, "Hkv": 2, "D": 64, "page": 16, "n_lo": 1,
         "n_hi": 1, "ctx_lo": 2, "ctx_hi": 19, "dtype": "fp16", "causal": True, "lse": True},
        # A decode step of the benchmark's batch and heads behind one long system prompt.
        {"name": "shared_decode_d128", "kind": "shared", "B": 32, "groups": 1, "alone": 0,
         "prefix_lo": 4096, "prefix_hi": 4096, "Hq": 32, "Hkv": 8, "D": 128, "page": 16, "n_lo": 1,
         "n_hi": 1, "ctx_lo": 100, "ctx_hi": 1000, "dtype": "fp16", "causal": True, "lse": False},
        # Many samples of the answer to one long document, eight query heads to a kv head.
        {"name": "shared_samples_bf16", "kind": "shared", "B": 64, "groups": 1, "alone": 0,
         "prefix_lo": 20001, "prefix_hi": 20001, "Hq": 64, "Hkv": 8, "D": 128, "page": 64,
         "n_lo": 1, "n_hi": 1, "ctx_lo": 1, "ctx_hi": 400, "dtype": "bf16", "causal": True,
         "lse": True},
        # Drafted tokens of several groups of sequences and of some that share nothing; wide
        # heads, odd pages.
        {"name": "shared_drafts_d256", "kind": "shared", "B": 24, "groups": 4, "alone": 3,
         "prefix_lo": 500, "prefix_hi": 3001, "Hq": 16, "Hkv": 4, "D": 256, "page": 24, "n_lo": 1,
         "n_hi": 6, "ctx_lo": 50, "ctx_hi": 600, "dtype": "fp16", "causal": True, "lse": True},
        # Prompts of different questions about one document.
        {"name": "shared_questions_d128", "kind": "shared", "B": 8, "groups": 1, "alone": 0,
         "prefix_lo": 8000, "prefix_hi": 8000, "Hq": 32, "Hkv": 8, "D": 128, "page": 32,
         "n_lo": 150, "n_hi": 350, "ctx_lo": 0, "ctx_hi": 0, "dtype": "bf16", "causal": True,
         "lse": False},
        # The first exchange of a conversation: five tokens after twelve, alone on the GPU.
        {"name": "weights_first_d64", "kind": "weights", "B": 1, "Hq": 8, "Hkv": 2, "D": 64,
         "page": 16, "n_lo": 5, "n_hi": 5, "ctx_lo": 12, "ctx_hi": 12, "L": 100, "dtype": "fp16",
         "causal": True},
        # A decode step of the benchmark's batch.
        {"name": "weights_decode_d128", "kind": "weights", "B": 32, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 16, "n_lo": 1, "n_hi": 1, "ctx_lo": 255, "ctx_hi": 8191, "L": 8200,
         "dtype": "fp16", "causal": True},
        # All tokens of a prompt's chunk count.
        {"name": "weights_prompt_bf16", "kind": "weights", "B": 1, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 32, "n_lo": 2048, "n_hi": 2048, "ctx_lo": 6000, "ctx_hi": 6000, "L": 8192,
         "dtype": "bf16", "causal": True},
        # Sequences a few tokens over their budget.
        {"name": "select_step", "kind": "select", "B": 16, "Hkv": 8, "len_lo": 1025,
         "len_hi": 1088, "L": 1100, "keep": 1024, "first": 4, "recent": 128, "ties": False},
        # Long prompts cut down to a tenth.
        {"name": "select_long", "kind": "select", "B": 8, "Hkv": 8, "len_lo": 20000,
         "len_hi": 40000, "L": 40000, "keep": 4000, "first": 4, "recent": 256, "ties": True},
        # The tokens that select_step's sequences keep close up.
        {"name": "keep_step_d128", "kind": "keep", "B": 16, "Hkv": 8, "D": 128, "page": 16,
         "len_lo": 1025, "len_hi": 1088, "L": 1100, "keep": 1024, "dtype": "fp16"},
        # Prompts cut to their budget.
        {"name": "keep_prompt_bf16", "kind": "keep", "B": 8, "Hkv": 8, "D": 128, "page": 64,
         "len_lo": 4000, "len_hi": 9000, "L": 9000, "keep": 2500, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


# A drawn case moves or computes no more than the largest listed ones, and the plain form's padded
# scores and gathered rows fit the card.
_MAX_FLOPS = 2.4e11
_MAX_BYTES = 4.5e8
_MAX_SCORES = 1.2e9
_MAX_GATHER = 4.0e8
_MAX_POOL = 3.0e8


def draw(rng):
    kind = rng.choice(["shared", "shared", "shared", "weights", "weights", "select", "keep"])
    while True:
        case = {"kind": kind, "Hkv": rng.choice([1, 2, 4, 8, 16])}
        Hkv = case["Hkv"]
        if kind != "select":
            D = rng.choice([64, 128, 128, 256])
            case.update(D=D, page=rng.choice([1, 8, 16, 16, 24, 32, 64, 128]),
                        dtype=rng.choice(["fp16", "bf16"]))
        if kind in ("shared", "weights"):
            case["Hq"] = Hkv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
            if case["Hq"] > 64:
                continue
            lo, hi = rng.choice([(1, 1), (1, 1), (1, 9), (10, 700)])
            case["n_hi"] = _log_int(rng, lo, hi)
            case["n_lo"] = rng.randint(lo, case["n_hi"])
            case["causal"] = rng.random() < 0.85
        if kind == "shared":
            case["groups"] = rng.choice([1, 1, 1, 2, 3, 5])
            case["alone"] = rng.choice([0, 0, 0, 1, 4])
            case["B"] = case["groups"] * _log_int(rng, 2, 64) + case["alone"] + rng.randint(0, 1)
            case["prefix_hi"] = _log_int(rng, 1, 20000)
            case["prefix_lo"] = rng.randint(1, case["prefix_hi"])
            case["ctx_hi"] = _log_int(rng, 1, 2000)
            case["ctx_lo"] = rng.randint(0, case["ctx_hi"])
            case["lse"] = rng.random() < 0.5
        elif kind == "weights":
            case["B"] = _log_int(rng, 1, 64)
            case["ctx_hi"] = _log_int(rng, 1, 20000)
            case["ctx_lo"] = rng.randint(0, case["ctx_hi"])
            case["L"] = case["ctx_hi"] + case["n_hi"] + rng.randint(0, 50)
        else:
            case["B"] = _log_int(rng, 1, 64)
            case["len_hi"] = _log_int(rng, 1, 40000 if kind == "select" else 9000)
            case["len_lo"] = rng.randint(1, case["len_hi"])
            case["L"] = case["len_hi"] + rng.randint(0, 50)
            case["keep"] = _log_int(rng, 1, case["len_hi"])
        if kind == "select":
            case["first"] = rng.choice([0, 0, 1, 4])
            case["recent"] = rng.choice([0, 0, 1, 32, 200])
            case["ties"] = rng.random() < 0.5
            if case["first"] + case["recent"] > case["keep"]:
                continue
        w = work(case)
        if w["flops"] > _MAX_FLOPS or w["bytes"] > _MAX_BYTES:
            continue
        if kind == "shared":
            rows = max(map(len, _members(case))) * case["n_hi"] * case["Hq"]
            if case["groups"] * rows * case["prefix_hi"] > _MAX_SCORES:
                continue
            if case["groups"] * case["prefix_hi"] * Hkv * D > _MAX_GATHER:
                continue
            if (_pages(case) + sum(_prefix_pages(case))) * 2 * Hkv * case["page"] * D > _MAX_POOL:
                continue
        if kind in ("shared", "weights"):
            longest = max(_lens(case))
            if case["B"] * case["Hq"] * case["n_hi"] * longest > _MAX_SCORES:
                continue
            if case["B"] * longest * Hkv * D > _MAX_GATHER:
                continue
        if kind != "select" and _pages(case) * 2 * Hkv * case["page"] * D > _MAX_POOL:
            continue
        return case


# --------------------------------------------------------------------------- sizes
def _spread(n, lo, hi, salt):
    """n whole numbers spread over [lo, hi], the same ones for the same case."""
    rng = random.Random(f"{salt} {n} {lo} {hi}")
    return [rng.randint(lo, hi) for _ in range(n)]


def _counts(case):
    """New tokens of each sequence."""
    return _spread(case["B"], case["n_lo"], case["n_hi"], "new")


def _lens(case):
    """Cached tokens of each sequence (behind its prefix), its new ones among them."""
    if "len_lo" in case:
        return _spread(case["B"], case["len_lo"], case["len_hi"], "length")
    ctx = _spread(case["B"], case["ctx_lo"], case["ctx_hi"], "context")
    return list(map(sum, zip(ctx, _counts(case))))


def _page_counts(case):
    return list(map(lambda n: -(-n // case["page"]), _lens(case)))


def _pages(case):
    return sum(_page_counts(case))


def _members(case):
    """The sequences of each group, as ranges; those behind the last group share nothing."""
    n, m = case["B"] - case["alone"], case["groups"]
    return [range(n * i // m, n * (i + 1) // m) for i in range(m)]


def _prefixes(case):
    """Tokens of each group's prefix."""
    return _spread(case["groups"], case["prefix_lo"], case["prefix_hi"], "prefix")


def _prefix_pages(case):
    return list(map(lambda n: -(-n // case["page"]), _prefixes(case)))


def _kept(case):
    """Tokens that each sequence keeps."""
    return list(map(lambda n: min(n, case["keep"]), _lens(case)))


def _pairs(case):
    """(new token, cached token of its sequence) pairs of which the first sees the second."""
    if case["causal"]:
        return sum(map(lambda n, m: n * (m - n) + n * (n + 1) // 2, _counts(case), _lens(case)))
    return sum(map(lambda n, m: n * m, _counts(case), _lens(case)))


def work(case):
    """Bytes: every input element that the call has to read once (the K/V rows, or K rows, that
    some new token sees) and every output element once.  FLOPs: 4 D per (query head, visible key)
    pair, 2 D where no V is multiplied.  Of the kept tokens' moves every one counts: the first
    dropped one of a head is near its front."""
    kind, Hkv, B = case["kind"], case["Hkv"], case["B"]
    if kind == "select":
        return {"bytes": 4 * (sum(_lens(case)) * Hkv + B * Hkv * (case["keep"] + 1) + 2 * B),
                "flops": 0}
    D = case["D"]
    table = 4 * (_pages(case) + 3 * B + 2)
    if kind == "keep":
        # The rows of K and V and the sums, read and written; the dropped sums, cleared.
        kept, dropped = sum(_kept(case)), sum(_lens(case)) - sum(_kept(case))
        return {"bytes": Hkv * (kept * (2 * D * 2 * 2 + 4 * 2 + 4) + 4 * dropped) + table,
                "flops": 0}
    Hq, new = case["Hq"], sum(_counts(case))
    if kind == "weights":
        return {"bytes": sum(_lens(case)) * Hkv * (D * 2 + 4 * 2) + new * Hq * (D * 2 + 4) + table,
                "flops": 2 * D * Hq * _pairs(case)}
    counts = _counts(case)
    pairs = _pairs(case) + sum(map(lambda m, p: sum(counts[m.start: m.stop]) * p, _members(case),
                                   _prefixes(case)))
    keys = sum(_lens(case)) + sum(_prefixes(case))
    table += 4 * (sum(_prefix_pages(case)) + 3 * case["groups"] + 2)
    return {"bytes": keys * Hkv * D * 2 * 2 + new * Hq * (D * 2 * 2 + (4 if case["lse"] else 0))
            + table, "flops": 4 * D * Hq * pairs}


# --------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 1000003 + 31)
    kind, Hkv, B, lens = case["kind"], case["Hkv"], case["B"], _lens(case)

    def randn(*shape, dt=torch.float32):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dt)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    def starts(v):
        return torch.tensor([0] + v, device=dev).cumsum(0).to(torch.int32)

    x = {"case": dict(case), "lengths": ints(lens), "longest": max(lens)}
    if kind != "shared":
        # What tokens drew so far: a few of them most of it, and nothing behind the last token.
        # Beside a step that adds to it, as much as steps like it draw.
        N = B + 3
        x["rows"] = torch.randperm(N, generator=g, device=dev)[:B].to(torch.int32)
        w = torch.exp(2.0 * randn(N, Hkv, case["L"]))
        if kind == "weights":
            w *= sum(_counts(case)) * case["Hq"] / Hkv / sum(lens)
        if case.get("ties"):
            w = torch.round(w * 8.0) / 8.0
        end = torch.zeros(N, dtype=torch.int32, device=dev)
        end[x["rows"].long()] = x["lengths"]
        x["weights"] = torch.where(torch.arange(case["L"], device=dev) < end[:, None, None], w, 0.0)
    if kind == "select":
        return x
    page, pages, D, dt = case["page"], _page_counts(case), case["D"], DTYPES[case["dtype"]]
    x["indptr"] = starts(pages)
    x["last"] = (x["lengths"] - 1) % page + 1
    more = sum(_prefix_pages(case)) if kind == "shared" else 0
    order = torch.randperm(sum(pages) + more, generator=g, device=dev).to(torch.int32)
    x["indices"] = order[: sum(pages)].contiguous()
    x["pool"] = randn(sum(pages) + more, 2, Hkv, page, D, dt=dt)
    if kind == "keep":
        # Kept tokens at random, in order, as a selection leaves them.
        K, M = case["keep"], x["longest"]
        r = torch.rand(B, Hkv, M, generator=g, device=dev)
        r = r.masked_fill_(torch.arange(M, device=dev) >= x["lengths"][:, None, None], 2.0)
        ind = r.topk(min(K, M), dim=-1, largest=False).indices.to(torch.int32)
        slot = torch.arange(K, device=dev, dtype=torch.int32)
        x["nnz"] = x["lengths"].clamp(max=K)[:, None, None].expand(B, Hkv, 1).contiguous()
        ind = torch.where(slot < x["nnz"], ind, M).sort(-1).values
        x["ind"] = torch.where(slot < x["nnz"], ind, -1).contiguous()
        return x
    counts = _counts(case)
    x["q"] = randn(sum(counts), case["Hq"], D, dt=dt)
    x["q_indptr"] = starts(counts)
    x["most_new"] = max(counts)
    if kind == "shared":
        members = _members(case)
        x["group_indptr"] = ints([m.start for m in members] + [members[-1].stop])
        x["prefix_indptr"] = starts(_prefix_pages(case))
        x["prefix_indices"] = order[sum(pages):].contiguous()
        x["prefix_lengths"] = ints(_prefixes(case))
        x["prefix_last"] = (x["prefix_lengths"] - 1) % page + 1
        x["longest_prefix"] = max(_prefixes(case))
        x["most_group"] = max(map(lambda m: sum(counts[m.start: m.stop]), members))
        return x
    # The normalisers that the step's attention returned.
    s = _scores(x)
    top = s.amax(-1, keepdim=True)
    lse = (top + s.sub_(top).exp_().sum(-1, keepdim=True).log()).view(B, Hkv, -1, x["most_new"])
    b, at = _new_tokens(x)
    x["lse"] = lse[b, :, :, at].reshape(-1, case["Hq"]).contiguous()
    return x


# --------------------------------------------------------------------------- plain forms
def _new_tokens(x):
    """Sequence of every new token, and its number in it."""
    qp = x["q_indptr"].long()
    t = torch.arange(x["q"].shape[0], device=qp.device)
    b = torch.searchsorted(qp[1:].contiguous(), t, right=True)
    return b, t - qp[:-1][b]


def _gather(x, indptr, indices, longest, planes=slice(None)):
    """Rows of the pool behind a page table, padded to the longest: [2 (or 1), B, Hkv, N, D]."""
    case = x["case"]
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    mp, ip = -(-longest // page), indptr.long()
    slots = (ip[:-1, None] + torch.arange(mp, device=ip.device)).clamp(max=indices.numel() - 1)
    kv = x["pool"][indices[slots].long(), planes]  # [B, mp, planes, Hkv, page, D]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(-1, ip.numel() - 1, Hkv, mp * page, D)
    return kv[:, :, :, :longest].float()


def _rows(x, starts, most):
    """Query rows from each start on, padded: [S, Hkv, G * most, D]."""
    case = x["case"]
    Hkv, D = case["Hkv"], case["D"]
    at = (starts[:, None] + torch.arange(most, device=starts.device)).clamp(max=x["q"].shape[0] - 1)
    q = x["q"][at].float().view(starts.numel(), most, Hkv, case["Hq"] // Hkv, D)
    return q.permute(0, 2, 3, 1, 4).reshape(starts.numel(), Hkv, -1, D)


def _scores(x, k=None):
    """Masked scores of the new tokens with their sequences' own keys [B, Hkv, G * n, N]."""
    case, lens, qp = x["case"], x["lengths"].long(), x["q_indptr"].long()
    n, N = x["most_new"], x["longest"]
    if k is None:
        k = _gather(x, x["indptr"], x["indices"], N, slice(0, 1))[0]
    s = torch.matmul(_rows(x, qp[:-1], n), k.transpose(-1, -2).contiguous()) / math.sqrt(case["D"])
    dev = lens.device
    limit = (lens - 1)[:, None].expand(-1, n)
    if case["causal"]:
        first = lens - (qp[1:] - qp[:-1])
        limit = torch.minimum(first[:, None] + torch.arange(n, device=dev), limit)
    B, Hkv = s.shape[:2]
    s.view(B, Hkv, -1, n, N).masked_fill_(
        torch.arange(N, device=dev) > limit[:, None, None, :, None], -math.inf)
    return s


def _plain_shared(x):
    """Attention over the groups' prefixes and over the sequences' own keys, each padded to the
    longest, and the sum of the two under one normaliser."""
    case = x["case"]
    Hkv, Hq, D = case["Hkv"], case["Hq"], case["D"]
    qp = x["q_indptr"].long()
    b, at = _new_tokens(x)

    def state(s, v, seq, row, most):
        """Max, sum of exponentials and weighted values of the rows of a padded batch."""
        top = s.amax(-1, keepdim=True)
        p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
        total, o = p.sum(-1, keepdim=True), torch.matmul(p, v)
        pick = lambda y: y.view(y.shape[0], Hkv, Hq // Hkv, most, -1)[seq, :, :, row].reshape(  # noqa: E731
            seq.numel(), Hq, -1)
        return pick(top), pick(total), pick(o)

    kv = _gather(x, x["indptr"], x["indices"], x["longest"])
    own_top, own_total, own_o = state(_scores(x, kv[0]), kv[1], b, at, x["most_new"])
    gp = x["group_indptr"].long()
    first = qp[gp]
    kv = _gather(x, x["prefix_indptr"], x["prefix_indices"], x["longest_prefix"])
    s = torch.matmul(_rows(x, first[:-1], x["most_group"]), kv[0].transpose(-1, -2).contiguous())
    s = (s / math.sqrt(D)).masked_fill_(
        torch.arange(x["longest_prefix"], device=qp.device)
        >= x["prefix_lengths"][:, None, None, None], -math.inf)
    grp = torch.searchsorted(gp[1:].contiguous(), b, right=True)
    has = grp < gp.numel() - 1
    grp = grp.clamp(max=gp.numel() - 2)
    row = torch.where(has, torch.arange(b.numel(), device=b.device) - first[grp], 0)
    top, total, o = state(s, kv[1], grp, row, x["most_group"])
    top = torch.where(has[:, None, None], top, -math.inf)
    both = torch.maximum(top, own_top)
    f, h = torch.exp(top - both), torch.exp(own_top - both)
    total = f * total + h * own_total
    out = ((f * o + h * own_o) / total).to(x["q"].dtype)
    if not case["lse"]:
        return out
    return {"out": out, "lse": (both + torch.log(total)).squeeze(-1)}


def _plain(x):
    case = x["case"]
    kind, Hkv, B = case["kind"], case["Hkv"], case["B"]
    if kind == "shared":
        return _plain_shared(x)
    dev, lens, rows = x["lengths"].device, x["lengths"].long(), x["rows"].long()
    if kind == "weights":
        s = _scores(x)
        qp, n = x["q_indptr"].long(), x["most_new"]
        at = (qp[:-1, None] + torch.arange(n, device=dev)).clamp(max=x["q"].shape[0] - 1)
        lse = x["lse"][at].view(B, n, Hkv, -1).permute(0, 2, 3, 1)  # [B, Hkv, G, n]
        lse = lse.masked_fill((torch.arange(n, device=dev) >= (qp[1:] - qp[:-1])[:, None])
                              [:, None, None], math.inf)  # padded tokens weigh nothing
        p = s.sub_(lse.reshape(B, Hkv, -1, 1)).exp_()
        x["weights"][rows, :, : x["longest"]] += p.sum(-2)
        return x["weights"]
    if kind == "select":
        N, keep = x["longest"], case["keep"]
        t = torch.arange(N, device=dev)
        w = x["weights"][rows, :, :N]
        sure = (t < case["first"]) | (t >= lens[:, None] - case["recent"])
        w = torch.where(sure[:, None], math.inf, w)
        w = torch.where((t < lens[:, None])[:, None], w, -math.inf)
        order = w.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
        nnz = lens.clamp(max=keep)[:, None, None].expand(B, Hkv, 1)
        order = torch.nn.functional.pad(order, (0, keep - order.shape[-1]), value=N)
        slot = torch.arange(keep, device=dev)
        ind = torch.where(slot < nnz, order, N).sort(-1).values
        return {"ind": torch.where(slot < nnz, ind, -1).to(torch.int32),
                "nnz": nnz.to(torch.int32)}
    # keep: gathered whole, then written.
    page, ind = case["page"], x["ind"].long()
    slot = torch.arange(case["keep"], device=dev)
    b, h, j = torch.nonzero(slot < x["nnz"], as_tuple=True)
    pages, ip = x["indices"].long(), x["indptr"].long()
    old = ind[b, h, j]
    src, dst = pages[ip[b] + old // page], pages[ip[b] + j // page]
    pool, w = x["pool"], x["weights"]
    pool[dst, :, h, j % page] = pool[src, :, h, old % page]
    sums = w[rows[b], h, old]
    w[rows] = w[rows].masked_fill_(
        torch.arange(case["L"], device=dev) < lens[:, None, None], 0.0)
    w[rows[b], h, j] = sums
    return {"pool": pool, "weights": w}


def run(x):
    if not own:
        return _plain(x)
    from attention_kernel_triton_amd import (attention_weights_paged, kept_index, paged_kv,
                                             shared_prefix_flash_attention_paged)

    case = x["case"]
    kind = case["kind"]
    if kind == "shared":
        out = shared_prefix_flash_attention_paged.flash_attention_shared_prefix_paged(
            x["q"], x["q_indptr"], x["pool"], x["indptr"], x["indices"], x["last"],
            x["group_indptr"], x["prefix_indptr"], x["prefix_indices"], x["prefix_last"],
            causal=case["causal"], return_lse=case["lse"])
        return {"out": out[0], "lse": out[1]} if case["lse"] else out
    if kind == "weights":
        attention_weights_paged.accumulate_attention_weights_paged(
            x["weights"], x["q"], x["q_indptr"], x["lse"], x["pool"], x["indptr"], x["indices"],
            x["last"], rows=x["rows"], causal=case["causal"])
        return x["weights"]
    if kind == "select":
        ind, nnz = kept_index.select_heaviest(x["weights"], x["lengths"], case["keep"],
                                              first=case["first"], recent=case["recent"],
                                              rows=x["rows"])
        return {"ind": ind, "nnz": nnz}
    paged_kv.keep_tokens(x["pool"], x["indptr"], x["indices"], x["last"], x["ind"], x["nnz"],
                         weights=x["weights"], rows=x["rows"])
    return {"pool": x["pool"], "weights": x["weights"]}


# --------------------------------------------------------------------------- exact results
def exact(case, seed):
    """The definitions in 64 bits, one sequence (and kv head) at a time."""
    x = prepare(case, seed)
    kind, Hkv, B, lens = case["kind"], case["Hkv"], case["B"], _lens(case)
    f64 = torch.float64
    if kind == "select":
        keep = case["keep"]
        ind = torch.full((B, Hkv, keep), -1, dtype=torch.int32)
        nnz = torch.empty((B, Hkv, 1), dtype=torch.int32)
        w = x["weights"][x["rows"].long()].cpu()
        for b in range(B):
            n, lo = lens[b], case["first"]
            hi = max(n - case["recent"], lo)
            for h in range(Hkv):
                got = list(range(n))
                if n > keep:
                    # The lowest of equal sums come first in a stable order.
                    best = torch.argsort(-w[b, h, lo:hi], stable=True)[: keep - lo - (n - hi)] + lo
                    got = sorted(list(range(lo)) + best.tolist() + list(range(hi, n)))
                ind[b, h, : len(got)] = torch.tensor(got, dtype=torch.int32)
                nnz[b, h, 0] = len(got)
        return {"ind": ind.cuda(), "nnz": nnz.cuda()}
    page, ip = case["page"], x["indptr"].tolist()
    if kind == "keep":
        pool, w, old_w = x["pool"].clone(), x["weights"].clone(), x["weights"]
        for b in range(B):
            pg, row = x["indices"][ip[b]: ip[b + 1]].long(), int(x["rows"][b])
            w[row, :, : lens[b]] = 0
            for h in range(Hkv):
                n = int(x["nnz"][b, h, 0])
                old, new = x["ind"][b, h, :n].long(), torch.arange(n, device="cuda")
                pool[pg[new // page], :, h, new % page] = x["pool"][pg[old // page], :, h, old % page]
                w[row, h, :n] = old_w[row, h, old]
        return {"pool": pool, "weights": w}
    D, G, counts, at = case["D"], case["Hq"] // Hkv, _counts(case), 0

    def rows_of(indices, start, stop, m):
        kv = x["pool"][indices[start:stop].long()]
        return kv.permute(1, 2, 0, 3, 4).reshape(2, Hkv, -1, D)[:, :, :m].to(f64)

    if kind == "weights":
        w = x["weights"].to(f64)
        for b in range(B):
            n, m = counts[b], lens[b]
            k = rows_of(x["indices"], ip[b], ip[b + 1], m)[0]
            hide = torch.arange(m, device="cuda") > torch.arange(m - n, m, device="cuda")[:, None]
            for h in range(case["Hq"]):
                s = torch.matmul(x["q"][at: at + n, h].to(f64), k[h // G].t()) * D ** -0.5
                s -= x["lse"][at: at + n, h, None].to(f64)
                if case["causal"]:
                    s.masked_fill_(hide, -math.inf)
                w[int(x["rows"][b]), h // G, :m] += s.exp_().sum(0)
            at += n
        return w
    out = torch.empty(x["q"].shape, dtype=f64, device="cuda")
    lse = torch.empty(x["q"].shape[:2], dtype=f64, device="cuda")
    pp, lens_p, members = x["prefix_indptr"].tolist(), _prefixes(case), _members(case)
    for i, group in enumerate(members + [range(members[-1].stop, B)]):
        shared = torch.empty(2, Hkv, 0, D, dtype=f64, device="cuda")
        if i < len(members):
            shared = rows_of(x["prefix_indices"], pp[i], pp[i + 1], lens_p[i])
        P = shared.shape[2]
        for b in group:
            n, m = counts[b], lens[b]
            kv = torch.cat((shared, rows_of(x["indices"], ip[b], ip[b + 1], m)), 2)
            hide = torch.arange(P + m, device="cuda") > torch.arange(P + m - n, P + m, device="cuda")[:, None]
            for h in range(Hkv):
                q = x["q"][at: at + n, h * G: h * G + G].to(f64).transpose(0, 1).reshape(G * n, D)
                s = torch.matmul(q, kv[0, h].t()).view(G, n, P + m) * D ** -0.5
                if case["causal"]:
                    s.masked_fill_(hide, -math.inf)
                e = torch.logsumexp(s, -1)
                o = torch.matmul(torch.exp_(s.sub_(e[..., None])).view(G * n, P + m), kv[1, h])
                lse[at: at + n, h * G: h * G + G] = e.t()
                out[at: at + n, h * G: h * G + G] = o.view(G, n, D).transpose(0, 1)
            at += n
    return {"out": out, "lse": lse} if case["lse"] else out
