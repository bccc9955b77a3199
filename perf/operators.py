"""Performance cases of the operators that serve a paged KV cache beyond single-token decode, and
the inputs, plain form, work and exact results of each.

A case is a dict of plain values.  Its "kind" names the call that a program makes:

  chunk          flash_attention_chunk_paged: several new tokens per sequence attend a paged cache
  append_rotary  append_paged_kv_rotary: new q and k rotated by their positions, k and v appended
  rotary         apply_rotary on dense Q and K, or its transpose (the gradient)
  copy           copy_pages: whole pages (compaction) or the filled part of pages (a fork's last page)

Tensors are N(0, 1); pools [P, 2, Hkv, page, D] lie behind a randomly permuted page table.
Sequence lengths follow from the case; everything else follows from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # The first exchange of a conversation: five tokens after twelve, alone on the GPU (latency).
        {"name": "chunk_first_d64", "kind": "chunk", "B": 1, "Hq": 8, "Hkv": 2, "D": 64, "page": 16,
         "first": 5, "n_lo": 5, "n_hi": 5, "ctx_lo": 12, "ctx_hi": 12, "dtype": "fp16",
         "causal": True, "lse": True},
        # One token per sequence: the decode batch of the benchmark through the chunk call.
        {"name": "chunk_single_d128", "kind": "chunk", "B": 32, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 16, "first": 1, "n_lo": 1, "n_hi": 1, "ctx_lo": 255, "ctx_hi": 8191,
         "dtype": "fp16", "causal": True, "lse": False},
        # Verification of drafted tokens, eight query heads to a kv head, with the normaliser.
        {"name": "chunk_verify_bf16", "kind": "chunk", "B": 16, "Hq": 64, "Hkv": 8, "D": 128,
         "page": 64, "first": 7, "n_lo": 3, "n_hi": 7, "ctx_lo": 500, "ctx_hi": 4000,
         "dtype": "bf16", "causal": True, "lse": True},
        # A mixed serving batch: one prompt of 777 tokens beside fifteen decoding sequences.
        {"name": "chunk_mixed_d128", "kind": "chunk", "B": 16, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 16, "first": 777, "n_lo": 1, "n_hi": 1, "ctx_lo": 0, "ctx_hi": 4096,
         "dtype": "fp16", "causal": True, "lse": False},
        # A piece of a long document against what is cached of it.
        {"name": "chunk_long_d128_bf16", "kind": "chunk", "B": 1, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 32, "first": 2048, "n_lo": 2048, "n_hi": 2048, "ctx_lo": 30000, "ctx_hi": 30000,
         "dtype": "bf16", "causal": True, "lse": False},
        # Every token sees the whole cache (another sequence's states), wide heads, odd pages.
        {"name": "chunk_full_d256", "kind": "chunk", "B": 3, "Hq": 16, "Hkv": 4, "D": 256,
         "page": 24, "first": 100, "n_lo": 100, "n_hi": 300, "ctx_lo": 1000, "ctx_hi": 3000,
         "dtype": "fp16", "causal": False, "lse": True},
        # A decode step's tokens, rotated and written.
        {"name": "append_rotary_step", "kind": "append_rotary", "B": 64, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 16, "first": 1, "n_lo": 1, "n_hi": 1, "ctx_lo": 100, "ctx_hi": 2000,
         "dtype": "fp16", "rot": 128, "base": 10000.0, "stretch": 1.0, "factor": 1.0,
         "interleaved": False},
        # Prompt chunks far into their contexts: half of each head rotated, neighbouring pairs,
        # positions stretched for a long context.
        {"name": "append_rotary_prompt", "kind": "append_rotary", "B": 4, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 64, "first": 3001, "n_lo": 1000, "n_hi": 3000, "ctx_lo": 0,
         "ctx_hi": 16000, "dtype": "bf16", "rot": 64, "base": 500000.0, "stretch": 8.0,
         "factor": 1.2, "interleaved": True},
        # Q and K of the benchmark's dense prefill.
        {"name": "rotary_dense_d64", "kind": "rotary", "B": 8, "Hq": 64, "Hkv": 16, "S": 1024,
         "D": 64, "dtype": "fp16", "rot": 64, "base": 10000.0, "stretch": 1.0, "factor": 1.0,
         "interleaved": False, "transpose": False, "far": 0},
        # The transposed map on a short bf16 batch at far positions, a quarter of each head.
        {"name": "rotary_transpose_d256", "kind": "rotary", "B": 2, "Hq": 16, "Hkv": 2, "S": 37,
         "D": 256, "dtype": "bf16", "rot": 64, "base": 1000000.0, "stretch": 4.0, "factor": 1.1,
         "interleaved": True, "transpose": True, "far": 1000000},
        # The last, partly filled pages of forked sequences.
        {"name": "copy_fork_tails", "kind": "copy", "N": 16, "P": 300, "Hkv": 8, "D": 128,
         "page": 16, "dtype": "fp16", "partial": True},
        # Compaction: a thousand pages to the front of the pool.
        {"name": "copy_compact", "kind": "copy", "N": 1000, "P": 2100, "Hkv": 8, "D": 128,
         "page": 64, "dtype": "bf16", "partial": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


# A drawn case moves or computes no more than the largest listed ones, and the plain form's padded
# scores and gathered rows fit the card.
_MAX_FLOPS = 1.05e12
_MAX_BYTES = 5.5e8
_MAX_SCORES = 2.2e9
_MAX_GATHER = 6.0e8
_MAX_POOL = 3.0e8


def _draw_rotation(rng, D):
    return {"rot": rng.choice([D, D, D // 2, D // 4, D // 2 - 4]),
            "base": rng.choice([10000.0, 500000.0, 1000000.0]),
            "stretch": rng.choice([1.0, 1.0, 4.0, 8.0]), "factor": rng.choice([1.0, 1.0, 1.2]),
            "interleaved": rng.random() < 0.5}


def draw(rng):
    kind = rng.choice(["chunk", "chunk", "chunk", "chunk", "append_rotary", "rotary", "copy"])
    while True:
        Hkv = rng.choice([1, 2, 4, 8, 16])
        G = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
        D = rng.choice([64, 128, 128, 256])
        case = {"kind": kind, "Hkv": Hkv, "D": D, "dtype": rng.choice(["fp16", "bf16"])}
        if kind != "copy":
            case.update(B=_log_int(rng, 1, 64), Hq=Hkv * G)
        if kind in ("chunk", "append_rotary"):
            shape = rng.choice(["single", "verify", "prompt", "mixed"])
            lo, hi = {"single": (1, 1), "verify": (1, 9), "prompt": (10, 3000), "mixed": (1, 2)}[shape]
            case["n_hi"] = _log_int(rng, lo, hi)
            case["n_lo"] = rng.randint(lo, case["n_hi"])
            case["first"] = _log_int(rng, 100, 2000) if shape == "mixed" else case["n_lo"]
            case["ctx_hi"] = _log_int(rng, 1, 32000)
            case["ctx_lo"] = round(case["ctx_hi"] * rng.uniform(0.0, 1.0))
            case["page"] = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
        if kind == "chunk":
            case.update(causal=rng.random() < 0.85, lse=rng.random() < 0.5)
        elif kind == "append_rotary":
            case.update(_draw_rotation(rng, D))
        elif kind == "rotary":
            case.update(S=_log_int(rng, 1, 8192), transpose=rng.random() < 0.4,
                        far=rng.choice([0, 0, 1000, 1000000]), **_draw_rotation(rng, D))
        else:
            N = _log_int(rng, 1, 3000)
            case.update(N=N, P=2 * N + rng.randint(0, 100), page=rng.choice([1, 8, 16, 24, 32, 64]),
                        partial=rng.random() < 0.5)
        if kind != "copy" and case["Hq"] > 64:
            continue
        w = work(case)
        if w["flops"] > _MAX_FLOPS or w["bytes"] > _MAX_BYTES:
            continue
        if kind == "chunk":
            longest = max(_lens(case))
            if case["B"] * case["Hq"] * max(_counts(case)) * longest > _MAX_SCORES:
                continue
            if case["B"] * longest * Hkv * D > _MAX_GATHER:
                continue
        if kind in ("chunk", "append_rotary"):
            if _pages(case) * 2 * Hkv * case["page"] * D > _MAX_POOL:
                continue
        if kind == "copy" and case["P"] * 2 * Hkv * case["page"] * D > _MAX_POOL:
            continue
        return case


# --------------------------------------------------------------------------- sizes
def _spread(n, lo, hi, salt):
    """n whole numbers spread over [lo, hi], the same ones for the same case."""
    rng = random.Random(f"{salt} {n} {lo} {hi}")
    return [rng.randint(lo, hi) for _ in range(n)]


def _counts(case):
    """New tokens of each sequence."""
    return [case["first"]] + _spread(case["B"] - 1, case["n_lo"], case["n_hi"], "new")


def _lens(case):
    """Cached tokens of each sequence, its new ones among them."""
    ctx = _spread(case["B"], case["ctx_lo"], case["ctx_hi"], "context")
    return list(map(sum, zip(ctx, _counts(case))))


def _page_counts(case):
    return list(map(lambda n: -(-n // case["page"]), _lens(case)))


def _pages(case):
    return sum(_page_counts(case))


def _copied(case):
    """Slots copied of each page: whole pages, or one to all of the slots."""
    if not case["partial"]:
        return [case["page"]] * case["N"]
    return _spread(case["N"], 1, case["page"], "slots")


def work(case):
    """Bytes: every input element that the call has to read once (the cached K/V rows that some
    new token sees) and every output element once.  FLOPs: 4 D per (query head, visible key) pair;
    three per element that a rotation writes."""
    kind, Hkv, D = case["kind"], case["Hkv"], case["D"]
    if kind == "copy":
        return {"bytes": sum(_copied(case)) * 2 * Hkv * D * 2 * 2 + 8 * case["N"], "flops": 0}
    Hq = case["Hq"]
    if kind == "rotary":
        rows = case["B"] * case["S"] * (Hq + Hkv)
        return {"bytes": rows * D * 2 * 2, "flops": 3 * rows * case["rot"]}
    counts, lens = _counts(case), _lens(case)
    new = sum(counts)
    table = 4 * (_pages(case) + 3 * case["B"] + 2)
    if kind == "append_rotary":
        # Of the page table only the pages that new tokens reach.
        touched = sum(map(lambda n: -(-n // case["page"]), counts))
        return {"bytes": new * D * 2 * 2 * (Hq + 2 * Hkv) + 4 * (touched + 3 * case["B"] + 2),
                "flops": 3 * new * (Hq + Hkv) * case["rot"]}
    if case["causal"]:
        pairs = sum(map(lambda n, m: n * (m - n) + n * (n + 1) // 2, counts, lens))
    else:
        pairs = sum(map(lambda n, m: n * m, counts, lens))
    return {"bytes": sum(lens) * Hkv * D * 2 * 2 + new * Hq * (D * 2 * 2 + (4 if case["lse"] else 0))
            + table, "flops": 4 * D * Hq * pairs}


# --------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 1000003 + 29)
    kind, Hkv, D, dt = case["kind"], case["Hkv"], case["D"], DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dt)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    x = {"case": dict(case)}
    if kind != "copy" and kind != "chunk":
        f = torch.arange(case["rot"] // 2, device=dev, dtype=torch.float64)
        x["inv_freq"] = case["base"] ** (-2.0 * f / case["rot"]) / case["stretch"]
    if kind == "rotary":
        B, S = case["B"], case["S"]
        x["Q"], x["K"] = randn(B, case["Hq"], S, D), randn(B, Hkv, S, D)
        x["positions"] = None
        if case["far"]:
            # Unequal starts, as in a batch of prompts that continue cached ones.
            x["positions"] = torch.randint(0, case["far"], (B, 1), generator=g, device=dev) + \
                torch.arange(S, device=dev)
        return x
    if kind == "copy":
        P, N = case["P"], case["N"]
        order = torch.randperm(P, generator=g, device=dev).to(torch.int32)
        x["pool"] = randn(P, 2, Hkv, case["page"], D)
        x["src"], x["dst"] = order[:N].contiguous(), order[N: 2 * N].contiguous()
        x["slots"] = ints(_copied(case)) if case["partial"] else None
        return x
    page, counts, lens = case["page"], _counts(case), _lens(case)
    pages = _page_counts(case)
    x["q"] = randn(sum(counts), case["Hq"], D)
    x["q_indptr"] = torch.tensor([0] + counts, device=dev).cumsum(0).to(torch.int32)
    x["indptr"] = torch.tensor([0] + pages, device=dev).cumsum(0).to(torch.int32)
    x["indices"] = torch.randperm(sum(pages), generator=g, device=dev).to(torch.int32)
    x["last"] = (ints(lens) - 1) % page + 1
    x["pool"] = randn(sum(pages), 2, Hkv, page, D)
    if kind == "append_rotary":
        x["k_new"], x["v_new"] = randn(sum(counts), Hkv, D), randn(sum(counts), Hkv, D)
    x["longest"], x["most_new"] = max(lens), max(counts)  # the sizes a program keeps on the host
    return x


# --------------------------------------------------------------------------- plain forms
def _token_positions(x, page):
    """Sequence and position of every new token, from the tables."""
    qp, ip = x["q_indptr"].long(), x["indptr"].long()
    t = torch.arange(x["q"].shape[0], device=qp.device)
    b = torch.searchsorted(qp[1:].contiguous(), t, right=True)
    lens = (ip[1:] - ip[:-1] - 1) * page + x["last"].long()
    return b, lens[b] - (qp[1:][b] - t), lens


def _rotate(x, positions, inv_freq, interleaved, factor):
    """Rotation of x [..., D] in 32 bits by 64-bit angles; positions broadcast against x's rows."""
    r = 2 * inv_freq.numel()
    angle = positions.double().unsqueeze(-1) * inv_freq
    cos, sin = (torch.cos(angle) * factor).float(), (torch.sin(angle) * factor).float()
    y = x.float()
    if interleaved:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        rotated = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = y[..., : r // 2], y[..., r // 2: r]
        rotated = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((rotated, y[..., r:]), -1).to(x.dtype)


def _plain_chunk(x):
    """Sequences padded to the longest: gathered keys and values, masked softmax, gathered rows."""
    case = x["case"]
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    G = case["Hq"] // Hkv
    b, pos, lens = _token_positions(x, page)
    B, n, N = lens.numel(), x["most_new"], x["longest"]
    ip, qp = x["indptr"].long(), x["q_indptr"].long()
    dev = lens.device
    mp = -(-N // page)
    slots = (ip[:-1, None] + torch.arange(mp, device=dev)).clamp(max=x["indices"].numel() - 1)
    kv = x["pool"][x["indices"][slots].long()]  # [B, mp, 2, Hkv, page, D]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, B, Hkv, mp * page, D)[:, :, :, :N].float()
    rows = (qp[:-1, None] + torch.arange(n, device=dev)).clamp(max=x["q"].shape[0] - 1)
    q = x["q"][rows].float().view(B, n, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * n, D)
    s = torch.matmul(q, kv[0].transpose(-1, -2).contiguous()) / math.sqrt(D)
    s = s.view(B, Hkv, G, n, N)
    key = torch.arange(N, device=dev)
    limit = lens - 1
    if case["causal"]:
        first = lens - (qp[1:] - qp[:-1])
        limit = torch.minimum(first[:, None] + torch.arange(n, device=dev), limit[:, None])
    else:
        limit = limit[:, None].expand(B, n)
    s.masked_fill_(key > limit[:, None, None, :, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, G * n, N), kv[1]).view(B, Hkv, G, n, D)
    o = torch.where(total > 0, o / total, 0.0)
    at = torch.arange(b.numel(), device=dev) - qp[:-1][b]
    out = o.permute(0, 3, 1, 2, 4)[b, at].reshape(-1, Hkv * G, D).to(x["q"].dtype)
    if not case["lse"]:
        return out
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2)[b, at].reshape(-1, Hkv * G)
    return {"out": out, "lse": lse}


def _plain(x):
    case = x["case"]
    kind = case["kind"]
    if kind == "chunk":
        return _plain_chunk(x)
    if kind == "append_rotary":
        page = case["page"]
        b, pos, _ = _token_positions(x, page)
        q, k = (_rotate(x[n], pos[:, None], x["inv_freq"], case["interleaved"], case["factor"])
                for n in ("q", "k_new"))
        pg = x["indices"][x["indptr"].long()[:-1][b] + pos // page].long()
        x["pool"][pg, 0, :, pos % page] = k
        x["pool"][pg, 1, :, pos % page] = x["v_new"]
        return {"q": q, "pool": x["pool"]}
    if kind == "rotary":
        positions = x["positions"]
        if positions is None:
            positions = torch.arange(case["S"], device=x["Q"].device)[None]
        sign = -1 if case["transpose"] else 1
        return tuple(_rotate(x[n], sign * positions[:, None], x["inv_freq"], case["interleaved"],
                             case["factor"]) for n in ("Q", "K"))
    src, dst, pool = x["src"].long(), x["dst"].long(), x["pool"]
    rows = pool[src]
    if x["slots"] is not None:
        keep = torch.arange(case["page"], device=src.device) < x["slots"][:, None]
        rows = torch.where(keep[:, None, None, :, None], rows, pool[dst])
    pool[dst] = rows
    return pool


def run(x):
    if not own:
        return _plain(x)
    from attention_kernel_triton_amd import chunk_flash_attention_paged, paged_kv, rotary

    case = x["case"]
    kind = case["kind"]
    if kind == "chunk":
        out = chunk_flash_attention_paged.flash_attention_chunk_paged(
            x["q"], x["q_indptr"], x["pool"], x["indptr"], x["indices"], x["last"],
            causal=case["causal"], return_lse=case["lse"])
        return {"out": out[0], "lse": out[1]} if case["lse"] else out
    if kind == "append_rotary":
        q = paged_kv.append_paged_kv_rotary(
            x["q"], x["k_new"], x["v_new"], x["q_indptr"], x["pool"], x["indptr"], x["indices"],
            x["last"], x["inv_freq"], interleaved=case["interleaved"], factor=case["factor"])
        return {"q": q, "pool": x["pool"]}
    if kind == "rotary":
        return rotary.apply_rotary(x["Q"], x["K"], x["inv_freq"], positions=x["positions"],
                                   interleaved=case["interleaved"], factor=case["factor"],
                                   transpose=case["transpose"])
    paged_kv.copy_pages(x["pool"], x["src"], x["dst"], num_tokens=x["slots"])
    return x["pool"]


# --------------------------------------------------------------------------- exact results
def exact(case, seed):
    """The definitions in 64 bits, one sequence (and kv head) at a time."""
    x = prepare(case, seed)
    kind, Hkv, D = case["kind"], case["Hkv"], case["D"]
    f64 = torch.float64

    def turn(t, pos):
        """t [rows, heads, D] at positions pos [rows], as complex numbers times e^(i angle)."""
        r = case["rot"]
        y = t.to(f64).clone()
        if case["interleaved"]:
            re, im = slice(0, r, 2), slice(1, r, 2)
        else:
            re, im = slice(0, r // 2), slice(r // 2, r)
        angle = pos.to(f64)[:, None, None] * x["inv_freq"]
        w = torch.complex(y[..., re], y[..., im]) * torch.polar(torch.full_like(angle, case["factor"]), angle)
        y[..., re], y[..., im] = w.real, w.imag
        return y

    if kind == "copy":
        pool = x["pool"]
        for s, d, n in zip(x["src"].tolist(), x["dst"].tolist(), _copied(case)):
            pool[d, :, :, :n] = pool[s, :, :, :n]
        return pool
    if kind == "rotary":
        out = []
        for name in ("Q", "K"):
            y = torch.empty(x[name].shape, dtype=f64, device="cuda")
            for b in range(case["B"]):
                pos = torch.arange(case["S"], device="cuda") if x["positions"] is None else x["positions"][b]
                y[b] = turn(x[name][b].transpose(0, 1), -pos if case["transpose"] else pos).transpose(0, 1)
            out.append(y)
        return tuple(out)
    page, counts, lens = case["page"], _counts(case), _lens(case)
    ip, at = x["indptr"].tolist(), 0
    if kind == "append_rotary":
        q = torch.empty(x["q"].shape, dtype=f64, device="cuda")
        pool = x["pool"].to(f64)
        for b in range(case["B"]):
            n = counts[b]
            pos = torch.arange(lens[b] - n, lens[b], device="cuda")
            q[at: at + n] = turn(x["q"][at: at + n], pos)
            pg = x["indices"][ip[b]: ip[b + 1]].long()[pos // page]
            pool[pg, 0, :, pos % page] = turn(x["k_new"][at: at + n], pos)
            pool[pg, 1, :, pos % page] = x["v_new"][at: at + n].to(f64)
            at += n
        return {"q": q, "pool": pool}
    G = case["Hq"] // Hkv
    out = torch.empty(x["q"].shape, dtype=f64, device="cuda")
    lse = torch.empty(x["q"].shape[:2], dtype=f64, device="cuda")
    for b in range(case["B"]):
        n, m = counts[b], lens[b]
        kv = x["pool"][x["indices"][ip[b]: ip[b + 1]].long()]
        kv = kv.permute(1, 2, 0, 3, 4).reshape(2, Hkv, -1, D)[:, :, :m]
        hide = torch.arange(m, device="cuda") > torch.arange(m - n, m, device="cuda")[:, None]
        for h in range(case["Hq"]):
            s = torch.matmul(x["q"][at: at + n, h].to(f64), kv[0, h // G].to(f64).t()) * D ** -0.5
            if case["causal"]:
                s.masked_fill_(hide, -math.inf)
            e = torch.logsumexp(s, -1)
            lse[at: at + n, h] = e
            out[at: at + n, h] = torch.matmul(torch.exp_(s.sub_(e[:, None])), kv[1, h // G].to(f64))
        at += n
    return {"out": out, "lse": lse} if case["lse"] else out
