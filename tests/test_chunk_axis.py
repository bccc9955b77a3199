"""The chunk attention's division of work (csrc/paged_chunk.hip), restated on the host: units on an
axis of keys, ranges, cuts, partial slots and arrival counters.

For random batches of every kind: each key of each unit is served once, parts of a cut unit go to
the ranges that its merge reads, slots and counters are used once and lie inside the workspace, whose
size is the library's own.
"""
import bisect
import itertools
import math
import random
import re
from pathlib import Path

import pytest

from attention_kernel_triton_amd import _native as N

CSRC = Path(__file__).resolve().parent.parent / "attention_kernel_triton_amd" / "csrc"


def _constant(name):
    text = (CSRC / "paged_chunk.hpp").read_text() + (CSRC / "paged_chunk.hip").read_text()
    return int(re.search(rf"constexpr int {name} = (\d+);", text).group(1))


BLOCK, COST, MIN_KEYS = _constant("kCkBlock"), _constant("kCkUnitCost"), _constant("kCkMinKeys")
ZERO = N.WORKSPACE_ZERO_BYTES
FEW, MANY = 1, 2


class Plan:
    """What the host computes from the sizes (without a device: 256 CUs)."""

    def __init__(self, batch, total_q, Hkv, G, D, page, total_pages):
        self.waves = 8 if D <= 128 else 4
        rows = 32 if D <= 128 else 64
        resident = -(-256 * (2 if D <= 128 else 1) * 4 // self.waves // 8) * 8
        seqs = min(batch, total_q)
        self.split = rows // G
        few = total_q <= self.split
        if not few and batch == 1:
            self.split = 0
        self.kinds = (FEW if self.split > 0 else 0) | (0 if few else MANY)
        self.TR = 32 * self.waves // G
        units = Hkv * seqs if self.kinds & FEW else 0
        if self.kinds & MANY:
            units += Hkv * (total_q // self.TR + seqs)
        wgs = math.ceil(units * (page * total_pages + COST) / MIN_KEYS)
        self.wgs = -(-wgs // 8) * 8 if wgs < resident else resident
        if self.kinds == FEW | MANY:
            self.wgs = max(self.wgs, 16)
        o = 32 * D * 4
        self.bytes = {FEW: o // (2 if rows > 32 else 4) + 512, MANY: o + 512}  # of a wave in a slot
        self.many_counter = self.wgs * self.waves if self.kinds & FEW else 0
        self.many_partial = 2 * self.wgs * self.waves * self.bytes[FEW] if self.kinds & FEW else 0
        self.counters, self.partial_bytes = self.many_counter, self.many_partial
        if self.kinds & MANY:
            self.counters += self.wgs * self.waves
            self.partial_bytes += 2 * self.wgs * self.waves * self.bytes[MANY]


class Axis:
    """The units of one kind, and the ranges that W workgroups cut the axis into."""

    def __init__(self, plan, kind, W, seqs, Hkv, causal):
        self.p, self.kind, self.W, self.Hkv, self.causal = plan, kind, W, Hkv, causal
        mine = lambda n: n > 0 and (n <= plan.split) == (kind == FEW)  # noqa: E731
        self.seqs = [(b, n, length) for b, (n, length) in enumerate(seqs) if mine(n)]
        self.starts = list(itertools.accumulate((self.head(n, m) * Hkv for _, n, m in self.seqs),
                                                initial=0))
        total = self.total = self.starts[-1]
        self.team = 4 if kind == FEW else plan.waves
        teams = plan.waves // self.team
        few_units = kind == FEW and sum(self.head(n, m) > 0 for _, n, m in self.seqs) * Hkv <= W // 8
        self.Lw = max(-(-total // (W if few_units else W * teams)), MIN_KEYS)
        self.ranges = W * teams

    def blocks(self, n):
        return -(-n // self.p.TR)

    def unit_start(self, n, m, r):
        if not self.causal:
            return r * (m + COST)
        return r * (max(m - n, 0) + COST) + self.p.TR * (r * (r + 1) // 2)

    def head(self, n, m):
        R = self.blocks(n)
        if not self.causal:
            return R * (m + COST)
        return self.unit_start(n, m, R - 1) + max(m - n, 0) + n + COST

    def kend(self, n, m, r):
        if not self.causal:
            return m
        t0 = r * self.p.TR
        return max(m - n + t0 + min(self.p.TR, n - t0), 0)

    def div(self, a):
        """As the device divides: in doubles."""
        q = int(float(a) / float(self.Lw))
        assert q == a // self.Lw
        return q

    def parts(self, x):
        """What range x does, in its order: (sequence, kv head, row block, first key, last + 1)."""
        x0 = x * self.Lw
        if x0 >= self.total:
            return []
        x1 = min(x0 + self.Lw, self.total)
        out, last = [], None
        for at in (x1 - 1, x0):
            i = bisect.bisect_right(self.starts, at) - 1
            b, n, m = self.seqs[i]
            U, hlen = self.starts[i], self.head(n, m)
            kvh = (at - U) // hlen
            hs = U + kvh * hlen
            r = max(q for q in range(self.blocks(n)) if self.unit_start(n, m, q) <= at - hs)
            while (i, kvh, r) != last:
                us, kend = hs + self.unit_start(n, m, r), self.kend(n, m, r)
                k0, k1 = (kend if y - us >= kend + BLOCK else 0 if y - us < BLOCK
                          else min((y - us) // BLOCK * BLOCK, kend) for y in (x0, x1))
                if kend == 0:
                    if x0 - us < BLOCK <= x1 - us:
                        out.append((b, kvh, r, 0, 0, us))
                elif k0 < k1:
                    out.append((b, kvh, r, k0, k1, us))
                if at == x1 - 1:
                    if us <= x0:
                        return out
                    last = (i, kvh, r)
                    break
                r += 1
                if r < self.blocks(n):
                    continue
                r, hs, kvh = 0, hs + hlen, kvh + 1
                if kvh < self.Hkv:
                    continue
                kvh, i = 0, i + 1
                if i == len(self.seqs):
                    return out
                b, n, m = self.seqs[i]
                assert hs == self.starts[i]
                hlen = self.head(n, m)
        return out

    def check(self):
        p, served, slots, counters = self.p, {}, set(), {}
        base = 0 if self.kind == FEW else p.many_counter
        counter_end = p.many_counter if self.kind == FEW else p.counters
        slot_bytes = self.team * p.bytes[self.kind]
        region = (0, p.many_partial) if self.kind == FEW else (p.many_partial, p.partial_bytes)
        for x in range(self.ranges):
            for b, kvh, r, k0, k1, us in self.parts(x):
                served.setdefault((b, kvh, r), []).append((k0, k1, x))
                n, m = next(s[1:] for s in self.seqs[bisect.bisect_left(self.seqs, (b,)):])
                kend = self.kend(n, m, r)
                if (k0, k1) == (0, kend):
                    continue
                wf = self.div(us + BLOCK - 1)
                wl = self.div(us + (kend - 1) // BLOCK * BLOCK + BLOCK - 1)
                assert wf <= x <= wl
                slot = 2 * x + (x == wf)
                assert slot not in slots
                slots.add(slot)
                assert region[0] + (slot + 1) * slot_bytes <= region[1]
                for w in range(self.team):
                    assert base <= base + self.team * wf + w < counter_end
                counters.setdefault(wf, []).append((b, kvh, r, wl - wf + 1))
        for wf, arrivals in counters.items():  # one unit to a counter, as many as it waits for
            assert len(set(arrivals)) == 1 and len(arrivals) == arrivals[0][3]
        for b, n, m in self.seqs:
            for kvh in range(self.Hkv):
                for r in range(self.blocks(n)):
                    got = sorted(served.pop((b, kvh, r)))
                    kend = self.kend(n, m, r)
                    assert got[0][0] == 0 and got[-1][1] == kend
                    assert all(a[1] == c[0] and a[2] + 1 == c[2] for a, c in zip(got, got[1:]))
        assert not served


def check(seqs, Hkv, G, D, page, causal, shares=()):
    """seqs: (new tokens, cached tokens) of each sequence."""
    total_q = sum(n for n, _ in seqs)
    pages = sum(-(-m // page) for _, m in seqs)
    plan = Plan(len(seqs), total_q, Hkv, G, D, page, pages)
    size = N.load().akt_chunk_paged_workspace_size(len(seqs), total_q, Hkv * G, Hkv, D, page, pages)
    assert size == -(-ZERO // 256) * 256 + plan.partial_bytes
    assert 4 * plan.counters <= ZERO - 256 and plan.wgs % 8 == 0
    assert all(n <= plan.split for n, _ in seqs) or plan.kinds & MANY
    if plan.kinds != FEW | MANY:
        shares = (plan.wgs if plan.kinds == FEW else 0,)
    else:  # a kind without sequences leaves the other all workgroups
        few = any(0 < n <= plan.split for n, _ in seqs)
        many = any(n > plan.split for n, _ in seqs)
        if not (few and many):
            shares = (plan.wgs if not many else 0,)
        else:
            shares = {min(max(8, s // 8 * 8), plan.wgs - 8) for s in (8, plan.wgs, *shares)}
    for S in shares:
        if S:
            Axis(plan, FEW, S, seqs, Hkv, causal).check()
        if S < plan.wgs:
            Axis(plan, MANY, plan.wgs - S, seqs, Hkv, causal).check()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("seed", range(40))
def test_random_batches(D, seed):
    rng = random.Random(1000 * D + seed)
    log = lambda lo, hi: round(math.exp(rng.uniform(math.log(lo), math.log(hi))))  # noqa: E731
    B = log(1, 90)
    most_new, most_ctx = log(1, 3000 // max(B // 8, 1)), log(1, 40000)
    seqs = []
    for _ in range(B):
        n = rng.choice([0, 1, 1, rng.randint(1, 9), rng.randint(0, most_new)])
        m = n + rng.choice([0, rng.randint(0, most_ctx)])
        if rng.random() < 0.05:
            m = rng.randint(0, n)  # a table with fewer tokens than new ones
        seqs.append((n, m))
    if not any(n for n, _ in seqs):
        seqs[0] = (1, 1)
    check(seqs, rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8, 16, 33, 64, 128]), D,
          rng.choice([1, 7, 16, 24, 64, 128]), rng.random() < 0.7, (rng.randint(8, 248),))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_edges(D, causal):
    """Single sequences and pairs whose lengths sit on both sides of blocks, ranges and units."""
    for m in (1, 127, 128, 129, 255, 256, 257, 383, 384, 385, 2 ** 15 - 1, 2 ** 15, 2 ** 15 + 1):
        for n in (1, 8, 9, 16, 17, 64, 65, 128, 300):
            check([(n, m + n)], 2, 4, D, 16, causal)
        check([(1, m + 1), (100, m + 100)], 2, 4, D, 16, causal, (64, 128))
        check([(1, m + 1)] * 9 + [(0, m)] * 3, 8, 1, D, 16, causal)


@pytest.mark.parametrize("causal", [True, False])
def test_far_axes(causal):
    """The longest tables that a call takes: quotients in doubles stay exact."""
    check([(1, 2 ** 29), (700, 2 ** 28), (3, 2 ** 27)], 8, 4, 128, 1 << 19, causal)
    check([(5000, 2 ** 30 - 2 ** 19)], 8, 16, 64, 1 << 19, causal)


def test_divisions_by_multiplication():
    """A row's token (rows below 256) and a key's page."""
    for G in range(1, 129):
        magic = (65536 + G - 1) // G
        assert all(n * magic >> 16 == n // G for n in range(256))
    rng = random.Random(1)
    for page in [1, 2, 3, 5, 7, 16, 24, 48, 100, 1000, 4096, (1 << 20) - 1] + rng.sample(range(1, 1 << 20), 200):
        magic = min(2 ** 32 // page, 2 ** 32 - 1)
        near = [k * page + d for k in (0, 1, 2, (2 ** 30) // page - 1) for d in (-1, 0, 1)]
        for n in [v for v in near if v >= 0] + [rng.randrange(2 ** 30) for _ in range(100)] + [2 ** 31 - 1]:
            q = n * magic >> 32
            q += n - q * page >= page
            assert q == n // page, (n, page)
