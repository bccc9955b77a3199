"""The division of work of shared-prefix attention (csrc/paged_chunk.hip with csrc/paged_shared_few.hpp)
and of the sums of attention weight (csrc/attention_weights.hip), restated on the host.

For random batches: every key of every unit is served once, the parts of a cut unit lie in the slots
that are read for it, slots and counters are used once and lie inside the workspace, whose size is
the library's own; blocks of rows that a tile of the sums leaves out see none of its keys.
"""
import math
import random
import re
from pathlib import Path

import pytest

from attention_kernel_triton_amd import _native as N

CSRC = Path(__file__).resolve().parent.parent / "attention_kernel_triton_amd" / "csrc"
ZERO = -(-N.WORKSPACE_ZERO_BYTES // 256) * 256


def _constants(*files):
    text = "".join((CSRC / f).read_text() for f in files)
    return {m[0]: int(m[1]) for m in re.findall(r"\b(k\w+) = (\d+)[;,]", text)}


CK = _constants("paged_chunk.hpp", "paged_chunk.hip")
WT = _constants("attention_weights.hip")


def _div(a, b):
    """As the device divides: in doubles."""
    q = int(float(a) / float(b))
    assert q == a // b
    return q


def _log(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


# ---- shared prefixes.

class Shared:
    """What the host computes from the sizes (without a device: 256 CUs)."""

    def __init__(self, batch, total_q, Hkv, G, D, page, total_pages, groups, prefix_pages):
        self.waves = 8 if D <= 128 else 4
        resident = -(-256 * (2 if D <= 128 else 1) * 4 // self.waves // 8) * 8
        seqs, self.split = min(batch, total_q) + min(groups, total_q), 32 // G
        few = total_q <= self.split
        if not few and batch == 1:
            self.split = 0
        self.few, self.many = self.split > 0, not few
        self.TR = 32 * self.waves // G
        units = Hkv * seqs * self.few + Hkv * (2 * total_q // self.TR + seqs) * self.many
        wgs = math.ceil(units * (page * (total_pages + prefix_pages) + CK["kCkUnitCost"]) / CK["kCkMinKeys"])
        self.wgs = -(-wgs // 8) * 8 if wgs < resident else resident
        if self.few and self.many:
            self.wgs = max(self.wgs, 16)
        self.ranges = self.wgs * self.waves
        self.state = 16 + 4 * D
        self.many_partial = 2 * self.ranges * 32 * self.state * self.few
        # A workgroup's slot of many rows holds a state of each of them.
        self.partial = self.many_partial + 2 * self.wgs * 32 * self.waves * self.state * self.many


def _check_parts(units, axis, ranges, block, slot_bytes, region):
    """units: (start, keys, end); each is cut at multiples of `block` by the ranges of `axis` keys."""
    slots, total = set(), units[-1][2]
    for start, keys, end in units:
        assert end - start >= keys + block  # its last block, too, lies before its end
        cut = lambda d: keys if d >= keys + block else 0 if d < block else min(d // block * block, keys)  # noqa: E731
        got = []
        for x in range(start // axis, min(ranges - 1, (end - 1) // axis) + 1):
            x0, x1 = x * axis, min((x + 1) * axis, total)
            k0, k1 = cut(x0 - start), cut(x1 - start)
            if k0 < k1 or (keys == 0 and x0 - start < block <= x1 - start):
                got.append((k0, k1, x))
        if keys == 0:
            assert len(got) == 1
            continue
        assert got[0][0] == 0 and got[-1][1] == keys
        assert all(a[1] == c[0] and a[2] + 1 == c[2] for a, c in zip(got, got[1:]))
        if len(got) == 1:
            continue
        wf = _div(start + block - 1, axis)
        wl = _div(start + (keys - 1) // block * block + block - 1, axis)
        assert (got[0][2], got[-1][2]) == (wf, wl)
        for _, _, x in got:
            slot = 2 * x + (x == wf)
            assert slot not in slots
            slots.add(slot)
            assert region[0] + (slot + 1) * slot_bytes <= region[1]
    assert total <= ranges * axis


def check_shared(seqs, groups, Hkv, G, D, page, causal, shares=()):
    """seqs: (new tokens, own keys) of each sequence; groups: (sequences, prefix keys), in order."""
    total_q = sum(n for n, _ in seqs)
    pages, prefix_pages = (sum(-(-m // page) for _, m in side) for side in (seqs, groups))
    plan = Shared(len(seqs), total_q, Hkv, G, D, page, pages, len(groups), prefix_pages)
    size = N.load().akt_shared_prefix_paged_workspace_size(
        len(seqs), total_q, Hkv * G, Hkv, D, page, pages, len(groups), prefix_pages)
    assert size == ZERO + plan.partial + 2 * total_q * Hkv * G * plan.state
    served, at = [], 0
    for n, m in seqs:
        served.append((n, m, causal))
    for count, m in groups:
        served.append((sum(n for n, _ in seqs[at:at + count]), m, False))
        at += count
    few = [s for s in served if 0 < s[0] <= plan.split]
    many = [s for s in served if s[0] > plan.split]
    assert plan.few or not few
    assert plan.many or not many
    if few and many:
        shares = {min(max(8, s // 8 * 8), plan.wgs - 8) for s in (8, plan.wgs, *shares)}
    else:
        shares = (plan.wgs if few else 0,)
    for S in shares:
        if few:
            units, x = [], 0
            for n, m, _ in few:
                for _ in range(Hkv):
                    units.append((x, m, x + m + CK["kWaveUnitCost"]))
                    x += m + CK["kWaveUnitCost"]
            axis = max(-(-x // (S * plan.waves)), CK["kCkWaveKeys"])
            # A wave's range: each is some wave's.
            mine = sorted(w * S + (b % 8) * (S // 8) + b // 8 for w in range(plan.waves) for b in range(S))
            assert mine == list(range(S * plan.waves))
            _check_parts(units, axis, S * plan.waves, CK["kCkWaveBlock"], 32 * plan.state,
                         (0, plan.many_partial))
        W = plan.wgs - S
        if many and W:
            units, x, cost = [], 0, CK["kSharedUnitCost"]
            for n, m, c in many:
                for _ in range(Hkv):
                    for t in range(0, n, plan.TR):
                        keys = max(m - n + min(t + plan.TR, n), 0) if c else m
                        # (Axis lengths are of a full block's limit, and never below what is served.)
                        length = (max(m - n, 0) + min(t + plan.TR, n) if c else m) + cost
                        units.append((x, keys, x + length))
                        x += length
            axis = max(-(-x // W), CK["kCkMinKeys"])
            _check_parts(units, axis, W, CK["kCkBlock"], 32 * plan.waves * plan.state,
                         (plan.many_partial, plan.partial))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("seed", range(30))
def test_shared_prefix_batches(D, seed):
    rng = random.Random(7000 * D + seed)
    seqs, groups = [], []
    most_new = _log(rng, 1, 400)
    for _ in range(_log(rng, 1, 12)):
        count = rng.choice([0, 1, 2, rng.randint(1, 20)])
        groups.append((count, rng.choice([0, 1, _log(rng, 1, 30000)])))
        for _ in range(count):
            n = rng.choice([0, 1, 1, rng.randint(1, 9), rng.randint(0, most_new)])
            seqs.append((n, rng.choice([n, n + _log(rng, 1, 3000), rng.randint(0, n)])))
    seqs += [(1, rng.randint(0, 500))] * rng.choice([0, 1, 5])
    if not any(n for n, _ in seqs):
        seqs.append((1, 1))
    check_shared(seqs, groups, rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8, 16, 33, 64]), D,
                 rng.choice([1, 7, 16, 24, 128]), rng.random() < 0.6, (rng.randint(8, 248),))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_shared_prefix_edges(D):
    for m in (1, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 2 ** 14 + 1):
        for n in (1, 4, 8, 9, 33, 64, 65):
            check_shared([(n, n)] * 3, [(2, m)], 2, 4, D, 16, True)
            check_shared([(n, m + n)], [(1, m)], 1, 4, D, 16, False, (64,))
    check_shared([(1, 2 ** 28), (1, 3), (200, 2 ** 27)], [(3, 2 ** 29)], 8, 4, D, 1 << 19, True, (64,))


# ---- sums of attention weight.

class Head:
    """The tiles of one (sequence, kv head)."""

    def __init__(self, n, m, G, causal):
        tile = WT["kWKeys"] * WT["kWWaves"]
        self.rows = -(-n * G // 32)
        self.full = self.rows + WT["kWTileCost"]
        self.tiles = -(-m // tile) if n else 0
        first = m - n
        self.t0 = self.tiles if not causal else 0 if first < 0 else min(first // tile + 1, self.tiles)
        self.f0 = max(self.t0 * tile - first, 0) * G // 32
        self.step, self.diag = tile // 32 * G, WT["kWDiagCost"] * G

    def skipped(self, t):
        return 0 if t < self.t0 else self.f0 + (t - self.t0) * self.step

    def start(self, t):
        i = max(t - self.t0, 0)
        return t * self.full - i * self.f0 - i * (i - 1) // 2 * self.step + i * self.diag

    def length(self, t):
        return self.full - self.skipped(t) + (self.diag if t >= self.t0 else 0)


@pytest.mark.parametrize("causal", [True, False])
def test_tiles_of_the_sums(causal):
    """Tiles begin where the ones before end; every row that sees a key of a tile is in its blocks."""
    tile = WT["kWKeys"] * WT["kWWaves"]
    rng = random.Random(5)
    for _ in range(400):
        G, n = rng.choice([1, 2, 3, 4, 7, 8, 16, 64, 128]), _log(rng, 1, 4000)
        m = rng.choice([n, rng.randint(0, n), n + _log(rng, 1, 5000), tile * rng.randint(0, 9)])
        if n * G <= WT["kWFew"]:
            continue
        h, at = Head(n, m, G, causal), 0
        for t in range(h.tiles):
            assert h.start(t) == at
            at += h.length(t)
            blocks = h.rows - h.skipped(t)
            assert h.length(t) >= blocks + WT["kWTileCost"] >= WT["kWTileCost"] + 1
            if causal:  # row r is token r / G, at position m - n + r / G
                rows = 32 * h.skipped(t)
                assert rows == 0 or m - n + (rows - 1) // G < t * tile
        assert h.start(h.tiles) == at


def check_weights(seqs, Hkv, G, D, page, causal, shares=()):
    total_q = sum(n for n, _ in seqs)
    pages = sum(-(-m // page) for _, m in seqs)
    tile, cost, diag = WT["kWKeys"] * WT["kWWaves"], WT["kWTileCost"], WT["kWDiagCost"]
    resident = 256 * (2 if D <= 128 else 1)
    tiles = (page * pages // tile + len(seqs)) * Hkv
    wgs = math.ceil(tiles * (total_q * G // 32 + 1 + cost + diag * G) / (cost + 1)) + 16
    wgs = -(-wgs // 8) * 8 if wgs < resident else resident
    size = N.load().akt_attention_weights_paged_workspace_size(len(seqs), total_q, Hkv * G, Hkv, D, page, pages)
    assert size == ZERO + 2 * wgs * tile * 4 and 4 * wgs <= N.WORKSPACE_ZERO_BYTES - 256
    few = [s for s in seqs if 0 < s[0] * G <= WT["kWFew"]]
    many = [s for s in seqs if s[0] * G > WT["kWFew"]]
    if few and many:
        shares = {min(max(8, s // 8 * 8), wgs - 8) for s in (8, wgs, *shares)}
    else:
        shares = (wgs if few else 0,)
    keys = 64 if D == 64 else 32
    for S in shares:
        if few:  # steps of a unit, each once
            units = [(-(-m // keys)) for n, m in few if m for _ in range(Hkv)]
            total = sum(u + 1 for u in units)
            axis = -(-total // (S * 4))
            at = 0
            for u in units:
                got = []
                for x in range(at // axis if axis else 0, (at + u) // axis + 1 if axis else 0):
                    j0, j1 = min(max(x * axis - at, 0), u), min(min((x + 1) * axis, total) - at, u)
                    if j0 < j1:
                        got.append((j0, j1))
                assert got[0][0] == 0 and got[-1][1] == u and x < S * 4
                assert all(a[1] == c[0] for a, c in zip(got, got[1:]))
                at += u + 1
        W = wgs - S
        heads = [h for h in (Head(n, m, G, causal) for n, m in many) if h.tiles]
        if not heads or not W:
            continue
        total = Hkv * sum(h.start(h.tiles) for h in heads)
        axis = max(-(-total // W), cost + 1)
        assert total <= axis * W
        at, slots, counters = 0, set(), set()
        for h in heads:
            for _ in range(Hkv):
                for t in range(h.tiles):
                    start, blocks = at + h.start(t), h.rows - h.skipped(t)
                    wf, wl = _div(start, axis), _div(start + blocks - 1, axis)
                    got = []
                    for x in range(wf, (start + h.length(t) - 1) // axis + 1):
                        j0 = min(max(x * axis - start, 0), blocks)
                        j1 = min(min((x + 1) * axis, total) - start, blocks)
                        if j0 < j1:
                            got.append((j0, j1, x))
                    assert got[0][0] == 0 and got[-1][1] == blocks
                    assert all(a[1] == c[0] for a, c in zip(got, got[1:]))
                    assert [x for _, _, x in got] == list(range(wf, wl + 1)) and wl < W
                    if len(got) > 1:
                        assert wf not in counters
                        counters.add(wf)
                        for x in range(wf, wl + 1):
                            slot = 2 * x + (x == wf)
                            assert slot not in slots and slot < 2 * wgs
                            slots.add(slot)
                at += h.start(h.tiles)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("seed", range(30))
def test_batches_of_the_sums(D, seed):
    rng = random.Random(9000 * D + seed)
    most_new, most_ctx, seqs = _log(rng, 1, 2000), _log(rng, 1, 20000), []
    for _ in range(_log(rng, 1, 40)):
        n = rng.choice([0, 1, 1, rng.randint(1, 9), rng.randint(0, most_new)])
        seqs.append((n, rng.choice([n, n + rng.randint(0, most_ctx), rng.randint(0, n)])))
    if not any(n for n, _ in seqs):
        seqs[0] = (1, 1)
    if not any(m for _, m in seqs):
        seqs[0] = (1, 1)
    check_weights(seqs, rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8, 16, 33, 64, 128]), D,
                  rng.choice([1, 7, 16, 24, 128]), rng.random() < 0.7, (rng.randint(8, 504),))
