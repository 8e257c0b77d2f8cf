"""The paged cache's plan, rope + append and decode attention on the GPU against their definitions in
64 bits on the host.

Tolerances, from the roundings on the way (u = 2^-24, half a step of f32):
- plan: whole numbers, equal.
- q_out: x0 cos - x1 sin with cos and sin good to 4 u, the angle rounded to f32 (pi u) and three
  roundings of the products and the sum: 12 u (|x0| + |x1|) magnitude.
- cache rows: half a step of f16 (2^-11 of the value, 2^-25 below its normal range) on top of that; v,
  which nothing precedes, is numpy's rounding to f16 bit for bit.
- attention, as a 2-norm over an output: a score's own error is about sqrt(head_dim) / 3 roundings of
  its partial sums (some 4 u of its size, up to 10 in magnitude) and one of its argument of exp2, so a
  weight is off by 5e-7 to 2e-6, independently from key to key; the weighted sum of values, whose signs
  are mixed, is off by the same share. 4e-6 for all. (Operands rounded to 11 bits, f16's, would give
  1e-4.)
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ATTENTION_RTOL = 4e-6


def dev(torch, array):
    return torch.from_numpy(np.ascontiguousarray(array)).cuda()


def host(t):
    return t.detach().cpu().numpy()


def stream(torch):
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------------------------------------
# Plan


def plan_reference(lengths, targets, tables, ring, pool, page_size, tokens):
    """The plan, one sequence after another."""
    tables, ring = tables.copy(), ring.copy()
    pages, width = len(ring), tables.shape[1]
    before, sound = ring.copy(), 0 <= pool[0] < pages and 0 <= pool[1] <= pages
    head, free = (int(pool[0]), int(pool[1])) if sound else (0, 0)
    cap = width * page_size
    granted, starts, listed, back = [], [0], [], []
    asked = needed = used = 0
    for b, (length, target) in enumerate(zip(lengths.tolist(), targets.tolist())):
        valid = 0 <= length <= cap and 0 <= target <= cap
        have, want = -(-length // page_size), -(-target // page_size)
        asked += max(0, target - length) if valid else 0
        fits = valid and asked <= tokens
        need = max(0, want - have) if fits else 0
        needed += need
        if not (fits and (need == 0 or needed <= free)):
            granted.append(length)
            starts.append(starts[-1])
            continue
        for j in range(need):
            tables[b, have + j] = before[(head + used + j) % pages]
        used += need
        back += tables[b, want:have].tolist() if want < have else []
        for pos in range(length, target):
            page = int(tables[b, pos // page_size])
            listed.append((b, pos, page * page_size + pos % page_size if 0 <= page < pages else -1))
        granted.append(target)
        starts.append(starts[-1] + max(0, target - length))
    back = back[:pages - free] if sound else []
    for i, page in enumerate(back):
        ring[(head + free + i) % pages] = page
    listed += [(-1, -1, -1)] * (tokens - len(listed))
    new_pool = [(head + used) % pages, free - used + len(back)] if sound else [int(v) for v in pool]
    return dict(tables=tables, free_pages=ring, granted=np.array(granted), pool_out=np.array(new_pool),
                starts=np.array(starts), lists=np.array(listed).reshape(tokens, 3).T)


def run_plan(mh, torch, lengths, targets, tables, ring, pool, page_size, tokens, in_place=False, times=1):
    d = {k: dev(torch, v.astype(np.int32)) for k, v in dict(lengths=lengths, targets=targets, tables=tables,
                                                            free_pages=ring, pool=np.asarray(pool)).items()}
    n, guard = len(lengths), 7
    starts = torch.full((n + 1 + guard,), 77, dtype=torch.int32, device="cuda")
    granted = d["lengths"] if in_place else torch.full((n + guard,), 77, dtype=torch.int32, device="cuda")
    pool_out = d["pool"] if in_place else torch.full((2 + guard,), 77, dtype=torch.int32, device="cuda")
    lists = torch.full((3, tokens + guard), 77, dtype=torch.int32, device="cuda")
    for _ in range(times):
        mh.check(mh.load().muyo_paged_plan(
            d["lengths"].data_ptr(), d["targets"].data_ptr(), n, d["tables"].data_ptr(), tables.shape[1],
            d["free_pages"].data_ptr(), d["pool"].data_ptr(), len(ring), page_size, tokens, granted.data_ptr(),
            pool_out.data_ptr(), starts.data_ptr(), lists[0].data_ptr(), lists[1].data_ptr(), lists[2].data_ptr(),
            stream(torch)))
    torch.cuda.synchronize()
    for t, used in ((starts, n + 1), (lists[0], tokens), (lists[1], tokens), (lists[2], tokens)):
        assert (host(t)[used:] == 77).all()
    if not in_place:
        assert (host(granted)[n:] == 77).all() and (host(pool_out)[2:] == 77).all()
    return dict(tables=host(d["tables"]), free_pages=host(d["free_pages"]), granted=host(granted)[:n],
                pool_out=host(pool_out)[:2], starts=host(starts)[:n + 1], lists=host(lists)[:, :tokens])


def plan_state(rng, lengths, width, page_size, spare):
    """Tables that hold the lengths with distinct pages, and a ring of `spare` others."""
    have = [-(-max(0, int(n)) // page_size) for n in lengths]
    pages = sum(have) + spare
    ids = rng.permutation(pages)
    tables, at = np.full((len(lengths), width), -1), 0
    for b, n in enumerate(have):
        tables[b, :n] = ids[at:at + n]
        at += n
    head = int(rng.integers(pages))
    ring = np.full(pages, -1)
    ring[(head + np.arange(spare)) % pages] = ids[at:]
    return tables, ring, [head, spare]


PLANS = [
    # sequences, longest, page_size, prompts' share, ended share, spare pages (of those needed), list room
    ("one_first_token", 1, 0, 16, 1.0, 0.0, 1.0, 1),
    ("one_step", 1, 33, 16, 0.0, 0.0, 1.0, 1),
    ("one_ends", 1, 300, 16, 0.0, 1.0, 1.0, 0),
    ("step_64", 64, 500, 16, 0.0, 0.0, 1.0, 64),
    ("step_255", 255, 100, 32, 0.0, 0.1, 1.0, 300),
    ("mixed_256", 256, 400, 16, 0.3, 0.2, 1.0, 100000),
    ("mixed_257", 257, 400, 64, 0.3, 0.2, 1.0, 100000),
    ("scarce_pages", 100, 300, 16, 0.4, 0.1, 0.5, 100000),
    ("scarce_room", 100, 300, 16, 0.4, 0.1, 1.0, 2000),
    ("no_pages", 40, 200, 16, 0.2, 0.2, 0.0, 100000),
    ("middle_1024", 1024, 60, 16, 0.2, 0.1, 0.9, 30000),
    ("middle_1025", 1025, 60, 16, 0.2, 0.1, 1.0, 30000),
    ("many_4096", 4096, 40, 16, 0.1, 0.1, 0.9, 30000),
    ("page_1024", 9, 5000, 1024, 0.3, 0.0, 1.0, 50000),
]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", PLANS, ids=[c[0] for c in PLANS])
def test_plan_matches_definition(mh, gpu, case, in_place):
    _, n, longest, page_size, new, done, share, room = case
    rng = np.random.default_rng(n * 7 + page_size)
    lengths = rng.integers(1, longest + 1, n) if longest else np.zeros(n, int)
    targets = lengths + 1
    kind = rng.random(n)
    prompts = kind < new
    lengths[prompts] = 0
    targets[prompts] = rng.integers(1, max(2, longest), prompts.sum())
    targets[(kind >= new) & (kind < new + done)] = 0
    width = -(-(longest + 2) // page_size) + 1
    need = np.maximum(0, -(-targets // page_size) - -(-lengths // page_size)).sum()
    tables, ring, pool = plan_state(rng, lengths, width, page_size, max(1, int(need * share)))
    want = plan_reference(lengths, targets, tables, ring, pool, page_size, room)
    got = run_plan(mh, gpu, lengths, targets, tables, ring, pool, page_size, room, in_place)
    for key in want:
        assert np.array_equal(got[key], want[key]), key


def test_plan_leaves_bad_requests_as_they_are(mh, gpu):
    """Negative lengths and targets, targets past the table, page ids outside the cache, and a pool that
    is none: no page, no token, nothing read or written out of range."""
    rng = np.random.default_rng(5)
    lengths = np.array([5, -1, 17, 40, 16, 2 ** 31 - 1, 0, 12, 64])
    targets = np.array([-3, 9, 65, 41, 17, 4, 2 ** 31 - 1, 0, 3])
    tables, ring, pool = plan_state(rng, np.minimum(lengths, 64), 4, 16, 6)
    tables[3, 2] = -7  # the page of sequence 3's next token
    for p in (pool, [-1, 3], [0, -1], [len(ring), 0], [0, len(ring) + 1], [2 ** 31 - 1, 2 ** 31 - 1]):
        want = plan_reference(lengths, targets, tables, ring, p, 16, 50)
        got = run_plan(mh, gpu, lengths, targets, tables, ring, p, 16, 50)
        for key in want:
            assert np.array_equal(got[key], want[key]), (p, key)
    assert want["lists"][2][0] == -1  # the token is listed, without a slot


def test_plan_life_of_a_batch(mh, gpu):
    """Fifty steps in place: sequences come, grow, shrink and end; every page is always in exactly one
    table row's live part or in the ring."""
    torch, rng = gpu, np.random.default_rng(11)
    n, width, size, pages = 33, 20, 16, 150
    lengths = np.zeros(n, np.int64)
    tables, ring, pool = np.full((n, width), -1), rng.permutation(pages), [0, pages]
    refused = 0
    for step in range(50):
        targets = lengths + 1
        chance = rng.random(n)
        targets[chance < 0.1] = 0
        shrink = (chance > 0.9) & (lengths > 3)
        targets[shrink] = lengths[shrink] - 3
        empty = lengths == 0
        targets[empty] = rng.integers(0, 120, empty.sum())
        got = run_plan(mh, torch, lengths, targets, tables, ring, pool, size, 700, in_place=True)
        want = plan_reference(lengths, targets, tables, ring, pool, size, 700)
        for key in want:
            assert np.array_equal(got[key], want[key]), (step, key)
        refused += int((got["granted"] != targets).sum())
        lengths, tables, ring, pool = got["granted"], got["tables"], got["free_pages"], got["pool_out"].tolist()
        held = [p for b in range(n) for p in tables[b, :-(-int(lengths[b]) // size)]]
        free = [ring[(pool[0] + i) % pages] for i in range(pool[1])]
        assert sorted(held + free) == list(range(pages)), step
    assert refused > 0


# ------------------------------------------------------------------------------------------------
# Rope and append


def rotate64(x, positions, turns, magnitude, layout, rotary):
    """x [tokens][heads][hd] rotated, and the bound 12 u (|x0| + |x1|) of each value."""
    x = x.astype(np.float64)
    angle = 2 * np.pi * np.mod(positions.astype(np.float64)[:, None] * turns, 1.0)
    c, s = np.cos(angle)[:, None] * magnitude, np.sin(angle)[:, None] * magnitude
    first = np.arange(rotary // 2) * (1 if layout == 0 else 2)
    second = first + (rotary // 2 if layout == 0 else 1)
    y, bound = x.copy(), np.zeros_like(x)
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., first] * s + x[..., second] * c
    bound[..., first] = bound[..., second] = 12 * U * magnitude * (np.abs(x[..., first]) + np.abs(x[..., second]))
    return y, bound


APPENDS = [
    # heads, kv_heads, head_dim, page_size, layout, rotary, tokens, last position, stacked
    (14, 2, 64, 16, 0, 64, 1, 0, True),
    (14, 2, 64, 16, 0, 64, 37, 300, True),
    (28, 4, 128, 64, 0, 128, 19, 1000003, False),
    (28, 4, 128, 32, 1, 128, 65, 40000, True),
    (28, 4, 128, 16, 1, 64, 9, 500, False),
    (28, 4, 128, 16, 0, 64, 9, 500, True),
    (14, 2, 64, 16, 0, 24, 5, 77, True),      # pairs of 12: whole quads
    (14, 2, 64, 16, 0, 20, 5, 77, True),      # pairs of 10: not
    (14, 2, 64, 128, 1, 6, 5, 77, False),
    (3, 3, 8, 16, 0, 2, 11, 2 ** 31 - 1, True),
    (5, 1, 40, 1024, 1, 40, 300, 299, True),
    (1, 1, 256, 16, 0, 256, 2, 9, False),
    (33, 16, 64, 16, 0, 32, 1000, 8000, True),
]


@pytest.mark.parametrize("case", APPENDS, ids=["-".join(map(str, c)) for c in APPENDS])
def test_rope_append_matches_definition(mh, gpu, case):
    heads, kv, hd, size, layout, rotary, tokens, last, stacked = case
    torch, rng = gpu, np.random.default_rng(hd + tokens)
    pages = -(-tokens // size) + 3
    turns, magnitude = mh.rope_frequencies(1e4, rotary, "YARN", factor=2.0, trained_context=4096)
    qd, kd = heads * hd, kv * hd
    width = qd + 2 * kd + 4  # and a gap behind each row
    if stacked:
        rows = rng.normal(0, 2, (tokens, width)).astype(np.float32)
        parts = [rows[:, :qd], rows[:, qd:qd + kd], rows[:, qd + kd:qd + 2 * kd]]
        d = dev(torch, rows)
        views, strides = [d[:, :qd], d[:, qd:qd + kd], d[:, qd + kd:]], [width] * 3
    else:
        parts = [rng.normal(0, 2, (tokens, n)).astype(np.float32) for n in (qd, kd, kd)]
        views, strides = [dev(torch, p) for p in parts], [qd, kd, kd]
    positions = rng.integers(0, last + 1, tokens) if tokens > 1 else np.array([last])
    positions[-1] = last
    slots = rng.permutation(pages * size)[:tokens]
    if tokens > 4:
        positions[1], slots[1] = -1, -1   # padding
        slots[2] = pages * size           # not appended
        slots[3] = -5
    fill = rng.normal(0, 1, (2, pages, kv, size, hd)).astype(np.float16)
    caches = [dev(torch, fill[i]) for i in range(2)]
    q_out = torch.full((tokens, qd), 9.0, device="cuda")
    dp, ds, dt = dev(torch, positions.astype(np.int32)), dev(torch, slots.astype(np.int32)), dev(torch, turns)
    mh.check(mh.load().muyo_paged_rope_append_f16kv(
        *(v.data_ptr() for v in views), *strides, q_out.data_ptr(), caches[0].data_ptr(), caches[1].data_ptr(),
        dp.data_ptr(), ds.data_ptr(), tokens, heads, kv, hd, pages, size, layout, rotary, dt.data_ptr(), magnitude,
        stream(torch)))
    torch.cuda.synchronize()
    live = positions >= 0
    q, q_bound = rotate64(parts[0].reshape(tokens, heads, hd), positions, turns, magnitude, layout, rotary)
    got = host(q_out).reshape(tokens, heads, hd)
    assert (np.abs(got - q) <= q_bound)[live].all()
    assert (got[~live] == 9.0).all()
    k, k_bound = rotate64(parts[1].reshape(tokens, kv, hd), positions, turns, magnitude, layout, rotary)
    want, bound = fill.astype(np.float64), np.zeros(fill.shape)
    for t in np.flatnonzero(live & (slots >= 0) & (slots < pages * size)):
        at = (slots[t] // size, slice(None), slots[t] % size)
        want[0][at], want[1][at] = k[t], parts[2][t].reshape(kv, hd).astype(np.float16)
        bound[0][at] = k_bound[t] * (1 + 2.0 ** -11) + np.maximum(np.abs(k[t]) * 2.0 ** -11, 2.0 ** -25)
    for i in range(2):
        assert (np.abs(host(caches[i]).astype(np.float64) - want[i]) <= bound[i]).all(), "kv"[i]


def test_rope_append_in_place_and_equal_layouts(mh, gpu):
    """q_out may be q; and the two layouts are the same rotation of differently placed values."""
    torch, rng = gpu, np.random.default_rng(3)
    tokens, heads, kv, hd, size, pages = 7, 4, 2, 64, 16, 4
    turns, _ = mh.rope_frequencies(1e6, hd)
    dt, zero = dev(torch, turns), torch.zeros((tokens, kv * hd), device="cuda")
    positions, slots = (torch.arange(tokens, dtype=torch.int32, device="cuda") + n for n in (1000, 3))
    caches = torch.zeros((2, pages, kv, size, hd), dtype=torch.float16, device="cuda")
    q = rng.normal(0, 1, (tokens, heads, hd)).astype(np.float32)
    order = np.arange(hd).reshape(2, hd // 2).T.flatten()  # interleaved place -> half place
    out = {}
    for layout in (0, 1):
        d = dev(torch, q if layout == 0 else q[..., order])
        mh.check(mh.load().muyo_paged_rope_append_f16kv(
            d.data_ptr(), zero.data_ptr(), zero.data_ptr(), heads * hd, kv * hd, kv * hd, d.data_ptr(),
            caches[0].data_ptr(), caches[1].data_ptr(), positions.data_ptr(), slots.data_ptr(), tokens, heads, kv, hd,
            pages, size, layout, hd, dt.data_ptr(), 1.0, stream(torch)))
        torch.cuda.synchronize()
        out[layout] = host(d)
    assert np.array_equal(out[0][..., order], out[1])
    want, bound = rotate64(q, np.arange(tokens) + 1000, turns, 1.0, 0, hd)
    assert (np.abs(out[0] - want) <= bound).all()


# ------------------------------------------------------------------------------------------------
# Attention


def attend64(q, kcache, vcache, table, position, window, scale):
    """One query's heads [heads][hd] over its pages, in 64 bits."""
    pages, kv, size, hd = kcache.shape
    heads = q.shape[0]
    end = min(position + 1, len(table) * size)
    first = max(0, position + 1 - window) if window else 0
    keys = [j for j in range(first, end) if 0 <= table[j // size] < pages]
    out = np.zeros((heads, hd))
    if not keys:
        return out
    keys = np.array(keys)
    at = table[keys // size], slice(None), keys % size
    k, v = kcache[at].astype(np.float64), vcache[at].astype(np.float64)
    for h in range(heads):
        g = h // (heads // kv)
        s = k[:, g] @ q[h].astype(np.float64) * scale
        p = np.exp(s - s.max())
        out[h] = (p / p.sum()) @ v[:, g]
    return out


class Attend:
    """A batch on the device and its call."""

    def __init__(self, mh, torch, rng, heads, kv, hd, size, positions, width=None, sequence=None, q_std=2.0,
                 spare=3):
        self.mh, self.torch = mh, torch
        self.shape = heads, kv, hd, size
        n = len(positions)
        self.positions, self.sequence = np.asarray(positions), np.arange(n) if sequence is None else sequence
        rows = int(max(self.sequence.max(), 0)) + 1
        longest = np.zeros(rows, int)
        for s, p in zip(self.sequence, self.positions):
            if 0 <= s < rows:
                longest[s] = max(longest[s], p + 1)
        counts = -(-longest // size)
        self.width = width or max(1, int(counts.max()))
        self.pages = int(counts.sum()) + spare
        ids, at = rng.permutation(self.pages), 0
        self.tables = np.full((rows, self.width), -1)
        for b, c in enumerate(counts):
            c = min(c, self.width)
            self.tables[b, :c] = ids[at:at + c]
            at += c
        self.q = rng.normal(0, q_std, (n, heads, hd)).astype(np.float32)
        self.caches = rng.normal(0, 1, (2, self.pages, kv, size, hd)).astype(np.float16)
        self.scale = 1 / math.sqrt(hd)

    def poison_unseen(self, window=0):
        """NaN and infinities wherever no query looks."""
        size = self.shape[3]
        seen = np.zeros((self.pages, size), bool)
        for s, p in zip(self.sequence, self.positions):
            if s >= 0 and p >= 0:
                j = np.arange(max(0, p + 1 - window) if window else 0, min(p + 1, self.width * size))
                seen[self.tables[s, j // size], j % size] = True
        bad = ~seen
        for cache in self.caches:
            cache.transpose(0, 2, 1, 3)[bad] = np.resize(np.array([np.nan, np.inf, -np.inf], np.float16),
                                                         cache.transpose(0, 2, 1, 3)[bad].shape)

    def call(self, window=0, where=None, out=None):
        torch, lib = self.torch, self.mh.load()
        heads, kv, hd, size = self.shape
        if where is None:
            self.d = [dev(torch, self.q), dev(torch, self.caches[0]), dev(torch, self.caches[1]),
                      dev(torch, self.tables.astype(np.int32)), dev(torch, self.sequence.astype(np.int32)),
                      dev(torch, self.positions.astype(np.int32))]
            nbytes = lib.muyo_paged_attention_decode_f16kv_workspace_bytes(len(self.q), heads, kv, hd)
            self.space = torch.full((nbytes + 256,), 0x5A, dtype=torch.uint8, device="cuda")
            self.nbytes = nbytes
        if out is None:
            out = torch.full((len(self.q), heads, hd), 9.0, device="cuda")
        q, k, v, tables, sequence, positions = self.d
        self.mh.check(lib.muyo_paged_attention_decode_f16kv(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), tables.data_ptr(), self.tables.shape[0],
            self.width, sequence.data_ptr(), positions.data_ptr(), len(self.q), heads, kv, hd, self.pages, size,
            window, self.scale, self.space.data_ptr(), self.nbytes, stream(torch)))
        return out

    def check(self, window=0, rtol=ATTENTION_RTOL):
        out = self.call(window)
        self.torch.cuda.synchronize()
        assert (host(self.space)[self.nbytes:] == 0x5A).all()
        self.compare(host(out), window, rtol)
        return out

    def compare(self, got, window=0, rtol=ATTENTION_RTOL):
        for i, (s, p) in enumerate(zip(self.sequence, self.positions)):
            if not 0 <= s < len(self.tables):
                assert (got[i] == 9.0).all(), i
                continue
            want = attend64(self.q[i], self.caches[0], self.caches[1], self.tables[s], int(p), window, self.scale)
            assert np.isfinite(got[i]).all(), i
            assert np.linalg.norm(got[i] - want) <= rtol * np.linalg.norm(want), (i, p)


LAYOUTS = [(14, 2, 64), (28, 4, 128), (16, 1, 64), (16, 1, 128), (4, 4, 128), (6, 2, 64), (9, 3, 128), (1, 1, 64)]


@pytest.mark.parametrize("heads, kv, hd", LAYOUTS)
def test_attention_of_all_head_layouts(mh, gpu, heads, kv, hd):
    """Lengths around pages, tiles and their multiples, one call; everything unseen is poisoned."""
    rng = np.random.default_rng(heads * hd)
    positions = np.array([0, 1, 14, 15, 16, 17, 30, 31, 32, 33, 62, 63, 64, 65, 127, 128, 129, 255, 256, 300, 511, 1000])
    batch = Attend(mh, gpu, rng, heads, kv, hd, 16, rng.permutation(positions))
    batch.poison_unseen()
    batch.check()


@pytest.mark.parametrize("size", [16, 32, 64, 128, 256, 512, 1024])
@pytest.mark.parametrize("window", [0, 1, 31, 100, 5000])
def test_attention_pages_and_windows(mh, gpu, size, window):
    rng = np.random.default_rng(size + window)
    batch = Attend(mh, gpu, rng, 14, 2, 64, size, np.array([0, 5, 99, 100, 101, 1023, 1024, 1500, 2222, 40]))
    batch.poison_unseen(window)
    batch.check(window)


@pytest.mark.parametrize("hd, positions", [
    (128, [20000]), (64, [20011]), (64, [32767]), (128, [3000, 1, 9000, 0, 150]),
    (64, [700] * 200), (128, list(range(0, 640, 5))),
    (64, [2000, 5] * 512), (64, [0, 40, 1300, 7, -1] * 250), (128, [9] * 1500 + [4000]),
])
def test_attention_long_and_many(mh, gpu, hd, positions):
    rng = np.random.default_rng(len(positions))
    heads, kv = (14, 2) if hd == 64 else (28, 4)
    batch = Attend(mh, gpu, rng, heads, kv, hd, 64, np.array(positions))
    batch.poison_unseen()
    batch.check()


@pytest.mark.parametrize("queries", [1, 5, 64, 65, 256, 300])
@pytest.mark.parametrize("longest", [512, 513])
def test_attention_of_short_sequences_in_wide_tables(mh, gpu, queries, longest):
    """Tables of 4096 keys, sequences up to `longest`, padding among them, on either side of what is cut."""
    rng = np.random.default_rng(queries + longest)
    positions = rng.integers(0, longest, queries)
    positions[0] = longest - 1
    sequence = rng.permutation(queries)
    if queries > 4:
        sequence[3] = -1
    batch = Attend(mh, gpu, rng, 14, 2, 64, 16, positions, width=256, sequence=sequence)
    batch.poison_unseen()
    batch.check()


def test_attention_padding_empty_rows_and_bad_pages(mh, gpu):
    """Padding rows stay, rows without keys are 0, pages outside the cache and keys past the table are
    left out, and several queries may share a sequence."""
    rng = np.random.default_rng(9)
    sequence = np.array([0, -1, 1, 2, 99, 2, 3, 3, 3, 4, -2 ** 31])
    positions = np.array([40, 7, -1, 100, 3, 101, 300, 17, 0, 63, 5])
    batch = Attend(mh, gpu, rng, 14, 2, 64, 16, positions, sequence=np.minimum(sequence, 4))
    batch.sequence = sequence  # 99 and below 0 name no row
    batch.tables[3, [1, 5, 6, 18]] = [-1, batch.pages, 2 ** 31 - 1, -2 ** 31]
    batch.tables[4, :] = -1    # a sequence whose every page is missing
    batch.positions[9] = 63
    out = host(batch.check())
    assert (out[2] == 0).all() and (out[9] == 0).all() and not (out[8] == 0).any()


def test_attention_positions_past_the_table(mh, gpu):
    rng = np.random.default_rng(10)
    batch = Attend(mh, gpu, rng, 28, 4, 128, 16, np.array([63, 20, 62]), spare=0)
    batch.positions = np.array([2 ** 31 - 1, 20, 64])
    batch.check()
    batch.check(window=1)     # the window lies past the table: nothing seen
    batch.check(window=2 ** 31)


def test_attention_of_large_small_and_negative_scales(mh, gpu):
    """q far outside f16's range in either direction, one sharp key, equal scores, a negative and a zero
    scale."""
    rng = np.random.default_rng(12)
    for q_std, scale in ((1e6, 1e-7), (1e-6, 1e5), (1e-20, 1e19), (1e20, 1e-21), (0.0, 1.0), (30.0, 0.125), (2.0, -0.125),
                         (2.0, 0.0)):
        batch = Attend(mh, gpu, rng, 14, 2, 64, 16, np.array([0, 33, 500]), q_std=q_std)
        batch.scale = scale
        # Scores of a standard deviation of 2, as elsewhere, at q_std * scale = 1 / 4; larger ones have larger
        # roundings, which are errors of the weights.
        batch.check(rtol=ATTENTION_RTOL * max(1.0, 4 * q_std * abs(scale)))


def test_attention_is_the_same_twice_and_on_another_stream(mh, gpu):
    torch, rng = gpu, np.random.default_rng(13)
    batch = Attend(mh, gpu, rng, 28, 4, 128, 32, np.array([5000, 3, 777, 12, 2500]))
    first = host(batch.check())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = batch.call(where=True)
    side.synchronize()
    assert np.array_equal(host(again).view(np.uint32), first.view(np.uint32))


def test_attention_past_four_gigabytes_of_cache(mh, gpu):
    """Pages whose values lie past 2^32 elements of the cache."""
    torch, rng = gpu, np.random.default_rng(14)
    heads, kv, hd, size = 28, 4, 128, 64
    pages = 2 ** 32 // (kv * size * hd) + 40
    caches = [torch.empty((pages, kv, size, hd), dtype=torch.float16, device="cuda") for _ in range(2)]
    batch = Attend(mh, gpu, rng, heads, kv, hd, size, np.array([400, 63, 130]), spare=0)
    call_tables = pages - 1 - batch.tables
    for i in range(2):
        caches[i][pages - batch.pages:] = dev(torch, batch.caches[i]).flip(0)
    batch.call()  # the small cache, for its buffers
    torch.cuda.synchronize()
    small, real = batch.tables, batch.pages
    batch.d[1], batch.d[2] = caches
    batch.d[3] = dev(torch, np.where(small >= 0, call_tables, -1).astype(np.int32))
    batch.pages = pages
    out = batch.call(where=True)
    torch.cuda.synchronize()
    batch.pages = real
    batch.compare(host(out))


def test_attention_replayed_with_other_lengths(mh, gpu):
    """A captured call whose positions, tables, q and padding change between replays, its workspace used by
    calls of other shapes in between."""
    torch, rng = gpu, np.random.default_rng(31)
    heads, kv, hd, size, width, n = 28, 4, 128, 16, 200, 9
    pages = n * width
    batch = Attend(mh, gpu, rng, heads, kv, hd, size, np.full(n, width * size - 1), spare=0)
    other = Attend(mh, gpu, rng, 14, 2, 64, 32, np.array([4000, 17, 900]))
    out = torch.full((n, heads, hd), 9.0, device="cuda")
    batch.call(out=out)
    other.call()
    assert other.nbytes <= batch.nbytes
    other.space = batch.space
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch.call(where=True, out=out)
    for replay in range(6):
        batch.positions = rng.integers(0, width * size, n) if replay % 2 else rng.integers(0, 50, n)
        batch.sequence = rng.permutation(n)
        batch.sequence[replay % n] = -1
        batch.tables = rng.permutation(pages).reshape(n, width)
        batch.q = rng.normal(0, 2, batch.q.shape).astype(np.float32)
        for d, value in zip((batch.d[0], batch.d[3], batch.d[4], batch.d[5]),
                            (batch.q, batch.tables, batch.sequence, batch.positions)):
            d.copy_(dev(torch, value.astype(np.float32 if value.dtype == np.float32 else np.int32)))
        out.fill_(9.0)
        other_out = other.call(where=True)
        graph.replay()
        torch.cuda.synchronize()
        batch.compare(host(out))
        other.compare(host(other_out))


def test_two_attentions_at_once(mh, gpu):
    """Two streams, a workspace each."""
    torch, rng = gpu, np.random.default_rng(32)
    batches = [Attend(mh, gpu, rng, 28, 4, 128, 16, rng.integers(0, 6000, 12)),
               Attend(mh, gpu, rng, 14, 2, 64, 64, rng.integers(0, 9000, 20))]
    alone = [host(b.check()) for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    together = []
    for _ in range(5):
        for b, s in zip(batches, streams):
            with torch.cuda.stream(s):
                together.append(b.call(where=True))
    torch.cuda.synchronize()
    for i, out in enumerate(together):
        assert np.array_equal(host(out).view(np.uint32), alone[i % 2].view(np.uint32)), i


def test_attention_in_place_and_most_heads(mh, gpu):
    """out may be q; 1024 heads of 64 kv heads, whole and split."""
    torch, rng = gpu, np.random.default_rng(33)
    for positions in ([5, 300], [1500, 3]):
        batch = Attend(mh, gpu, rng, 1024, 64, 64, 16, np.array(positions))
        batch.poison_unseen()
        want = host(batch.check())
        got = batch.call(where=True, out=batch.d[0].view(len(positions), 1024, 64))
        torch.cuda.synchronize()
        assert np.array_equal(host(got).view(np.uint32), want.view(np.uint32))


def test_attention_of_more_heads_than_a_launch_has_workgroups_in_a_row(mh, gpu):
    """16400 queries of 1024 kv heads: 2^24 + 16384 (query, kv head), 256 threads each. One key is visible, so a
    head's output is that key's value."""
    torch = gpu
    queries, heads, hd = 16400, 1024, 64
    keys = torch.randn(heads, 16, hd, device="cuda").half()
    values = torch.randn(heads, 16, hd, device="cuda").half()
    q = torch.randn(1, heads, hd, device="cuda").expand(queries, heads, hd).contiguous()
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    zeros = torch.zeros(queries, dtype=torch.int32, device="cuda")
    lib = mh.load()
    need = lib.muyo_paged_attention_decode_f16kv_workspace_bytes(queries, heads, heads, hd)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    mh.check(lib.muyo_paged_attention_decode_f16kv(
        q.data_ptr(), keys.data_ptr(), values.data_ptr(), q.data_ptr(), table.data_ptr(), 1, 1, zeros.data_ptr(),
        zeros.data_ptr(), queries, heads, heads, hd, 1, 16, 0, 0.125, work.data_ptr(), need, stream(torch)))
    torch.cuda.synchronize()
    want = values[:, 0].float()
    # The weight of the only key cancels but for its low plane's rounding (2^-25, u / 2), the sum with the high
    # plane's product (u), the reciprocal and the product with it (u / 2 to u each).
    assert ((q - want).abs() <= 4 * U * want.abs()).all()


def test_plan_of_the_longest_lists(mh, gpu):
    """2^24 list entries, nearly all of them padding, and a long sequence that ends."""
    rng = np.random.default_rng(34)
    lengths, targets = np.array([100000, 3, 0]), np.array([0, 5, 40000])
    tables, ring, pool = plan_state(rng, lengths, 7000, 16, 3000)
    want = plan_reference(lengths, targets, tables, ring, pool, 16, 60000)
    for in_place in (False, True):
        got = run_plan(mh, gpu, lengths, targets, tables, ring, pool, 16, 1 << 24, in_place)
        for key in want:
            if key == "lists":
                assert np.array_equal(got[key][:, :60000], want[key]) and (got[key][:, 60000:] == -1).all()
            else:
                assert np.array_equal(got[key], want[key]), key


def test_a_steps_operators_in_one_graph(mh, gpu):
    """Plan, append, attention, a head's product and the log probabilities captured together, in place, and
    replayed: each replay is the next token of every sequence, against the same steps in 64 bits."""
    torch, rng, lib = gpu, np.random.default_rng(21), mh.load()
    heads, kv, hd, size, pages, width, n = 14, 2, 64, 16, 60, 8, 5
    lengths = np.array([0, 15, 16, 40, 99])
    tables, ring, pool = plan_state(rng, lengths, width, size, pages - sum(-(-lengths // size)))
    turns, _ = mh.rope_frequencies(1e6, hd)
    caches = rng.normal(0, 1, (2, pages, kv, size, hd)).astype(np.float16)
    d = {k: dev(torch, np.asarray(v, dtype=np.int32)) for k, v in dict(lengths=lengths, tables=tables, ring=ring,
                                                                       pool=pool).items()}
    targets = torch.empty(n, dtype=torch.int32, device="cuda")
    starts = torch.empty(n + 1, dtype=torch.int32, device="cuda")
    lists = torch.empty((3, n + 1), dtype=torch.int32, device="cuda")  # one row of padding
    qkv = torch.zeros((n + 1, (heads + 2 * kv) * hd), device="cuda")
    q_out, out = torch.full((n + 1, heads * hd), 9.0, device="cuda"), torch.full((n + 1, heads * hd), 9.0, device="cuda")
    dc, dt = [dev(torch, c) for c in caches], dev(torch, turns)
    nbytes = lib.muyo_paged_attention_decode_f16kv_workspace_bytes(n + 1, heads, kv, hd)
    space = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    vocab, top = 1000, 4
    head = dev(torch, rng.normal(0, 0.1, (vocab, heads * hd)).astype(np.float16))
    planes = torch.empty((2, n + 1, heads * hd), dtype=torch.float16, device="cuda")
    logits, given = torch.empty((n + 1, vocab), device="cuda"), torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    answers = torch.empty((2, n + 1), device="cuda")
    ranks, best = torch.empty(n + 1, dtype=torch.int32, device="cuda"), torch.empty((n + 1, top), device="cuda")
    best_ids = torch.empty((n + 1, top), dtype=torch.int32, device="cuda")
    more_bytes = lib.muyo_token_logprobs_workspace_bytes(n + 1, vocab, top)
    more = torch.empty(more_bytes, dtype=torch.uint8, device="cuda")

    def step():
        torch.add(d["lengths"], 1, out=targets)
        mh.check(lib.muyo_paged_plan(
            d["lengths"].data_ptr(), targets.data_ptr(), n, d["tables"].data_ptr(), width, d["ring"].data_ptr(),
            d["pool"].data_ptr(), pages, size, n + 1, d["lengths"].data_ptr(), d["pool"].data_ptr(),
            starts.data_ptr(), lists[0].data_ptr(), lists[1].data_ptr(), lists[2].data_ptr(), stream(torch)))
        q, k, v = (qkv.data_ptr() + 4 * hd * i for i in (0, heads, heads + kv))
        stride = qkv.shape[1]
        mh.check(lib.muyo_paged_rope_append_f16kv(
            q, k, v, stride, stride, stride, q_out.data_ptr(), dc[0].data_ptr(), dc[1].data_ptr(),
            lists[1].data_ptr(), lists[2].data_ptr(), n + 1, heads, kv, hd, pages, size, 0, hd, dt.data_ptr(), 1.0,
            stream(torch)))
        mh.check(lib.muyo_paged_attention_decode_f16kv(
            q_out.data_ptr(), dc[0].data_ptr(), dc[1].data_ptr(), out.data_ptr(), d["tables"].data_ptr(), n, width,
            lists[0].data_ptr(), lists[1].data_ptr(), n + 1, heads, kv, hd, pages, size, 0, 0.125, space.data_ptr(),
            nbytes, stream(torch)))
        mh.check(lib.muyo_split_f32_f16x2(out.data_ptr(), out.numel(), planes[0].data_ptr(), planes[1].data_ptr(),
                                          stream(torch)))
        mh.check(lib.muyo_gemm_split_f16(planes[0].data_ptr(), planes[1].data_ptr(), head.data_ptr(), None, None,
                                         logits.data_ptr(), n + 1, vocab, heads * hd, stream(torch)))
        mh.check(lib.muyo_token_logprobs_f32(
            logits.data_ptr(), vocab, n + 1, vocab, given.data_ptr(), answers[0].data_ptr(), ranks.data_ptr(),
            answers[1].data_ptr(), top, best_ids.data_ptr(), best.data_ptr(), more.data_ptr(), more_bytes,
            stream(torch)))

    saved = {k: t.clone() for k, t in d.items()}
    step()  # once eagerly, then back to the start
    torch.cuda.synchronize()
    for k, t in saved.items():
        d[k].copy_(t)
    dc[0].copy_(dev(torch, caches[0]))
    dc[1].copy_(dev(torch, caches[1]))
    out.fill_(9.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    want_caches = caches.astype(np.float64)
    for replay in range(20):
        rows = rng.normal(0, 1, (n + 1, qkv.shape[1])).astype(np.float32)
        qkv.copy_(dev(torch, rows))
        tokens = rng.integers(0, vocab, n + 1)
        given.copy_(dev(torch, tokens.astype(np.int32)))
        want = plan_reference(lengths, lengths + 1, tables, ring, pool, size, n + 1)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(lists), want["lists"]), replay
        lengths, tables, ring, pool = want["granted"], want["tables"], want["free_pages"], want["pool_out"].tolist()
        positions, slots = want["lists"][1], want["lists"][2]
        rows = rows.reshape(n + 1, heads + 2 * kv, hd)
        q, _ = rotate64(rows[:, :heads], positions, turns, 1.0, 0, hd)
        k, _ = rotate64(rows[:, heads:heads + kv], positions, turns, 1.0, 0, hd)
        got, cached = host(out).reshape(n + 1, heads, hd), [host(c) for c in dc]
        for t in range(n):
            at = (slots[t] // size, slice(None), slots[t] % size)
            want_caches[0][at], want_caches[1][at] = k[t], rows[t, heads + kv:]
            # The keys as they are stored: their rounding is the cache's, checked here.
            assert np.abs(cached[0][at] - k[t]).max() <= 2.0 ** -10 * np.abs(k[t]).max()
            ref = attend64(q[t], cached[0], cached[1], tables[t], int(positions[t]), 0, 0.125)
            assert np.linalg.norm(got[t] - ref) <= ATTENTION_RTOL * np.linalg.norm(ref), (replay, t)
        assert (got[n] == 9.0).all() and (host(q_out)[n] == 9.0).all()  # the padding row
        x = host(logits).astype(np.float64)
        product = got.reshape(n + 1, -1).astype(np.float64) @ host(head).astype(np.float64).T
        assert np.linalg.norm(x - product) <= 1e-6 * np.linalg.norm(product)  # two planes: some 21 bits
        lp = x - np.log(np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True)) - x.max(1, keepdims=True)
        order = np.argsort(-x, 1, kind="stable")
        # Logits of a few units: some eight roundings of that size.
        assert np.abs(host(answers)[0] - lp[np.arange(n + 1), tokens]).max() <= 64 * U * np.abs(lp).max()
        assert np.abs(host(answers)[1] + (np.exp(lp) * lp).sum(1)).max() <= 64 * U * np.abs(lp).max()
        assert np.array_equal(host(best_ids), order[:, :top])
        assert np.array_equal(host(ranks), np.argsort(order, 1)[np.arange(n + 1), tokens])
    assert lengths.tolist() == [20, 35, 36, 60, 119]


def with_sinks(batch, rng, nats, value, last=False):
    """Key 0 (or the last one) of each sequence scores `nats[i]` for every head of its query i, the others as
    they were, a standard deviation of 2 about 0; its value row is `value` times one of theirs."""
    heads, kv, hd, size = batch.shape
    for i, (b, p) in enumerate(zip(batch.sequence, batch.positions)):
        key = int(p) if last else 0
        at = batch.tables[b, key // size], slice(None), key % size
        for g, q in enumerate(batch.q[i].astype(np.float64).reshape(kv, heads // kv, hd)):
            batch.caches[0][at][g] = np.linalg.pinv(q) @ np.full(heads // kv, nats[i] / batch.scale)
        batch.caches[1][at] = rng.normal(0, value, (kv, hd))


SINKS = [
    # heads, kv_heads, head_dim, page_size, keys: whole, cut, and (300 queries) several to a workgroup
    (14, 2, 64, 16, [302] * 8),
    (28, 4, 128, 16, [300, 1000] * 4),
    (14, 2, 64, 64, [16384] * 8),
    (28, 4, 128, 64, [16384, 4096] * 4),
    (14, 2, 64, 16, [1500] * 300),
    (4, 4, 128, 16, [1100] * 300),
    (16, 1, 128, 32, [5000] * 4),
]


@pytest.mark.parametrize("value, last, spread", [(0.0, False, 1.0), (0.0, False, 0.1), (0.01, False, 1.0),
                                                 (0.01, False, 0.1), (1.0, False, 1.0), (0.0, True, 1.0)])
@pytest.mark.parametrize("heads, kv, hd, size, keys", SINKS, ids=["-".join(map(str, (*s[:4], s[4][0], len(s[4]))))
                                                                 for s in SINKS])
def test_attention_with_a_key_that_has_most_of_the_weight(mh, gpu, heads, kv, hd, size, keys, value, last,
                                                          spread):
    """One key 8 to 20 nats above the mean of the others, which differ much or little, with a value row that is 0,
    small or ordinary: the output is that of the many small weights. A score of S is off by some 4 u S, as
    above, where 10 was taken for S; a sink's own S is larger, and its error is one of the sum of weights."""
    rng = np.random.default_rng(hd + len(keys) + keys[0])
    nats = np.resize(np.array([20.0, 8.0, 17.0, 14.0, 12.0, 0.0]), len(keys))
    batch = Attend(mh, gpu, rng, heads, kv, hd, size, np.array(keys) - 1)
    batch.caches[0] *= np.float16(spread)
    with_sinks(batch, rng, nats, value, last)
    out = batch.call()
    gpu.cuda.synchronize()
    got, some = host(out), np.unique(np.concatenate([np.arange(8) % len(keys), rng.integers(0, len(keys), 16)]))
    worst = 0.0
    for i in some:
        want = attend64(batch.q[i], *batch.caches, batch.tables[batch.sequence[i]], keys[i] - 1, 0, batch.scale)
        off = np.linalg.norm(got[i] - want) / np.linalg.norm(want)
        worst = max(worst, off / max(1.0, nats[i] / 10))
    assert worst <= ATTENTION_RTOL, worst


@pytest.mark.parametrize("heads, kv, hd, positions", [(14, 2, 64, [0, 40, 300]), (28, 4, 128, [700, 1000]),
                                                      (14, 2, 64, [5000, 7]), (28, 4, 128, [3000, 16383])])
@pytest.mark.parametrize("ratio", [300.0, 1e4, 1e5])
def test_attention_with_one_large_component_of_q(mh, gpu, heads, kv, hd, positions, ratio):
    """A component of q far above the others meets a component of K that is 0: the scores are those of the others,
    with their own roundings."""
    rng = np.random.default_rng(hd)
    batch = Attend(mh, gpu, rng, heads, kv, hd, 16, np.array(positions))
    batch.q[..., 5] *= ratio
    batch.caches[0][..., 5] = 0
    batch.check()


@pytest.mark.parametrize("heads, kv, hd, positions", [(14, 2, 64, [0, 33, 500]), (28, 4, 128, [900, 1023]),
                                                      (14, 2, 64, [3000, 40, 20000]), (28, 4, 128, [16383, 1100])])
@pytest.mark.parametrize("q_std, scale", [(2.0, 1e9), (2.0, -1e12), (2.0, 1e30), (2.0, 3e38), (1e20, 1e25),
                                          (1e-20, 1e38)])
def test_attention_of_scores_far_past_any_exponent(mh, gpu, heads, kv, hd, positions, q_std, scale):
    """Scaled scores from 1e10 on: the largest one's value is the output, exactly but for the reciprocal of the sum
    and the product with it; and keys that are all the same share the weight."""
    rng = np.random.default_rng(hd + len(positions))
    batch = Attend(mh, gpu, rng, heads, kv, hd, 64, np.array(positions), q_std=q_std)
    batch.scale = scale
    for i, p in enumerate(positions):  # no close second: a score's roundings are some 2^-20 of these
        keys = np.arange(p + 1)
        k = batch.caches[0][batch.tables[i, keys // 64], :, keys % 64].astype(np.float64)
        scores = np.sort(np.einsum("hd,khd->hk", batch.q[i] / q_std, np.repeat(k, heads // kv, 1)) * np.sign(scale), 1)
        if p:
            small = (scores[:, -1] - scores[:, -2]) < 1e-4 * scores[:, -1]
            assert not small.any()
    batch.check(rtol=4 * U)
    batch.caches[0][:] = batch.caches[0][:1, :, :1]
    batch.check()
