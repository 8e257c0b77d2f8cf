"""Rope + append into a paged cache of 8-bit values and decode attention over it, on the GPU against their
definitions in 64 bits on the host.

Tolerances:
- q_out: as the fp16 cache's append, 12 u (|x0| + |x1|) magnitude (u = 2^-24, half a step of f32).
- codes and scales: those of values in 64 bits, equal. Both sides' values are good to some 2^-50, and of a few
  million values one lies that near a border between two codes with a chance of about 2^-50 * 2^8 * 2^22.
- attention: as the fp16 cache's, 4e-6 of a 2-norm over an output; a score and a weight have one rounding more
  (of the product with a scale), u each.
"""
import numpy as np
import pytest

from test_paged_gpu import (ATTENTION_RTOL, LAYOUTS, SINKS, U, Attend, attend64, dev, host, plan_reference,
                            plan_state, rotate64, stream, with_sinks)

pytestmark = pytest.mark.gpu

INT8, E4M3 = 0, 1
FORMATS = [INT8, E4M3]
LARGEST = {INT8: 127.0, E4M3: 448.0}


def _e4m3():
    code = np.arange(128)
    exponent, fraction = code >> 3, code & 7
    size = np.where(exponent == 0, fraction * 2.0 ** -9, (8 + fraction) * 2.0 ** (exponent - 10.0))
    size[127] = np.nan
    return np.concatenate([size, -size])


E4M3_VALUES = _e4m3()  # of each byte


def decode(codes, form):
    return codes.view(np.int8).astype(np.float64) if form == INT8 else E4M3_VALUES[codes]


def quantise(rows, form):
    """(codes, scales) of rows [..., hd] in 64 bits, by the definition."""
    rows = np.asarray(rows, dtype=np.float64)
    with np.errstate(all="ignore"):
        size = np.abs(rows).max(-1)
        finite = np.isfinite(rows).all(-1)
        scales = np.where(finite, size / LARGEST[form], np.nan).astype(np.float32)
        ok = finite & (scales > 0)
        x = np.where(ok[..., None], rows / scales.astype(np.float64)[..., None], 0.0)
    x = np.clip(x, -LARGEST[form], LARGEST[form])
    if form == INT8:
        return np.rint(x).astype(np.int8).view(np.uint8), scales
    values = E4M3_VALUES[:127]
    middle = (values[1:] + values[:-1]) / 2
    low = np.searchsorted(middle, np.abs(x))           # a half step goes to the code below it here
    tie = (low < 126) & (np.abs(x) == middle[np.minimum(low, 125)])
    code = np.where(tie & (low % 2 == 1), low + 1, low)  # and to the even one in the end
    return (code + np.where(np.signbit(x), 128, 0)).astype(np.uint8), scales


# ------------------------------------------------------------------------------------------------
# Append

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
    (3, 3, 64, 16, 0, 2, 11, 2 ** 31 - 1, True),
    (5, 1, 128, 1024, 1, 100, 300, 299, True),
    (1, 1, 128, 16, 0, 126, 2, 9, False),
    (33, 16, 64, 16, 0, 32, 1000, 8000, True),
    (2, 1, 128, 16, 1, 64, 3001, 5000, False),
]


class Append:
    """Tokens on the device, their caches and their call."""

    def __init__(self, mh, torch, rng, heads, kv, hd, size, form, parts, positions, slots, pages, stacked=False):
        self.mh, self.torch, self.form = mh, torch, form
        self.shape = heads, kv, hd, size, pages
        tokens, self.parts = len(positions), [p.astype(np.float32) for p in parts]
        if stacked:
            gap = np.zeros((tokens, 4), np.float32)  # and a gap behind each row
            d = dev(torch, np.concatenate([*(p.reshape(tokens, -1) for p in self.parts), gap], 1))
            ends = np.cumsum([p[0].size for p in self.parts])
            self.views, self.strides = [d[:, :ends[0]], d[:, ends[0]:ends[1]], d[:, ends[1]:ends[2]]], [d.shape[1]] * 3
        else:
            self.views = [dev(torch, p) for p in self.parts]
            self.strides = [p[0].size for p in self.parts]
        self.positions, self.slots = np.asarray(positions), np.asarray(slots)
        self.codes = rng.integers(0, 256, (2, pages, kv, size, hd)).astype(np.uint8)
        self.scales = rng.normal(1, 0.1, (2, pages, kv, size)).astype(np.float32)
        self.d = [dev(torch, x) for x in (*self.codes, *self.scales)]
        self.lists = [dev(torch, x.astype(np.int32)) for x in (self.positions, self.slots)]
        self.q_out = torch.full((tokens, heads * hd), 9.0, device="cuda")

    def call(self, layout, rotary, turns, magnitude, q_out=None):
        heads, kv, hd, size, pages = self.shape
        self.turns = dev(self.torch, turns)
        self.mh.check(self.mh.load().muyo_paged_rope_append_q8kv(
            *(v.data_ptr() for v in self.views), *self.strides, (self.q_out if q_out is None else q_out).data_ptr(),
            *(t.data_ptr() for t in self.d), *(t.data_ptr() for t in self.lists), len(self.positions), heads, kv, hd,
            pages, size, self.form, layout, rotary, self.turns.data_ptr(), magnitude, stream(self.torch)))

    def check(self, layout, rotary, turns, magnitude):
        self.call(layout, rotary, turns, magnitude)
        self.torch.cuda.synchronize()
        heads, kv, hd, size, pages = self.shape
        tokens, live = len(self.positions), self.positions >= 0
        q, bound = rotate64(self.parts[0].reshape(tokens, heads, hd), self.positions, turns, magnitude, layout, rotary)
        got = host(self.q_out).reshape(tokens, heads, hd)
        assert (np.abs(got - q) <= bound)[live].all()
        assert (got[~live] == 9.0).all()
        with np.errstate(invalid="ignore"):
            k, _ = rotate64(self.parts[1].reshape(tokens, kv, hd), self.positions, turns, magnitude, layout, rotary)
        new = [quantise(k, self.form), quantise(self.parts[2].reshape(tokens, kv, hd), self.form)]
        codes, scales = self.codes.copy(), self.scales.copy()
        for t in np.flatnonzero(live & (self.slots >= 0) & (self.slots < pages * size)):
            at = (self.slots[t] // size, slice(None), self.slots[t] % size)
            for i in range(2):
                codes[i][at], scales[i][at] = new[i][0][t], new[i][1][t]
        for i in range(2):
            assert np.array_equal(host(self.d[2 + i]), scales[i], equal_nan=True), "kv"[i]
            assert np.array_equal(host(self.d[i]), codes[i]), "kv"[i]


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("case", APPENDS, ids=["-".join(map(str, c)) for c in APPENDS])
def test_append_matches_definition(mh, gpu, case, form):
    heads, kv, hd, size, layout, rotary, tokens, last, stacked = case
    rng = np.random.default_rng(hd + tokens)
    pages = -(-tokens // size) + 3
    turns, magnitude = mh.rope_frequencies(1e4, rotary, "YARN", factor=2.0, trained_context=4096)
    parts = [rng.normal(0, 2, (tokens, n, hd)) for n in (heads, kv, kv)]
    positions = rng.integers(0, last + 1, tokens)
    positions[-1] = last
    slots = rng.permutation(pages * size)[:tokens]
    if tokens > 4:
        positions[1], slots[1] = -1, -1   # padding
        slots[2] = pages * size           # not appended
        slots[3] = -5
    batch = Append(mh, gpu, rng, heads, kv, hd, size, form, parts, positions, slots, pages, stacked)
    batch.check(layout, rotary, turns, magnitude)


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("hd", [64, 128])
def test_append_of_borders_and_extreme_rows(mh, gpu, hd, form):
    """Values of v on and next to every border between two codes, rows of zeros, of sizes from f32's smallest to
    its largest, and rows with an infinity or a NaN."""
    rng = np.random.default_rng(hd)
    most = LARGEST[form]
    values = np.arange(128.0) if form == INT8 else E4M3_VALUES[:127]
    middle = ((values[1:] + values[:-1]) / 2).astype(np.float32)
    near = np.concatenate([middle, np.nextafter(middle, np.float32(0)), np.nextafter(middle, np.float32(1e9))])
    near = np.concatenate([near, -near])
    rows = []
    for i in range(0, len(near), hd - 1):
        row = np.resize(near[i:i + hd - 1], hd).astype(np.float32)
        row[0] = most  # scale 1
        rows.append(row)
    for exponent in range(-149, 128, 7):
        rows.append((rng.uniform(-1, 1, hd) * 2.0 ** exponent).astype(np.float32))
    rows += [np.zeros(hd, np.float32), np.full(hd, -0.0, np.float32), np.full(hd, 3.0e38, np.float32)]
    for bad in (np.nan, np.inf, -np.inf):
        row = rng.normal(0, 1, hd).astype(np.float32)
        row[rng.integers(hd)] = bad
        rows.append(row)
    rows = np.stack(rows)
    n, size = len(rows), 16
    pages = -(-n // size)
    turns, _ = mh.rope_frequencies(1e4, hd)
    parts = [np.zeros((n, 1, hd)), rows[:, None], rows[:, None]]
    batch = Append(mh, gpu, rng, 1, 1, hd, size, form, parts, np.zeros(n, int), np.arange(n), pages)
    batch.check(0, hd, turns, 1.0)


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("layout, rotary", [(0, 64), (1, 64), (0, 20)])
def test_append_of_rows_past_f32(mh, gpu, layout, rotary, form):
    """A magnitude that takes some rows of k to where f32 ends, and past it: their scale is infinite, their codes 0."""
    rng = np.random.default_rng(5)
    n, hd, size = 40, 64, 16
    turns, _ = mh.rope_frequencies(1e4, rotary)
    k = rng.uniform(0.5, 1, (n, 1, hd)) * 2.0 ** (np.arange(n) + 88.0)[:, None, None]
    batch = Append(mh, gpu, rng, 1, 1, hd, size, form, [np.zeros((n, 1, hd)), k, np.ones((n, 1, hd))],
                   rng.integers(0, 3000, n), rng.permutation(48)[:n], 3)
    batch.call(layout, rotary, turns, 2.0 ** 30)
    gpu.cuda.synchronize()
    rotated, _ = rotate64(batch.parts[1].reshape(n, 1, hd), batch.positions, turns, 2.0 ** 30, layout, rotary)
    codes, scales = quantise(rotated[:, 0], form)
    codes[np.isinf(scales)] = 0  # of either sign
    assert np.isinf(scales).any() and (scales < np.inf).any()
    at = batch.slots // size, 0, batch.slots % size
    assert np.array_equal(host(batch.d[2])[at], scales)
    assert np.array_equal(host(batch.d[0])[at], codes)


def test_append_in_place_is_the_fp16_caches_rotation(mh, gpu):
    """q_out may be q, and q is rotated as by the fp16 cache's append, bit for bit."""
    torch, rng = gpu, np.random.default_rng(3)
    heads, kv, hd, size, pages, tokens = 28, 4, 128, 16, 5, 70
    turns, magnitude = mh.rope_frequencies(1e6, hd, "LINEAR", factor=4.0)
    parts = [rng.normal(0, 1, (tokens, n, hd)) for n in (heads, kv, kv)]
    for layout in (0, 1):
        batch = Append(mh, torch, rng, heads, kv, hd, size, INT8, parts, rng.integers(0, 9000, tokens),
                       rng.permutation(pages * size)[:tokens], pages)
        batch.check(layout, hd, turns, magnitude)
        half = torch.zeros((2, pages, kv, size, hd), dtype=torch.float16, device="cuda")
        other = torch.empty_like(batch.q_out)
        mh.check(mh.load().muyo_paged_rope_append_f16kv(
            *(v.data_ptr() for v in batch.views), *batch.strides, other.data_ptr(), half[0].data_ptr(),
            half[1].data_ptr(), *(t.data_ptr() for t in batch.lists), tokens, heads, kv, hd, pages, size, layout, hd,
            batch.turns.data_ptr(), magnitude, stream(torch)))
        batch.call(layout, hd, turns, magnitude, q_out=batch.views[0])
        torch.cuda.synchronize()
        assert np.array_equal(host(other), host(batch.q_out))
        assert np.array_equal(host(batch.views[0]).reshape(tokens, -1), host(batch.q_out))


# ------------------------------------------------------------------------------------------------
# Attention


class Attend8(Attend):
    """Attend over codes and scales; `caches` holds the values that they stand for."""

    def __init__(self, *args, form, **more):
        super().__init__(*args, **more)
        self.form = form
        # Normal codes, and rows of different sizes, V's very; K's at most as elsewhere, so that scores are.
        order, shape = np.random.default_rng(1), self.caches.shape
        torch = self.torch
        codes = torch.randn(shape, generator=torch.Generator().manual_seed(1)) * (LARGEST[form] / 4)
        codes = codes.clamp(-LARGEST[form], LARGEST[form])
        codes = codes.round().to(torch.int8) if form == INT8 else codes.to(torch.float8_e4m3fn)
        self.codes = codes.view(torch.uint8).numpy()
        self.scales = order.uniform(0.7, 1.0, shape[:-1]) * (4 / LARGEST[form])
        self.scales[0] *= 2.0 ** order.integers(-2, 1, shape[1:-1])
        self.scales[1] *= 2.0 ** order.integers(-3, 4, shape[1:-1])
        self.scales = self.scales.astype(np.float32)
        self.caches = self.values()

    def values(self):
        return decode(self.codes, self.form) * self.scales.astype(np.float64)[..., None]

    def requantise(self):
        """Rows of `caches` that are no longer what is stored, stored."""
        changed = (self.caches != self.values()).any(-1)
        self.codes[changed], self.scales[changed] = quantise(self.caches[changed], self.form)
        self.caches = self.values()

    def poison_unseen(self, window=0):
        """NaN and infinities wherever no query looks."""
        size = self.shape[3]
        seen = np.zeros((self.pages, size), bool)
        for s, p in zip(self.sequence, self.positions):
            if s >= 0 and p >= 0:
                j = np.arange(max(0, p + 1 - window) if window else 0, min(p + 1, self.width * size))
                seen[self.tables[s, j // size], j % size] = True
        for codes, scales in zip(self.codes, self.scales):
            codes.transpose(0, 2, 1, 3)[~seen] = 0x7F  # e4m3's NaN
            view = scales.transpose(0, 2, 1)
            view[~seen] = np.resize(np.array([np.nan, np.inf, -np.inf], np.float32), view[~seen].shape)

    def call(self, window=0, where=None, out=None):
        torch, lib = self.torch, self.mh.load()
        heads, kv, hd, size = self.shape
        if where is None:
            self.d = [dev(torch, x) for x in (self.q, *self.codes, *self.scales, self.tables.astype(np.int32),
                                              self.sequence.astype(np.int32), self.positions.astype(np.int32))]
            self.nbytes = lib.muyo_paged_attention_decode_q8kv_workspace_bytes(len(self.q), heads, kv, hd)
            self.space = torch.full((self.nbytes + 256,), 0x5A, dtype=torch.uint8, device="cuda")
        if out is None:
            out = torch.full((len(self.q), heads, hd), 9.0, device="cuda")
        q, k, v, ks, vs, tables, sequence, positions = self.d
        self.mh.check(lib.muyo_paged_attention_decode_q8kv(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), out.data_ptr(), tables.data_ptr(),
            self.tables.shape[0], self.width, sequence.data_ptr(), positions.data_ptr(), len(self.q), heads, kv, hd,
            self.pages, size, self.form, window, self.scale, self.space.data_ptr(), self.nbytes, stream(torch)))
        return out


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("heads, kv, hd", LAYOUTS)
def test_attention_of_all_head_layouts(mh, gpu, heads, kv, hd, form):
    """Lengths around pages, tiles and their multiples, one call; everything unseen is poisoned."""
    rng = np.random.default_rng(heads * hd)
    positions = np.array([0, 1, 14, 15, 16, 17, 31, 32, 62, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 511, 1000])
    batch = Attend8(mh, gpu, rng, heads, kv, hd, 16, rng.permutation(positions), form=form)
    batch.poison_unseen()
    batch.check()


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("size", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("window", [0, 1, 63, 100, 5000])
def test_attention_pages_and_windows(mh, gpu, size, window, form):
    rng = np.random.default_rng(size + window)
    batch = Attend8(mh, gpu, rng, 14, 2, 64, size, np.array([0, 5, 99, 100, 101, 1023, 1024, 1500, 2222, 40]), form=form)
    batch.poison_unseen(window)
    batch.check(window)


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("hd, positions", [
    (128, [20000]), (64, [20011]), (128, [3000, 1, 9000, 0, 150]), (128, [1100] * 70),
    (64, [700] * 200), (128, list(range(0, 640, 5))), (64, [2000, 5] * 512), (64, [0, 40, 1300, 7, -1] * 250),
])
def test_attention_long_and_many(mh, gpu, hd, positions, form):
    rng = np.random.default_rng(len(positions))
    heads, kv = (14, 2) if hd == 64 else (28, 4)
    batch = Attend8(mh, gpu, rng, heads, kv, hd, 64, np.array(positions), form=form)
    batch.poison_unseen()
    batch.check()


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("queries", [1, 5, 65, 300])
def test_attention_of_short_sequences_in_wide_tables(mh, gpu, queries, form):
    """Tables of 4096 keys, sequences of up to 513, padding among them."""
    rng = np.random.default_rng(queries)
    positions = rng.integers(0, 513, queries)
    positions[0] = 512
    sequence = rng.permutation(queries)
    if queries > 4:
        sequence[3] = -1
    batch = Attend8(mh, gpu, rng, 14, 2, 64, 16, positions, width=256, sequence=sequence, form=form)
    batch.poison_unseen()
    batch.check()


@pytest.mark.parametrize("form", FORMATS)
def test_attention_padding_empty_rows_and_bad_pages(mh, gpu, form):
    """Padding rows stay, rows without keys are 0, pages outside the cache and keys past the table are
    left out, and several queries may share a sequence."""
    rng = np.random.default_rng(9)
    sequence = np.array([0, -1, 1, 2, 99, 2, 3, 3, 3, 4, -2 ** 31])
    positions = np.array([40, 7, -1, 100, 3, 101, 300, 17, 0, 63, 5])
    batch = Attend8(mh, gpu, rng, 14, 2, 64, 16, positions, sequence=np.minimum(sequence, 4), form=form)
    batch.sequence = sequence  # 99 and below 0 name no row
    batch.tables[3, [1, 5, 6, 18]] = [-1, batch.pages, 2 ** 31 - 1, -2 ** 31]
    batch.tables[4, :] = -1    # a sequence whose every page is missing
    out = host(batch.check())
    assert (out[2] == 0).all() and (out[9] == 0).all() and (out[8] != 0).any()


def test_attention_positions_past_the_table(mh, gpu):
    batch = Attend8(mh, gpu, np.random.default_rng(10), 28, 4, 128, 16, np.array([63, 20, 62]), spare=0, form=INT8)
    batch.positions = np.array([2 ** 31 - 1, 20, 64])
    batch.check()
    batch.check(window=1)     # the window lies past the table: nothing seen
    batch.check(window=2 ** 31)


@pytest.mark.parametrize("form", FORMATS)
def test_attention_of_large_small_and_negative_scales(mh, gpu, form):
    """q, and a cache's scales, far from 1 in either direction, equal scores, a negative and a zero scale."""
    rng = np.random.default_rng(12)
    for q_std, scale, k_size, v_size in ((1e6, 1e-7, 1, 1), (1e-6, 1e5, 1, 1), (1e-20, 1e19, 1, 1e20),
                                         (1e20, 1e-21, 1, 1e-20), (0.0, 1.0, 1, 1), (2.0, -0.125, 1, 1),
                                         (2.0, 0.0, 1, 1), (1e20, 0.125, 1e-20, 1e25), (1e-20, 0.125, 1e20, 1e-25)):
        for position in (500, 3000):
            batch = Attend8(mh, gpu, rng, 14, 2, 64, 16, np.array([0, 33, position]), q_std=q_std, form=form)
            batch.scale = scale
            batch.caches[0] *= k_size
            batch.caches[1] *= v_size
            batch.requantise()
            # Scores of a standard deviation of 2, as elsewhere, at q_std * scale * k_size = 1 / 4; larger ones
            # have larger roundings, which are errors of the weights.
            batch.check(rtol=ATTENTION_RTOL * max(1.0, 4 * q_std * k_size * abs(scale)))


HERE = [s for s in SINKS if len(s[4]) < 100] + [(4, 4, 128, 16, [1100] * 70)]


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("value, last", [(0.0, False), (0.01, False), (1.0, False), (0.0, True)])
@pytest.mark.parametrize("heads, kv, hd, size, keys", HERE, ids=["-".join(map(str, (*s[:4], s[4][0], len(s[4]))))
                                                                for s in HERE])
def test_attention_with_a_key_that_has_most_of_the_weight(mh, gpu, heads, kv, hd, size, keys, value, last, form):
    """One key up to 20 nats above the others with a value row that is 0, small or ordinary: the output is that
    of the many small weights. A score of S is off by some 4 u S, where 10 was taken for S."""
    rng = np.random.default_rng(hd + len(keys) + keys[0])
    nats = np.resize(np.array([20.0, 8.0, 17.0, 14.0, 12.0, 0.0]), len(keys))
    batch = Attend8(mh, gpu, rng, heads, kv, hd, size, np.array(keys) - 1, form=form)
    with_sinks(batch, rng, nats, value, last)
    batch.requantise()
    out = batch.call()
    gpu.cuda.synchronize()
    got, worst = host(out), 0.0
    for i in np.unique(np.concatenate([np.arange(8) % len(keys), rng.integers(0, len(keys), 8)])):
        want = attend64(batch.q[i], *batch.caches, batch.tables[batch.sequence[i]], keys[i] - 1, 0, batch.scale)
        off = np.linalg.norm(got[i] - want) / np.linalg.norm(want)
        worst = max(worst, off / max(1.0, nats[i] / 10))
    assert worst <= ATTENTION_RTOL, worst


@pytest.mark.parametrize("heads, kv, hd, positions", [(14, 2, 64, [0, 40, 300]), (28, 4, 128, [3000, 700])])
def test_attention_with_one_large_component_of_q(mh, gpu, heads, kv, hd, positions):
    """A component of q far above the others meets a component of K that is 0: the scores are those of the others,
    with their own roundings."""
    for ratio in (300.0, 1e5):
        batch = Attend8(mh, gpu, np.random.default_rng(hd), heads, kv, hd, 16, np.array(positions), form=INT8)
        batch.q[..., 5] *= ratio
        batch.caches[0][..., 5] = 0
        batch.requantise()
        batch.check()


@pytest.mark.parametrize("q_std, scale", [(2.0, 1e9), (2.0, -1e12), (2.0, 3e38), (1e20, 1e25), (1e-20, 1e38)])
def test_attention_of_scores_far_past_any_exponent(mh, gpu, q_std, scale):
    """The largest score's value is the output, exactly but for the weights' planes and the division; keys that are
    all the same share the weight."""
    for form in FORMATS:
        batch = Attend8(mh, gpu, np.random.default_rng(5), 14, 2, 64, 64, np.array([3000, 40, 700]), q_std=q_std,
                        form=form)
        batch.scale = scale
        for i, p in enumerate(batch.positions):  # no close second: a score's roundings are some 2^-20 of these
            keys = np.arange(p + 1)
            k = batch.caches[0][batch.tables[i, keys // 64], :, keys % 64]
            scores = np.einsum("hd,khd->hk", batch.q[i] / q_std, np.repeat(k, 7, 1)) * np.sign(scale)
            scores = np.sort(scores, 1)
            assert not ((scores[:, -1] - scores[:, -2]) < 1e-4 * scores[:, -1]).any()
        # The product of the value's scale and code and of the reciprocal, u to 2 u each.
        batch.check(rtol=6 * U)
        batch.caches[:] = batch.caches[:, :1, :, :1]
        batch.requantise()
        batch.check()


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("heads, kv, hd, position", [(14, 2, 64, 700), (28, 4, 128, 3000)])
def test_attention_of_the_largest_and_smallest_scales(mh, gpu, heads, kv, hd, position, form):
    """Scales at the ends that the call is stated for."""
    rng = np.random.default_rng(7)
    for k_most, v_most in ((96, 110 - np.log2(position + 1)), (96, -72), (-140, -72), (-140, 96)):
        batch = Attend8(mh, gpu, rng, heads, kv, hd, 16, np.array([position, 40]), form=form)
        k_size, v_size = (2.0 ** np.floor(most - np.log2(float(batch.scales[i].max())))
                          for i, most in enumerate((k_most, v_most)))
        # K's rows are then of that size, and scores as elsewhere.
        batch.scales[0] *= np.float32(k_size)
        batch.scales[1] *= np.float32(v_size)
        assert batch.scales[0].max() <= 2.0 ** 96 and batch.scales[1].max() <= 2.0 ** 110 / (position + 1)
        batch.scale /= max(k_size, 2.0 ** -120)
        batch.q *= np.float32(max(k_size, 2.0 ** -120) / k_size)
        batch.caches = batch.values()
        batch.check()


@pytest.mark.parametrize("form", FORMATS)
@pytest.mark.parametrize("keys", [1000, 3000])
def test_attention_of_equal_values_at_the_largest_scale(mh, gpu, keys, form):
    """Weights that a later maximum leaves above 1, each of the largest code and scale: the sum is the largest that a
    call is stated for, and the output that value."""
    heads, kv, hd = 28, 4, 128
    batch = Attend8(mh, gpu, np.random.default_rng(2), heads, kv, hd, 16, np.array([keys - 1]), form=form)
    batch.q[:] = 1.0
    batch.scale = 0.125 / hd
    batch.codes[1] = 127 if form == INT8 else 126  # the largest
    batch.scales[1] = 2.0 ** 110 / keys
    batch.codes[0] = 56 if form == E4M3 else 1     # 1
    batch.scales[0] = 1.0
    later = batch.tables[0][np.arange(128, keys) // 16], slice(None), np.arange(128, keys) % 16
    batch.scales[0][later] = 8.0 * 5.4             # nats above the first 128 keys' 1 / 8: 2^7.6 of their weight
    batch.caches = batch.values()
    want = LARGEST[form] * float(np.float32(2.0 ** 110 / keys))
    out = host(batch.call())
    assert np.abs(out / want - 1).max() <= ATTENTION_RTOL


@pytest.mark.parametrize("form", FORMATS)
def test_attention_of_vanishing_scales(mh, gpu, form):
    for most in (-80, -100, -120, -126, -140):
        batch = Attend8(mh, gpu, np.random.default_rng(3), 14, 2, 64, 16, np.array([2000, 15]), form=form)
        batch.scales[1] = batch.scales[1] / batch.scales[1].max() * 2.0 ** most
        batch.caches = batch.values()
        out = host(batch.call())
        for i, p in enumerate(batch.positions):
            want = attend64(batch.q[i], *batch.caches, batch.tables[i], int(p), 0, batch.scale)
            assert np.abs(out[i] - want).max() <= 2.0 ** -84 + ATTENTION_RTOL * np.abs(want).max(), most


def test_attention_past_four_gigabytes_of_cache(mh, gpu):
    """Pages whose codes lie past 2^32 bytes of the cache."""
    torch, rng = gpu, np.random.default_rng(14)
    heads, kv, hd, size = 28, 4, 128, 64
    pages = 2 ** 32 // (kv * size * hd) + 40
    batch = Attend8(mh, gpu, rng, heads, kv, hd, size, np.array([400, 63, 1130]), spare=0, form=E4M3)
    codes = [torch.empty((pages, kv, size, hd), dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.empty((pages, kv, size), device="cuda") for _ in range(2)]
    for i in range(2):
        codes[i][pages - batch.pages:] = dev(torch, batch.codes[i]).flip(0)
        scales[i][pages - batch.pages:] = dev(torch, batch.scales[i]).flip(0)
    batch.call()  # the small cache, for its buffers
    torch.cuda.synchronize()
    small, real = batch.tables, batch.pages
    batch.d[1:5] = [*codes, *scales]
    batch.d[5] = dev(torch, np.where(small >= 0, pages - 1 - small, -1).astype(np.int32))
    batch.pages = pages
    out = batch.call(where=True)
    torch.cuda.synchronize()
    batch.pages = real
    batch.compare(host(out))


def test_attention_in_place_twice_and_on_other_streams(mh, gpu):
    """out may be q; the same bits on another stream, and two calls at once with a workspace each."""
    torch, rng = gpu, np.random.default_rng(33)
    batches = [Attend8(mh, gpu, rng, 28, 4, 128, 16, rng.integers(0, 6000, 12), form=INT8),
               Attend8(mh, gpu, rng, 14, 2, 64, 64, rng.integers(0, 900, 20), form=E4M3)]
    alone = [host(b.check()) for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    together = []
    for _ in range(4):
        for b, s in zip(batches, streams):
            with torch.cuda.stream(s):
                together.append(b.call(where=True))
    torch.cuda.synchronize()
    for i, out in enumerate(together):
        assert np.array_equal(host(out).view(np.uint32), alone[i % 2].view(np.uint32)), i
    for b, want in zip(batches, alone):
        got = b.call(where=True, out=b.d[0])
        torch.cuda.synchronize()
        assert np.array_equal(host(got).view(np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("form", FORMATS)
def test_a_steps_operators_in_one_graph(mh, gpu, form):
    """Plan, append and attention captured together, in place, and replayed: each replay is the next token of
    every sequence, against the same steps in 64 bits."""
    torch, rng, lib = gpu, np.random.default_rng(21), mh.load()
    heads, kv, hd, size, pages, width, n = 14, 2, 64, 16, 200, 70, 5
    lengths = np.array([0, 15, 16, 40, 1100])
    tables, ring, pool = plan_state(rng, lengths, width, size, pages - sum(-(-lengths // size)))
    turns, _ = mh.rope_frequencies(1e6, hd)
    codes, scales = quantise(rng.normal(0, 1, (2, pages, kv, size, hd)), form)
    d = {k: dev(torch, np.asarray(v, dtype=np.int32)) for k, v in dict(lengths=lengths, tables=tables, ring=ring,
                                                                       pool=pool).items()}
    targets = torch.empty(n, dtype=torch.int32, device="cuda")
    starts = torch.empty(n + 1, dtype=torch.int32, device="cuda")
    lists = torch.empty((3, n + 1), dtype=torch.int32, device="cuda")  # one row of padding
    qkv = torch.zeros((n + 1, (heads + 2 * kv) * hd), device="cuda")
    q_out, out = torch.full((n + 1, heads * hd), 9.0, device="cuda"), torch.full((n + 1, heads * hd), 9.0, device="cuda")
    cache, dt = [dev(torch, x) for x in (*codes, *scales)], dev(torch, turns)
    start = [t.clone() for t in cache]
    nbytes = lib.muyo_paged_attention_decode_q8kv_workspace_bytes(n + 1, heads, kv, hd)
    space = torch.empty(nbytes, dtype=torch.uint8, device="cuda")

    def step():
        torch.add(d["lengths"], 1, out=targets)
        mh.check(lib.muyo_paged_plan(
            d["lengths"].data_ptr(), targets.data_ptr(), n, d["tables"].data_ptr(), width, d["ring"].data_ptr(),
            d["pool"].data_ptr(), pages, size, n + 1, d["lengths"].data_ptr(), d["pool"].data_ptr(),
            starts.data_ptr(), lists[0].data_ptr(), lists[1].data_ptr(), lists[2].data_ptr(), stream(torch)))
        q, k, v = (qkv.data_ptr() + 4 * hd * i for i in (0, heads, heads + kv))
        stride = qkv.shape[1]
        mh.check(lib.muyo_paged_rope_append_q8kv(
            q, k, v, stride, stride, stride, q_out.data_ptr(), *(t.data_ptr() for t in cache), lists[1].data_ptr(),
            lists[2].data_ptr(), n + 1, heads, kv, hd, pages, size, form, 0, hd, dt.data_ptr(), 1.0, stream(torch)))
        mh.check(lib.muyo_paged_attention_decode_q8kv(
            q_out.data_ptr(), *(t.data_ptr() for t in cache), out.data_ptr(), d["tables"].data_ptr(), n, width,
            lists[0].data_ptr(), lists[1].data_ptr(), n + 1, heads, kv, hd, pages, size, form, 0, 0.125,
            space.data_ptr(), nbytes, stream(torch)))

    saved = {k: t.clone() for k, t in d.items()}
    step()  # once eagerly, then back to the start
    torch.cuda.synchronize()
    for k, t in saved.items():
        d[k].copy_(t)
    for t, was in zip(cache, start):
        t.copy_(was)
    out.fill_(9.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for replay in range(20):
        rows = rng.normal(0, 1, (n + 1, qkv.shape[1])).astype(np.float32)
        qkv.copy_(dev(torch, rows))
        want = plan_reference(lengths, lengths + 1, tables, ring, pool, size, n + 1)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(lists), want["lists"]), replay
        lengths, tables, ring, pool = want["granted"], want["tables"], want["free_pages"], want["pool_out"].tolist()
        positions, slots = want["lists"][1], want["lists"][2]
        rows = rows.reshape(n + 1, heads + 2 * kv, hd)
        q, _ = rotate64(rows[:, :heads], positions, turns, 1.0, 0, hd)
        k, _ = rotate64(rows[:, heads:heads + kv], positions, turns, 1.0, 0, hd)
        for t in range(n):
            at = (slots[t] // size, slice(None), slots[t] % size)
            for i, x in enumerate((k[t], rows[t, heads + kv:])):
                codes[i][at], scales[i][at] = quantise(x, form)
        for got, x in zip(cache, (*codes, *scales)):
            assert np.array_equal(host(got), x), replay
        values = [decode(c, form) * s.astype(np.float64)[..., None] for c, s in zip(codes, scales)]
        got = host(out).reshape(n + 1, heads, hd)
        for t in range(n):
            ref = attend64(q[t], *values, tables[t], int(positions[t]), 0, 0.125)
            assert np.linalg.norm(got[t] - ref) <= ATTENTION_RTOL * np.linalg.norm(ref), (replay, t)
        assert (got[n] == 9.0).all() and (host(q_out)[n] == 9.0).all()  # the padding row
