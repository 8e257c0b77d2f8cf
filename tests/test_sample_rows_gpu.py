"""The batch sampler on the GPU against its definition in 64 bits on the host.

Tokens are equal. Weights and their sums are good to 2^-39 here and to some 2^-50 on the host, so that a given
number lands on another token with a chance of about (tokens kept) * 2^-39 * (largest weight / total): 2^-22 at
most for each row. A log probability p is good to 2^-39 before it is rounded to f32, u |p| (u = 2^-24), u more for
those near 0, whose share of the weight is rounded before the log.
"""
import math

import numpy as np
import pytest

from test_paged_gpu import dev, host, stream

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def kept_of(row, temperature, top_k, top_p, min_p):
    """(indices kept by rising index, their weights), by the definition."""
    x = np.where(np.isnan(row), -np.inf, np.minimum(row, np.finfo(np.float32).max)).astype(np.float64)
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not len(order):
        return order, np.zeros(0)
    if not temperature > 0:
        return order[:1], np.ones(1)
    with np.errstate(over="ignore"):
        w = np.exp((x[order] - x[order[0]]) / np.float64(np.float32(temperature)))
    count = min(top_k, len(order)) if top_k > 0 else len(order)
    mass = np.cumsum(w)
    if top_p < 1:
        share = np.float64(np.float32(top_p)) * mass[count - 1]
        count = min(count, max(1, int((mass - w < share).sum())))
    if min_p > 0:
        count = min(count, max(1, int((w >= np.float64(np.float32(min_p))).sum())))
    kept = np.sort(order[:count])
    back = np.empty(len(row))
    back[order] = w
    return kept, back[kept]


def sample64(row, setting, random):
    kept, w = kept_of(row, *setting)
    if not len(kept):
        return -1, -math.inf
    mass = np.cumsum(w)
    at = min(int((mass <= max(random, 0.0) * mass[-1]).sum()), int(np.flatnonzero(w > 0)[-1]))
    return int(kept[at]), math.log(w[at] / mass[-1])


class Batch:
    def __init__(self, mh, torch, logits, settings, randoms, stride=None, off=()):
        self.mh, self.torch, self.logits, self.off = mh, torch, logits.astype(np.float32), off
        rows, self.vocab = logits.shape
        self.stride = stride or self.vocab
        wide = np.full((rows, self.stride), 1e9, np.float32)  # what lies between rows is no logit
        wide[:, :self.vocab] = self.logits
        self.settings, self.randoms = settings, np.asarray(randoms, np.float64)
        columns = [np.asarray(c) for c in zip(*settings)]
        self.d = [dev(torch, wide), *(None if i in off else dev(torch, c.astype(t)) for i, (c, t) in enumerate(
            zip(columns, (np.float32, np.int32, np.float32, np.float32)))), dev(torch, self.randoms)]
        defaults = (1.0, 0, 1.0, 0.0)
        self.settings = [tuple(defaults[i] if i in off else v for i, v in enumerate(s)) for s in settings]
        self.tokens = torch.full((rows + 3,), 77, dtype=torch.int32, device="cuda")
        self.logprobs = torch.full((rows + 3,), 77.0, device="cuda")
        self.nbytes = mh.load().muyo_sample_rows_workspace_bytes(rows, self.vocab)
        self.space = torch.full((self.nbytes + 256,), 0x5A, dtype=torch.uint8, device="cuda")

    def call(self, logprobs=True):
        ptr = [None if t is None else t.data_ptr() for t in self.d]
        self.mh.check(self.mh.load().muyo_sample_rows_f32(
            ptr[0], self.stride, len(self.logits), self.vocab, *ptr[1:6], self.tokens.data_ptr(),
            self.logprobs.data_ptr() if logprobs else None, self.space.data_ptr(), self.nbytes, stream(self.torch)))

    def check(self):
        self.call()
        self.torch.cuda.synchronize()
        self.compare()

    def compare(self):
        rows = len(self.logits)
        tokens, logprobs = host(self.tokens), host(self.logprobs)
        assert (tokens[rows:] == 77).all() and (logprobs[rows:] == 77).all()
        assert (host(self.space)[self.nbytes:] == 0x5A).all()
        for r in range(rows):
            token, lp = sample64(self.logits[r], self.settings[r], self.randoms[r])
            assert tokens[r] == token, (r, self.settings[r], self.randoms[r], tokens[r], token)
            if math.isinf(lp):
                assert logprobs[r] == lp
            else:
                assert abs(logprobs[r] - lp) <= 2 * U * max(1.0, abs(lp)), (r, logprobs[r], lp)


SETTINGS = [
    (1.0, 0, 1.0, 0.0), (0.7, 40, 0.95, 0.0), (1.0, 0, 0.9, 0.0), (0.0, 5, 0.5, 0.5), (-1.0, 0, 1.0, 0.0),
    (1.0, 1, 1.0, 0.0), (1.5, 100, 1.0, 0.02), (0.3, 0, 0.999, 0.0), (1.0, 0, 1.0, 0.05), (2.0, 7, 0.3, 0.9),
    (1.0, 0, 0.0, 0.0), (1.0, 0, -1.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 2.0), (0.05, 3, 0.8, 0.0),
    (10.0, 10 ** 9, 0.97, 0.0001), (1.0, 2000, 0.99, 0.0), (math.inf, 0, 0.5, 0.0), (1e-30, 0, 0.9, 0.1),
    (1e30, 0, 1.0, 0.0), (1.0, -5, 1.5, -1.0), (math.nan, 3, 0.5, 0.0),
]


def logits_of(rng, rows, vocab, std=2.5):
    x = rng.normal(0, std, (rows, vocab))
    if vocab > 40:
        for row in x:
            row[rng.integers(0, vocab, 12)] += rng.normal(8, 4, 12)
    return x.astype(np.float32)


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 1000, 1023, 1025, 4097, 32000, 151936])
def test_settings_and_vocabularies(mh, gpu, vocab):
    rng = np.random.default_rng(vocab)
    rows = len(SETTINGS)
    Batch(mh, gpu, logits_of(rng, rows, vocab), SETTINGS, rng.random(rows)).check()


@pytest.mark.parametrize("rows, vocab", [(1, 152064), (2, 151937), (64, 20000), (300, 5003), (1700, 999), (3000, 40),
                                         (1, 1), (5, 2), (7, 3), (4095, 7)])
def test_rows(mh, gpu, rows, vocab):
    """From many workgroups a row to one."""
    rng = np.random.default_rng(rows)
    settings = [SETTINGS[i] for i in rng.integers(0, len(SETTINGS), rows)]
    Batch(mh, gpu, logits_of(rng, rows, vocab), settings, rng.random(rows), stride=vocab + 5).check()


@pytest.mark.parametrize("vocab", [1, 70, 1501, 4999])
def test_thousands_of_rows(mh, gpu, vocab):
    """More rows than get workgroups of their own for their lists, the first of them also in a call that has these."""
    rng = np.random.default_rng(vocab)
    rows = 4100
    settings = [SETTINGS[i] for i in rng.integers(0, len(SETTINGS), rows)]
    x = logits_of(rng, 41, vocab)[rng.integers(0, 41, rows)]
    x[rng.random(rows) < 0.05] = -np.inf
    randoms = rng.random(rows)
    batch = Batch(mh, gpu, x, settings, randoms, stride=vocab + 3)
    batch.check()
    less = Batch(mh, gpu, x[:4096], settings[:4096], randoms[:4096], stride=vocab + 1)
    less.call()
    gpu.cuda.synchronize()
    assert np.array_equal(host(less.tokens)[:4096], host(batch.tokens)[:4096])


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_logits_that_begin_anywhere(mh, gpu, shift):
    """Rows at any multiple of four bytes."""
    torch, rng = gpu, np.random.default_rng(shift)
    for rows, vocab, stride in ((22, 5001, 5001), (22, 151936, 151937), (3, 3, 7)):
        batch = Batch(mh, torch, logits_of(rng, rows, vocab), SETTINGS[:rows], rng.random(rows), stride=stride)
        wide = torch.full((rows * stride + 8,), 1e9, device="cuda")
        wide[shift:shift + rows * stride] = batch.d[0].flatten()
        batch.d[0] = wide[shift:]
        batch.check()


def test_results_between_rows_of_logits(mh, gpu):
    torch, rng = gpu, np.random.default_rng(11)
    rows, vocab = 22, 4999
    batch = Batch(mh, torch, logits_of(rng, rows, vocab), SETTINGS, rng.random(rows), stride=vocab + 60)
    wide = batch.d[0].flatten()
    before = host(wide).copy()
    first, second = vocab + 2, 3 * (vocab + 60) + vocab + 1
    batch.tokens, batch.logprobs = wide[first:first + rows].view(torch.int32), wide[second:second + rows]
    batch.call()
    torch.cuda.synchronize()
    after = host(wide)
    changed = np.flatnonzero(after.view(np.uint32) != before.view(np.uint32))
    assert np.isin(changed, np.r_[first:first + rows, second:second + rows]).all()
    for r in range(rows):
        token, lp = sample64(batch.logits[r], SETTINGS[r], batch.randoms[r])
        assert after[first + r].view(np.int32) == token
        assert abs(after[second + r] - lp) <= 2 * U * max(1.0, abs(lp))


def test_settings_that_are_off(mh, gpu):
    rng = np.random.default_rng(2)
    settings = [(0.6, 9, 0.8, 0.1)] * 8
    for off in ((0,), (1,), (2,), (3,), (0, 1, 2, 3)):
        Batch(mh, gpu, logits_of(rng, 8, 3001), settings, rng.random(8), off=off).check()
    batch = Batch(mh, gpu, logits_of(rng, 8, 3001), settings, rng.random(8))
    batch.call(logprobs=False)
    gpu.cuda.synchronize()
    assert (host(batch.logprobs) == 77).all()
    batch.check()


@pytest.mark.parametrize("step", [0.0, 0.0625, 0.5, 8.0])
@pytest.mark.parametrize("vocab", [700, 9000, 70000])
def test_equal_logits(mh, gpu, vocab, step):
    """Logits of few values (as widened bf16 has them): cuts fall among equal ones, the lowest index first; in
    steps of more than a listing holds, too."""
    rng = np.random.default_rng(vocab)
    settings = [s for s in SETTINGS if s[0] == s[0]] + [(1.0, vocab // 2, 0.5, 0.0), (0.8, vocab - 3, 1.0, 0.0),
                                                        (1.0, 0, 0.25, 0.0), (3.0, vocab // 3, 0.9, 0.5)]
    x = rng.normal(0, 2, (len(settings), vocab))
    x = np.round(x / step) * step if step else np.zeros_like(x)
    Batch(mh, gpu, x, settings, rng.random(len(settings))).check()


@pytest.mark.parametrize("std", [1.0, 0.3, 0.01, 1e-4])
def test_flat_rows(mh, gpu, std):
    """Tens of thousands of logits in the steps of the cuts, few of them equal."""
    rng = np.random.default_rng(int(1 / std))
    more = [(1.0, 30000, 1.0, 0.0), (1.0, 30000, 0.5, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 0, 0.999, 0.0), (1.0, 0, 1.0, 0.7),
            (0.9, 40000, 0.9, 0.5), (2.0, 69999, 0.9999, 0.0), (1.0, 0, 1e-6, 0.0), (1.0, 5000, 0.99, 0.001)]
    settings = SETTINGS + more
    rows = len(settings)
    x = rng.normal(0, std, (rows, 70000)).astype(np.float32)
    Batch(mh, gpu, x, settings, rng.random(rows)).check()
    x[:, ::3] = -np.inf
    batch = Batch(mh, gpu, np.tile(x, (9, 1)), settings * 9, rng.random(9 * rows))
    batch.check()


@pytest.mark.parametrize("vocab", [61, 4000, 4096, 4150, 4300])
def test_equal_logits_at_tiny_temperatures(mh, gpu, vocab):
    """Places so far out that what a step leaves of them is any number: as many as a list holds, and more."""
    rng = np.random.default_rng(vocab)
    x = np.repeat(rng.normal(0, 3, (24, 1)), vocab, 1)
    settings = [(1e-20, 0, 1.0, 0.0), (1e-18, 0, 0.9, 0.0), (1e-25, 4140, 1.0, 0.0), (1e-20, 0, 1.0, 0.5)] * 6
    Batch(mh, gpu, x, settings, rng.random(24)).check()


def test_masked_infinite_and_missing_logits(mh, gpu):
    rng = np.random.default_rng(4)
    vocab = 5000
    base = logits_of(rng, 9, vocab)
    base[0] = -np.inf                       # a mask that leaves nothing
    base[1] = np.nan
    base[2, rng.random(vocab) < 0.99] = -np.inf
    base[3, :] = -np.inf
    base[3, 4321] = -7.0                    # and one that leaves one
    base[4, [17, 40, 4000]] = np.inf
    base[5, rng.random(vocab) < 0.5] = np.nan
    base[6] = -np.finfo(np.float32).max     # the type's lowest value as a mask
    base[6, [5, 99]] = [1.0, 0.5]
    base[7] = -np.finfo(np.float32).max
    base[8, ::2] = np.finfo(np.float32).max
    for setting in SETTINGS:
        Batch(mh, gpu, base, [setting] * 9, rng.random(9)).check()


def test_given_numbers(mh, gpu):
    """0, the last below 1, and numbers outside of [0, 1); the numbers of a fine row of them share the tokens out by
    their weights."""
    rng = np.random.default_rng(5)
    edge = [0.0, -0.0, -3.0, math.nan, np.nextafter(1.0, 0.0), 1.0, 7.5, math.inf, 5e-324, 0.5]
    x = np.repeat(logits_of(rng, 1, 2011), len(edge), 0)
    for setting in ((1.0, 0, 1.0, 0.0), (0.7, 40, 0.95, 0.0), (2.0, 0, 0.9, 0.01)):
        batch = Batch(mh, gpu, x, [setting] * len(edge), edge)
        batch.randoms = np.array([0.0 if not e > 0 else min(e, 1.0) for e in edge])
        batch.check()
    n = 4000
    x = np.repeat(np.array([[0.0, 1.0, -1.0, 2.0, 0.5, -np.inf, 3.0]]), n, 0)
    batch = Batch(mh, gpu, x, [(0.9, 0, 1.0, 0.0)] * n, (np.arange(n) + 0.5) / n)
    batch.check()
    p = np.exp(x[0] / np.float64(np.float32(0.9)))
    counts = np.bincount(host(batch.tokens)[:n], minlength=7)
    assert (np.abs(counts / n - p / p.sum()) <= 1.0 / n).all()  # a border's place between two numbers


def test_a_large_vocabulary(mh, gpu):
    """2^21 + 7 logits in few and in many workgroups of a row."""
    rng = np.random.default_rng(6)
    vocab = 2 ** 21 + 7
    settings = [(1.0, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (0.7, 40, 0.95, 0.0)]
    Batch(mh, gpu, logits_of(rng, 3, vocab), settings, [0.9999, 0.3, 0.6]).check()
    x = np.repeat(logits_of(rng, 1, vocab), 3, 0)
    few = Batch(mh, gpu, x, settings, [1.0 - 2.0 ** -53, 0.7, 0.2])
    few.check()


def test_the_largest_vocabulary(mh, gpu):
    """2^24 logits, of a few values so that steps hold millions, and of as many as there are."""
    rng = np.random.default_rng(8)
    x = rng.normal(0, 1, (2, 2 ** 24)).astype(np.float32)
    x[0] = np.round(x[0])
    Batch(mh, gpu, x, [(1.0, 0, 0.97, 0.0), (1.0, 5000, 0.8, 0.0)], [0.6, 0.7]).check()


@pytest.mark.parametrize("rows, vocab, stride", [(5, 5003, 2 ** 29 + 3), (4101, 700, 270001)])
def test_rows_past_four_gigabytes(mh, gpu, rows, vocab, stride):
    torch, rng = gpu, np.random.default_rng(rows)
    settings = [SETTINGS[i] for i in rng.integers(0, len(SETTINGS), rows)]
    x = logits_of(rng, 41, vocab)[rng.integers(0, 41, rows)]
    batch = Batch(mh, torch, x, settings, rng.random(rows))
    wide = torch.empty((rows - 1) * stride + vocab, device="cuda")
    torch.as_strided(wide, (rows, vocab), (stride, 1)).copy_(batch.d[0])
    batch.d[0], batch.stride = wide, stride
    batch.check()


def test_the_same_twice_and_on_other_streams(mh, gpu):
    torch, rng = gpu, np.random.default_rng(7)
    batches = []
    for rows, vocab in ((5, 151936), (700, 3000)):
        settings = [SETTINGS[i] for i in rng.integers(0, len(SETTINGS), rows)]
        batches.append(Batch(mh, torch, logits_of(rng, rows, vocab), settings, rng.random(rows)))
    for b in batches:
        b.check()
    first = [host(b.logprobs).view(np.uint32).copy() for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    for _ in range(4):
        for b, s in zip(batches, streams):
            with torch.cuda.stream(s):
                b.logprobs.fill_(77.0)
                b.call()
    torch.cuda.synchronize()
    for b, bits in zip(batches, first):
        b.compare()
        assert np.array_equal(host(b.logprobs).view(np.uint32), bits)


def test_replayed_with_other_logits_and_settings(mh, gpu):
    """A captured call whose inputs change between replays, its workspace used by other calls in between."""
    torch, rng = gpu, np.random.default_rng(8)
    rows, vocab = 12, 30011
    batch = Batch(mh, torch, logits_of(rng, rows, vocab), SETTINGS[:rows], rng.random(rows))
    other = Batch(mh, torch, logits_of(rng, 3, 5000), SETTINGS[:3], rng.random(3))
    other.space = batch.space
    batch.call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch.call()
    for _ in range(5):
        batch.logits = logits_of(rng, rows, vocab, rng.uniform(0.1, 5))
        batch.settings = [SETTINGS[i] for i in rng.integers(0, len(SETTINGS), rows)]
        batch.randoms = rng.random(rows)
        columns = [np.asarray(c) for c in zip(*batch.settings)]
        for d, value in zip(batch.d, (batch.logits, *columns, batch.randoms)):
            d.copy_(dev(torch, value).to(d.dtype))
        other.call()
        graph.replay()
        torch.cuda.synchronize()
        batch.compare()


def test_agrees_with_the_log_probabilities(mh, gpu):
    """Without cuts a token's log probability is muyo_token_logprobs_f32's of the same row."""
    torch, rng, lib = gpu, np.random.default_rng(9), mh.load()
    rows, vocab = 20, 50021
    batch = Batch(mh, torch, logits_of(rng, rows, vocab), [(1.0, 0, 1.0, 0.0)] * rows, rng.random(rows))
    batch.check()
    out = torch.empty(rows, device="cuda")
    need = lib.muyo_token_logprobs_workspace_bytes(rows, vocab, 0)
    space = torch.empty(need, dtype=torch.uint8, device="cuda")
    mh.check(lib.muyo_token_logprobs_f32(batch.d[0].data_ptr(), vocab, rows, vocab, batch.tokens.data_ptr(),
                                         out.data_ptr(), None, None, 0, None, None, space.data_ptr(), need,
                                         stream(torch)))
    torch.cuda.synchronize()
    # Logits of a few units: some eight roundings of that size.
    assert np.abs(host(out) - host(batch.logprobs)[:rows]).max() <= 64 * U * np.abs(host(out)).max()


def peaked_rows(rng, rows, vocab, ties):
    """Rows whose largest logit is alone or 37 times there, 23 others the next f32 numbers below it; some have masked
    and missing logits."""
    x = rng.normal(0, 2.5, (rows, vocab)).astype(np.float32)
    for r, row in enumerate(x):
        peak = np.float32([3.3, 20.3, 1000.7, -20.3][(r // 5 + r) % 4])
        row[:] = np.minimum(row, 2.0) if peak > 0 else np.minimum(row, 2.0) - np.float32(30.0)
        if r % 3:
            row[rng.random(vocab) < 0.2] = -np.inf
            row[rng.random(vocab) < 0.1] = np.nan
        at = rng.choice(vocab, 60, replace=False)
        row[at[:37 if ties[r] else 1]] = peak
        row[at[37:]] = peak - np.spacing(peak) * np.arange(1, 24, dtype=np.float32)
    return x


@pytest.mark.parametrize("rows, vocab", [(1, 151936), (61, 151936), (500, 151936), (55, 3001), (4100, 500)])
def test_small_temperatures(mh, gpu, rows, vocab):
    """Where a unit in the last place of the largest logit is less than a step of weights, as many, and more than all
    of them."""
    rng = np.random.default_rng(rows)
    temperatures = [1e-4, 1e-5, 1e-6, 1e-7, 2e-8, 1e-8, 1e-9, 1e-10, 1e-11, 1e-12, 1e-13, 1e-14]
    cuts = [(0, 1.0, 0.0), (0, 1.0, 0.5), (0, 0.6, 0.0), (3000, 1.0, 0.0), (40, 0.9, 0.0)]
    settings = [(t, *c) for t in temperatures for c in cuts]
    for first in range(0, len(settings) if rows == 1 else 1):
        these = [settings[(first + r) % len(settings)] for r in range(rows)]
        x = peaked_rows(rng, rows, vocab, [s[2] == 0.6 or r % 2 for r, s in enumerate(these)])
        Batch(mh, gpu, x, these, rng.random(rows)).check()


# Temperatures at which the largest f32's place on a grid of eighths of an octave, cut to 32 bits, is that of ordinary
# logits.
WRAPPED = [0.037677984684705734, 0.04902310296893120, 0.07893555611371994, 0.12279371172189713, 0.17001739144325256]


@pytest.mark.parametrize("rows", [1, 61, 600])
@pytest.mark.parametrize("temperature", WRAPPED)
def test_missing_logits_are_not_large_ones(mh, gpu, temperature, rows):
    """NaN at temperatures and peaks where the largest number's place would be one that counts."""
    rng = np.random.default_rng(rows)
    per_unit = 8.0 * 1.44269504088896340736 / temperature
    assert np.float32(temperature) == temperature
    wrapped = (np.float64(np.finfo(np.float32).max) * per_unit + 1.5 * 2.0 ** 52).view(np.int64).astype(np.int32)
    cuts = [(0, 1.0, 0.0), (0, 0.9, 0.0), (3000, 1.0, 0.0), (40, 0.95, 0.0), (0, 1.0, 0.1)]
    nans = np.array([0x7FC00000, 0xFFC00000, 0x7FFFFFFF], np.uint32).view(np.float32)
    vocab = 20011
    x = rng.normal(0, 2.5, (rows, vocab)).astype(np.float32)
    for r, row in enumerate(x):
        below = (8, 9, 40, 300, 500)[r % 5]  # steps that the wrapped place is below the first one
        peak = np.float32((wrapped + below - 8) / per_unit)
        row[:] = peak - np.abs(row) * np.float32(4.0 * temperature)
        row[rng.integers(vocab)] = peak
        missing = np.flatnonzero(rng.random(vocab) < (0.0002, 0.01, 0.3)[r // 5 % 3])
        missing = missing[row[missing] != peak]
        row[missing] = np.resize(nans, len(missing))
    settings = [(temperature, *cuts[(r // 15 + r) % 5]) for r in range(rows)]
    Batch(mh, gpu, x, settings, rng.random(rows)).check()


@pytest.mark.parametrize("temperature", [1e24, 1e28, 1e33, 1e36, 1e38])
def test_infinite_and_missing_logits_at_huge_temperatures(mh, gpu, temperature):
    """The largest number, as which an infinity counts, near enough to the others for a step of its own or theirs."""
    rng = np.random.default_rng(3)
    vocab = 9001
    most = np.finfo(np.float32).max
    x = rng.normal(0, 1, (20, vocab)).astype(np.float32)
    for r, row in enumerate(x):
        row *= np.float32([1.0, 1e30, 1e36, 3e37][r % 4])
        row[rng.integers(0, vocab, 30)] = (np.inf, most)[r // 4 % 2]
        row[rng.integers(0, vocab, 2000)] = np.nan
        row[rng.integers(0, vocab, 20)] = -np.inf
    cuts = [(0, 1.0, 0.0), (0, 0.9, 0.0), (3000, 1.0, 0.0), (40, 0.95, 0.0), (0, 1.0, 0.1)]
    Batch(mh, gpu, x, [(temperature, *cuts[r // 4]) for r in range(20)], rng.random(20)).check()


@pytest.mark.parametrize("rows, vocab", [(1, 151936), (61, 20011), (700, 5003), (4100, 300)])
def test_signalling_missing_logits(mh, gpu, rows, vocab):
    """NaN of every kind before, behind and between the largest logits, in all settings."""
    rng = np.random.default_rng(rows)
    nans = np.array([0x7F800001, 0xFFBFFFFF, 0x7FC00000, 0xFFC00000, 0x7FA00000], np.uint32).view(np.float32)
    for first in range(0, len(SETTINGS) if rows == 1 else 1):
        x = logits_of(rng, rows, vocab)
        for r, row in enumerate(x):
            missing = np.flatnonzero(rng.random(vocab) < (0.001, 0.05, 0.6)[r % 3])
            row[missing] = np.resize(nans, len(missing))
            order = np.argsort(np.where(np.isnan(row), -np.inf, -row))[:40]  # and next to the largest
            row[np.minimum(order[::2] + 1, vocab - 1)] = nans[0]
        settings = [SETTINGS[(first + r) % len(SETTINGS)] for r in range(rows)]
        Batch(mh, gpu, x, settings, rng.random(rows)).check()
