"""Attention over a shared prefix and each query's own keys on the GPU against its definition in 64 bits on the host,
to the tolerance of the attention over own keys (4e-6 of a 2-norm over an output, from the same roundings)."""
import numpy as np
import pytest

from test_paged_gpu import (ATTENTION_RTOL, LAYOUTS, U, Attend, dev, host, plan_reference, plan_state, rotate64, stream,
                            with_sinks)

pytestmark = pytest.mark.gpu


def rows_of(caches, table, count):
    """K and V [keys][kv][hd] of a row's first `count` keys, in 64 bits; those without a page left out."""
    pages, _, size, _ = caches[0].shape
    keys = np.arange(min(count, len(table) * size))
    keys = keys[(table[keys // size] >= 0) & (table[keys // size] < pages)]
    return [c[table[keys // size], :, keys % size].astype(np.float64) for c in caches]


def attend_rows(q, k, v, scale):
    heads, hd = q.shape
    out = np.zeros((heads, hd))
    if len(k):
        for h in range(heads):
            g = h // (heads // k.shape[1])
            s = k[:, g] @ q[h].astype(np.float64) * scale
            p = np.exp(s - s.max())
            out[h] = (p / p.sum()) @ v[:, g]
    return out


class Shared(Attend):
    """A batch whose sequences go on from the last row of the tables, `prefix` keys long."""

    def __init__(self, mh, torch, rng, heads, kv, hd, size, positions, prefix, sequence=None, **more):
        n = len(positions)
        sequence = np.arange(n) if sequence is None else np.asarray(sequence)
        rows = int(max(sequence.max(), 0)) + 1
        super().__init__(mh, torch, rng, heads, kv, hd, size, np.append(positions, prefix - 1),
                         sequence=np.append(sequence, rows), **more)
        self.q, self.sequence, self.positions = self.q[:n], self.sequence[:n], self.positions[:n]
        self.prefix = np.array([rows, prefix])

    def poison_unseen(self, window=0):
        """NaN and infinities wherever no query looks."""
        size = self.shape[3]
        seen = np.zeros((self.pages, size), bool)
        for s, p in [*zip(self.sequence, self.positions), (self.prefix[0], self.prefix[1] - 1)]:
            if s >= 0 and p >= 0:
                j = np.arange(min(p + 1, self.width * size))
                seen[self.tables[s, j // size], j % size] = True
        for cache in self.caches:
            view = cache.transpose(0, 2, 1, 3)
            view[~seen] = np.resize(np.array([np.nan, np.inf, -np.inf], np.float16), view[~seen].shape)

    def call(self, window=0, where=None, out=None):
        assert window == 0
        torch, lib = self.torch, self.mh.load()
        heads, kv, hd, size = self.shape
        if where is None:
            self.d = [dev(torch, x) for x in (self.q, *self.caches, self.tables.astype(np.int32),
                                              self.sequence.astype(np.int32), self.positions.astype(np.int32),
                                              self.prefix.astype(np.int32))]
            self.nbytes = lib.muyo_paged_attention_prefix_f16kv_workspace_bytes(len(self.q), heads, kv, hd)
            self.space = torch.full((self.nbytes + 256,), 0x5A, dtype=torch.uint8, device="cuda")
        if out is None:
            out = torch.full((len(self.q), heads, hd), 9.0, device="cuda")
        q, k, v, tables, sequence, positions, prefix = self.d
        self.mh.check(lib.muyo_paged_attention_prefix_f16kv(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), tables.data_ptr(), self.tables.shape[0],
            self.width, sequence.data_ptr(), positions.data_ptr(), len(self.q), prefix.data_ptr(), heads, kv, hd,
            self.pages, size, self.scale, self.space.data_ptr(), self.nbytes, stream(torch)))
        return out

    def compare(self, got, window=0, rtol=ATTENTION_RTOL, some=None):
        sound = 0 <= self.prefix[0] < len(self.tables) and self.prefix[1] > 0
        k0, v0 = rows_of(self.caches, self.tables[self.prefix[0] if sound else 0], int(self.prefix[1]) if sound else 0)
        for i in range(len(self.q)) if some is None else some:
            s, p = self.sequence[i], int(self.positions[i])
            if not 0 <= s < len(self.tables):
                assert (got[i] == 9.0).all(), i
                continue
            k1, v1 = rows_of(self.caches, self.tables[s], max(0, p + 1))
            want = attend_rows(self.q[i], np.concatenate([k0, k1]), np.concatenate([v0, v1]), self.scale)
            assert np.isfinite(got[i]).all(), i
            assert np.linalg.norm(got[i] - want) <= rtol * np.linalg.norm(want), (i, p)


@pytest.mark.parametrize("heads, kv, hd", LAYOUTS)
def test_all_head_layouts(mh, gpu, heads, kv, hd):
    """Own keys around pages and tiles, none among them; everything unseen is poisoned."""
    rng = np.random.default_rng(heads * hd)
    positions = np.array([-1, 0, 1, 14, 15, 16, 31, 32, 63, 64, 127, 128, 300, 1000])
    batch = Shared(mh, gpu, rng, heads, kv, hd, 16, rng.permutation(positions), 777)
    batch.poison_unseen()
    batch.check()


@pytest.mark.parametrize("size", [16, 64, 1024])
@pytest.mark.parametrize("prefix", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 1000, 5003])
def test_prefix_lengths(mh, gpu, size, prefix):
    rng = np.random.default_rng(size + prefix)
    for heads, kv, hd in ((14, 2, 64), (28, 4, 128)):
        batch = Shared(mh, gpu, rng, heads, kv, hd, size, np.array([0, 40, 99, -1, 7]), prefix)
        batch.poison_unseen()
        batch.check()


@pytest.mark.parametrize("queries", [1, 4, 5, 9, 18, 19, 37, 100, 400])
def test_numbers_of_queries(mh, gpu, queries):
    """Rows that fill a wave, a workgroup and several, and do not."""
    rng = np.random.default_rng(queries)
    for heads, kv, hd in ((14, 2, 64), (28, 4, 128)):
        batch = Shared(mh, gpu, rng, heads, kv, hd, 32, rng.integers(0, 200, queries), 1500)
        batch.poison_unseen()
        out = batch.call()
        gpu.cuda.synchronize()
        assert (host(batch.space)[batch.nbytes:] == 0x5A).all()
        batch.compare(host(out), some=np.unique(np.r_[:min(queries, 12), rng.integers(0, queries, 12), queries - 1]))


def test_long_prefixes_and_own_keys(mh, gpu):
    rng = np.random.default_rng(6)
    for heads, kv, hd, positions, prefix in ((28, 4, 128, [5000, 3, 1500], 20011), (14, 2, 64, [9000], 32768),
                                             (14, 2, 64, [2000] * 20, 12345), (64, 64, 64, [100, 3000], 2500)):
        batch = Shared(mh, gpu, rng, heads, kv, hd, 64, np.array(positions), prefix)
        batch.poison_unseen()
        batch.check()


def test_padding_bad_pages_and_missing_prefixes(mh, gpu):
    """Padding rows stay, pages outside the cache and keys past the table are left out, and without a prefix the
    result is that of the own keys, which may be none (0)."""
    rng = np.random.default_rng(9)
    for heads, kv, hd in ((14, 2, 64), (28, 4, 128)):
        sequence = np.array([0, -1, 1, 2, 99, 2, 3, 3, -2 ** 31])
        positions = np.array([40, 7, -1, 100, 3, 101, 300, 17, 5])
        batch = Shared(mh, gpu, rng, heads, kv, hd, 16, positions, 500, sequence=np.minimum(sequence, 3))
        batch.sequence = sequence
        batch.tables[3, [1, 5, 18]] = [-1, batch.pages, -2 ** 31]
        batch.tables[4, [0, 3, 17, 30, 31]] = [-1, batch.pages, 2 ** 31 - 1, -7, -1]  # of the prefix
        batch.check()
        for prefix in ([4, 0], [4, -5], [-1, 500], [5, 500], [2 ** 31 - 1, 500], [-2 ** 31, 500]):
            batch.prefix = np.array(prefix)
            out = host(batch.check())
            assert (out[2] == 0).all()
        batch.prefix = np.array([4, 2 ** 31 - 1])  # past the table: its whole row
        batch.tables[4, 32:] = -1
        batch.check()
        batch.tables[4, :] = -1                    # a prefix whose every page is missing
        out = host(batch.check())
        assert (out[2] == 0).all()


def test_a_prefix_of_poisoned_neighbours(mh, gpu):
    """Missing pages among seen ones, and page 0 (which stands in for them) full of NaN."""
    rng = np.random.default_rng(10)
    for heads, kv, hd in ((14, 2, 64), (28, 4, 128)):
        batch = Shared(mh, gpu, rng, heads, kv, hd, 16, np.array([33, 5]), 400)
        for row, column in ((2, 0), (2, 5), (2, 24), (0, 1)):
            batch.tables[row, column] = -1
        batch.tables[batch.tables == 0] = -1
        batch.caches[:, 0] = np.nan
        batch.check()


def test_large_small_and_negative_scales(mh, gpu):
    rng = np.random.default_rng(12)
    for q_std, scale in ((1e6, 1e-7), (1e-6, 1e5), (1e-20, 1e19), (1e20, 1e-21), (0.0, 1.0), (30.0, 0.125), (2.0, -0.125),
                         (2.0, 0.0)):
        batch = Shared(mh, gpu, rng, 14, 2, 64, 16, np.array([0, 33, 500]), 300, q_std=q_std)
        batch.scale = scale
        # Scores of a standard deviation of 2, as elsewhere, at q_std * scale = 1 / 4; larger ones have larger
        # roundings, which are errors of the weights.
        batch.check(rtol=ATTENTION_RTOL * max(1.0, 4 * q_std * abs(scale)))


@pytest.mark.parametrize("heads, kv, hd", [(14, 2, 64), (28, 4, 128), (16, 1, 128)])
@pytest.mark.parametrize("value", [0.0, 0.01, 1.0])
def test_a_key_that_has_most_of_the_weight(mh, gpu, heads, kv, hd, value):
    """One key up to 20 nats above the others, among a query's own or in the prefix, with a value row that is 0, small or
    ordinary: the output is that of the many small weights. A score of S is off by some 4 u S, where 10 was taken
    for S."""
    rng = np.random.default_rng(hd + heads)
    nats = np.array([20.0, 8.0, 17.0, 14.0, 12.0, 0.0])
    batch = Shared(mh, gpu, rng, heads, kv, hd, 16, np.array([100, 300, 1000, 20, 2000, 64]), 3000)
    with_sinks(batch, rng, nats, value)
    batch.check(rtol=ATTENTION_RTOL * 2.0)
    # In the prefix a key can have that score for one query's heads.
    for which in range(3):
        batch = Shared(mh, gpu, rng, heads, kv, hd, 16, np.array([100, 300, -1]), 3000)
        key = [0, 1700, 2999][which]
        at = batch.tables[batch.prefix[0], key // 16], slice(None), key % 16
        for g, q in enumerate(batch.q[which].astype(np.float64).reshape(kv, heads // kv, hd)):
            batch.caches[0][at][g] = np.linalg.pinv(q) @ np.full(heads // kv, nats[which] / batch.scale)
        batch.caches[1][at] = rng.normal(0, value, (kv, hd))
        batch.check(rtol=ATTENTION_RTOL * 2.0)


@pytest.mark.parametrize("heads, kv, hd", [(14, 2, 64), (28, 4, 128), (16, 1, 128)])
@pytest.mark.parametrize("value, spread", [(0.0, 0.1), (0.01, 0.1), (0.0, 1.0)])
def test_small_weights_as_in_the_attention_over_own_keys(mh, gpu, heads, kv, hd, value, spread):
    """Its test of a key with most of the weight, at its tolerance, with that key a query's own or the prefix's."""
    rng = np.random.default_rng(hd + heads)
    nats = np.array([20.0, 8.0, 17.0, 14.0, 12.0, 0.0])
    batch = Shared(mh, gpu, rng, heads, kv, hd, 16, np.array([100, 300, 1000, 20, 2000, 64]), 3000)
    batch.caches[0] *= np.float16(spread)
    with_sinks(batch, rng, nats, value)
    out = batch.call()
    gpu.cuda.synchronize()
    for i in range(len(nats)):
        batch.compare(host(out), rtol=ATTENTION_RTOL * max(1.0, nats[i] / 10), some=[i])
    for which in range(3):
        batch = Shared(mh, gpu, rng, heads, kv, hd, 16, np.array([100, 300, -1]), 3000)
        batch.caches[0] *= np.float16(spread)
        key = [0, 1700, 2999][which]
        at = batch.tables[batch.prefix[0], key // 16], slice(None), key % 16
        for g, q in enumerate(batch.q[which].astype(np.float64).reshape(kv, heads // kv, hd)):
            batch.caches[0][at][g] = np.linalg.pinv(q) @ np.full(heads // kv, nats[which] / batch.scale)
        batch.caches[1][at] = rng.normal(0, value, (kv, hd))
        out = batch.call()
        gpu.cuda.synchronize()
        batch.compare(host(out), rtol=ATTENTION_RTOL * max(1.0, nats[which] / 10), some=[which])


@pytest.mark.parametrize("q_std, scale", [(2.0, 1e9), (2.0, -1e12), (2.0, 3e38), (1e20, 1e25), (1e-20, 1e38)])
def test_scores_far_past_any_exponent(mh, gpu, q_std, scale):
    """The largest score's value is the output, but for the weights' planes and the joins' products, and keys that are
    all the same share the weight."""
    for heads, kv, hd in ((14, 2, 64), (28, 4, 128)):
        batch = Shared(mh, gpu, np.random.default_rng(5), heads, kv, hd, 64, np.array([900, 40, 7]), 1500, q_std=q_std)
        batch.scale = scale
        k0, _ = rows_of(batch.caches, batch.tables[3], 1500)
        for i, p in enumerate(batch.positions):  # no close second: a score's roundings are some 2^-20 of these
            k = np.concatenate([k0, rows_of(batch.caches, batch.tables[i], p + 1)[0]])
            scores = np.einsum("hd,khd->hk", batch.q[i] / q_std, np.repeat(k, heads // kv, 1)) * np.sign(scale)
            scores = np.sort(scores, 1)
            assert not ((scores[:, -1] - scores[:, -2]) < 1e-4 * scores[:, -1]).any()
        # The planes' rounding (u), a reciprocal and two divisions with their products (u / 2 to u each).
        batch.check(rtol=8 * U)
        batch.caches[:] = batch.caches[:, :1, :, :1]
        batch.check()


def test_in_place_twice_and_on_other_streams(mh, gpu):
    torch, rng = gpu, np.random.default_rng(33)
    batches = [Shared(mh, gpu, rng, 28, 4, 128, 16, rng.integers(0, 2000, 12), 3001),
               Shared(mh, gpu, rng, 14, 2, 64, 64, rng.integers(0, 900, 50), 700)]
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


def test_past_four_gigabytes_of_cache(mh, gpu):
    torch, rng = gpu, np.random.default_rng(14)
    heads, kv, hd, size = 28, 4, 128, 64
    pages = 2 ** 32 // (kv * size * hd) + 40
    batch = Shared(mh, gpu, rng, heads, kv, hd, size, np.array([400, 63]), 1000, spare=0)
    caches = [torch.empty((pages, kv, size, hd), dtype=torch.float16, device="cuda") for _ in range(2)]
    for i in range(2):
        caches[i][pages - batch.pages:] = dev(torch, batch.caches[i]).flip(0)
    batch.call()  # the small cache, for its buffers
    torch.cuda.synchronize()
    small, real = batch.tables, batch.pages
    batch.d[1:3] = caches
    batch.d[3] = dev(torch, np.where(small >= 0, pages - 1 - small, -1).astype(np.int32))
    batch.pages = pages
    out = batch.call(where=True)
    torch.cuda.synchronize()
    batch.pages = real
    batch.compare(host(out))


def test_more_queries_than_are_scanned(mh, gpu):
    """Shares whose sums a kernel of its own makes, and a last sequence that shares cut."""
    rng = np.random.default_rng(21)
    positions = rng.integers(-1, 60, 1300)
    positions[[3, 700, 1299]] = [1400, 1100, 2047]
    for heads, kv, hd in ((14, 2, 64), (28, 4, 128)):
        batch = Shared(mh, gpu, rng, heads, kv, hd, 16, positions, 90)
        batch.poison_unseen()
        out = batch.call()
        gpu.cuda.synchronize()
        batch.compare(host(out), some=np.r_[:8, 700, rng.integers(0, 1300, 12), 1298, 1299])


def test_the_largest_batch(mh, gpu):
    """65535 queries of 264 heads: more workgroups than a dimension of a launch takes."""
    torch, rng = gpu, np.random.default_rng(22)
    heads, hd, n = 264, 64, 65535
    small = np.array([5, 0, -1, 17, 30])
    batch = Shared(mh, torch, rng, heads, heads, hd, 16, small, 20)
    batch.poison_unseen()
    batch.call()
    batch.d[0] = torch.randn((n, heads, hd), device="cuda")
    which = np.arange(n) % len(small)
    some = np.r_[:6, 4095:4100, rng.integers(0, n, 6), n - 6:n]
    batch.sequence, batch.positions = batch.sequence[which], batch.positions[which]
    batch.d[4], batch.d[5] = (dev(torch, x.astype(np.int32)) for x in (batch.sequence, batch.positions))
    batch.q = np.zeros((n, 1))
    batch.nbytes = mh.load().muyo_paged_attention_prefix_f16kv_workspace_bytes(n, heads, heads, hd)
    batch.space = torch.empty(batch.nbytes, dtype=torch.uint8, device="cuda")
    out = batch.call(where=True)
    torch.cuda.synchronize()
    pick = torch.from_numpy(some).cuda()
    batch.q, got = host(batch.d[0][pick]), host(out[pick])
    batch.sequence, batch.positions = batch.sequence[some], batch.positions[some]
    batch.compare(got)


def test_a_steps_operators_in_one_graph(mh, gpu):
    """Plan, append, attention and sampling of chats that share a prompt, captured together and replayed: the prompt is
    a sequence of the plan with its own pages, the chats' rope positions go on behind it."""
    torch, rng, lib = gpu, np.random.default_rng(21), mh.load()
    heads, kv, hd, size, pages, width, n, prompt, vocab = 14, 2, 64, 16, 200, 40, 6, 333, 500
    lengths = np.array([0, 15, 16, 40, 200, prompt])  # the last row is the prompt's
    tables, ring, pool = plan_state(rng, lengths, width, size, pages - sum(-(-lengths // size)))
    turns, _ = mh.rope_frequencies(1e6, hd)
    caches = rng.normal(0, 1, (2, pages, kv, size, hd)).astype(np.float16)
    d = {k: dev(torch, np.asarray(v, dtype=np.int32)) for k, v in dict(
        lengths=lengths, tables=tables, ring=ring, pool=pool, prefix=[n - 1, prompt], grow=[1] * (n - 1) + [0]).items()}
    targets, starts = (torch.empty(n + i, dtype=torch.int32, device="cuda") for i in (0, 1))
    lists = torch.empty((3, n), dtype=torch.int32, device="cuda")  # the chats' tokens and one row of padding
    rope_positions = torch.empty(n, dtype=torch.int32, device="cuda")
    qkv = torch.zeros((n, (heads + 2 * kv) * hd), device="cuda")
    q_out, out = torch.full((n, heads * hd), 9.0, device="cuda"), torch.full((n, heads * hd), 9.0, device="cuda")
    dc, dt = [dev(torch, c) for c in caches], dev(torch, turns)
    nbytes = lib.muyo_paged_attention_prefix_f16kv_workspace_bytes(n, heads, kv, hd)
    space = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    head = dev(torch, rng.normal(0, 0.5, (vocab, heads * hd)).astype(np.float16))
    planes = torch.empty((2, n, heads * hd), dtype=torch.float16, device="cuda")
    logits = torch.empty((n, vocab), device="cuda")
    top_ks = dev(torch, np.full(n, 5, np.int32))
    numbers, tokens = torch.empty(n, dtype=torch.float64, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
    more_bytes = lib.muyo_sample_rows_workspace_bytes(n, vocab)
    more = torch.empty(more_bytes, dtype=torch.uint8, device="cuda")

    def step():
        torch.add(d["lengths"], d["grow"], out=targets)
        mh.check(lib.muyo_paged_plan(
            d["lengths"].data_ptr(), targets.data_ptr(), n, d["tables"].data_ptr(), width, d["ring"].data_ptr(),
            d["pool"].data_ptr(), pages, size, n, d["lengths"].data_ptr(), d["pool"].data_ptr(), starts.data_ptr(),
            lists[0].data_ptr(), lists[1].data_ptr(), lists[2].data_ptr(), stream(torch)))
        torch.where(lists[1] < 0, lists[1], lists[1] + prompt, out=rope_positions)
        q, k, v = (qkv.data_ptr() + 4 * hd * i for i in (0, heads, heads + kv))
        stride = qkv.shape[1]
        mh.check(lib.muyo_paged_rope_append_f16kv(
            q, k, v, stride, stride, stride, q_out.data_ptr(), dc[0].data_ptr(), dc[1].data_ptr(),
            rope_positions.data_ptr(), lists[2].data_ptr(), n, heads, kv, hd, pages, size, 0, hd, dt.data_ptr(), 1.0,
            stream(torch)))
        mh.check(lib.muyo_paged_attention_prefix_f16kv(
            q_out.data_ptr(), dc[0].data_ptr(), dc[1].data_ptr(), out.data_ptr(), d["tables"].data_ptr(), n, width,
            lists[0].data_ptr(), lists[1].data_ptr(), n, d["prefix"].data_ptr(), heads, kv, hd, pages, size, 0.125,
            space.data_ptr(), nbytes, stream(torch)))
        mh.check(lib.muyo_split_f32_f16x2(out.data_ptr(), out.numel(), planes[0].data_ptr(), planes[1].data_ptr(),
                                          stream(torch)))
        mh.check(lib.muyo_gemm_split_f16(planes[0].data_ptr(), planes[1].data_ptr(), head.data_ptr(), None, None,
                                         logits.data_ptr(), n, vocab, heads * hd, stream(torch)))
        mh.check(lib.muyo_sample_rows_f32(
            logits.data_ptr(), vocab, n, vocab, None, top_ks.data_ptr(), None, None, numbers.data_ptr(),
            tokens.data_ptr(), None, more.data_ptr(), more_bytes, stream(torch)))

    saved = {k: t.clone() for k, t in d.items()}
    step()  # once eagerly, then back to the start
    torch.cuda.synchronize()
    for k, t in saved.items():
        d[k].copy_(t)
    for t, c in zip(dc, caches):
        t.copy_(dev(torch, c))
    out.fill_(9.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for replay in range(12):
        rows = rng.normal(0, 1, (n, qkv.shape[1])).astype(np.float32)
        qkv.copy_(dev(torch, rows))
        u = rng.random(n)
        numbers.copy_(dev(torch, u))
        want = plan_reference(lengths, lengths + np.r_[[1] * (n - 1), 0], tables, ring, pool, size, n)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(lists), want["lists"]), replay
        lengths, tables, ring, pool = want["granted"], want["tables"], want["free_pages"], want["pool_out"].tolist()
        positions = want["lists"][1]
        q, _ = rotate64(rows.reshape(n, heads + 2 * kv, hd)[:, :heads], positions + prompt, turns, 1.0, 0, hd)
        got, cached = host(out).reshape(n, heads, hd), [host(c) for c in dc]
        for t in range(n - 1):
            k0, v0 = rows_of(cached, tables[n - 1], prompt)
            k1, v1 = rows_of(cached, tables[want["lists"][0][t]], int(positions[t]) + 1)
            ref = attend_rows(q[t], np.concatenate([k0, k1]), np.concatenate([v0, v1]), 0.125)
            assert np.linalg.norm(got[t] - ref) <= ATTENTION_RTOL * np.linalg.norm(ref), (replay, t)
        assert (got[n - 1] == 9.0).all()  # the padding row
        x = host(logits).astype(np.float64)
        for t in range(n):
            best = np.sort(np.argsort(-x[t], kind="stable")[:5])
            mass = np.cumsum(np.exp(x[t, best] - x[t].max()))
            assert host(tokens)[t] == best[(mass <= u[t] * mass[-1]).sum()], (replay, t)
    assert lengths.tolist() == [12, 27, 28, 52, 212, prompt]
