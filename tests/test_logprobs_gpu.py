"""Token log probabilities, ranks, entropies and alternatives on the GPU against 64 bits on the host.

Ids and ranks are equal: they depend on the order of the given f32 logits alone. Tolerances (u = 2^-24):
a row's sum of weights is made in f32 in chains of at most vocab / 64 terms, each weight with a few
roundings of its own and one of its exponent's argument (up to `spread` = the largest distance that
still counts, 20, in log2 units 29 u), so its logarithm is good to (vocab / 64 + 64) u; x - m and the
last subtraction round at their own sizes. The entropy is the same with sums of weight times distance.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def host(t):
    return t.detach().cpu().numpy()


def run(mh, torch, x, tokens, top, stride=None, offset=0, given=True, entropy=True):
    """The call on rows `stride` apart, `offset` values into an allocation; buffers with room behind
    them, which has to stay as it is."""
    rows, vocab = x.shape
    stride = stride or vocab
    buffer = torch.full((offset + rows * stride + 8,), 1e30, device="cuda")
    view = buffer[offset:offset + rows * stride].view(rows, stride)
    view[:, :vocab] = torch.from_numpy(x).cuda()
    lib = mh.load()
    ids = torch.full((rows * top + 5,), 77, dtype=torch.int32, device="cuda")
    ranks = torch.full((rows + 5,), 77, dtype=torch.int32, device="cuda")
    logprobs, entropies = (torch.full((rows + 5,), 77.0, device="cuda") for _ in range(2))
    tops = torch.full((rows * top + 5,), 77.0, device="cuda")
    t = torch.tensor(np.asarray(tokens), dtype=torch.int32, device="cuda")
    size = lib.muyo_token_logprobs_workspace_bytes(rows, vocab, top)
    space = torch.full((size + 64,), 0x5A, dtype=torch.uint8, device="cuda")
    mh.check(lib.muyo_token_logprobs_f32(
        view.data_ptr(), stride, rows, vocab, t.data_ptr() if given else None, logprobs.data_ptr() if given else None,
        ranks.data_ptr() if given else None, entropies.data_ptr() if entropy else None, top,
        ids.data_ptr() if top else None, tops.data_ptr() if top else None, space.data_ptr(), size,
        torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert (host(space)[size:] == 0x5A).all()
    for buf, used in ((ids, rows * top), (tops, rows * top), (ranks, rows if given else 0),
                      (logprobs, rows if given else 0), (entropies, rows if entropy else 0)):
        assert (host(buf)[used:] == 77).all()
    return dict(logprobs=host(logprobs)[:rows], ranks=host(ranks)[:rows], entropy=host(entropies)[:rows],
                ids=host(ids)[:rows * top].reshape(rows, top), tops=host(tops)[:rows * top].reshape(rows, top))


def reference(x, tokens, top):
    x = x.astype(np.float64)
    m = x.max(1, keepdims=True)
    d = x - m
    e = np.exp(d)
    s = e.sum(1)
    lp = d - np.log(s)[:, None]
    order = np.argsort(-x, 1, kind="stable")
    place = np.empty_like(order)
    np.put_along_axis(place, order, np.arange(x.shape[1])[None].repeat(len(x), 0), 1)
    at = np.arange(len(x)), np.asarray(tokens)
    with np.errstate(invalid="ignore"):
        entropy = np.log(s) - np.where(e > 0, e * d, 0.0).sum(1) / s
    return dict(logprobs=lp[at], ranks=place[at], entropy=entropy, ids=order[:, :top],
                tops=np.take_along_axis(lp, order[:, :top], 1)), m[:, 0]


def check(got, x, tokens, top, given=True, entropy=True):
    want, m = reference(x, tokens, top)
    chain = (x.shape[1] / 64 + 64) * U
    size = np.abs(m) + np.abs(x).max(1, where=np.isfinite(x), initial=0.0)
    assert np.array_equal(got["ids"], want["ids"])
    with np.errstate(invalid="ignore"):  # -inf as it is
        off = np.where(got["tops"] == want["tops"], 0.0, np.abs(got["tops"] - want["tops"]))
        assert (off <= chain + 4 * U * (size[:, None] + 16)).all(), off.max()
        if given:
            assert np.array_equal(got["ranks"], want["ranks"])
            off = np.where(got["logprobs"] == want["logprobs"], 0.0, np.abs(got["logprobs"] - want["logprobs"]))
            assert (off <= chain + 4 * U * (size + 16)).all(), off.max()
    if entropy:
        assert (np.abs(got["entropy"] - want["entropy"]) <= chain * (2 + want["entropy"]) + 64 * U).all()


SHAPES = [
    # rows, vocab, top, std, stride, offset
    (1, 1, 1, 1.0, None, 0),
    (3, 2, 2, 1.0, None, 0),
    (5, 63, 63, 1.0, None, 0),
    (4, 64, 64, 3.0, None, 0),
    (2, 65, 64, 3.0, 67, 1),
    (7, 1000, 20, 3.0, None, 0),
    (7, 1001, 20, 3.0, None, 3),     # rows on every alignment
    (2, 8191, 5, 1.0, 8192, 0),
    (2, 8192, 64, 1.0, None, 0),
    (2, 8193, 64, 1.0, 8196, 2),
    (1, 151936, 20, 3.0, None, 0),
    (1, 151936, 64, 0.01, None, 0),  # almost flat
    (1, 151936, 0, 30.0, None, 0),   # one token has nearly everything
    (61, 152064, 5, 3.0, None, 0),
    (17, 151937, 3, 3.0, 151940, 1),
    (300, 32001, 1, 2.0, None, 0),
    (1500, 5000, 10, 2.0, None, 0),
    (2100, 129, 2, 2.0, None, 0),
    (1, 600001, 7, 3.0, None, 0),
    (70000, 40, 3, 2.0, 41, 1),
    (3000, 1024, 64, 2.0, None, 0),
    (2, 2000000, 33, 3.0, None, 2),
]


@pytest.mark.parametrize("rows, vocab, top, std, stride, offset", SHAPES)
def test_logprobs_match_definition(mh, gpu, rows, vocab, top, std, stride, offset):
    rng = np.random.default_rng(rows + vocab)
    x = rng.normal(0, std, (rows, vocab)).astype(np.float32)
    tokens = rng.integers(0, vocab, rows)
    tokens[::3] = x[::3].argmax(1)
    check(run(mh, gpu, x, tokens, top, stride, offset), x, tokens, top)


@pytest.mark.parametrize("rows, vocab", [(2, 500), (3, 20000), (600, 3001)])
def test_equal_logits_go_by_index(mh, gpu, rows, vocab):
    """Rows of one value, of a few values, and of zeros of both signs: the order is by index where values
    are equal, over whole slices of equal ones."""
    rng = np.random.default_rng(vocab)
    x = rng.integers(-2, 3, (rows, vocab)).astype(np.float32)
    x[0] = 1.25
    x[1] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)
    tokens = rng.integers(0, vocab, rows)
    tokens[0] = vocab - 1
    check(run(mh, gpu, x, tokens, 64), x, tokens, 64)
    rising = np.arange(vocab, dtype=np.float32)[None].repeat(2, 0) * 0.01
    rising[1] = rising[1][::-1]
    check(run(mh, gpu, rising, [0, 0], 64), rising, [0, 0], 64)


@pytest.mark.parametrize("rows", [1, 61, 300, 1100])
def test_first_tokens_close_together_and_far_apart(mh, gpu, rows):
    """The first tokens in a stretch that one thread or one wave reads, spread so that one thread's loads have
    them all, and tied in numbers past any list of candidates."""
    vocab = 151936
    rng = np.random.default_rng(rows)
    x = np.repeat(rng.normal(0, 1, (1, vocab)).astype(np.float32), rows, 0)
    for row in range(rows):
        kind = row % 6 if rows > 1 else 1
        if kind == 0:
            x[row, 70000:70064] += 20
        elif kind == 1:
            x[row, 5::1024] += 20                     # a lane of every wave
        elif kind == 2:
            x[row, 4096:5120] = 20                    # more equal ones than are ranked at once
        elif kind == 3:
            x[row, rng.integers(0, vocab, 3000)] = 20
        elif kind == 4:
            x[row, -40:] = 20 - np.arange(40) % 7
        else:
            x[row, 8192 + 3::16384] = 30 + np.arange(len(x[row, 8192 + 3::16384]))
    tokens = rng.integers(0, vocab, rows)
    tokens[0] = 70001
    got = run(mh, gpu, x, tokens, 20)
    some = np.unique(np.concatenate([np.arange(min(rows, 12)), rng.integers(0, rows, 12)]))
    check({k: v[some] for k, v in got.items()}, x[some], tokens[some], 20)


@pytest.mark.parametrize("rows, vocab, top", [(1, 151936, 20), (61, 152064, 5), (300, 151936, 20), (1100, 40000, 64)])
def test_few_tokens_left_by_a_mask(mh, gpu, rows, vocab, top):
    """Ten tokens allowed, anywhere or in one stretch, the others -inf or the lowest value; and logits rounded to
    8 bits, with their ties."""
    rng = np.random.default_rng(rows + top)
    x = rng.normal(0, 3, (rows, vocab)).astype(np.float32)
    bits = x[::4].view(np.uint32)
    x[::4] = ((bits + 0x8000) & 0xFFFF0000).view(np.float32)
    for row in range(rows):
        if row % 4 != 0:
            at = rng.integers(0, vocab, 10) if row % 2 else 5000 + np.arange(10)
            keep = x[row, at]
            x[row] = -np.inf if row % 4 != 3 else np.finfo(np.float32).min
            x[row, at] = keep
    tokens = rng.integers(0, vocab, rows)
    got = run(mh, gpu, x, tokens, top)
    some = np.unique(np.concatenate([np.arange(min(rows, 12)), rng.integers(0, rows, 12)]))
    check({k: v[some] for k, v in got.items()}, x[some], tokens[some], top)


@pytest.mark.parametrize("vocab", [100, 9001, 151936])
def test_masked_logits(mh, gpu, vocab):
    """-inf and the type's lowest value among the logits, a row with one token left, a row with none."""
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 2, (6, vocab)).astype(np.float32)
    x[0, rng.random(vocab) < 0.9] = -np.inf
    x[1, rng.random(vocab) < 0.9] = np.finfo(np.float32).min
    x[2] = -np.inf
    x[2, vocab - 3] = 5.0
    x[3] = np.finfo(np.float32).min
    x[4] = -np.inf
    x[5, ::2] = -np.inf
    tokens = np.array([int(np.flatnonzero(x[0] == -np.inf)[0]), int(x[1].argmax()), vocab - 3, 7, 9, 1])
    got = run(mh, gpu, x, tokens, 20)
    live = [0, 1, 2, 3, 5]
    check({k: v[live] for k, v in got.items()}, x[live], tokens[live], 20)
    assert got["logprobs"][0] == -np.inf and got["logprobs"][2] == 0.0 and got["entropy"][2] == 0.0
    assert got["logprobs"][4] == -np.inf and got["entropy"][4] == 0.0 and got["ranks"][4] == 9
    assert (got["tops"][4] == -np.inf).all() and np.array_equal(got["ids"][4], np.arange(20))


def test_largest_and_smallest_logits(mh, gpu):
    """Logits at the ends of the type's range, alone and beside ordinary ones."""
    rng = np.random.default_rng(3)
    big = np.finfo(np.float32).max
    x = rng.normal(0, 2, (7, 3000)).astype(np.float32)
    x[0, 100] = big
    x[1, ::7] = big
    x[2, :] = -big
    x[2, 5] = -big * np.float32(0.999)
    x[3] *= np.float32(1e-42)
    x[4, 1:] = -big
    x[5] = x[5] * np.float32(1e37)
    x[6] = x[6] * np.float32(1e-3) + np.float32(2e5)
    tokens = np.array([100, 1, 5, 7, 0, int(x[5].argmax()), 9])
    check(run(mh, gpu, x, tokens, 20), x, tokens, 20)


def test_logits_that_are_no_numbers(mh, gpu):
    """NaN or +inf in a row makes its log probabilities and entropy NaN, and only its; in the order NaN is
    last and +inf first."""
    rng = np.random.default_rng(4)
    for vocab in (50, 20001):
        x = rng.normal(0, 2, (4, vocab)).astype(np.float32)
        clean = x.copy()
        x[1, 17] = np.nan
        x[2, 30] = np.inf
        x[3] = np.nan
        tokens = np.array([3, 17, 30, 0])
        got = run(mh, gpu, x, tokens, 5)
        check({k: v[:1] for k, v in got.items()}, clean[:1], tokens[:1], 5)
        for r in (1, 2, 3):
            assert np.isnan(got["logprobs"][r]) and np.isnan(got["entropy"][r]) and np.isnan(got["tops"][r]).all()
        assert got["ranks"].tolist()[1:] == [vocab - 1, 0, 0]
        assert got["ids"][2][0] == 30 and 17 not in got["ids"][1] and got["ids"][3].tolist() == list(range(5))


def test_tokens_outside_the_vocabulary_and_absent_outputs(mh, gpu):
    rng = np.random.default_rng(6)
    x = rng.normal(0, 2, (5, 777)).astype(np.float32)
    tokens = np.array([-1, 777, 2 ** 31 - 1, -2 ** 31, 5])
    got = run(mh, gpu, x, tokens, 3)
    assert (got["logprobs"][:4] == -np.inf).all() and (got["ranks"][:4] == -1).all()
    check({k: v[4:] for k, v in got.items()}, x[4:], tokens[4:], 3)
    inside = np.zeros(5, int)
    check(run(mh, gpu, x, inside, 3, given=False), x, inside, 3, given=False)
    check(run(mh, gpu, x, inside, 3, entropy=False), x, inside, 3, entropy=False)
    check(run(mh, gpu, x, inside, 0), x, inside, 0)


def test_logprobs_in_a_graph_and_on_another_stream(mh, gpu):
    torch, lib = gpu, mh.load()
    rows, vocab, top = 9, 151936, 8
    x = torch.empty((rows, vocab), device="cuda")
    tokens = torch.empty(rows, dtype=torch.int32, device="cuda")
    logprobs, entropy = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ranks, ids = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty((rows, top), dtype=torch.int32,
                                                                                 device="cuda")
    tops = torch.empty((rows, top), device="cuda")
    size = lib.muyo_token_logprobs_workspace_bytes(rows, vocab, top)
    space = torch.empty(size, dtype=torch.uint8, device="cuda")

    def call():
        mh.check(lib.muyo_token_logprobs_f32(
            x.data_ptr(), vocab, rows, vocab, tokens.data_ptr(), logprobs.data_ptr(), ranks.data_ptr(),
            entropy.data_ptr(), top, ids.data_ptr(), tops.data_ptr(), space.data_ptr(), size,
            torch.cuda.current_stream().cuda_stream))

    rng = np.random.default_rng(8)
    graph = torch.cuda.CUDAGraph()
    x.zero_()
    tokens.zero_()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call()
    side = torch.cuda.Stream()
    for i in range(6):
        values = rng.normal(0, 3, (rows, vocab)).astype(np.float32)
        given = rng.integers(0, vocab, rows)
        x.copy_(torch.from_numpy(values))
        tokens.copy_(torch.from_numpy(given.astype(np.int32)))
        torch.cuda.synchronize()
        if i % 2 == 0:
            graph.replay()
        else:
            with torch.cuda.stream(side):
                call()
        torch.cuda.synchronize()
        check(dict(logprobs=host(logprobs), ranks=host(ranks), entropy=host(entropy), ids=host(ids), tops=host(tops)),
              values, given, top)


def test_logprobs_past_four_gigabytes_of_rows(mh, gpu):
    """Rows whose values lie past 2^31 elements."""
    torch, lib = gpu, mh.load()
    rows, stride, vocab = 3, 1100000000, 5000
    buffer = torch.empty(2 * stride + vocab, device="cuda")
    rng = np.random.default_rng(9)
    values = rng.normal(0, 2, (rows, vocab)).astype(np.float32)
    for r in range(rows):
        buffer[r * stride:r * stride + vocab] = torch.from_numpy(values[r]).cuda()
    ids, ranks = torch.empty((rows, 2), dtype=torch.int32, device="cuda"), torch.empty(rows, dtype=torch.int32,
                                                                                      device="cuda")
    tops, out = torch.empty((rows, 2), device="cuda"), torch.empty((2, rows), device="cuda")
    tokens = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    size = lib.muyo_token_logprobs_workspace_bytes(rows, vocab, 2)
    space = torch.empty(size, dtype=torch.uint8, device="cuda")
    mh.check(lib.muyo_token_logprobs_f32(
        buffer.data_ptr(), stride, rows, vocab, tokens.data_ptr(), out[0].data_ptr(), ranks.data_ptr(),
        out[1].data_ptr(), 2, ids.data_ptr(), tops.data_ptr(), space.data_ptr(), size,
        torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    check(dict(logprobs=host(out)[0], entropy=host(out)[1], ranks=host(ranks), ids=host(ids), tops=host(tops)), values,
          [1, 2, 3], 2)


def test_results_between_rows_of_logits(mh, gpu):
    """Rows of a wider buffer whose further columns hold the results and the workspace of the call."""
    torch, lib = gpu, mh.load()
    rows, vocab, top = 3, 20001, 4
    size = lib.muyo_token_logprobs_workspace_bytes(rows, vocab, top)
    stride = vocab + 3 + size // 4 + 64
    stride += -stride % 4
    rng = np.random.default_rng(12)
    x, given = rng.normal(0, 2, (rows, vocab)).astype(np.float32), rng.integers(0, vocab, rows)
    buffer = torch.zeros((rows, stride), device="cuda")
    buffer[:, :vocab] = torch.from_numpy(x).cuda()
    tokens = torch.from_numpy(given.astype(np.int32)).cuda()
    gaps = [buffer.data_ptr() + 4 * (r * stride + vocab) for r in range(rows)]
    mh.check(lib.muyo_token_logprobs_f32(
        buffer.data_ptr(), stride, rows, vocab, tokens.data_ptr(), gaps[0], gaps[0] + 12, gaps[0] + 24, top, gaps[2],
        gaps[2] + 48, gaps[1] + 12, size, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    got = host(buffer)
    assert np.array_equal(got[:, :vocab], x)
    first, last = got[0, vocab:vocab + 9], got[2, vocab:vocab + 24]
    check(dict(logprobs=first[:3], ranks=first[3:6].view(np.int32), entropy=first[6:9],
               ids=last[:12].view(np.int32).reshape(rows, top), tops=last[12:].reshape(rows, top)), x, given, top)
