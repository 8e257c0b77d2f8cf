"""The paged-cache and log-probability entry points without a device: what they refuse, and the rope
frequencies (host arithmetic) against their formulas in 64 bits."""
import ctypes
import math

import numpy as np
import pytest


def fake(i):
    """A distinct, aligned, never-read address per buffer (1 GiB apart)."""
    return ctypes.c_void_p((i + 1) << 30)


PLAN = dict(lengths=fake(0), targets=fake(1), sequences=4, tables=fake(2), table_pages=8, free_pages=fake(3),
            pool=fake(4), pages=64, page_size=16, tokens=10, granted=fake(5), pool_out=fake(6), starts=fake(7),
            token_sequence=fake(8), positions=fake(9), slots=fake(10), stream=None)
APPEND = dict(q=fake(0), k=fake(1), v=fake(2), q_stride=896, k_stride=128, v_stride=128, q_out=fake(3),
              kcache=fake(4), vcache=fake(5), positions=fake(6), slots=fake(7), tokens=3, heads=14, kv_heads=2,
              head_dim=64, pages=64, page_size=16, rope_layout=0, rotary_dim=64, turns=fake(8), magnitude=1.0,
              stream=None)
ATTEND = dict(q=fake(0), kcache=fake(1), vcache=fake(2), out=fake(3), tables=fake(4), sequences=3, table_pages=8,
              query_sequence=fake(5), positions=fake(6), queries=3, heads=14, kv_heads=2, head_dim=64, pages=64,
              page_size=16, window=0, scale=0.125, workspace=fake(7), workspace_bytes=1 << 30, stream=None)
LOGPROBS = dict(logits=fake(0), row_stride=1000, rows=3, vocab=1000, tokens=fake(1), logprobs=fake(2), ranks=fake(3),
                entropy=fake(4), top=5, top_ids=fake(5), top_logprobs=fake(6), workspace=fake(7),
                workspace_bytes=1 << 30, stream=None)

REFUSALS = [
    *[("paged_plan", PLAN, {k: None}, "MUYO_E_NULL")
      for k in ("lengths", "targets", "tables", "free_pages", "pool", "granted", "pool_out", "starts",
                "token_sequence", "positions", "slots")],
    ("paged_plan", PLAN, dict(sequences=0), "MUYO_E_RANGE"),
    ("paged_plan", PLAN, dict(sequences=4097), "MUYO_E_RANGE"),
    ("paged_plan", PLAN, dict(tokens=(1 << 24) + 1), "MUYO_E_RANGE"),
    ("paged_plan", PLAN, dict(pages=0), "MUYO_E_RANGE"),
    ("paged_plan", PLAN, dict(pages=1 << 27), "MUYO_E_RANGE"),
    ("paged_plan", PLAN, dict(table_pages=0), "MUYO_E_RANGE"),
    ("paged_plan", PLAN, dict(table_pages=1 << 27), "MUYO_E_RANGE"),
    ("paged_plan", PLAN, dict(table_pages=1 << 26, sequences=32), "MUYO_E_RANGE"),
    ("paged_plan", PLAN, dict(page_size=0), "MUYO_E_UNSUPPORTED"),
    ("paged_plan", PLAN, dict(page_size=8), "MUYO_E_UNSUPPORTED"),
    ("paged_plan", PLAN, dict(page_size=48), "MUYO_E_UNSUPPORTED"),
    ("paged_plan", PLAN, dict(page_size=2048), "MUYO_E_UNSUPPORTED"),
    ("paged_plan", PLAN, dict(granted=PLAN["targets"]), "MUYO_E_CONTRACT"),
    ("paged_plan", PLAN, dict(granted=ctypes.c_void_p(PLAN["lengths"].value + 4)), "MUYO_E_CONTRACT"),
    ("paged_plan", PLAN, dict(pool_out=ctypes.c_void_p(PLAN["pool"].value + 4)), "MUYO_E_CONTRACT"),
    ("paged_plan", PLAN, dict(slots=PLAN["positions"]), "MUYO_E_CONTRACT"),
    ("paged_plan", PLAN, dict(starts=ctypes.c_void_p(PLAN["tables"].value + 4 * 31)), "MUYO_E_CONTRACT"),
    *[("paged_rope_append_f16kv", APPEND, {k: None}, "MUYO_E_NULL")
      for k in ("q", "k", "v", "q_out", "kcache", "vcache", "positions", "slots", "turns")],
    ("paged_rope_append_f16kv", APPEND, dict(tokens=0), "MUYO_E_RANGE"),
    ("paged_rope_append_f16kv", APPEND, dict(heads=0), "MUYO_E_RANGE"),
    ("paged_rope_append_f16kv", APPEND, dict(kv_heads=0), "MUYO_E_RANGE"),
    ("paged_rope_append_f16kv", APPEND, dict(heads=1025), "MUYO_E_RANGE"),
    ("paged_rope_append_f16kv", APPEND, dict(pages=0), "MUYO_E_RANGE"),
    ("paged_rope_append_f16kv", APPEND, dict(page_size=24), "MUYO_E_UNSUPPORTED"),
    ("paged_rope_append_f16kv", APPEND, dict(head_dim=60), "MUYO_E_UNSUPPORTED"),
    ("paged_rope_append_f16kv", APPEND, dict(rotary_dim=0), "MUYO_E_UNSUPPORTED"),
    ("paged_rope_append_f16kv", APPEND, dict(rotary_dim=33), "MUYO_E_UNSUPPORTED"),
    ("paged_rope_append_f16kv", APPEND, dict(rotary_dim=66), "MUYO_E_UNSUPPORTED"),
    ("paged_rope_append_f16kv", APPEND, dict(rope_layout=2), "MUYO_E_UNSUPPORTED"),
    ("paged_rope_append_f16kv", APPEND, dict(q_stride=895), "MUYO_E_CONTRACT"),
    ("paged_rope_append_f16kv", APPEND, dict(q_stride=898), "MUYO_E_CONTRACT"),
    ("paged_rope_append_f16kv", APPEND, dict(k_stride=124), "MUYO_E_CONTRACT"),
    ("paged_rope_append_f16kv", APPEND, dict(v_stride=130), "MUYO_E_CONTRACT"),
    ("paged_rope_append_f16kv", APPEND, dict(q=ctypes.c_void_p(8)), "MUYO_E_CONTRACT"),
    ("paged_rope_append_f16kv", APPEND, dict(kcache=ctypes.c_void_p((5 << 30) + 2)), "MUYO_E_CONTRACT"),
    ("paged_rope_append_f16kv", APPEND, dict(turns=ctypes.c_void_p(4)), "MUYO_E_CONTRACT"),
    ("paged_rope_append_f16kv", APPEND, dict(magnitude=math.nan), "MUYO_E_CONTRACT"),
    ("paged_rope_append_f16kv", APPEND, dict(vcache=APPEND["kcache"]), "MUYO_E_CONTRACT"),
    ("paged_rope_append_f16kv", APPEND, dict(q_out=APPEND["q"], k=APPEND["q"]), "MUYO_E_CONTRACT"),
    ("paged_rope_append_f16kv", APPEND, dict(tokens=1 << 24, q_out=APPEND["q"]), "MUYO_E_RANGE"),
    ("paged_rope_append_f16kv", APPEND, dict(tokens=1 << 22, rotary_dim=60, q_out=APPEND["q"]), "MUYO_E_RANGE"),
    ("paged_rope_append_f16kv", APPEND, dict(q_out=APPEND["k"]), "MUYO_E_CONTRACT"),
    ("paged_rope_append_f16kv", APPEND, dict(q_out=APPEND["q"], q_stride=1152), "MUYO_E_CONTRACT"),
    *[("paged_attention_decode_f16kv", ATTEND, {k: None}, "MUYO_E_NULL")
      for k in ("q", "kcache", "vcache", "out", "tables", "query_sequence", "positions")],
    ("paged_attention_decode_f16kv", ATTEND, dict(queries=0), "MUYO_E_UNSUPPORTED"),
    ("paged_attention_decode_f16kv", ATTEND, dict(queries=65536), "MUYO_E_UNSUPPORTED"),
    ("paged_attention_decode_f16kv", ATTEND, dict(kv_heads=3), "MUYO_E_UNSUPPORTED"),
    ("paged_attention_decode_f16kv", ATTEND, dict(heads=34), "MUYO_E_UNSUPPORTED"),
    ("paged_attention_decode_f16kv", ATTEND, dict(heads=0), "MUYO_E_UNSUPPORTED"),
    ("paged_attention_decode_f16kv", ATTEND, dict(head_dim=96), "MUYO_E_UNSUPPORTED"),
    ("paged_attention_decode_f16kv", ATTEND, dict(page_size=20), "MUYO_E_UNSUPPORTED"),
    ("paged_attention_decode_f16kv", ATTEND, dict(sequences=0), "MUYO_E_RANGE"),
    ("paged_attention_decode_f16kv", ATTEND, dict(table_pages=0), "MUYO_E_RANGE"),
    ("paged_attention_decode_f16kv", ATTEND, dict(table_pages=1 << 27), "MUYO_E_RANGE"),
    ("paged_attention_decode_f16kv", ATTEND, dict(pages=1 << 27), "MUYO_E_RANGE"),
    ("paged_attention_decode_f16kv", ATTEND, dict(q=ctypes.c_void_p(4)), "MUYO_E_CONTRACT"),
    ("paged_attention_decode_f16kv", ATTEND, dict(vcache=ctypes.c_void_p(8)), "MUYO_E_CONTRACT"),
    ("paged_attention_decode_f16kv", ATTEND, dict(scale=math.inf), "MUYO_E_CONTRACT"),
    ("paged_attention_decode_f16kv", ATTEND, dict(scale=math.nan), "MUYO_E_CONTRACT"),
    ("paged_attention_decode_f16kv", ATTEND, dict(workspace=None), "MUYO_E_CONTRACT"),
    ("paged_attention_decode_f16kv", ATTEND, dict(workspace=ctypes.c_void_p(8)), "MUYO_E_CONTRACT"),
    ("paged_attention_decode_f16kv", ATTEND, dict(workspace_bytes=15), "MUYO_E_CONTRACT"),
    ("paged_attention_decode_f16kv", ATTEND, dict(out=ctypes.c_void_p(ATTEND["q"].value + 3584)), "MUYO_E_CONTRACT"),
    ("paged_attention_decode_f16kv", ATTEND, dict(out=ATTEND["kcache"]), "MUYO_E_CONTRACT"),
    ("paged_attention_decode_f16kv", ATTEND, dict(out=ATTEND["vcache"]), "MUYO_E_CONTRACT"),
    ("paged_attention_decode_f16kv", ATTEND, dict(out=ATTEND["workspace"]), "MUYO_E_CONTRACT"),
    ("token_logprobs_f32", LOGPROBS, dict(logits=None), "MUYO_E_NULL"),
    ("token_logprobs_f32", LOGPROBS, dict(tokens=None), "MUYO_E_NULL"),
    ("token_logprobs_f32", LOGPROBS, dict(top_ids=None), "MUYO_E_NULL"),
    ("token_logprobs_f32", LOGPROBS, dict(top_logprobs=None), "MUYO_E_NULL"),
    ("token_logprobs_f32", LOGPROBS, dict(rows=0), "MUYO_E_RANGE"),
    ("token_logprobs_f32", LOGPROBS, dict(rows=1 << 24), "MUYO_E_RANGE"),
    ("token_logprobs_f32", LOGPROBS, dict(rows=(1 << 24) - 1, vocab=0x7FFFFFFF, row_stride=0x7FFFFFFF,
                                          workspace_bytes=1 << 62), "MUYO_E_RANGE"),
    ("token_logprobs_f32", LOGPROBS, dict(vocab=0, row_stride=0, top=0), "MUYO_E_RANGE"),
    ("token_logprobs_f32", LOGPROBS, dict(top=65), "MUYO_E_RANGE"),
    ("token_logprobs_f32", LOGPROBS, dict(vocab=4), "MUYO_E_RANGE"),
    ("token_logprobs_f32", LOGPROBS, dict(logits=ctypes.c_void_p(2)), "MUYO_E_CONTRACT"),
    ("token_logprobs_f32", LOGPROBS, dict(row_stride=999), "MUYO_E_CONTRACT"),
    ("token_logprobs_f32", LOGPROBS, dict(workspace=None), "MUYO_E_CONTRACT"),
    ("token_logprobs_f32", LOGPROBS, dict(workspace_bytes=0), "MUYO_E_CONTRACT"),
]


@pytest.mark.parametrize("case", REFUSALS, ids=[f"{i}-{c[0]}-{'-'.join(c[2])}" for i, c in enumerate(REFUSALS)])
def test_refused_before_anything_is_launched(mh, case):
    entry, good, change, status = case
    call = getattr(mh.load(), "muyo_" + entry)
    assert call(*{**good, **change}.values()) == getattr(mh, status)
    assert entry.encode() in mh.load().muyo_last_error()


def test_workspace_sizes_of_unsupported_shapes_are_zero(mh):
    lib = mh.load()
    size = lib.muyo_paged_attention_decode_f16kv_workspace_bytes
    assert size(1, 14, 2, 64) > 0 and size(65535, 28, 4, 128) > 0
    for shape in ((0, 14, 2, 64), (1, 14, 3, 64), (1, 34, 2, 64), (1, 14, 2, 80), (65536, 14, 2, 64), (1, 0, 1, 64),
                  (1, 14, 0, 64)):
        assert size(*shape) == 0, shape
    size = lib.muyo_token_logprobs_workspace_bytes
    assert size(1, 151936, 64) > 0 and size(5000, 1, 0) > 0
    for shape in ((0, 100, 1), (1, 0, 0), (1, 100, 65), (1, 4, 5), (1, 1 << 31, 1)):
        assert size(*shape) == 0, shape


# ------------------------------------------------------------------------------------------------
# Rope frequencies. 64-bit arithmetic on both sides: a handful of roundings, 1e-14 relative.


def plain_turns(base, dim):
    return [base ** (-2.0 * j / dim) / (2 * math.pi) for j in range(dim // 2)]


def test_rope_frequencies_unscaled_linear_and_base(mh):
    for base, dim in ((1e6, 64), (1e4, 128), (500000.0, 2), (1e6, 34)):
        turns, magnitude = mh.rope_frequencies(base, dim)
        assert magnitude == 1.0
        np.testing.assert_allclose(turns, plain_turns(base, dim), rtol=1e-14)
        turns, magnitude = mh.rope_frequencies(base, dim, "LINEAR", factor=8.0)
        assert magnitude == 1.0
        np.testing.assert_allclose(turns, np.array(plain_turns(base, dim)) / 8, rtol=1e-14)
    turns, magnitude = mh.rope_frequencies(1e4, 64, "BASE", factor=4.0)
    np.testing.assert_allclose(turns, plain_turns(1e4 * 4.0 ** (64 / 62), 64), rtol=1e-13)
    # The slowest pair turns a quarter as fast, the fastest as before.
    np.testing.assert_allclose(turns[[0, -1]] / np.array(plain_turns(1e4, 64))[[0, -1]], [1.0, 0.25], rtol=1e-13)


def test_rope_frequencies_yarn_is_the_rope_contracts(mh):
    """The ramp and the magnitude of rope_funcs.glsl:17-35 with ext_factor 1, freq_scale 1 / factor, and
    ggml's corr_dims: pair j's angle per position is extrapolated * (1 - mix) + interpolated * mix ..."""
    base, dim, context, factor = 1e6, 128, 32768, 4.0
    turns, magnitude = mh.rope_frequencies(base, dim, "YARN", factor=factor, low=1.0, high=32.0, attn_factor=1.25,
                                           trained_context=context)
    low = max(0, math.floor(dim * math.log(context / (32 * 2 * math.pi)) / (2 * math.log(base))))
    high = min(dim - 1, math.ceil(dim * math.log(context / (1 * 2 * math.pi)) / (2 * math.log(base))))
    assert 0 < low < high < dim // 2
    for j, plain in enumerate(plain_turns(base, dim)):
        mix = 1.0 - min(1.0, max(0.0, (j - low) / max(0.001, high - low)))
        assert turns[j] == pytest.approx(plain / factor * (1 - mix) + plain * mix, rel=1e-13)
    assert magnitude == np.float32(1.25 * (1 + 0.1 * math.log(factor)))


def test_rope_frequencies_by_wavelength_and_divisors(mh):
    base, dim, context, factor, low, high = 5e5, 128, 8192, 8.0, 1.0, 4.0
    turns, magnitude = mh.rope_frequencies(base, dim, "WAVELENGTH", factor=factor, low=low, high=high,
                                           trained_context=context)
    kinds = set()
    for j, plain in enumerate(plain_turns(base, dim)):
        wavelength = 1 / plain
        if wavelength < context / high:
            want, kind = plain, "kept"
        elif wavelength > context / low:
            want, kind = plain / factor, "scaled"
        else:
            smooth = (context / wavelength - low) / (high - low)
            want, kind = (1 - smooth) * plain / factor + smooth * plain, "between"
        kinds.add(kind)
        assert turns[j] == pytest.approx(want, rel=1e-12)
    assert kinds == {"kept", "scaled", "between"} and magnitude == 1.0
    divisors = np.linspace(1.0, 30.0, 32, dtype=np.float32)
    turns, _ = mh.rope_frequencies(1e4, 64, pair_divisors=divisors)
    np.testing.assert_allclose(turns, np.array(plain_turns(1e4, 64)) / divisors.astype(np.float64), rtol=1e-14)


@pytest.mark.parametrize("args, kwargs, status", [
    ((1e6, 0), {}, "MUYO_E_CONTRACT"),
    ((1e6, 7), {}, "MUYO_E_CONTRACT"),
    ((1.0, 64), {}, "MUYO_E_CONTRACT"),
    ((math.nan, 64), {}, "MUYO_E_CONTRACT"),
    ((math.inf, 64), {}, "MUYO_E_CONTRACT"),
    ((1e6, 64), dict(scaling="LINEAR", factor=0.0), "MUYO_E_CONTRACT"),
    ((1e6, 64), dict(scaling="LINEAR", factor=math.nan), "MUYO_E_CONTRACT"),
    ((1e6, 2), dict(scaling="BASE", factor=2.0), "MUYO_E_CONTRACT"),
    ((1e6, 64), dict(scaling="YARN", factor=2.0), "MUYO_E_CONTRACT"),
    ((1e6, 64), dict(scaling="YARN", factor=2.0, low=0.0, trained_context=4096), "MUYO_E_CONTRACT"),
    ((1e6, 64), dict(scaling="WAVELENGTH", factor=2.0, low=4.0, high=4.0, trained_context=4096), "MUYO_E_CONTRACT"),
    ((1e6, 64), dict(pair_divisors=np.zeros(32)), "MUYO_E_CONTRACT"),
])
def test_rope_frequencies_refusals(mh, args, kwargs, status):
    with pytest.raises(mh.MuyoError) as error:
        mh.rope_frequencies(*args, **kwargs)
    assert error.value.status == getattr(mh, status)


def test_rope_frequencies_unknown_kind_and_nulls(mh):
    lib, magnitude = mh.load(), ctypes.c_float()
    turns = np.empty(32)
    s = mh.MuyoRopeScaling(5, 1.0, 1.0, 32.0, 1.0, 4096)
    assert lib.muyo_rope_frequencies(1e6, 64, mh.ref(s), None, turns.ctypes.data,
                                     ctypes.byref(magnitude)) == mh.MUYO_E_UNSUPPORTED
    assert lib.muyo_rope_frequencies(1e6, 64, None, None, None, ctypes.byref(magnitude)) == mh.MUYO_E_NULL
    assert lib.muyo_rope_frequencies(1e6, 64, None, None, turns.ctypes.data, None) == mh.MUYO_E_NULL
    with pytest.raises(ValueError):
        mh.rope_frequencies(1e6, 64, pair_divisors=np.ones(31))


# ------------------------------------------------------------------------------------------------
# Buffers that a call writes and others that it uses: no two of them may share a byte.


def moved(pointer, nbytes):
    return ctypes.c_void_p(pointer.value + nbytes)


APPEND_BYTES = dict(kcache=2 * 2 * 64 * 64 * 16, vcache=2 * 2 * 64 * 64 * 16, q_out=4 * 896 * 3, positions=12,
                    slots=12, turns=256)


@pytest.mark.parametrize("written, other", [(w, o) for w in ("q_out", "kcache", "vcache")
                                            for o in ("q_out", "kcache", "vcache", "positions", "slots", "turns")
                                            if w != o])
def test_append_refuses_written_buffers_over_others(mh, written, other):
    """At the other's beginning, over its last 16 bytes, and ending inside it."""
    call = mh.load().muyo_paged_rope_append_f16kv
    for at in (0, (APPEND_BYTES[other] - 1) // 16 * 16, 16 - APPEND_BYTES[written]):
        change = {written: moved(APPEND[other], at)}
        assert call(*{**APPEND, **change}.values()) == mh.MUYO_E_CONTRACT, at
        assert b"overlaps" in mh.load().muyo_last_error()


@pytest.mark.parametrize("source, width", [("q", 896), ("k", 128), ("v", 128)])
@pytest.mark.parametrize("cache", ["kcache", "vcache"])
def test_append_refuses_caches_over_the_rows_that_it_reads(mh, source, width, cache):
    """Over a row's beginning, its last 16 bytes, and the last row, where rows are far apart."""
    call, stride = mh.load().muyo_paged_rope_append_f16kv, 1 << 20
    for at in (0, 4 * width - 16, 8 * stride + 4 * width - 16, 4 * stride + 16 - APPEND_BYTES[cache]):
        change = {source + "_stride": stride, cache: moved(APPEND[source], at)}
        assert call(*{**APPEND, **change}.values()) == mh.MUYO_E_CONTRACT, at
        assert b"overlaps " + source.encode() in mh.load().muyo_last_error()


ATTEND_BYTES = dict(out=4 * 3 * 896, q=4 * 3 * 896, kcache=2 * 2 * 64 * 64 * 16, vcache=2 * 2 * 64 * 64 * 16,
                    tables=4 * 3 * 8, query_sequence=12, positions=12)


@pytest.mark.parametrize("written, other", [(w, o) for w in ("out", "workspace")
                                            for o in ("out", "q", "kcache", "vcache", "tables", "query_sequence",
                                                      "positions") if w != o])
def test_attention_refuses_written_buffers_over_others(mh, written, other):
    """At the other's beginning (out over q may be there), over its last 16 bytes, and ending inside it."""
    lib = mh.load()
    call = lib.muyo_paged_attention_decode_f16kv
    own = dict(ATTEND_BYTES, workspace=lib.muyo_paged_attention_decode_f16kv_workspace_bytes(3, 14, 2, 64))[written]
    for at in (0, (ATTEND_BYTES[other] - 1) // 16 * 16, 16 - own // 16 * 16):
        if (written, other, at) != ("out", "q", 0):
            assert call(*{**ATTEND, written: moved(ATTEND[other], at)}.values()) == mh.MUYO_E_CONTRACT, at
            assert b"overlaps" in lib.muyo_last_error()


LOGPROB_BYTES = dict(logits=4 * 3 * 1000, tokens=12, logprobs=12, ranks=12, entropy=12, top_ids=60, top_logprobs=60)


@pytest.mark.parametrize("written, other", [(w, o) for w in ("logprobs", "ranks", "entropy", "top_ids", "top_logprobs",
                                                             "workspace")
                                            for o in LOGPROB_BYTES if w != o])
def test_logprobs_refuse_written_buffers_over_others(mh, written, other):
    """At the other's beginning, over its last 16 bytes, and ending inside it."""
    lib = mh.load()
    own = dict(LOGPROB_BYTES, workspace=lib.muyo_token_logprobs_workspace_bytes(3, 1000, 5))[written]
    for at in (0, (LOGPROB_BYTES[other] - 1) // 16 * 16, 16 - max(16, own // 16 * 16)):
        change = {written: moved(LOGPROBS[other], at)}
        assert lib.muyo_token_logprobs_f32(*{**LOGPROBS, **change}.values()) == mh.MUYO_E_CONTRACT, at
        assert b"overlaps" in lib.muyo_last_error()


@pytest.mark.parametrize("at", [4 * 999, 4 * (1 << 20), 8 * (1 << 20) + 3996, 4 * (1 << 20) - 56])
def test_logprobs_refuse_outputs_over_rows_far_apart(mh, at):
    """A row's last logit, another's first, the last row's last, and an output that ends in a row."""
    change = dict(row_stride=1 << 20, top_ids=moved(LOGPROBS["logits"], at))
    assert mh.load().muyo_token_logprobs_f32(*{**LOGPROBS, **change}.values()) == mh.MUYO_E_CONTRACT
    assert b"top_ids overlaps logits" in mh.load().muyo_last_error()


@pytest.mark.parametrize("change", [dict(low=32.0, high=1.0), dict(low=33.0), dict(factor=1e-5), dict(factor=4e-5),
                                    dict(attn_factor=0.0), dict(attn_factor=-1.0)],
                         ids=lambda c: "-".join(f"{k}={v}" for k, v in c.items()))
def test_rope_frequencies_yarn_without_a_ramp_or_magnitude(mh, change):
    """Ends in the wrong order, and factors whose 1 + ln(factor) / 10 (with attn_factor) is not above 0."""
    with pytest.raises(mh.MuyoError) as error:
        mh.rope_frequencies(1e6, 64, "YARN", **{**dict(factor=4.0, trained_context=4096), **change})
    assert error.value.status == mh.MUYO_E_CONTRACT


def test_rope_frequencies_yarn_at_the_ends_of_what_is_taken(mh):
    """low = high: pairs on one side keep their speed, on the other turn 1 / factor as fast, but for one on the border
    (its place is rounded down for one end and up for the other). A factor just above e^-10 has a magnitude."""
    turns, _ = mh.rope_frequencies(1e6, 64, "YARN", factor=4.0, low=8.0, high=8.0, trained_context=4096)
    plain = np.array(plain_turns(1e6, 64))
    border = 64 * math.log(4096 / (8 * 2 * math.pi)) / (2 * math.log(1e6))
    j = np.arange(32)
    np.testing.assert_allclose(turns, np.where(j <= border, plain, plain / 4), rtol=1e-14)
    _, magnitude = mh.rope_frequencies(1e6, 64, "YARN", factor=5e-5, trained_context=4096)
    assert magnitude == np.float32(1 + 0.1 * math.log(np.float32(5e-5))) and 0 < magnitude < 0.01


def test_rope_frequencies_of_a_base_stretched_past_any_number(mh):
    with pytest.raises(mh.MuyoError) as error:
        mh.rope_frequencies(1e300, 4, "BASE", factor=1e30)
    assert error.value.status == mh.MUYO_E_CONTRACT
