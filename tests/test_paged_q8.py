"""The 8-bit paged cache's entry points without a device: what they refuse."""
import ctypes
import math

import pytest

from test_paged import fake

APPEND = dict(q=fake(0), k=fake(1), v=fake(2), q_stride=896, k_stride=128, v_stride=128, q_out=fake(3),
              kcache=fake(4), vcache=fake(5), kscales=fake(6), vscales=fake(7), positions=fake(8), slots=fake(9),
              tokens=3, heads=14, kv_heads=2, head_dim=64, pages=64, page_size=16, format=0, rope_layout=0,
              rotary_dim=64, turns=fake(10), magnitude=1.0, stream=None)
ATTEND = dict(q=fake(0), kcache=fake(1), vcache=fake(2), kscales=fake(3), vscales=fake(4), out=fake(5),
              tables=fake(6), sequences=3, table_pages=8, query_sequence=fake(7), positions=fake(8), queries=3,
              heads=14, kv_heads=2, head_dim=64, pages=64, page_size=16, format=0, window=0, scale=0.125,
              workspace=fake(9), workspace_bytes=1 << 30, stream=None)


def past(pointer, nbytes):
    return ctypes.c_void_p(pointer.value + nbytes)


REFUSALS = [
    *[("paged_rope_append_q8kv", APPEND, {k: None}, "MUYO_E_NULL")
      for k in ("q", "k", "v", "q_out", "kcache", "vcache", "kscales", "vscales", "positions", "slots", "turns")],
    ("paged_rope_append_q8kv", APPEND, dict(tokens=0), "MUYO_E_RANGE"),
    ("paged_rope_append_q8kv", APPEND, dict(tokens=(1 << 24) + 1), "MUYO_E_RANGE"),
    ("paged_rope_append_q8kv", APPEND, dict(tokens=1 << 24), "MUYO_E_RANGE"),
    ("paged_rope_append_q8kv", APPEND, dict(heads=0), "MUYO_E_RANGE"),
    ("paged_rope_append_q8kv", APPEND, dict(kv_heads=0), "MUYO_E_RANGE"),
    ("paged_rope_append_q8kv", APPEND, dict(heads=1025), "MUYO_E_RANGE"),
    ("paged_rope_append_q8kv", APPEND, dict(pages=0), "MUYO_E_RANGE"),
    ("paged_rope_append_q8kv", APPEND, dict(pages=1 << 27), "MUYO_E_RANGE"),
    ("paged_rope_append_q8kv", APPEND, dict(page_size=24), "MUYO_E_UNSUPPORTED"),
    ("paged_rope_append_q8kv", APPEND, dict(head_dim=96), "MUYO_E_UNSUPPORTED"),
    ("paged_rope_append_q8kv", APPEND, dict(head_dim=256), "MUYO_E_UNSUPPORTED"),
    ("paged_rope_append_q8kv", APPEND, dict(format=2), "MUYO_E_UNSUPPORTED"),
    ("paged_rope_append_q8kv", APPEND, dict(rotary_dim=0), "MUYO_E_UNSUPPORTED"),
    ("paged_rope_append_q8kv", APPEND, dict(rotary_dim=33), "MUYO_E_UNSUPPORTED"),
    ("paged_rope_append_q8kv", APPEND, dict(rotary_dim=66), "MUYO_E_UNSUPPORTED"),
    ("paged_rope_append_q8kv", APPEND, dict(rope_layout=2), "MUYO_E_UNSUPPORTED"),
    ("paged_rope_append_q8kv", APPEND, dict(q_stride=892), "MUYO_E_CONTRACT"),
    ("paged_rope_append_q8kv", APPEND, dict(k_stride=130), "MUYO_E_CONTRACT"),
    ("paged_rope_append_q8kv", APPEND, dict(q=ctypes.c_void_p(8)), "MUYO_E_CONTRACT"),
    *[("paged_rope_append_q8kv", APPEND, {k: past(APPEND[k], 8)}, "MUYO_E_CONTRACT")
      for k in ("kcache", "vcache", "kscales", "vscales")],
    ("paged_rope_append_q8kv", APPEND, dict(turns=ctypes.c_void_p(4)), "MUYO_E_CONTRACT"),
    ("paged_rope_append_q8kv", APPEND, dict(magnitude=math.inf), "MUYO_E_CONTRACT"),
    ("paged_rope_append_q8kv", APPEND, dict(vcache=APPEND["kcache"]), "MUYO_E_CONTRACT"),
    ("paged_rope_append_q8kv", APPEND, dict(vscales=APPEND["kscales"]), "MUYO_E_CONTRACT"),
    # A scale behind the last byte of the cache but one row's, and the one behind it all.
    ("paged_rope_append_q8kv", APPEND, dict(kscales=past(APPEND["kcache"], 64 * 2 * 16 * 64 - 16)), "MUYO_E_CONTRACT"),
    ("paged_rope_append_q8kv", APPEND, dict(vscales=past(APPEND["slots"], -64 * 2 * 16 * 4 + 16)), "MUYO_E_CONTRACT"),
    ("paged_rope_append_q8kv", APPEND, dict(kscales=APPEND["q"]), "MUYO_E_CONTRACT"),
    ("paged_rope_append_q8kv", APPEND, dict(vcache=APPEND["v"]), "MUYO_E_CONTRACT"),
    ("paged_rope_append_q8kv", APPEND, dict(q_out=APPEND["kscales"]), "MUYO_E_CONTRACT"),
    ("paged_rope_append_q8kv", APPEND, dict(q_out=APPEND["q"], q_stride=1152), "MUYO_E_CONTRACT"),
    *[("paged_attention_decode_q8kv", ATTEND, {k: None}, "MUYO_E_NULL")
      for k in ("q", "kcache", "vcache", "kscales", "vscales", "out", "tables", "query_sequence", "positions")],
    ("paged_attention_decode_q8kv", ATTEND, dict(queries=0), "MUYO_E_UNSUPPORTED"),
    ("paged_attention_decode_q8kv", ATTEND, dict(queries=65536), "MUYO_E_UNSUPPORTED"),
    ("paged_attention_decode_q8kv", ATTEND, dict(kv_heads=3), "MUYO_E_UNSUPPORTED"),
    ("paged_attention_decode_q8kv", ATTEND, dict(heads=34), "MUYO_E_UNSUPPORTED"),
    ("paged_attention_decode_q8kv", ATTEND, dict(head_dim=32), "MUYO_E_UNSUPPORTED"),
    ("paged_attention_decode_q8kv", ATTEND, dict(format=2), "MUYO_E_UNSUPPORTED"),
    ("paged_attention_decode_q8kv", ATTEND, dict(page_size=8), "MUYO_E_UNSUPPORTED"),
    ("paged_attention_decode_q8kv", ATTEND, dict(sequences=0), "MUYO_E_RANGE"),
    ("paged_attention_decode_q8kv", ATTEND, dict(table_pages=0), "MUYO_E_RANGE"),
    ("paged_attention_decode_q8kv", ATTEND, dict(pages=1 << 27), "MUYO_E_RANGE"),
    *[("paged_attention_decode_q8kv", ATTEND, {k: past(ATTEND[k], 4)}, "MUYO_E_CONTRACT")
      for k in ("q", "kcache", "vcache", "kscales", "vscales", "out", "workspace")],
    ("paged_attention_decode_q8kv", ATTEND, dict(scale=math.nan), "MUYO_E_CONTRACT"),
    ("paged_attention_decode_q8kv", ATTEND, dict(workspace=None), "MUYO_E_CONTRACT"),
    ("paged_attention_decode_q8kv", ATTEND, dict(workspace_bytes=15), "MUYO_E_CONTRACT"),
    ("paged_attention_decode_q8kv", ATTEND, dict(out=past(ATTEND["q"], 3584)), "MUYO_E_CONTRACT"),
    *[("paged_attention_decode_q8kv", ATTEND, dict(out=ATTEND[k]), "MUYO_E_CONTRACT")
      for k in ("kcache", "vcache", "kscales", "vscales", "tables", "query_sequence", "positions", "workspace")],
    *[("paged_attention_decode_q8kv", ATTEND, dict(workspace=ATTEND[k]), "MUYO_E_CONTRACT")
      for k in ("q", "kcache", "vcache", "kscales", "vscales", "tables", "query_sequence", "positions")],
]


@pytest.mark.parametrize("case", REFUSALS, ids=[f"{i}-{c[0]}-{'-'.join(c[2])}" for i, c in enumerate(REFUSALS)])
def test_refused_before_anything_is_launched(mh, case):
    entry, good, change, status = case
    call = getattr(mh.load(), "muyo_" + entry)
    assert call(*{**good, **change}.values()) == getattr(mh, status)
    assert entry.encode() in mh.load().muyo_last_error()


def test_workspace_sizes_of_unsupported_shapes_are_zero(mh):
    size = mh.load().muyo_paged_attention_decode_q8kv_workspace_bytes
    assert size(1, 14, 2, 64) > 0 and size(65535, 28, 4, 128) > 0
    for shape in ((0, 14, 2, 64), (1, 14, 3, 64), (1, 34, 2, 64), (1, 14, 2, 80), (65536, 14, 2, 64), (1, 0, 1, 64)):
        assert size(*shape) == 0, shape
