"""The shared-prefix attention's entry point without a device: what it refuses."""
import math

import pytest

from test_paged import fake
from test_paged_q8 import past

ATTEND = dict(q=fake(0), kcache=fake(1), vcache=fake(2), out=fake(3), tables=fake(4), sequences=4, table_pages=8,
              query_sequence=fake(5), positions=fake(6), queries=3, prefix=fake(7), heads=14, kv_heads=2, head_dim=64,
              pages=64, page_size=16, scale=0.125, workspace=fake(8), workspace_bytes=1 << 30, stream=None)
READ = ("kcache", "vcache", "tables", "query_sequence", "positions", "prefix")
REFUSALS = [
    *[({k: None}, "MUYO_E_NULL") for k in ("q", "out", *READ)],
    (dict(queries=0), "MUYO_E_UNSUPPORTED"),
    (dict(queries=65536), "MUYO_E_UNSUPPORTED"),
    (dict(kv_heads=3), "MUYO_E_UNSUPPORTED"),
    (dict(heads=34), "MUYO_E_UNSUPPORTED"),
    (dict(head_dim=96), "MUYO_E_UNSUPPORTED"),
    (dict(page_size=20), "MUYO_E_UNSUPPORTED"),
    (dict(sequences=0), "MUYO_E_RANGE"),
    (dict(table_pages=0), "MUYO_E_RANGE"),
    (dict(pages=1 << 27), "MUYO_E_RANGE"),
    *[({k: past(ATTEND[k], 4)}, "MUYO_E_CONTRACT") for k in ("q", "kcache", "vcache", "out", "workspace")],
    (dict(scale=math.inf), "MUYO_E_CONTRACT"),
    (dict(workspace=None), "MUYO_E_CONTRACT"),
    (dict(workspace_bytes=15), "MUYO_E_CONTRACT"),
    (dict(out=past(ATTEND["q"], 3584)), "MUYO_E_CONTRACT"),
    *[({w: ATTEND[k]}, "MUYO_E_CONTRACT") for w in ("out", "workspace") for k in READ],
    (dict(workspace=ATTEND["q"]), "MUYO_E_CONTRACT"),
    (dict(out=ATTEND["workspace"]), "MUYO_E_CONTRACT"),
]


@pytest.mark.parametrize("case", REFUSALS, ids=[f"{i}-{'-'.join(c[0])}" for i, c in enumerate(REFUSALS)])
def test_refused_before_anything_is_launched(mh, case):
    change, status = case
    assert mh.load().muyo_paged_attention_prefix_f16kv(*{**ATTEND, **change}.values()) == getattr(mh, status)
    assert b"paged_attention_prefix_f16kv" in mh.load().muyo_last_error()


def test_workspace_sizes(mh):
    lib = mh.load()
    size = lib.muyo_paged_attention_prefix_f16kv_workspace_bytes
    for shape in ((1, 14, 2, 64), (250, 28, 4, 128), (65535, 28, 4, 128)):
        assert size(*shape) > lib.muyo_paged_attention_decode_f16kv_workspace_bytes(*shape)
    for shape in ((0, 14, 2, 64), (1, 14, 3, 64), (1, 34, 2, 64), (1, 14, 2, 80), (65536, 14, 2, 64)):
        assert size(*shape) == 0, shape
