"""The batch sampler's entry point without a device: what it refuses."""
import ctypes

import pytest

from test_paged import fake
from test_paged_q8 import past

SAMPLE = dict(logits=fake(0), row_stride=1000, rows=3, vocab=1000, temperatures=fake(1), top_ks=fake(2),
              top_ps=fake(3), min_ps=fake(4), randoms=fake(5), tokens=fake(6), logprobs=fake(7), workspace=fake(8),
              workspace_bytes=1 << 30, stream=None)
READ = ("logits", "temperatures", "top_ks", "top_ps", "min_ps", "randoms")
REFUSALS = [
    *[({k: None}, "MUYO_E_NULL") for k in ("logits", "randoms", "tokens")],
    (dict(rows=0), "MUYO_E_RANGE"),
    (dict(rows=1 << 22), "MUYO_E_RANGE"),
    (dict(vocab=0), "MUYO_E_RANGE"),
    (dict(vocab=(1 << 24) + 1, row_stride=1 << 25), "MUYO_E_RANGE"),
    (dict(row_stride=999), "MUYO_E_CONTRACT"),
    (dict(logits=ctypes.c_void_p(2)), "MUYO_E_CONTRACT"),
    (dict(randoms=past(SAMPLE["randoms"], 4)), "MUYO_E_CONTRACT"),
    (dict(workspace=None), "MUYO_E_CONTRACT"),
    (dict(workspace=past(SAMPLE["workspace"], 8)), "MUYO_E_CONTRACT"),
    (dict(workspace_bytes=15), "MUYO_E_CONTRACT"),
    *[({w: SAMPLE[k]}, "MUYO_E_CONTRACT") for w in ("tokens", "logprobs", "workspace") for k in READ],
    (dict(tokens=SAMPLE["logprobs"]), "MUYO_E_CONTRACT"),
    (dict(tokens=past(SAMPLE["workspace"], 16)), "MUYO_E_CONTRACT"),
    (dict(logprobs=past(SAMPLE["randoms"], 20)), "MUYO_E_CONTRACT"),
    (dict(tokens=past(SAMPLE["logits"], 4 * 2999)), "MUYO_E_CONTRACT"),
]


@pytest.mark.parametrize("case", REFUSALS, ids=[f"{i}-{'-'.join(c[0])}" for i, c in enumerate(REFUSALS)])
def test_refused_before_anything_is_launched(mh, case):
    change, status = case
    assert mh.load().muyo_sample_rows_f32(*{**SAMPLE, **change}.values()) == getattr(mh, status)
    assert b"sample_rows_f32" in mh.load().muyo_last_error()


def test_workspace_sizes_of_unsupported_shapes_are_zero(mh):
    size = mh.load().muyo_sample_rows_workspace_bytes
    assert size(1, 1) > 0 and size((1 << 22) - 1, 1000) > 0 and size(1, 1 << 24) > 0
    for shape in ((0, 100), (1, 0), (1 << 22, 100), (1, (1 << 24) + 1)):
        assert size(*shape) == 0, shape


def test_lists_take_no_more_than_their_rows_have(mh):
    """What rows that are listed need beside others: a row's steps, and a key for each logit up to 4096."""
    size = mh.load().muyo_sample_rows_workspace_bytes
    for vocab in (1, 7, 1000, 4096, 30000):
        assert size(4096, vocab) - size(4097, vocab) <= 4096 * (6200 + 8 * min(vocab, 4096)), vocab
