"""Rows that are written have a place each: strides that lead two rows or heads to the same bytes are refused before anything asks for a device, and layouts that do not are taken as far as
that.  Addresses here are never read."""
import numpy as np
import pytest

import slhav2_b200 as S
from tests.test_cache4_refusals_cpu import A, cache, heads, refused, rows, turn

SEG = S.make_segments([(0, 100, 0, 4, 0)])
KV = 4
D = 256  # codes 128 bytes, scales 16, bfloat16 rows 256 elements

SAME = [dict(row=16, head=128), dict(row=512, head=16), dict(row=112, head=128 * 100), dict(row=128, head=128), dict(row=384, head=128), dict(row=128, head=256), dict(row=128, head=288), dict(row=1024, head=64),
        dict(row=160, head=144), dict(row=1 << 40, head=1 << 41)]
APART = [dict(row=512, head=128), dict(row=128, head=12800), dict(row=1 << 40, head=128), dict(row=128, head=1 << 40), dict(row=528, head=128), dict(row=144, head=14400), dict(row=256, head=25600 + 128),
         dict(row=256, head=25600 - 128), dict(row=1024, head=256), dict(row=1 << 50, head=1 << 48)]


def read(to):
    S.read_cache4(cache(n_kv_heads=KV, head_dim=D), SEG, to)


def taken(call, *args):
    if S.device_count() == 0:
        refused(S.ERR_DEVICE, "", call, *args)


@pytest.mark.parametrize("k", SAME)
def test_strides_that_lead_to_the_same_place(k):
    near = S.make_segments([(0, 100, 0, 100, 0)])
    row, head = k["row"], k["head"]
    refused(S.ERR_DIMENSION, "place", lambda: S.write_cache4(cache(n_kv_heads=KV, head_dim=D, code_row_stride=row, code_head_stride=head), near, rows(n_kv_heads=KV, head_dim=D), 100))
    refused(S.ERR_DIMENSION, "keys", read, rows(n_kv_heads=KV, head_dim=D, values=None, key_row_stride=row * 2, key_head_stride=head * 2))
    refused(S.ERR_DIMENSION, "values", read, rows(n_kv_heads=KV, head_dim=D, keys=None, value_row_stride=row * 2, value_head_stride=head * 2))
    refused(S.ERR_DIMENSION, "keys", lambda: S.rotate_heads(heads(q=None, v=None, n_tokens=100, n_kv_heads=KV, head_dim=D), to=rows(n_kv_heads=KV, head_dim=D, values=None, key_row_stride=row * 2,
                                                                                                                                 key_head_stride=head * 2)))
    refused(S.ERR_DIMENSION, "q_out", lambda: S.rotate_heads(heads(k=None, v=None, n_heads=KV, n_tokens=100, head_dim=D), q_out=A, q_out_token_stride=row * 2, q_out_head_stride=head * 2))


@pytest.mark.parametrize("k", APART)
def test_strides_that_do_not(k):
    near = S.make_segments([(0, 100, 0, 100, 0)])
    row, head = k["row"], k["head"]
    taken(lambda: S.write_cache4(cache(n_kv_heads=KV, head_dim=D, code_row_stride=row, code_head_stride=head), near, rows(n_kv_heads=KV, head_dim=D), 100))
    taken(read, rows(n_kv_heads=KV, head_dim=D, values=None, key_row_stride=row * 2, key_head_stride=head * 2))
    taken(lambda: S.rotate_heads(heads(k=None, v=None, n_heads=KV, n_tokens=100, head_dim=D), q_out=A, q_out_token_stride=row * 2, q_out_head_stride=head * 2))


def test_only_rows_that_are_written_count():
    # two rows by heads: 100 rows of 128 bytes would reach into the next head, two do not
    k = cache(n_kv_heads=KV, head_dim=D, code_row_stride=128, code_head_stride=256)
    taken(lambda: S.write_cache4(k, S.make_segments([(50, 2, 0, 2, 0)]), rows(n_kv_heads=KV, head_dim=D), 2))
    refused(S.ERR_DIMENSION, "codes", lambda: S.write_cache4(k, S.make_segments([(50, 3, 0, 3, 0)]), rows(n_kv_heads=KV, head_dim=D), 3))
    refused(S.ERR_DIMENSION, "codes", lambda: S.write_cache4(k, S.make_segments([(50, 1, 0, 1, 0), (52, 1, 1, 1, 0)]), rows(n_kv_heads=KV, head_dim=D), 2))
    # one row, whatever its stride
    taken(lambda: S.write_cache4(cache(n_kv_heads=KV, head_dim=D, code_row_stride=16, code_head_stride=128), S.make_segments([(0, 1, 0, 1, 0)]), rows(n_kv_heads=KV, head_dim=D), 1))
    # counts of rows on the host say which are written
    few = cache(n_kv_heads=KV, head_dim=D, code_row_stride=128, code_head_stride=256, rows=np.array([2], np.uint32))
    taken(lambda: S.write_cache4(few, S.make_segments([(0, 100, 0, 2, 0)]), rows(n_kv_heads=KV, head_dim=D), 2))
    # no row
    taken(lambda: S.write_cache4(cache(n_kv_heads=KV, head_dim=D, code_row_stride=16, code_head_stride=16), S.make_segments([(0, 0, 0, 4, 0)]), rows(n_kv_heads=KV, head_dim=D), 4))


def test_one_head_and_default_strides():
    taken(lambda: S.write_cache4(cache(n_kv_heads=1, head_dim=D, code_row_stride=128, code_head_stride=16), SEG, rows(n_kv_heads=1, head_dim=D), 4))
    refused(S.ERR_DIMENSION, "codes", lambda: S.write_cache4(cache(n_kv_heads=1, head_dim=D, code_row_stride=112), SEG, rows(n_kv_heads=1, head_dim=D), 4))
    refused(S.ERR_DIMENSION, "scales", lambda: S.write_cache4(cache(n_kv_heads=2, head_dim=D, scale_row_stride=16), SEG, rows(n_kv_heads=2, head_dim=D), 4))
    refused(S.ERR_DIMENSION, "scales", lambda: S.write_cache4(cache(n_kv_heads=2, head_dim=80, scale_row_stride=8, scale_head_stride=24), SEG, rows(n_kv_heads=2, head_dim=80), 4))
    for d in (16, 48, 64, 80, 128, 208, 256):
        for kv in (1, 3, 8):
            taken(lambda: S.write_cache4(cache(n_kv_heads=kv, head_dim=d), SEG, rows(n_kv_heads=kv, head_dim=d), 4))
            taken(lambda: S.rotate_heads(heads(n_heads=kv, n_kv_heads=kv, head_dim=d), q_out=A, to=rows(n_kv_heads=kv, head_dim=d)))


def test_strides_at_random():
    if S.device_count() > 0:
        pytest.skip("a GPU is present")
    rng = np.random.default_rng(1)
    found = [0, 0]
    for _ in range(3000):
        kv, n, d = int(rng.integers(1, 6)), int(rng.integers(1, 9)), 16 * int(rng.integers(1, 9))
        row, head = (16 * int(x) for x in rng.integers(1, 40, 2))
        at = sorted(r * row + h * head for r in range(n) for h in range(kv))
        same = any(b - a < d // 2 for a, b in zip(at, at[1:]))
        found[same] += 1
        with pytest.raises(S.SlhaError) as e:
            S.write_cache4(cache(n_kv_heads=kv, head_dim=d, code_row_stride=row, code_head_stride=head), S.make_segments([(7, n, 0, n, 0)]), rows(n_kv_heads=kv, head_dim=d), n)
        assert e.value.code == (S.ERR_DIMENSION if same else S.ERR_DEVICE), (kv, n, d, row, head)
    assert min(found) > 300
