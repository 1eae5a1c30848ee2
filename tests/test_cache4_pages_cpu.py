"""Caches that lie sequence by sequence, or page by page, [sequence][head][row]: a sequence's rows begin at sequence * heads * room, heads are `room` rows apart.  The rows between two sequences'
first heads are other heads', which no call takes for shared places unless it writes them as rows too.  Addresses here are never read."""
import numpy as np
import pytest

import slhav2_b200 as S
from tests.test_cache4_refusals_cpu import A, cache, heads, refused, rows

KV, ROOM, D = 8, 64, 128
PAGES = dict(n_kv_heads=KV, head_dim=D, code_row_stride=D // 2, code_head_stride=ROOM * D // 2, scale_row_stride=8, scale_head_stride=ROOM * 8)
TO = dict(n_kv_heads=KV, head_dim=D, key_row_stride=D, key_head_stride=ROOM * D, value_row_stride=D, value_head_stride=ROOM * D)


def taken(call):
    if S.device_count() == 0:
        refused(S.ERR_DEVICE, "", call)


@pytest.mark.parametrize("tokens", [1, 5, ROOM])
def test_sequences_that_lie_head_by_head(tokens):
    segs = S.make_segments([(i * KV * ROOM, ROOM, i * tokens, tokens, 0) for i in (0, 1, 2, 5)][:3] + [(5 * KV * ROOM, ROOM, 3 * tokens, tokens, 0)])
    taken(lambda: S.write_cache4(cache(**PAGES), segs, rows(n_kv_heads=KV, head_dim=D), 4 * tokens))
    taken(lambda: S.write_cache4(cache(rows=np.full(4, 40, np.uint32), **PAGES), segs, rows(n_kv_heads=KV, head_dim=D), 4 * tokens))
    taken(lambda: S.read_cache4(cache(**PAGES), segs, rows(**TO)))
    taken(lambda: S.rotate_heads(heads(q=None, n_tokens=4 * tokens, n_kv_heads=KV, head_dim=D), to=rows(**TO), segments=segs))


def test_rows_that_reach_into_the_next_head():
    for begin, n in ((0, ROOM + 1), (3 * KV * ROOM - 1, 2)):
        segs = S.make_segments([(0, ROOM, 0, 1, 0), (begin + KV * ROOM, n, 1, n, 0)])
        if begin == 0:
            refused(S.ERR_DIMENSION, "codes", lambda: S.write_cache4(cache(**PAGES), segs, rows(n_kv_heads=KV, head_dim=D), n + 1))
            refused(S.ERR_DIMENSION, "keys", lambda: S.rotate_heads(heads(q=None, n_tokens=n + 1, n_kv_heads=KV, head_dim=D), to=rows(**TO), segments=segs))
        else:
            taken(lambda: S.write_cache4(cache(**PAGES), segs, rows(n_kv_heads=KV, head_dim=D), n + 1))
    # the first head of one sequence in the second head of another
    segs = S.make_segments([(0, ROOM, 0, ROOM, 0), (ROOM + 10, 3, ROOM, 3, 0)])
    refused(S.ERR_DIMENSION, "codes", lambda: S.write_cache4(cache(**PAGES), segs, rows(n_kv_heads=KV, head_dim=D), ROOM + 3))
    refused(S.ERR_DIMENSION, "keys", lambda: S.read_cache4(cache(n_kv_heads=KV, head_dim=D), segs, rows(**TO)))


def test_queries_of_some_tokens():
    # [token][head], tokens half a head apart: those of the segments are even ones
    segs = S.make_segments([(0, 1, 2 * i, 1, 0) for i in range(4)])
    taken(lambda: S.rotate_heads(heads(k=None, v=None, n_heads=1, n_tokens=8, head_dim=64), q_out=A, q_out_token_stride=32, q_out_head_stride=64, segments=segs))
    refused(S.ERR_DIMENSION, "q_out", lambda: S.rotate_heads(heads(k=None, v=None, n_heads=1, n_tokens=8, head_dim=64), q_out=A, q_out_token_stride=32, q_out_head_stride=64))


def test_segments_at_random():
    if S.device_count() > 0:
        pytest.skip("a GPU is present")
    rng = np.random.default_rng(2)
    found = [0, 0]
    for _ in range(3000):
        kv, d = int(rng.integers(1, 6)), 16 * int(rng.integers(1, 9))
        row, head = (16 * int(x) for x in rng.integers(1, 12, 2))
        segs, at, q = [], int(rng.integers(0, 50)), 0
        for _ in range(int(rng.integers(1, 5))):
            n, t = int(rng.integers(0, 5)), int(rng.integers(0, 5))
            segs.append((at, n, q, t, 0))
            at += n + int(rng.choice([0, 1, 3, 10, 40]))
            q += t
        if q == 0:
            continue
        written = [b + n - min(n, t) + j for b, n, _, t, _ in segs for j in range(min(n, t))]
        rng.shuffle(segs)
        places = sorted(r * row + h * head for r in written for h in range(kv))
        same = any(b - a < d // 2 for a, b in zip(places, places[1:]))
        found[same] += 1
        with pytest.raises(S.SlhaError) as e:
            S.write_cache4(cache(n_kv_heads=kv, head_dim=d, code_row_stride=row, code_head_stride=head), S.make_segments(segs), rows(n_kv_heads=kv, head_dim=d), q)
        assert e.value.code == (S.ERR_DIMENSION if same else S.ERR_DEVICE), (kv, d, row, head, segs)
    assert min(found) > 300
