"""What the calls on a cache of rows refuse before they ask for a device: addresses here are never read."""
import numpy as np
import pytest

import slhav2_b200 as S

A = 1 << 20  # an aligned address that nothing is read from


def cache(**more):
    kind = dict(keys=A, values=A, n_kv_heads=2, head_dim=64, dtype=S.BF16)
    kind.update(more)
    return S.KvCache(**kind)


def queries(**more):
    kind = dict(q=A, n_tokens=4, n_heads=4, head_dim=64)
    kind.update(more)
    return S.CacheQueries(**kind)


SEG = S.make_segments([(0, 100, 0, 4, 0)])


def refused(code, word, call, *args, **more):
    with pytest.raises(S.SlhaError) as e:
        call(*args, **more)
    assert e.value.code == code and word in e.value.message, e.value.message


@pytest.mark.parametrize("call", [lambda k, s, q: S.attend_cache(k, s, q, A), lambda k, s, q: S.attend_tree(k, s, q, np.zeros(4, np.uint32), A),
                                  lambda k, s, q: S.observe_cache(k, s, q, A, A, 100)])
def test_what_no_call_with_queries_takes(call):
    refused(S.ERR_NULL, "NULL", call, cache(keys=None), SEG, queries())
    for bad in (dict(dtype=7), dict(head_dim=0), dict(head_dim=60), dict(head_dim=264), dict(n_kv_heads=0), dict(n_kv_heads=70000), dict(key_row_stride=65),
                dict(key_head_stride=4), dict(keys=A + 2)):
        refused(S.ERR_DIMENSION, "", call, cache(**bad), SEG, queries())
    refused(S.ERR_DIMENSION, "head_dim", call, cache(dtype=S.F32, head_dim=66), SEG, queries())
    refused(S.ERR_NULL, "q is NULL", call, cache(), SEG, queries(q=None))
    for bad in (dict(n_heads=0), dict(n_heads=3), dict(token_stride=3), dict(head_stride=1), dict(q=A + 8)):
        refused(S.ERR_DIMENSION, "", call, cache(), SEG, queries(**bad))
    for bad in (dict(scale=float("nan")), dict(softcap=-1.0), dict(softcap=float("inf")), dict(softcap=1e-42, scale=1.0)):
        refused(S.ERR_NONFINITE, "finite", call, cache(), SEG, queries(**bad))
    refused(S.ERR_NULL, "positions", call, cache(positions=A), SEG, queries())
    refused(S.ERR_NULL, "documents", call, cache(documents=A), SEG, queries())
    refused(S.ERR_NULL, "documents", call, cache(), SEG, queries(documents=np.zeros(4, np.uint32)))
    refused(S.ERR_DIMENSION, "n_tokens", call, cache(), S.make_segments([(0, 100, 1, 4, 0)]), queries())
    refused(S.ERR_DIMENSION, "n_tokens", call, cache(), S.make_segments([(0, 100, 0xFFFFFFFF, 4, 0)]), queries())
    refused(S.ERR_DIMENSION, "2^32", call, cache(), S.make_segments([(0, 100, 0, 4, 0xFFFFFFF0)]), queries())


def test_what_attention_refuses():
    refused(S.ERR_NULL, "NULL", S.attend_cache, cache(), SEG, queries(), None)
    refused(S.ERR_NULL, "values", S.attend_cache, cache(values=None), SEG, queries(), A)
    refused(S.ERR_DIMENSION, "out", S.attend_cache, cache(), SEG, queries(), A + 4)
    refused(S.ERR_DIMENSION, "out", S.attend_cache, cache(), SEG, queries(), A, out_token_stride=5)
    refused(S.ERR_DIMENSION, "value", S.attend_cache, cache(values=A + 2), SEG, queries(), A)
    refused(S.ERR_DIMENSION, "strides", S.attend_cache, cache(value_row_stride=1), SEG, queries(), A)
    assert S.attend_cache(cache(), S.make_segments([]), queries(), A) == A  # nothing to do


def test_what_trees_refuse():
    refused(S.ERR_NULL, "NULL", lambda: S.api._check(S.load_library().slha_b200_attend_tree(cache().address, SEG.ctypes.data, 1, queries().address, None, A, 256, 64, None)))
    refused(S.ERR_DIMENSION, "256", S.attend_tree, cache(), S.make_segments([(0, 400, 0, 257, 0)]), queries(n_tokens=257), np.zeros(257, np.uint32), A)
    refused(S.ERR_DIMENSION, "last rows", S.attend_tree, cache(), S.make_segments([(0, 3, 0, 4, 0)]), queries(), np.zeros(4, np.uint32), A)


def test_what_observation_refuses():
    refused(S.ERR_NULL, "NULL", S.observe_cache, cache(), SEG, queries(), None, A, 100)
    refused(S.ERR_NULL, "NULL", S.observe_cache, cache(), SEG, queries(), A, None, 100)
    refused(S.ERR_NONFINITE, "decay", S.observe_cache, cache(), SEG, queries(), A, A, 100, decay=float("inf"))


def test_what_removal_refuses():
    seg = S.make_segments([(0, 100, 0, 0, 0)])
    to = cache(positions=A, entry_head_stride=50)
    to_seg = S.make_segments([(0, 50, 0, 0, 0)])
    refused(S.ERR_NULL, "NULL", S.evict_cache, cache(), seg, None, 100, 50)
    refused(S.ERR_DIMENSION, "budget", S.evict_cache, cache(), seg, A, 100, 0)
    refused(S.ERR_NULL, "NULL", S.evict_cache, cache(), seg, A, 100, 50, to=cache())
    refused(S.ERR_DIMENSION, "same", S.evict_cache, cache(), seg, A, 100, 50, to=cache(head_dim=128), to_segments=to_seg)
    refused(S.ERR_NULL, "positions", S.evict_cache, cache(), seg, A, 100, 50, to=to, to_segments=to_seg)
    refused(S.ERR_DIMENSION, "entry_head_stride", S.evict_cache, cache(positions=A), seg, A, 100, 50)
    refused(S.ERR_DIMENSION, "entry_head_stride", S.evict_cache, cache(positions=A), seg, A, 100, 50, to=cache(positions=A), to_segments=to_seg)
    refused(S.ERR_NULL, "tiles_to", S.evict_cache, cache(), seg, A, 100, 50, to=cache(), to_segments=to_seg, tiles=A)
    refused(S.ERR_DIMENSION, "tiles", S.evict_cache, cache(), seg, A, 100, 50, tiles=A + 4)
    refused(S.ERR_DIMENSION, "weights_to", S.evict_cache, cache(), seg, A, 100, 50, weights_to=A + 64, weights_to_head_stride=100)
    refused(S.ERR_CAPACITY, "room", S.evict_cache, cache(), seg, A, 100, 51, to=cache(), to_segments=to_seg)
    refused(S.ERR_DIMENSION, "2^32", S.evict_cache, cache(), S.make_segments([(0, 100, 0, 0, 0xFFFFFFFF)]), A, 100, 50)


def test_calls_that_pass_their_checks_need_a_device():
    if S.device_count() > 0:
        pytest.skip("a GPU is present")
    refused(S.ERR_DEVICE, "", S.attend_cache, cache(), SEG, queries(), A)
    refused(S.ERR_DEVICE, "", S.observe_cache, cache(values=None), SEG, queries(), A, A, 100)
    refused(S.ERR_DEVICE, "", S.evict_cache, cache(), SEG, A, 100, 50)
