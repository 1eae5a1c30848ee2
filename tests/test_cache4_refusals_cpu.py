"""What the calls on rows of 4 bits, and the rotation of heads, refuse before they ask for a device: addresses here are never read."""
import numpy as np
import pytest

import slhav2_b200 as S

A = 1 << 20  # an aligned address that nothing is read from
SEG = S.make_segments([(0, 100, 0, 4, 0)])


def cache(**more):
    kind = dict(key_codes=A, value_codes=A, key_scales=A, value_scales=A, n_kv_heads=2, head_dim=64)
    kind.update(more)
    return S.KvCache4(**kind)


def rows(**more):
    kind = dict(keys=A, values=A, n_kv_heads=2, head_dim=64)
    kind.update(more)
    return S.KvCache(**kind)


def queries(**more):
    kind = dict(q=A, n_tokens=4, n_heads=4, head_dim=64)
    kind.update(more)
    return S.CacheQueries(**kind)


def heads(**more):
    kind = dict(q=A, k=A, v=A, n_tokens=4, n_heads=4, n_kv_heads=2, head_dim=64)
    kind.update(more)
    return S.HeadRows(**kind)


def turn(**more):
    kind = dict(frequencies=np.ones(32, np.float32), positions=np.zeros(4, np.uint32), rotary_dim=64)
    kind.update(more)
    return S.Rotation(**kind)


def refused(code, word, call, *args, **more):
    with pytest.raises(S.SlhaError) as e:
        call(*args, **more)
    assert e.value.code == code and word in e.value.message, e.value.message


CALLS = [lambda k, s=SEG: S.attend_cache4(k, s, queries(head_dim=k.head_dim, scale=1.0), A), lambda k, s=SEG: S.attend_tree4(k, s, queries(head_dim=k.head_dim, scale=1.0), np.zeros(4, np.uint32), A),
         lambda k, s=SEG: S.write_cache4(k, s, rows(head_dim=max(16, k.head_dim), n_kv_heads=k.n_kv_heads), 4), lambda k, s=SEG: S.read_cache4(k, s, rows(head_dim=max(16, k.head_dim), n_kv_heads=k.n_kv_heads))]


@pytest.mark.parametrize("call", CALLS)
def test_caches_that_no_call_takes(call):
    for name in ("key_codes", "value_codes", "key_scales", "value_scales"):
        refused(S.ERR_NULL, "NULL", call, cache(**{name: None}))
        refused(S.ERR_DIMENSION, "begin", call, cache(**{name: A + 2}))
    for bad in (dict(dtype=7), dict(head_dim=0), dict(head_dim=24), dict(head_dim=272), dict(n_kv_heads=0), dict(n_kv_heads=70000), dict(code_row_stride=72), dict(code_head_stride=40),
                dict(scale_row_stride=6), dict(scale_head_stride=2), dict(key_exponent=65), dict(value_exponent=-65), dict(key_exponent=-2 ** 31)):
        refused(S.ERR_DIMENSION, "", call, cache(**bad))
    refused(S.ERR_DIMENSION, "8 bytes", call, cache(head_dim=80, scale_row_stride=12))
    refused(S.ERR_DIMENSION, "16 bytes", call, cache(head_dim=256, scale_head_stride=24))
    refused(S.ERR_DIMENSION, "4 bytes", call, cache(rows=A + 2))


@pytest.mark.parametrize("call", [lambda k, s, q: S.attend_cache4(k, s, q, A), lambda k, s, q: S.attend_tree4(k, s, q, np.zeros(4, np.uint32), A)])
def test_queries_that_attention_refuses(call):
    refused(S.ERR_NULL, "q is NULL", call, cache(), SEG, queries(q=None))
    for bad in (dict(n_heads=0), dict(n_heads=3), dict(token_stride=3), dict(head_stride=1), dict(q=A + 8)):
        refused(S.ERR_DIMENSION, "", call, cache(), SEG, queries(**bad))
    for bad in (dict(scale=float("nan")), dict(softcap=-1.0), dict(softcap=float("inf")), dict(softcap=1e-42, scale=1.0)):
        refused(S.ERR_NONFINITE, "finite", call, cache(), SEG, queries(**bad))
    refused(S.ERR_NONFINITE, "key_exponent", call, cache(key_exponent=64), SEG, queries(scale=1e30))
    refused(S.ERR_NONFINITE, "key_exponent", call, cache(key_exponent=-64), SEG, queries(scale=1e-25))
    refused(S.ERR_NULL, "positions", call, cache(positions=A), SEG, queries())
    refused(S.ERR_NULL, "documents", call, cache(), SEG, queries(documents=np.zeros(4, np.uint32)))
    refused(S.ERR_DIMENSION, "n_tokens", call, cache(), S.make_segments([(0, 100, 1, 4, 0)]), queries())
    refused(S.ERR_DIMENSION, "2^32", call, cache(), S.make_segments([(0, 100, 0, 4, 0xFFFFFFF0)]), queries())
    refused(S.ERR_DIMENSION, "same query tokens", call, cache(), S.make_segments([(0, 100, 0, 3, 0), (100, 100, 2, 2, 0)]), queries())


def test_what_else_attention_refuses():
    refused(S.ERR_NULL, "NULL", S.attend_cache4, cache(), SEG, queries(), None)
    refused(S.ERR_DIMENSION, "out", S.attend_cache4, cache(), SEG, queries(), A + 4)
    refused(S.ERR_DIMENSION, "out", S.attend_cache4, cache(), SEG, queries(), A, out_token_stride=5)
    refused(S.ERR_DIMENSION, "4 bytes", S.attend_cache4, cache(), SEG, queries(), A, A + 1)
    assert S.attend_cache4(cache(), S.make_segments([]), queries(), A) == A
    refused(S.ERR_DIMENSION, "256", S.attend_tree4, cache(), S.make_segments([(0, 400, 0, 257, 0)]), queries(n_tokens=257), np.zeros(257, np.uint32), A)
    refused(S.ERR_DIMENSION, "last rows", S.attend_tree4, cache(), S.make_segments([(0, 3, 0, 4, 0)]), queries(), np.zeros(4, np.uint32), A)
    with pytest.raises(TypeError):
        cache(key_scales=np.zeros(4, np.float32))


def test_what_writing_refuses():
    write = lambda k, s, r, n=4: S.write_cache4(k, s, r, n)  # noqa: E731
    refused(S.ERR_NULL, "NULL", write, cache(), SEG, rows(values=None))
    for bad in (dict(dtype=3), dict(head_dim=128), dict(n_kv_heads=1), dict(keys=A + 8), dict(value_row_stride=4), dict(key_head_stride=2)):
        refused(S.ERR_DIMENSION, "from", write, cache(), SEG, rows(**bad))
    for bad in (dict(code_row_stride=0), dict(code_head_stride=0), dict(scale_row_stride=0), dict(scale_head_stride=0)):
        refused(S.ERR_DIMENSION, "place", write, cache(**bad), SEG, rows())
    refused(S.ERR_DIMENSION, "n_tokens", write, cache(), S.make_segments([(0, 100, 1, 4, 0)]), rows())
    refused(S.ERR_DIMENSION, "same rows", write, cache(), S.make_segments([(0, 100, 0, 3, 0), (90, 9, 3, 1, 0)]), rows())
    write(cache(), S.make_segments([]), rows())
    # rows that two segments share in front of their tokens' are no fault
    if S.device_count() == 0:
        refused(S.ERR_DEVICE, "", write, cache(rows=np.array([50, 60], np.uint32)), S.make_segments([(0, 100, 0, 3, 0), (0, 100, 3, 1, 0)]), rows())
    refused(S.ERR_DIMENSION, "same rows", write, cache(rows=np.array([60, 60], np.uint32)), S.make_segments([(0, 100, 0, 3, 0), (0, 100, 3, 1, 0)]), rows())


def test_what_reading_refuses():
    refused(S.ERR_NULL, "NULL", S.read_cache4, cache(), SEG, rows(keys=None, values=None))
    for bad in (dict(dtype=3), dict(head_dim=128), dict(keys=A + 8), dict(value_row_stride=4)):
        refused(S.ERR_DIMENSION, "to", S.read_cache4, cache(), SEG, rows(**bad))
    for bad in (dict(key_row_stride=0), dict(value_head_stride=0)):
        refused(S.ERR_DIMENSION, "place", S.read_cache4, cache(), SEG, rows(**bad))
    refused(S.ERR_CAPACITY, "room", S.read_cache4, cache(), SEG, rows(), S.make_segments([(0, 99, 0, 0, 0)]))
    two = S.make_segments([(0, 100, 0, 0, 0), (100, 50, 0, 0, 0)])
    refused(S.ERR_DIMENSION, "same rows", S.read_cache4, cache(), two, rows(), S.make_segments([(0, 100, 0, 0, 0), (99, 50, 0, 0, 0)]))
    with pytest.raises(ValueError):
        S.read_cache4(cache(), two, rows(), SEG)


def test_what_rotation_refuses():
    go = lambda h, r=None, **more: S.rotate_heads(h, r, **dict(dict(q_out=A, to=rows()), **more))  # noqa: E731
    refused(S.ERR_NULL, "no heads", go, heads(q=None, k=None, v=None), turn())
    refused(S.ERR_NULL, "q_out", go, heads(), turn(), q_out=None)
    refused(S.ERR_NULL, "rows", go, heads(), turn(), to=None)
    refused(S.ERR_NULL, "to", go, heads(), turn(), to=rows(values=None))
    for bad in (dict(dtype=5), dict(head_dim=60), dict(head_dim=264), dict(n_heads=0), dict(n_kv_heads=0), dict(q=A + 8), dict(token_stride=4), dict(head_stride=12)):
        refused(S.ERR_DIMENSION, "", go, heads(**bad), turn())
    refused(S.ERR_DIMENSION, "q_out", go, heads(), turn(), q_out=A + 4)
    refused(S.ERR_DIMENSION, "q_out", go, heads(), turn(), q_out_head_stride=0)
    refused(S.ERR_DIMENSION, "dtype", go, heads(), turn(), to=rows(dtype=S.F32))
    refused(S.ERR_DIMENSION, "head_dim", go, heads(), turn(), to=rows(head_dim=128))
    refused(S.ERR_DIMENSION, "place", go, heads(), turn(), to=rows(key_head_stride=0))
    refused(S.ERR_NONFINITE, "eps", go, heads(norm=True, eps=float("nan")), turn())
    refused(S.ERR_NONFINITE, "eps", go, heads(norm=True, eps=-1.0), turn())
    refused(S.ERR_DIMENSION, "norm", go, heads(q_weight=np.ones(64, np.float32)), turn())
    refused(S.ERR_DIMENSION, "weights", go, heads(norm=True, q_weight=A + 8), turn())
    refused(S.ERR_NULL, "NULL", go, heads(), turn(frequencies=None))
    refused(S.ERR_NULL, "NULL", go, heads(), turn(positions=None))
    for bad in (dict(rotary_dim=0), dict(rotary_dim=72), dict(rotary_dim=60), dict(n_axes=0), dict(n_axes=2), dict(n_axes=3, axes=np.full(32, 3, np.uint8))):
        refused(S.ERR_DIMENSION, "", go, heads(), turn(**bad))
    refused(S.ERR_NONFINITE, "magnitude", go, heads(), turn(magnitude=float("inf")))
    refused(S.ERR_DIMENSION, "n_tokens", go, heads(), turn(), segments=S.make_segments([(0, 10, 2, 3, 0)]))
    refused(S.ERR_DIMENSION, "same rows", go, heads(), turn(), segments=S.make_segments([(0, 10, 0, 2, 0), (5, 5, 2, 1, 0)]))
    refused(S.ERR_DIMENSION, "same tokens", go, heads(), turn(), segments=S.make_segments([(0, 10, 0, 2, 0), (10, 5, 1, 1, 0)]))
    with pytest.raises(TypeError):
        heads(k=np.zeros(4, np.float64))


def test_calls_that_pass_their_checks_need_a_device():
    if S.device_count() > 0:
        pytest.skip("a GPU is present")
    for call in CALLS:
        refused(S.ERR_DEVICE, "", call, cache())
    refused(S.ERR_DEVICE, "", S.rotate_heads, heads(), turn(), q_out=A, to=rows(), segments=SEG)
