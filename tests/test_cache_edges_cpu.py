"""What the calls on a cache of rows refuse because there is no right answer: the same tokens or rows in two segments, scales that float32 cannot hold in units of log 2,
positions that wrap, rows that go to one place from several KV heads.  Addresses here are never read."""
import numpy as np
import pytest

import slhav2_b200 as S
from tests.test_cache_refusals_cpu import A, SEG, cache, queries, refused


def passes(call, *args, **more):
    """Past its checks of arguments: without a GPU the device is what is missing (with one the addresses would be)."""
    with pytest.raises(S.SlhaError) as e:
        call(*args, **more)
    assert e.value.code == S.ERR_DEVICE, e.value.message


# ---- the same tokens or rows twice
TWICE = [(0, 100, 0, 2, 0), (100, 100, 2, 2, 0), (300, 100, 1, 1, 0)]


def test_query_tokens_of_two_segments():
    segs = S.make_segments(TWICE)
    refused(S.ERR_DIMENSION, "tokens", S.attend_cache, cache(), segs, queries(), A)
    refused(S.ERR_DIMENSION, "tokens", S.attend_cache, cache(), segs[::-1], queries(), A)
    refused(S.ERR_DIMENSION, "tokens", S.attend_tree, cache(), segs, queries(), np.zeros(4, np.uint32), A)
    passes(S.observe_cache, cache(), segs, queries(), A, A, 400)  # (which only reads them)
    passes(S.attend_cache, cache(), S.make_segments([(0, 100, 2, 2, 0), (0, 100, 0, 2, 0), (0, 100, 1, 0, 0)]), queries(), A)  # any order, one prompt's rows for several, no tokens


def test_rows_of_two_segments():
    over, beside = S.make_segments([(50, 51, 0, 2, 0), (0, 50, 2, 1, 0), (100, 50, 3, 1, 0)]), S.make_segments([(50, 50, 0, 2, 0), (0, 50, 2, 1, 0), (100, 50, 3, 1, 0), (60, 0, 0, 0, 0)])
    refused(S.ERR_DIMENSION, "rows", S.observe_cache, cache(), over, queries(), A, A, 400)
    refused(S.ERR_DIMENSION, "rows", S.evict_cache, cache(), over, A, 400, 10)
    passes(S.attend_cache, cache(), over, queries(), A)
    for call, more in ((lambda k, s: S.observe_cache(k, s, queries(), A, A, 400), {}), (lambda k, s: S.evict_cache(k, s, A, 400, 10), {})):
        passes(call, cache(), beside)
        passes(call, cache(rows=np.array([50, 50, 50], np.uint32)), over)  # the table's room overlaps, the rows do not
        refused(S.ERR_DIMENSION, "rows", call, cache(rows=np.array([51, 50, 50], np.uint32)), over)
    # to another cache: where the rows go
    to = dict(to=cache(), to_segments=S.make_segments([(0, 10, 0, 0, 0), (9, 10, 0, 0, 0), (30, 10, 0, 0, 0)]))
    refused(S.ERR_DIMENSION, "rows", S.evict_cache, cache(), over, A, 400, 10, **to)
    passes(S.evict_cache, cache(), over, A, 400, 9, **to)


# ---- numbers that float32 does not hold
@pytest.mark.parametrize("call", [lambda k, s, q: S.attend_cache(k, s, q, A), lambda k, s, q: S.attend_tree(k, s, q, np.zeros(4, np.uint32), A),
                                  lambda k, s, q: S.observe_cache(k, s, q, A, A, 100)])
def test_scales_and_caps_at_the_ends_of_their_range(call):
    # scores are held in units of log 2, and a capped one as tanh(scale / softcap * product): neither factor may overflow or lose bits
    for bad in (dict(scale=3e38), dict(scale=-3e38), dict(softcap=3e38), dict(softcap=2.0 ** 101), dict(scale=1e-20, softcap=1e19), dict(scale=-1e-20, softcap=2e18)):
        refused(S.ERR_NONFINITE, "finite" if "softcap" not in bad else "softcap", call, cache(), SEG, queries(**bad))
    for good in (dict(scale=2e38), dict(softcap=2.0 ** 100), dict(scale=0.0, softcap=1e19), dict(scale=1e-20), dict(scale=1e-20, softcap=1e17)):
        passes(call, cache(), SEG, queries(**good))


# ---- positions that wrap
def test_tokens_whose_positions_would_wrap():
    # more tokens than rows, and no positions of their own: token i has position index_base + i
    top = 2 ** 32
    refused(S.ERR_DIMENSION, "2^32", S.attend_cache, cache(), S.make_segments([(0, 2, 0, 4, top - 3)]), queries(), A)
    refused(S.ERR_DIMENSION, "2^32", S.observe_cache, cache(), S.make_segments([(0, 0, 0, 4, top - 3)]), queries(), A, A, 100)
    passes(S.attend_cache, cache(), S.make_segments([(0, 2, 0, 4, top - 4)]), queries(), A)
    passes(S.attend_cache, cache(), S.make_segments([(0, 2, 0, 4, top - 3)]), queries(positions=np.zeros(4, np.uint32)), A)


# ---- places that several KV heads would write
def test_weights_and_tiles_of_heads_that_keep_different_rows():
    seg, to_seg = S.make_segments([(0, 100, 0, 0, 0)]), S.make_segments([(0, 50, 0, 0, 0)])
    to = dict(to=cache(), to_segments=to_seg)
    refused(S.ERR_DIMENSION, "weights_to", S.evict_cache, cache(), seg, A, 100, 50, weights_to=A, weights_to_head_stride=0, **to)
    refused(S.ERR_DIMENSION, "tiles", S.evict_cache, cache(), seg, A, 100, 50, tiles=A, tile_head_stride=100, tiles_to=A, tiles_to_head_stride=0, **to)
    refused(S.ERR_DIMENSION, "tiles", S.evict_cache, cache(), seg, A, 100, 50, tiles=A, tile_head_stride=0)  # in place
    # weights of the heads' own, or of all heads with positions of the heads' own that count
    own = dict(positions=A, entry_head_stride=100)
    refused(S.ERR_DIMENSION, "weights_to", S.evict_cache, cache(**own), seg, A, 0, 50, weights_to=A, weights_to_head_stride=0, sink_window=4)
    for bad in (dict(key_head_stride=0), dict(value_head_stride=0)):
        refused(S.ERR_DIMENSION, "rows", S.evict_cache, cache(), seg, A, 100, 50, to=cache(**bad), to_segments=to_seg)
    # every head keeps the same rows; a single head
    passes(S.evict_cache, cache(), seg, A, 0, 50, weights_to=A, weights_to_head_stride=0, tiles=A, tile_head_stride=0, sink_window=4)
    passes(S.evict_cache, cache(**own), seg, A, 0, 50, weights_to=A, weights_to_head_stride=0)
    passes(S.evict_cache, cache(n_kv_heads=1), seg, A, 0, 50, weights_to=A, tiles=A, to=cache(n_kv_heads=1), to_segments=to_seg, tiles_to=A)


# ---- tensors of other types and orders
def test_tensors_are_what_a_call_reads_them_as():
    torch = pytest.importorskip("torch")
    rows, heads, d = 8, 2, 64
    kv = torch.zeros(rows, heads, d, dtype=torch.bfloat16)
    u32, f32 = torch.zeros(heads * rows, dtype=torch.int32), torch.zeros(heads * rows)
    seg = S.make_segments([(0, rows, 0, 4, 0)])
    for what, more in (("keys", dict(keys=kv.float())), ("keys", dict(keys=kv.half())), ("values", dict(values=kv.float())), ("keys", dict(dtype=S.F32)), ("positions", dict(positions=u32.long())),
                       ("documents", dict(documents=f32)), ("rows", dict(rows=u32.long())), ("keys", dict(keys=np.zeros((rows, heads, d))))):
        with pytest.raises(TypeError, match=what):
            cache(**{**dict(keys=kv, values=kv), **more})
    for what, more in (("q", dict(q=torch.zeros(4, 4, d, dtype=torch.float64))), ("slopes", dict(slopes=f32.double())), ("prefix", dict(prefix=u32.short())), ("positions", dict(positions=u32.long())),
                       ("documents", dict(documents=f32))):
        with pytest.raises(TypeError, match=what):
            queries(**more)
    with pytest.raises(ValueError, match="keys"):
        cache(keys=kv.transpose(0, 1), values=kv)
    with pytest.raises(ValueError, match="q"):
        queries(q=kv.transpose(0, 1))
    cache(keys=kv.transpose(0, 1), values=kv, key_row_stride=heads * d)  # strides that are given are the caller's
    k, q = cache(keys=kv, values=kv.view(torch.int16)), queries(q=torch.zeros(4, 4, d, dtype=torch.bfloat16))
    for what, call in (("q", lambda: S.attend_cache(k, seg, queries(q=torch.zeros(4, 4, d)), A)), ("out", lambda: S.attend_cache(k, seg, q, torch.zeros(4, 4, d))),
                       ("lse_out", lambda: S.attend_cache(k, seg, q, A, torch.zeros(4, 4, dtype=torch.bfloat16))), ("parents", lambda: S.attend_tree(k, seg, q, u32.long(), A)),
                       ("q", lambda: S.observe_cache(k, seg, queries(q=torch.zeros(4, 4, d)), A, A, 8)), ("lse", lambda: S.observe_cache(k, seg, q, f32.double(), A, 8)),
                       ("weights_out", lambda: S.observe_cache(k, seg, q, A, f32.double(), 8)), ("weights", lambda: S.evict_cache(k, seg, u32, 8, 4)),
                       ("rows_out", lambda: S.evict_cache(k, seg, A, 8, 4, rows_out=u32.long())), ("source_out", lambda: S.evict_cache(k, seg, A, 8, 4, source_out=f32))):
        with pytest.raises(TypeError, match=what):
            call()
    passes(S.attend_cache, k, seg, q, torch.zeros(4, 4, d, dtype=torch.bfloat16), torch.zeros(4, 4))


# ---- arrays that begin within a word
def test_arrays_of_words_begin_on_one():
    bad, word = A + 2, "multiple of 4"
    seg, one = SEG, S.make_segments([(0, 100, 0, 0, 0)])
    for more in (dict(positions=bad), dict(documents=bad), dict(rows=type("Raw", (), {"data_ptr": lambda self: bad})())):
        k = cache(**more)
        q = queries(positions=type("Raw", (), {"data_ptr": lambda self: A})(), documents=type("Raw", (), {"data_ptr": lambda self: A})() if "documents" in more else None)
        refused(S.ERR_DIMENSION, word, S.attend_cache, k, seg, q, A)
        refused(S.ERR_DIMENSION, word, S.observe_cache, k, seg, q, A, A, 100)
        refused(S.ERR_DIMENSION, word, S.evict_cache, cache(entry_head_stride=100, **more), one, A, 100, 50)
    raw = type("Raw", (), {"data_ptr": lambda self: bad})()
    for more in (dict(slopes=raw), dict(prefix=raw), dict(positions=raw)):
        refused(S.ERR_DIMENSION, word, S.attend_cache, cache(), seg, queries(**more), A)
    refused(S.ERR_DIMENSION, word, S.attend_cache, cache(), seg, queries(), A, bad)
    refused(S.ERR_DIMENSION, word, S.attend_tree, cache(), seg, queries(), raw, A)
    for args in ((bad, A), (A, bad)):
        refused(S.ERR_DIMENSION, word, S.observe_cache, cache(), seg, queries(), *args, 100)
    refused(S.ERR_DIMENSION, word, S.observe_cache, cache(), seg, queries(), A, A, 100, weights_in=bad)
    refused(S.ERR_DIMENSION, word, S.evict_cache, cache(), one, bad, 100, 50)
    for more in (dict(source_out=bad), dict(rows_out=bad)):
        refused(S.ERR_DIMENSION, word, S.evict_cache, cache(), one, A, 100, 50, **more)
