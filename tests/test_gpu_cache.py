"""Exact attention over a cache of rows (slha_b200_attend_cache, slha_b200_attend_tree), the weight that rows receive (slha_b200_observe_cache) and
their removal (slha_b200_evict_cache) against plain forms in 64 bits; the bounds are those of tests/cache_cases.py."""
import ctypes as C

import numpy as np
import pytest

from tests import cache_cases as K
from tests import helpers as H

pytestmark = pytest.mark.gpu
S = pytest.importorskip("slhav2_b200")
F = np.float32


def make(rng, lens, tokens, kv, group, d, bf16, q_scale=1.5, bases=None, **more):
    total = int(sum(lens))
    keys, dk = K.as_type(rng.standard_normal((max(total, 1), kv, d)) * np.exp(0.5 * rng.standard_normal(d)), bf16)
    values, dv = K.as_type(rng.standard_normal((max(total, 1), kv, d)), bf16)
    toks = [tokens] * len(lens) if np.isscalar(tokens) else list(tokens)
    q, dq = K.as_type(q_scale * rng.standard_normal((max(sum(toks), 1), kv * group, d)), bf16)
    segs, at, q0 = [], 0, 0
    for i, (n, t) in enumerate(zip(lens, toks)):
        segs.append((at, int(n), q0, t, 0 if bases is None else bases[i]))
        at += int(n)
        q0 += t
    return K.Call(keys, values, q, segs, d ** -0.5, **more), (dk, dv, dq)


def on_device(call, raw, bf16):
    """The handles of a call whose arrays lie as the defaults say."""
    up = lambda x, t: None if x is None else S.to_device(np.ascontiguousarray(x, t))  # noqa: E731
    per_head = call.row_pos is not None or call.row_doc is not None
    total = call.keys.shape[0]
    cache = S.KvCache(S.to_device(raw[0]), S.to_device(raw[1]), call.kv, call.d, dtype=S.BF16 if bf16 else S.F32, positions=up(call.row_pos, np.uint32),
                      documents=up(call.row_doc, np.uint32), entry_head_stride=total if per_head else 0, rows=call.rows)
    queries = S.CacheQueries(S.to_device(raw[2]), call.q.shape[0], call.heads, call.d, scale=call.scale, softcap=call.softcap, window=call.window, causal=call.causal,
                             slopes=call.slopes, prefix=call.prefix, positions=up(call.q_pos, np.uint32), documents=up(call.q_doc, np.uint32))
    return cache, S.make_segments(call.segs), queries


def results(call, bf16, cache, segs, queries):
    n = call.q.size
    out, lse = S.to_device(np.full(n, 7.0, F) if not bf16 else np.full(n, 0x40E0, np.uint16)), S.to_device(np.full(call.q.shape[:2], 7.0, F))
    if call.parents is not None:
        S.attend_tree(cache, segs, queries, call.parents, out, lse)
    else:
        S.attend_cache(cache, segs, queries, out, lse)
    o = out.download(np.uint16 if bf16 else F, n)
    return (K.from_bf16(o) if bf16 else o).reshape(call.q.shape), lse.download(F, call.q.shape[0] * call.heads).reshape(call.q.shape[:2])


def held(got, want, tol):
    """Values within their bound; infinities, NaN and what no segment writes (7) in their places."""
    want = np.where(np.isnan(want), 7.0, want)
    with np.errstate(invalid="ignore"):
        same = (got == want) | (np.abs(got - want) <= tol)
    assert same.all(), (int((~same).sum()), np.argwhere(~same)[:3], got[~same][:3], want[~same][:3], np.broadcast_to(tol, got.shape)[~same][:3])


def check(call, raw, bf16):
    got = results(call, bf16, *on_device(call, raw, bf16))
    out, lse, out_tol, lse_tol = call.attend(bf16)
    held(got[1], lse, lse_tol)
    held(got[0], out, out_tol)
    return got


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("d", [8, 64, 80, 128, 200, 256])
@pytest.mark.parametrize("kv,group,tokens,lens", [(2, 4, 1, (1, 63, 64, 65, 700)), (1, 1, 1, (5000,)), (2, 3, 9, (9, 10, 130, 257)), (1, 8, 37, (37, 300)), (3, 5, 5, (200, 33))])
def test_attention_of_every_type_and_width(bf16, d, kv, group, tokens, lens):
    rng = np.random.default_rng(d * 10 + tokens)
    check(*make(rng, lens, tokens, kv, group, d, bf16), bf16)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("tokens", [1, 3, 40, 150])
@pytest.mark.parametrize("more", [dict(softcap=5.0), dict(alibi=True), dict(window=17), dict(prefix=True), dict(prefix=True, window=9, alibi=True), dict(causal=False),
                                  dict(causal=False, window=30), dict(docs=True), dict(docs=True, prefix=True, softcap=20.0), dict(moved=True, alibi=True, window=90),
                                  dict(moved=True, docs=True, prefix=True)])
def test_attention_s_masks_bias_and_cap(bf16, tokens, more):
    rng = np.random.default_rng(len(str(more)) * 7 + tokens)
    lens, kv, group, d = (tokens, 150 + tokens, 300 + tokens), 2, 3, 64
    total = sum(lens)
    kind = {k: v for k, v in more.items() if k in ("softcap", "window", "causal")}
    if more.get("alibi"):
        kind["slopes"] = (2.0 ** -np.arange(1, kv * group + 1)).astype(F)
    if more.get("prefix"):
        kind["prefix"] = np.array([0, 70, 40], np.uint32)
    if more.get("docs"):
        doc = np.concatenate([np.sort(rng.integers(1, 4, n)) for n in lens]).astype(np.uint32)
        kind["row_doc"] = np.stack([doc] * kv)
        kind["q_doc"] = np.concatenate([doc[e - tokens:e] for e in np.cumsum(lens)])
    if more.get("moved"):
        kind["row_pos"] = np.stack([np.concatenate([rng.permutation(2 * n)[:n] for n in lens]) for _ in range(kv)]).astype(np.uint32)
        kind["q_pos"] = np.concatenate([2 * n - tokens + np.arange(tokens) for n in lens]).astype(np.uint32)
    check(*make(rng, lens, tokens, kv, group, d, bf16, **kind), bf16)


@pytest.mark.parametrize("bf16", [True, False])
def test_lengths_of_zero_tokens_without_a_row_and_tokens_of_no_segment(bf16):
    rng = np.random.default_rng(3)
    call, raw = make(rng, (0, 40, 0, 100), (2, 3, 0, 0), 2, 2, 128, bf16)
    check(call, raw, bf16)
    # rows of another document, rows behind the token, nothing below the prefix: a token that sees no row
    call, raw = make(rng, (40, 90), (2, 30), 2, 2, 64, bf16, row_doc=np.full((2, 130), 5, np.uint32), q_doc=np.full(32, 6, np.uint32))
    o, z = check(call, raw, bf16)
    assert np.all(o == 0) and np.all(z == -np.inf)
    call, raw = make(rng, (70,), (20,), 1, 1, 64, bf16, row_pos=np.full((1, 70), 900, np.uint32), q_pos=np.arange(890, 910, dtype=np.uint32))
    o, z = check(call, raw, bf16)
    assert np.all(o[:10] == 0) and np.all(np.isfinite(z[10:]))
    # the segments that have rows are the last of a token array: tokens before and behind them keep what they held
    call, raw = make(rng, (50, 60), (4, 40), 2, 2, 64, bf16)
    call.segs = [(0, 50, 3, 1, 0), (50, 60, 10, 20, 0)]
    check(call, raw, bf16)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("tokens", [1, 6, 100])
def test_rows_that_a_token_does_not_see_may_hold_anything(bf16, tokens):
    rng = np.random.default_rng(tokens)
    lens, kv, group, d = (300, 411), 2, 2, 64
    doc = rng.integers(0, 3, sum(lens)).astype(np.uint32)
    for b, n in ((0, 300), (300, 411)):
        doc[b + n - tokens:b + n] = rng.integers(0, 2, tokens)
    call, raw = make(rng, lens, tokens, kv, group, d, bf16, row_doc=np.stack([doc] * kv), q_doc=np.concatenate([doc[300 - tokens:300], doc[711 - tokens:711]]))
    want = call.attend(bf16)
    hidden = doc == 2  # no token's document
    for a, r in ((call.keys, raw[0]), (call.values, raw[1])):
        odd = rng.choice(np.array([np.nan, np.inf, -np.inf], F), a[hidden].shape)
        r[hidden] = K.as_type(odd, bf16)[1]
    got = results(call, bf16, *on_device(call, raw, bf16))
    held(got[1], want[1], want[3])
    held(got[0], want[0], want[2])
    # an infinity that tokens of document 1 see, and those of document 0 do not
    at = int(np.flatnonzero((doc[:300] == 1))[0])
    raw[1][at, :, 3] = K.as_type(np.full(kv, np.inf), bf16)[1]
    got = results(call, bf16, *on_device(call, raw, bf16))
    sees = np.zeros(call.q.shape[0], bool)
    sees[:tokens] = call.q_doc[:tokens] == 1
    if bf16:
        assert np.all(got[0][sees][:, :, 3] == np.inf)
    assert not np.isfinite(got[0][sees][:, :, 3]).any()
    keep = np.ones(got[0].shape, bool)
    keep[sees, :, 3] = False
    assert np.all((np.abs(got[0] - want[0]) <= want[2])[keep])


@pytest.mark.parametrize("bf16", [True, False])
def test_layouts_strides_and_device_row_counts(bf16):
    rng = np.random.default_rng(11)
    kv, group, d, lens, tokens = 2, 2, 64, (130, 75), 5
    call, raw = make(rng, lens, tokens, kv, group, d, bf16)
    call.rows = np.array([100, 900], np.uint32)  # fewer than the table says, and more
    e = 2 if bf16 else 4
    # keys [kv_head][row][d] with a gap behind each row, values [row][d][..] of both heads with a gap, queries and outputs [head][token]
    total = 205
    k = np.zeros((kv, total, d + 8), raw[0].dtype)
    k[:, :, :d] = raw[0].transpose(1, 0, 2)
    v = np.zeros((total, kv, d + 16), raw[1].dtype)
    v[:, :, :d] = raw[1]
    q = np.zeros((kv * group, 10, d + 8), raw[2].dtype)
    q[:, :, :d] = raw[2].transpose(1, 0, 2)
    rows = S.to_device(call.rows)
    cache = S.KvCache(S.to_device(k), S.to_device(v), kv, d, dtype=S.BF16 if bf16 else S.F32, key_row_stride=d + 8, key_head_stride=total * (d + 8),
                      value_row_stride=kv * (d + 16), value_head_stride=d + 16, rows=rows)
    queries = S.CacheQueries(S.to_device(q), 10, kv * group, d, token_stride=d + 8, head_stride=10 * (d + 8))
    out = S.to_device(np.zeros((kv * group, 10, d + 24), np.uint16 if bf16 else F))
    lse = S.DeviceBuffer(10 * kv * group * 4)
    S.attend_cache(cache, S.to_device(S.make_segments(call.segs)).download(S.SEGMENT_DTYPE, 2), queries, out, lse, out_token_stride=d + 24, out_head_stride=10 * (d + 24))
    o = out.download(np.uint16 if bf16 else F, kv * group * 10 * (d + 24)).reshape(kv * group, 10, d + 24)
    assert np.all(o[:, :, d:] == 0)
    o = o[:, :, :d].transpose(1, 0, 2)
    want = call.attend(bf16)
    held(K.from_bf16(o).reshape(want[0].shape) if bf16 else o, want[0], want[2])
    assert e


def test_tables_in_device_memory_and_of_many_segments():
    rng = np.random.default_rng(12)
    lens = rng.integers(1, 200, 90)
    call, raw = make(rng, lens, 1, 2, 2, 64, True)
    cache, segs, queries = on_device(call, raw, True)
    got = results(call, True, cache, segs, queries)
    want = call.attend(True)
    held(got[0], want[0], want[2])
    dev = S.to_device(segs)
    out, lse = S.DeviceBuffer(call.q.size * 2), S.DeviceBuffer(call.q.size)
    lib = S.load_library()
    assert lib.slha_b200_attend_cache(cache.address, dev.data_ptr(), len(segs), queries.address, out.data_ptr(), call.heads * 64, 64, lse.data_ptr()) == 0
    assert np.array_equal(K.from_bf16(out.download(np.uint16, call.q.size)).reshape(call.q.shape), got[0])


def test_rows_of_a_few_and_of_many_tokens_in_one_call():
    rng = np.random.default_rng(13)
    call, raw = make(rng, (500, 900, 333, 64, 2000), (1, 70, 9, 64, 1), 2, 3, 128, True)
    a = check(call, raw, True)
    b = results(call, True, *on_device(call, raw, True))
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])  # the same bits again


@pytest.mark.parametrize("bf16", [True, False])
def test_scores_far_from_zero_and_weights_that_vanish(bf16):
    rng = np.random.default_rng(14)
    for q_scale in (1e-6, 30.0, 300.0):
        check(*make(rng, (400, 129), 3, 2, 2, 64, bf16, q_scale=q_scale), bf16)
    call, raw = make(rng, (300,), 2, 1, 2, 64, bf16, slopes=np.array([3.0, 0.0], F))
    check(call, raw, bf16)


def test_positions_near_the_end_of_their_range():
    rng = np.random.default_rng(15)
    top = 2 ** 32
    check(*make(rng, (200,), 5, 1, 2, 64, True, bases=[top - 200]), True)
    pos = (top - 1 - rng.permutation(200)).astype(np.uint32)
    call, raw = make(rng, (200,), 5, 1, 2, 64, True, row_pos=pos[None], q_pos=np.array([0, 5, top - 100, top - 50, top - 1], np.uint32), window=60)
    check(call, raw, True)


def test_element_offsets_beyond_32_bits():
    # rows 2^27 elements apart: the last ones lie 10 GB behind the first
    rng = np.random.default_rng(16)
    call, raw = make(rng, (40,), 1, 1, 2, 64, True)
    step, n = 1 << 27, 40
    big = S.DeviceBuffer(((n - 1) * step + 2 * 64) * 2)
    for r in range(n):
        lib = S.load_library()
        both = np.concatenate([raw[0][r, 0], raw[1][r, 0]])
        assert lib.slha_b200_memcpy(big.data_ptr() + r * step * 2, both.ctypes.data, 256) == 0
    cache = S.KvCache(big, big.view(128, big.nbytes - 128), 1, 64, key_row_stride=step, value_row_stride=step)
    queries = S.CacheQueries(S.to_device(raw[2]), 1, 2, 64)
    got = results(call, True, cache, S.make_segments(call.segs), queries)
    want = call.attend(True)
    held(got[0], want[0], want[2])
    # the same offsets on the way through removal: rows 8.. to the first places of a small cache
    w = np.arange(40, dtype=F)
    small_k, small_v = S.DeviceBuffer(8 * 128), S.DeviceBuffer(8 * 128)
    to = S.KvCache(small_k, small_v, 1, 64)
    S.evict_cache(cache, S.make_segments([(0, 40, 0, 0, 0)]), S.to_device(w), 40, 8, to=to, to_segments=S.make_segments([(0, 8, 0, 0, 0)]))
    src = K.evict(w, np.arange(40), 8, 0, 0)
    assert np.array_equal(small_k.download(np.uint16, 512).reshape(8, 64), raw[0][src, 0])
    assert np.array_equal(small_v.download(np.uint16, 512).reshape(8, 64), raw[1][src, 0])
    big.free()


# ---- trees of drafted tokens
def tree(rng, kind, t):
    if kind == "chain":
        return np.arange(-1, t - 1).astype(np.int64).astype(np.uint32)
    if kind == "star":
        return np.concatenate([[K.NONE], np.zeros(t - 1)]).astype(np.uint32) if t > 1 else np.array([K.NONE], np.uint32)
    p = np.array([-1] + [int(rng.integers(-1, i)) for i in range(1, t)], np.int64)
    return p.astype(np.uint32)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("kind", ["chain", "star", "random"])
@pytest.mark.parametrize("t,lens,kv,group,d", [(1, (1, 50), 2, 4, 64), (7, (7, 100, 513), 2, 4, 128), (64, (64, 200), 1, 2, 64), (256, (300,), 1, 1, 64), (33, (90, 700), 2, 8, 80)])
def test_trees_of_drafted_tokens(bf16, kind, t, lens, kv, group, d):
    rng = np.random.default_rng(t + len(kind))
    call, raw = make(rng, lens, t, kv, group, d, bf16, parents=np.concatenate([tree(rng, kind, t) for _ in lens]))
    got = check(call, raw, bf16)
    if kind == "chain":  # a chain is an ordinary continuation
        call.parents = None
        want = call.attend(bf16)
        held(got[0], want[0], want[2])


@pytest.mark.parametrize("more", [dict(softcap=8.0), dict(window=6), dict(prefix=np.array([3, 60], np.uint32), window=4), dict(alibi=True), dict(moved=True)])
def test_trees_under_the_other_rules(more):
    rng = np.random.default_rng(31)
    t, lens, kv, group = 21, (90, 130), 2, 2
    kind = {k: v for k, v in more.items() if k not in ("alibi", "moved")}
    if more.get("alibi"):
        kind["slopes"] = np.array([0.5, 0.1, 0.0, 2.0], F)
    if more.get("moved"):
        kind["row_pos"] = rng.integers(0, 500, (kv, sum(lens))).astype(np.uint32)
        kind["q_pos"] = rng.integers(200, 500, 2 * t).astype(np.uint32)
    check(*make(rng, lens, t, kv, group, 64, True, parents=np.concatenate([tree(rng, "random", t) for _ in lens]), **kind), True)


def test_parents_that_are_no_earlier_token_are_roots():
    rng = np.random.default_rng(32)
    p = np.array([0, 1, 7, 2, 4000000000, 3], np.uint32)  # itself, itself, a later one, an earlier one, far away, an earlier one
    check(*make(rng, (50,), 6, 1, 2, 64, True, parents=p), True)


# ---- received weights
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("tokens,lens,kv,group,d", [(1, (1, 127, 128, 129, 700), 2, 4, 128), (1, (300,), 1, 1, 256), (40, (40, 500), 2, 3, 64), (17, (170,), 2, 2, 200), (200, (333,), 1, 4, 80), (70, (500,), 1, 4, 128)])
@pytest.mark.parametrize("more", [dict(), dict(softcap=6.0, window=50), dict(alibi=True, prefix=True), dict(docs=True, moved=True)])
def test_weights_that_rows_receive(bf16, tokens, lens, kv, group, d, more):
    rng = np.random.default_rng(tokens + d)
    total = sum(lens)
    kind = {k: v for k, v in more.items() if k in ("softcap", "window")}
    if more.get("alibi"):
        kind["slopes"] = rng.random(kv * group).astype(F)
    if more.get("prefix"):
        kind["prefix"] = np.array([min(n, 30) for n in lens], np.uint32)
    if more.get("docs"):
        kind["row_doc"] = rng.integers(0, 2, (kv, total)).astype(np.uint32)
        kind["q_doc"] = rng.integers(0, 3, tokens * len(lens)).astype(np.uint32)
    if more.get("moved"):
        kind["row_pos"] = rng.integers(0, 2 * max(lens), (kv, total)).astype(np.uint32)
        kind["q_pos"] = rng.integers(0, 2 * max(lens), tokens * len(lens)).astype(np.uint32)
    call, raw = make(rng, lens, tokens, kv, group, d, bf16, **kind)
    cache, segs, queries = on_device(call, raw, bf16)
    _, lse = results(call, bf16, cache, segs, queries)
    dl = S.to_device(lse)
    pitch = total + 5
    before = rng.random((kv, pitch)).astype(F)
    w = S.to_device(before)
    S.observe_cache(cache, segs, queries, dl, w, pitch, weights_in=w, decay=0.75)
    want, tol = call.received(lse, before, 0.75)
    held(w.download(F, kv * pitch).reshape(kv, pitch), want, tol)
    # nothing received before: what the array held does not count, entries of no row stay
    fresh = S.to_device(np.full((kv, pitch), np.nan, F))
    S.observe_cache(cache, segs, queries, dl, fresh, pitch)
    want, tol = call.received(lse, np.zeros((kv, pitch), F), 0.0)
    got = fresh.download(F, kv * pitch).reshape(kv, pitch)
    assert np.isnan(got[:, total:]).all()
    held(got[:, :total], want[:, :total], tol[:, :total])
    for h in range(kv):  # every token that sees a row hands out a weight of one a head
        for (b, n, q0, t, _) in segs:
            seen = np.isfinite(lse[q0:q0 + t, h * group:(h + 1) * group]).sum()
            assert abs(float(got[h, b:b + n].astype(np.float64).sum()) - seen) <= 1e-3 * max(seen, 1)


def test_received_weights_where_hidden_rows_hold_anything_and_tokens_see_nothing():
    rng = np.random.default_rng(41)
    n, t = 200, 9
    doc = rng.integers(0, 2, n).astype(np.uint32)
    q_doc = np.array([0] * 5 + [9] * 4, np.uint32)
    call, raw = make(rng, (n,), t, 1, 2, 64, True, row_doc=doc[None], q_doc=q_doc)
    raw[0][doc == 1] = K.as_type(np.full((int((doc == 1).sum()), 1, 64), np.nan), True)[1]
    cache, segs, queries = on_device(call, raw, True)
    _, lse = results(call, True, cache, segs, queries)
    assert np.all(lse[5:] == -np.inf)
    w = S.to_device(np.zeros(n, F))
    S.observe_cache(cache, segs, queries, S.to_device(lse), w, n)
    want, tol = call.received(lse, np.zeros((1, n), F), 1.0)
    got = w.download(F, n)[None]
    held(got, want, tol)
    assert np.all(got[0, doc == 1] == 0)


# ---- removal
def removal(rng, lens, kv, d, bf16, moved, tiles, ties):
    total = sum(lens)
    _, k = K.as_type(rng.standard_normal((total, kv, d)), bf16)
    _, v = K.as_type(rng.standard_normal((total, kv, d)), bf16)
    w = rng.random((kv, total)).astype(F) if not ties else rng.integers(0, 3, (kv, total)).astype(F)
    pos = np.stack([np.concatenate([rng.permutation(3 * n)[:n] for n in lens]) for _ in range(kv)]).astype(np.uint32) if moved else None
    doc = rng.integers(0, 9, (kv, total)).astype(np.uint32) if moved else None
    t = rng.integers(0, 256, (kv, total, 128)).astype(np.uint8) if tiles else None
    begins = np.concatenate([[0], np.cumsum(lens)])
    return k, v, w, pos, doc, t, begins


@pytest.mark.parametrize("bf16,d", [(True, 128), (True, 8), (True, 64), (False, 64), (False, 256), (True, 200)])
@pytest.mark.parametrize("lens,budget,sink,recent", [((1, 40, 41, 100), 40, 0, 0), ((5000, 300), 257, 4, 30), ((4097, 8193), 4096, 0, 100), ((700,), 699, 2, 0), ((300, 10), 1, 0, 0),
                                                     ((90,), 50, 40, 40)])
@pytest.mark.parametrize("moved,ties", [(False, False), (True, True)])
def test_rows_of_least_weight_leave(bf16, d, lens, budget, sink, recent, moved, ties):
    rng = np.random.default_rng(budget + d)
    kv, tiles = 2, d == 128
    total = sum(lens)
    k, v, w, pos, doc, t, begins = removal(rng, lens, kv, d, bf16, moved, tiles, ties)
    if ties:
        w[0, ::7] = np.nan
        w[1, ::11] = -0.0
        w[1, 3::50] = np.inf
    want = {}
    for i, n in enumerate(lens):
        for h in range(kv):
            at = slice(begins[i], begins[i] + n)
            want[i, h] = K.evict(w[h, at], pos[h, at] if moved else np.arange(n), budget, sink, recent)
    segs = [(int(begins[i]), n, 0, 0, 0) for i, n in enumerate(lens)]
    dt, each = (S.BF16, np.uint16) if bf16 else (S.F32, F)
    up = lambda x: None if x is None else S.to_device(x)  # noqa: E731
    dk, dv, dw, dp, dd, dtile = (up(x) for x in (k, v, w, pos, doc, t))
    cache = S.KvCache(dk, dv, kv, d, dtype=dt, positions=dp, documents=dd, entry_head_stride=total if moved else 0)
    # into another cache: its own strides, something in every place
    room = [min(n, budget) + 3 for n in lens]
    to_begin = np.concatenate([[2], 2 + np.cumsum(room)])
    wide = int(to_begin[-1])
    ok, ov = (S.to_device(np.full((kv, wide, d), 9, each)) for _ in range(2))
    ow, op, od = (S.to_device(np.full((kv, wide), 9, x)) for x in (F, np.uint32, np.uint32))
    ot = S.to_device(np.full((kv, wide, 128), 9, np.uint8))
    src, cnt = S.to_device(np.full((len(lens), kv, budget), K.NONE, np.uint32)), S.DeviceBuffer(4 * len(lens))
    to = S.KvCache(ok, ov, kv, d, dtype=dt, key_row_stride=d, key_head_stride=wide * d, value_row_stride=d, value_head_stride=wide * d,
                   positions=op if moved else None, documents=od if moved else None, entry_head_stride=wide)
    S.evict_cache(cache, S.make_segments(segs), dw, total, budget, sink, recent, to=to,
                  to_segments=S.make_segments([(int(b), r - 3, 0, 0, 0) for b, r in zip(to_begin, room)]), weights_to=ow, weights_to_head_stride=wide, tiles=dtile,
                  tile_head_stride=total, tiles_to=ot, tiles_to_head_stride=wide, source_out=src, rows_out=cnt)
    assert cnt.download(np.uint32, len(lens)).tolist() == [min(n, budget) for n in lens]
    got_src = src.download(np.uint32, len(lens) * kv * budget).reshape(len(lens), kv, budget)
    gk, gv = (x.download(each, kv * wide * d).reshape(kv, wide, d) for x in (ok, ov))
    gw, gp, gd = (x.download(y, kv * wide).reshape(kv, wide) for x, y in ((ow, F), (op, np.uint32), (od, np.uint32)))
    gt = ot.download(np.uint8, kv * wide * 128).reshape(kv, wide, 128)
    ek, ev, ew, ep, ed, et = (np.full_like(x, 9) for x in (gk, gv, gw, gp, gd, gt))
    for (i, h), s in want.items():
        assert np.array_equal(got_src[i, h, :len(s)], s) and np.all(got_src[i, h, len(s):] == K.NONE)
        place, row = to_begin[i] + np.arange(len(s)), begins[i] + s
        ek[h, place], ev[h, place], ew[h, place] = k[row, h], v[row, h], w[h, row]
        if moved:
            ep[h, place], ed[h, place] = pos[h, row], doc[h, row]
        if tiles:
            et[h, place] = t[h, row]
    for a, b in ((gk, ek), (gv, ev), (gp, ep), (gd, ed), (gt, et)):
        assert np.array_equal(a, b)
    assert gw.tobytes() == ew.tobytes()
    # in place: what lies behind the rows that stay, and everything of other rows, keeps its bytes
    S.evict_cache(cache, S.make_segments(segs), dw, total, budget, sink, recent, weights_to=dw, weights_to_head_stride=total, tiles=dtile, tile_head_stride=total)
    for (i, h), s in want.items():
        place, row = begins[i] + np.arange(len(s)), begins[i] + s
        for x in (k, v):
            x[place, h] = x[row, h]
        w[h, place] = w[h, row]
        if moved:
            pos[h, place], doc[h, place] = pos[h, row], doc[h, row]
        if tiles:
            t[h, place] = t[h, row]
    assert np.array_equal(dk.download(each, k.size).reshape(k.shape), k) and np.array_equal(dv.download(each, v.size).reshape(v.shape), v)
    assert dw.download(F, w.size).tobytes() == w.tobytes()
    if moved:
        assert np.array_equal(dp.download(np.uint32, pos.size).reshape(pos.shape), pos) and np.array_equal(dd.download(np.uint32, doc.size).reshape(doc.shape), doc)
    if tiles:
        assert np.array_equal(dtile.download(np.uint8, t.size).reshape(t.shape), t)


@pytest.mark.parametrize("n,budget", [(60000, 5000), (49152, 49151), (49153, 1000), (200000, 150000)])
def test_removal_from_long_segments(n, budget):
    # keys that do not fit into shared memory, and around the border
    rng = np.random.default_rng(n)
    w = rng.random(n).astype(F)
    w[rng.random(n) < 0.3] = 0.25
    k = rng.integers(0, 65536, (n, 8)).astype(np.uint16)
    cache = S.KvCache(S.to_device(k), S.to_device(k), 1, 8)
    src = S.DeviceBuffer(4 * budget)
    S.evict_cache(cache, S.make_segments([(0, n, 0, 0, 0)]), S.to_device(w), n, budget, sink_window=3, recent_window=11, source_out=src)
    assert np.array_equal(src.download(np.uint32, budget), K.evict(w, np.arange(n), budget, 3, 11))


def test_row_counts_on_the_device_go_through_a_removal():
    rng = np.random.default_rng(51)
    lens, rows, budget, kv, d = (100, 200, 50), np.array([80, 170, 20], np.uint32), 60, 2, 64
    k, v, w, _, _, _, begins = removal(rng, lens, kv, d, True, False, False, False)
    dk, dv, dw, drows = S.to_device(k), S.to_device(v), S.to_device(w), S.to_device(rows)
    cache = S.KvCache(dk, dv, kv, d, rows=drows)
    segs = S.make_segments([(int(begins[i]), n, 0, 0, 0) for i, n in enumerate(lens)])
    S.evict_cache(cache, segs, dw, sum(lens), budget, recent_window=5, weights_to=dw, weights_to_head_stride=sum(lens), rows_out=drows)
    assert drows.download(np.uint32, 3).tolist() == [60, 60, 20]
    for i in range(3):
        for h in range(kv):
            n, b = int(rows[i]), int(begins[i])
            s = K.evict(w[h, b:b + n], np.arange(n), budget, 0, 5)
            k[b + np.arange(len(s)), h] = k[b + s, h]
    assert np.array_equal(dk.download(np.uint16, k.size).reshape(k.shape), k)


# ---- together, as a decode loop uses them
def test_a_decode_loop_attends_observes_and_evicts_with_its_tiles():
    rng = np.random.default_rng(61)
    kv, group, d, seqs, budget, room, steps = 2, 2, 128, 2, 96, 160, 40
    heads = kv * group
    _, proj = H.make_model_pair(d)
    model = S.Model.from_projection(proj, d, 7)
    k = np.zeros((kv, seqs * room, d), np.uint16)
    v = np.zeros_like(k)
    dk, dv = S.to_device(k), S.to_device(v)
    dpos, dw = S.to_device(np.zeros((kv, seqs * room), np.uint32)), S.to_device(np.zeros((kv, seqs * room), F))
    tiles = S.DeviceBuffer(kv * seqs * room * 128)
    lib = S.load_library()
    cache = S.KvCache(dk, dv, kv, d, key_row_stride=d, key_head_stride=seqs * room * d, value_row_stride=d, value_head_stride=seqs * room * d, positions=dpos,
                      entry_head_stride=seqs * room)
    pos = np.zeros((kv, seqs * room), np.uint32)
    w = np.zeros((kv, seqs * room))
    n = [0, 0]
    put = lambda buf, at, x: lib.slha_b200_memcpy(buf.data_ptr() + at, np.ascontiguousarray(x).ctypes.data, np.ascontiguousarray(x).nbytes)  # noqa: E731
    vals = np.zeros((kv, seqs * room, d), F)
    keys = np.zeros((kv, seqs * room, d), F)
    for step in range(steps):
        new = 30 if step == 0 else 3  # a prompt, then a few tokens a step
        at_pos = 0 if step == 0 else 30 + 3 * (step - 1)
        for s in range(seqs):
            for h in range(kv):
                kx, kr = K.as_type(rng.standard_normal((new, d)), True)
                vx, vr = K.as_type(rng.standard_normal((new, d)), True)
                row = s * room + n[s]
                at = h * seqs * room + row
                keys[h, row:row + new], vals[h, row:row + new] = kx, vx
                pos[h, row:row + new] = at_pos + np.arange(new)
                assert put(dk, at * d * 2, kr) == 0 and put(dv, at * d * 2, vr) == 0 and put(dpos, at * 4, pos[h, row:row + new]) == 0
                assert put(dw, at * 4, np.zeros(new, F)) == 0
                w[h, row:row + new] = 0
                model.encode_keys(kx, S.CODEC_MIXED, positions=pos[h, row:row + new], out=tiles.view(at * 128, new * 128))
            n[s] += new
        q, dq = K.as_type(1.5 * rng.standard_normal((seqs * new, heads, d)), True)
        segs = S.make_segments([(s * room, n[s], s * new, new, 0) for s in range(seqs)])
        qp = np.concatenate([at_pos + np.arange(new)] * seqs).astype(np.uint32)
        queries = S.CacheQueries(S.to_device(dq), seqs * new, heads, d, softcap=20.0, positions=S.to_device(qp))
        call = K.Call(keys.transpose(1, 0, 2), vals.transpose(1, 0, 2), q, [tuple(int(x) for x in s) for s in segs.tolist()], d ** -0.5, softcap=20.0, row_pos=pos, q_pos=qp)
        call.segs = [(a, b, c, e, f) for a, b, c, e, f in call.segs]
        got = results(call, True, cache, segs, queries)
        want = call.attend(True)
        held(got[0], want[0], want[2])
        S.observe_cache(cache, segs, queries, S.to_device(got[1]), dw, seqs * room, weights_in=dw, decay=0.9)
        w, tol = call.received(got[1], w.astype(F), 0.9)
        now = dw.download(F, kv * seqs * room).reshape(kv, seqs * room)
        held(now, w, tol + 1e-6 * np.abs(w))
        w = now.astype(np.float64)
        S.evict_cache(cache, segs, dw, seqs * room, budget, sink_window=2, recent_window=16, weights_to=dw, weights_to_head_stride=seqs * room, tiles=tiles,
                      tile_head_stride=seqs * room)
        for s in range(seqs):
            b = s * room
            for h in range(kv):
                src = K.evict(now[h, b:b + n[s]], pos[h, b:b + n[s]], budget, 2, 16)
                place = b + np.arange(len(src))
                for x in (keys, vals, pos, w):
                    x[h, place] = x[h, b + src]
            n[s] = min(n[s], budget)
    assert n == [budget, budget]
    # the tiles went along: each is the one its key is encoded to, and scoring and the decode tail run on what is left
    lay = tiles.download(S.TILE_DTYPE, kv * seqs * room).reshape(kv, seqs * room)
    for h in range(kv):
        for s in range(seqs):
            at = slice(s * room, s * room + budget)
            assert lay[h, at].tobytes() == model.encode_keys(keys[h, at], S.CODEC_MIXED, positions=pos[h, at]).tobytes()
    qc, qs = model.prepare_queries(rng.standard_normal((1, d)).astype(F))
    idx, sc, cnt = S.score_topk(tiles, S.make_segments([(room, budget, 0, 1, 0)]), qc, qs, 1, 16)
    out = S.attend_topk(idx, sc, 16, d ** -0.5, dv, d, value_dtype=S.BF16, top_count=cnt, value_row_base=np.array([room], np.uint64))
    assert cnt[0] == 16 and np.isfinite(out).all()


# ---- streams, graphs, threads
def test_calls_on_two_streams_and_captured_calls_keep_their_working_memory_apart():
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(71)
    calls, handles, wants = [], [], []
    for i in range(2):
        call, raw = make(rng, (9000,), 1, 2, 4, 128, True)
        calls.append(call)
        handles.append(on_device(call, raw, True))
        wants.append(call.attend(True))
    S.synchronize()
    outs = [(torch.empty(call.q.shape, dtype=torch.bfloat16, device="cuda"), torch.empty(call.q.shape[:2], device="cuda")) for call in calls]
    streams = [torch.cuda.Stream() for _ in range(2)]
    try:
        for _ in range(20):
            for h, o, st in zip(handles, outs, streams):
                S.set_stream(st.cuda_stream)
                S.attend_cache(h[0], h[1], h[2], o[0], o[1])
        torch.cuda.synchronize()
        for o, w in zip(outs, wants):
            held(o[0].float().cpu().numpy(), w[0], w[2])
            o[0].zero_()
        torch.cuda.synchronize()
        graphs = []
        for h, o, st in zip(handles, outs, streams):
            S.set_stream(st.cuda_stream)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                S.attend_cache(h[0], h[1], h[2], o[0], o[1])
            graphs.append(g)
        for _ in range(20):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, wants):
            held(o[0].float().cpu().numpy(), w[0], w[2])
            held(o[1].cpu().numpy(), w[1], w[3])
    finally:
        S.set_stream(None)


def test_a_captured_decode_step_follows_the_row_counts_on_the_device():
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(72)
    kv, group, d, most, budget = 2, 2, 64, 600, 200
    call, raw = make(rng, (most,), 1, kv, group, d, True, row_pos=np.stack([np.arange(most)] * kv), q_pos=np.array([5000], np.uint32))
    call.rows = np.array([300], np.uint32)
    up = lambda x: torch.from_numpy(np.ascontiguousarray(x).view(np.int16) if x.dtype == np.uint16 else x.astype(np.int32)).cuda()  # noqa: E731
    k, v, q, rows, qp, pos = (up(x) for x in (raw[0], raw[1], raw[2], call.rows, call.q_pos, call.row_pos))
    out, lse = torch.empty(1, kv * group, d, dtype=torch.bfloat16, device="cuda"), torch.empty(1, kv * group, device="cuda")
    w = torch.zeros(kv, most, device="cuda")
    cache = S.KvCache(k, v, kv, d, positions=pos, entry_head_stride=most, rows=rows)
    queries = S.CacheQueries(q, 1, kv * group, d, positions=qp)
    segs = S.make_segments([(0, most, 0, 1, 0)])
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        S.set_stream(st.cuda_stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            S.attend_cache(cache, segs, queries, out, lse)
            S.observe_cache(cache, segs, queries, lse, w, most, weights_in=w, decay=1.0)
            S.evict_cache(cache, segs, w, most, budget, weights_to=w, weights_to_head_stride=most, rows_out=rows)
        for n in (300, 450):
            call.rows[0] = n
            k.copy_(up(raw[0]))
            v.copy_(up(raw[1]))
            pos.copy_(up(call.row_pos))
            w.zero_()
            rows.fill_(n)
            torch.cuda.synchronize()
            with torch.cuda.stream(st):
                g.replay()
            torch.cuda.synchronize()
            want = call.attend(True)
            held(out.float().cpu().numpy(), want[0], want[2])
            assert int(rows.item()) == budget
            z = lse.cpu().numpy()
            full, tol = call.received(z, np.zeros((kv, most), F), 1.0)
            kept = w.cpu().numpy()[:, :budget]
            for h in range(kv):
                best = np.sort(full[h, :n])[::-1][:budget]
                assert np.all(np.abs(np.sort(kept[h])[::-1] - best) <= tol[h].max() + 1e-6 * best)
    finally:
        S.set_stream(None)


def test_a_call_that_cannot_be_captured_says_so():
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(73)
    call, raw = make(rng, (100,), 1, 1, 2, 64, True, slopes=np.array([0.5, 0.25], F))
    cache, segs, queries = on_device(call, raw, True)  # (slopes in host memory)
    out = torch.empty(1, 2, 64, dtype=torch.bfloat16, device="cuda")
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    try:
        S.set_stream(st.cuda_stream)
        g = torch.cuda.CUDAGraph()
        with pytest.raises(Exception):
            with torch.cuda.graph(g, stream=st):
                S.attend_cache(cache, segs, queries, out)
        torch.cuda.synchronize()
        S.attend_cache(cache, segs, queries, out)
        torch.cuda.synchronize()
        want = call.attend(True)
        held(out.float().cpu().numpy(), want[0], want[2])
    finally:
        S.set_stream(None)


def test_calls_from_several_threads():
    import threading

    rng = np.random.default_rng(74)
    made = [make(rng, (int(rng.integers(50, 6000)),), int(rng.integers(1, 30)), 2, 2, 64, True) for _ in range(6)]
    wants = [c.attend(True) for c, _ in made]
    bad = []

    def work(i):
        try:
            for _ in range(5):
                got = results(made[i][0], True, *on_device(made[i][0], made[i][1], True))
                held(got[0], wants[i][0], wants[i][2])
        except BaseException as e:  # noqa: BLE001
            bad.append(repr(e)[:300])

    ts = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad, bad


def test_host_arrays_where_device_memory_is_asked_for_are_refused():
    rng = np.random.default_rng(75)
    call, raw = make(rng, (100,), 1, 1, 2, 64, True)
    cache, segs, queries = on_device(call, raw, True)
    out = np.zeros(1 * 2 * 64 * 4, np.uint16)
    at = (out.ctypes.data + 15) // 16 * 16
    with pytest.raises(S.SlhaError) as e:
        S.attend_cache(cache, segs, queries, at)
    assert e.value.code == S.ERR_DEVICE and "out" in e.value.message
    w = S.DeviceBuffer(400)
    with pytest.raises(S.SlhaError) as e:
        S.observe_cache(cache, segs, queries, np.zeros(2, F), w, 100)
    assert e.value.code == S.ERR_DEVICE and "lse" in e.value.message
    assert C.sizeof(type(cache.c)) == 96


# ---- many query rows: two tiles of 128 a block
@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("tokens,lens,kv,group", [(33, (33, 100), 1, 1), (128, (128, 129, 500), 1, 1), (129, (129, 700), 2, 1), (64, (1000, 64), 2, 4), (100, (100, 3001), 1, 8), (300, (300,), 2, 3)])
def test_blocks_of_many_query_rows(d, tokens, lens, kv, group):
    rng = np.random.default_rng(tokens * d)
    call, raw = make(rng, lens, tokens, kv, group, d, True)
    a = check(call, raw, True)
    b = results(call, True, *on_device(call, raw, True))
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("q_scale", [1e-6, 1.0, 12.0, 100.0])
@pytest.mark.parametrize("cap", [0.0, 1.0, 30.0])
def test_many_query_rows_whose_largest_scores_come_late(q_scale, cap):
    # keys grow along the segment, so that the running maximum rises tile after tile
    rng = np.random.default_rng(int(q_scale * 10) + int(cap))
    call, raw = make(rng, (1500,), 70, 1, 4, 64, True, q_scale=q_scale, softcap=cap)
    grow = np.linspace(0.05, 2.0, 1500)[:, None, None]
    call.keys, raw = K.as_type(call.keys * grow, True)[0], (K.as_type(call.keys * grow, True)[1], raw[1], raw[2])
    check(call, raw, True)


@pytest.mark.parametrize("more", [dict(), dict(softcap=9.0), dict(softcap=0.7), dict(alibi=True), dict(window=200), dict(window=40, prefix=True, softcap=5.0), dict(prefix=True, alibi=True), dict(causal=False),
                                  dict(causal=False, window=111, alibi=True), dict(docs=True), dict(docs=True, alibi=True, softcap=8.0), dict(moved=True), dict(moved=True, docs=True, window=700),
                                  dict(q_only=True), dict(negative=True), dict(zero=True)])
@pytest.mark.parametrize("d", [64, 128])
def test_wide_blocks_under_every_rule(more, d):
    rng = np.random.default_rng(len(str(more)) + d)
    lens, kv, group, tokens = (130, 700, 1290), 2, 4, 70
    total = sum(lens)
    kind = {k: v for k, v in more.items() if k in ("softcap", "window", "causal")}
    if more.get("alibi"):
        kind["slopes"] = (2.0 ** -np.arange(1, kv * group + 1)).astype(F)
    if more.get("prefix"):
        kind["prefix"] = np.array([130, 300, 17], np.uint32)
    if more.get("docs"):
        doc = np.concatenate([np.sort(rng.integers(1, 5, n)) for n in lens]).astype(np.uint32)
        kind["row_doc"] = np.stack([doc] * kv)
        kind["q_doc"] = np.concatenate([doc[e - tokens:e] for e in np.cumsum(lens)])
    if more.get("moved"):
        kind["row_pos"] = np.stack([np.concatenate([rng.permutation(2 * n)[:n] for n in lens]) for _ in range(kv)]).astype(np.uint32)
        kind["q_pos"] = np.concatenate([2 * n - tokens + np.arange(tokens) for n in lens]).astype(np.uint32)
    if more.get("q_only"):
        kind["q_pos"] = np.concatenate([np.sort(rng.integers(0, n, tokens)) for n in lens]).astype(np.uint32)
    call, raw = make(rng, lens, tokens, kv, group, d, True, **kind)
    if more.get("negative"):
        call.scale = -call.scale
    if more.get("zero"):
        call.scale = 0.0
    check(call, raw, True)
    if not more.get("negative") and total:
        cache, segs, queries = on_device(call, raw, True)
        _, lse = results(call, True, cache, segs, queries)
        w = S.to_device(np.zeros((kv, total), F))
        S.observe_cache(cache, segs, queries, S.to_device(lse), w, total)
        want, tol = call.received(lse, np.zeros((kv, total), F), 1.0)
        held(w.download(F, kv * total).reshape(kv, total), want, tol)


@pytest.mark.parametrize("tokens,group,lens", [(100, 4, (900, 130)), (33, 1, (500,)), (512, 1, (600,))])
def test_wide_blocks_where_hidden_rows_hold_anything(tokens, group, lens):
    rng = np.random.default_rng(tokens)
    kv, d, total = 2, 128, sum(lens)
    ends = np.cumsum(lens)
    doc = rng.integers(0, 3, total).astype(np.uint32)
    for e in ends:
        doc[e - tokens:e] = rng.integers(0, 2, tokens)
    call, raw = make(rng, lens, tokens, kv, group, d, True, row_doc=np.stack([doc] * kv), q_doc=np.concatenate([doc[e - tokens:e] for e in ends]))
    want = call.attend(True)
    before = np.zeros((kv, total), F)
    for r in raw[:2]:
        r[doc == 2] = K.as_type(rng.choice(np.array([np.nan, np.inf, -np.inf], F), r[doc == 2].shape), True)[1]
    cache, segs, queries = on_device(call, raw, True)
    got = results(call, True, cache, segs, queries)
    held(got[1], want[1], want[3])
    held(got[0], want[0], want[2])
    w = S.to_device(before)
    S.observe_cache(cache, segs, queries, S.to_device(got[1]), w, total)
    weights, tol = call.received(got[1], before, 1.0)
    held(w.download(F, kv * total).reshape(kv, total), weights, tol)
    # rows behind a segment's end, and the rest of the last tile, belong to nobody
    call, raw = make(rng, (tokens + 70, 400), tokens, kv, group, d, True)
    call.segs[1:] = []
    want = call.attend(True)
    for r in raw[:2]:
        r[tokens + 70:] = K.as_type(np.full(r[tokens + 70:].shape, np.nan), True)[1]
    got = results(call, True, *on_device(call, raw, True))
    held(got[0][:tokens], want[0][:tokens], want[2][:tokens])


def test_wide_blocks_of_other_layouts_and_row_counts_on_the_device():
    # keys [kv_head][row][d] with gaps, values [row][kv_head][d], queries [head][token]: no boxes of queries and outputs; then strides that no map of rows takes
    rng = np.random.default_rng(81)
    kv, group, d, lens, tokens = 2, 4, 128, (900, 333), 40
    call, raw = make(rng, lens, tokens, kv, group, d, True)
    call.rows = np.array([777, 4000], np.uint32)
    total, heads = sum(lens), kv * group
    want = call.attend(True)
    for head_gap, row_gap in ((0, 8), (24, 40)):
        k = np.zeros((kv, total * (d + row_gap) + head_gap), np.uint16)
        k[:, :total * (d + row_gap)].reshape(kv, total, d + row_gap)[:, :, :d] = raw[0].transpose(1, 0, 2)
        q = np.ascontiguousarray(raw[2].transpose(1, 0, 2))
        rows = S.to_device(call.rows)
        cache = S.KvCache(S.to_device(k), S.to_device(raw[1]), kv, d, key_row_stride=d + row_gap, key_head_stride=total * (d + row_gap) + head_gap, rows=rows)
        queries = S.CacheQueries(S.to_device(q), 2 * tokens, heads, d, token_stride=d, head_stride=2 * tokens * d)
        out, lse = S.to_device(np.zeros((heads, 2 * tokens, d), np.uint16)), S.DeviceBuffer(8 * tokens * heads)
        S.attend_cache(cache, S.make_segments(call.segs), queries, out, lse, out_token_stride=d, out_head_stride=2 * tokens * d)
        o = K.from_bf16(out.download(np.uint16, heads * 2 * tokens * d)).reshape(heads, 2 * tokens, d).transpose(1, 0, 2)
        held(o, want[0], want[2])
        held(lse.download(F, 2 * tokens * heads).reshape(2 * tokens, heads), want[1], want[3])
        w = S.to_device(np.zeros((kv, total), F))
        S.observe_cache(cache, S.make_segments(call.segs), queries, lse, w, total)
        weights, tol = call.received(lse.download(F, 2 * tokens * heads).reshape(2 * tokens, heads), np.zeros((kv, total), F), 1.0)
        held(w.download(F, kv * total).reshape(kv, total), weights, tol)


def test_wide_blocks_of_many_segments_and_of_long_ones_in_parts():
    rng = np.random.default_rng(82)
    lens = rng.integers(40, 160, 70)
    check(*make(rng, lens, 40, 1, 1, 64, True), True)
    call, raw = make(rng, (20000, 300), (64, 33), 1, 1, 64, True, window=9000)
    check(call, raw, True)
    call, raw = make(rng, (6000,), 64, 1, 2, 128, True, parents=tree(rng, "random", 64), softcap=12.0)
    check(call, raw, True)


@pytest.mark.parametrize("n", [140000, 1300])
def test_many_tokens_over_a_long_cache_agree_with_few(n):
    # the same token among 40 and alone: two kernels, splits of more tiles than a run holds
    rng = np.random.default_rng(n)
    kv, group, d = 1, 1, 64
    call, raw = make(rng, (n,), 40, kv, group, d, True)
    cache, segs, queries = on_device(call, raw, True)
    many = results(call, True, cache, segs, queries)
    one = S.CacheQueries(S.to_device(raw[2][39:]), 1, 1, d)
    out, lse = S.DeviceBuffer(2 * d), S.DeviceBuffer(4)
    S.attend_cache(cache, S.make_segments([(0, n, 0, 1, 0)]), one, out, lse)
    got = K.from_bf16(out.download(np.uint16, d))
    assert abs(float(lse.download(F, 1)[0]) - float(many[1][39, 0])) <= 2e-5
    mag = np.abs(call.values).max()
    assert np.all(np.abs(got - many[0][39, 0]) <= 2.0 ** -7 * mag)


@pytest.mark.parametrize("n_kv,n,budget", [(1, 700, 90), (3, 5000, 4000), (40, 9000, 100), (200, 300, 150), (1, 131072, 70000)])
def test_removal_by_clusters_of_every_size(n_kv, n, budget):
    rng = np.random.default_rng(n)
    w = rng.integers(0, 50, (n_kv, n)).astype(F)
    k = rng.integers(0, 65536, (n, n_kv, 8)).astype(np.uint16)
    cache = S.KvCache(S.to_device(k), S.to_device(k), n_kv, 8)
    src = S.DeviceBuffer(4 * n_kv * budget)
    S.evict_cache(cache, S.make_segments([(0, n, 0, 0, 0)]), S.to_device(w), n, budget, sink_window=3, recent_window=11, source_out=src)
    got = src.download(np.uint32, n_kv * budget).reshape(n_kv, budget)
    for h in range(0, n_kv, max(1, n_kv // 4)):
        assert np.array_equal(got[h], K.evict(w[h], np.arange(n), budget, 3, 11))


@pytest.mark.parametrize("n_kv,n,budget", [(1, 16384, 90), (3, 20001, 20000), (60, 17000, 500), (13, 70000, 600), (2, 65536, 65535)])
def test_removal_from_long_caches(n_kv, n, budget):
    test_removal_by_clusters_of_every_size(n_kv, n, budget)


@pytest.mark.parametrize("tokens,group,lens", [(1, 4, (20000, 77)), (8, 4, (19990, 130)), (5, 1, (12000, 9000)), (9, 4, (10000,)), (64, 4, (9999,)), (43, 3, (5000, 129, 6000)), (65, 4, (3000,))])
@pytest.mark.parametrize("more", [dict(), dict(softcap=5.0, alibi=True), dict(docs=True), dict(window=3000)])
def test_weights_of_rows_in_long_runs_of_tiles(tokens, group, lens, more):
    rng = np.random.default_rng(tokens * 7 + group)
    kv, d, total = 8, 64, sum(lens)
    kind = {k: v for k, v in more.items() if k in ("softcap", "window")}
    if more.get("alibi"):
        kind["slopes"] = (2.0 ** -np.arange(1, kv * group + 1) / 64).astype(F)
    if more.get("docs"):
        doc = np.sort(rng.integers(1, 4, total)).astype(np.uint32)
        kind["row_doc"] = np.stack([doc] * kv)
        kind["q_doc"] = rng.integers(1, 5, tokens * len(lens)).astype(np.uint32)
    call, raw = make(rng, lens, tokens, kv, group, d, True, **kind)
    cache, segs, queries = on_device(call, raw, True)
    _, lse = results(call, True, cache, segs, queries)
    before = rng.random((kv, total)).astype(F)
    w = S.to_device(before)
    S.observe_cache(cache, segs, queries, S.to_device(lse), w, total, weights_in=w, decay=0.5)
    want, tol = call.received(lse, before, 0.5)
    held(w.download(F, kv * total).reshape(kv, total), want, tol)


@pytest.mark.parametrize("more", [dict(), dict(causal=False), dict(window=333), dict(docs=True), dict(prefix=np.array([200, 0, 650], np.uint32)), dict(softcap=9.0), dict(ahead=True)])
@pytest.mark.parametrize("size", [0.003, 0.3, -0.05, 3.0])
def test_wide_blocks_whose_bias_grows_by_the_row(more, size):
    # slopes that differ by head, some zero: tiles before, behind and around the tokens; sizes on both sides of where the largest score is only bounded
    rng = np.random.default_rng(91)
    lens, tokens, kv, group, d = (1500, 131, 700), 70, 2, 4, 64
    kind = {k: v for k, v in more.items() if k in ("causal", "window", "prefix", "softcap")}
    kind["slopes"] = (size * np.array([1, 0.5, 0, 0.25, 1, 1, 0.9, 0.7])).astype(F)
    if more.get("docs"):
        doc = np.concatenate([np.sort(rng.integers(1, 3, n)) for n in lens]).astype(np.uint32)
        kind["row_doc"] = np.stack([doc] * kv)
        kind["q_doc"] = np.concatenate([doc[e - tokens:e] for e in np.cumsum(lens)])
    if more.get("ahead"):  # tokens far before and far behind all rows
        kind["q_pos"] = np.concatenate([np.arange(tokens), 5000000 + np.arange(tokens), 300 + 3 * np.arange(tokens)]).astype(np.uint32)
        kind["causal"] = False
    check(*make(rng, lens, tokens, kv, group, d, True, **kind), True)


@pytest.mark.parametrize("d,group,tokens", [(128, 4, 40), (64, 1, 300), (128, 8, 33)])
def test_wide_blocks_without_a_row_among_others(d, group, tokens):
    # sequences whose rows are gone, and tokens of a document that no row has: zeros, while blocks beside them work
    rng = np.random.default_rng(d + tokens)
    lens, kv = (600, 400, 700, 333, 512, 64) * 4, 3
    call, raw = make(rng, lens, tokens, kv, group, d, True)
    call.rows = np.array([600, 0, 350, 0, 512, 0] * 4, np.uint32)
    out, lse = check(call, raw, True)
    for i in range(1, len(lens), 2):
        assert np.all(out[i * tokens:(i + 1) * tokens] == 0) and np.all(lse[i * tokens:(i + 1) * tokens] == -np.inf)
    total = sum(lens)
    call, raw = make(rng, lens, tokens, kv, group, d, True, row_doc=np.ones((kv, total), np.uint32), q_doc=np.repeat(np.arange(len(lens)) % 2, tokens).astype(np.uint32))
    out, lse = check(call, raw, True)
    assert np.all(out.reshape(len(lens), tokens, -1)[::2] == 0) and np.all(lse.reshape(len(lens), tokens, -1)[::2] == -np.inf)
