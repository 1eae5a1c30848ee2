"""Rows of keys and values in 4 bits: written and read back (slha_b200_write_cache4, slha_b200_read_cache4) bit for bit as the formula says, and attention over
them (slha_b200_attend_cache4, slha_b200_attend_tree4) against plain forms in 64 bits; the bounds are those of tests/cache4_cases.py."""
import numpy as np
import pytest

from tests import cache4_cases as Q
from tests import cache_cases as K

pytestmark = pytest.mark.gpu
S = pytest.importorskip("slhav2_b200")
F = np.float32


def type_of(bf16):
    return S.BF16 if bf16 else S.F32


# --------------------------------------------------------------------------- written and read back
class Stored:
    """A cache [row][head] of `total` rows with known bytes in every gap and row, on the device."""

    def __init__(self, total, kv, d, bf16=True, key_exponent=0, value_exponent=0, rows=None):
        self.total, self.kv, self.d = total, kv, d
        a, b = Q.laid_out(np.zeros((total, kv, d), np.uint8), np.zeros((total, kv, d // 16), np.uint8))
        self.shapes = a.shape, b.shape
        self.arrays = [S.to_device(np.full(s, 0xA5, np.uint8)) for s in (a.shape, a.shape, b.shape, b.shape)]
        self.cache = S.KvCache4(*self.arrays, kv, d, dtype=type_of(bf16), key_exponent=key_exponent, value_exponent=value_exponent, rows=rows)

    def bytes(self, x):
        """Keys' (0) or values' (1) code and scale bytes."""
        return [self.arrays[i + x].download(np.uint8, int(np.prod(s))).reshape(s) for i, s in ((0, self.shapes[0]), (2, self.shapes[1]))]


def odd_rows(rng, n, kv, d, bf16, exponent):
    """Rows of many sizes, with blocks of zeros, of borders between codes, of the smallest and the largest sizes."""
    x = rng.standard_normal((n, kv, d)) * np.exp2(rng.integers(-12, 12, (n, kv, d // 16)).repeat(16, -1)) * np.exp(rng.standard_normal((n, kv, d)))
    blocks = x.reshape(n, kv, -1, 16)
    pick = lambda p: rng.random(blocks.shape[:3]) < p  # noqa: E731
    border = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    on = pick(0.3)  # on the borders of the codes, for every one of the eight fractions a scale has, and the scale itself between two
    blocks[on] = (rng.choice(border, (int(on.sum()), 16)) * rng.choice([-1, 1], (int(on.sum()), 16)) * (1 + rng.integers(0, 16, (int(on.sum()), 1)) / 16) *
                  np.exp2(rng.integers(-7, 8, (int(on.sum()), 1))))
    near = pick(0.2)  # the largest is six times a scale, the others next to the borders
    step = 2.0 ** -7 if bf16 else 2.0 ** -23
    k = int(near.sum())
    blocks[near] = rng.choice(border, (k, 16)) * (1 + rng.integers(0, 8, (k, 1)) / 8) * (1 + step * rng.integers(-1, 2, (k, 16)))
    blocks[near, 0] = 6 * (1 + rng.integers(0, 8, k) / 8)
    blocks[pick(0.05)] = 0.0
    blocks[pick(0.05)] *= 2.0 ** -30
    blocks[pick(0.05)] *= 2.0 ** 30
    with np.errstate(over="ignore"):
        return K.as_type(blocks.reshape(n, kv, d) * 2.0 ** exponent, bf16)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("d", [16, 48, 64, 80, 96, 128, 208, 256])
@pytest.mark.parametrize("kv,tokens,exponent", [(1, 1, 0), (2, 7, -3), (3, 50, 5), (8, 200, 0), (5, 33, -64), (5, 33, 64)])
def test_codes_and_scales_are_what_the_formula_gives(bf16, d, kv, tokens, exponent):
    rng = np.random.default_rng(d + tokens)
    total = tokens + 9
    keys, dk = odd_rows(rng, tokens, kv, d, bf16, exponent)
    vals, dv = odd_rows(rng, tokens, kv, d, bf16, 0)
    st = Stored(total, kv, d, key_exponent=exponent)
    S.write_cache4(st.cache, S.make_segments([(3, tokens + 4, 0, tokens, 0)]), S.KvCache(S.to_device(dk), S.to_device(dv), kv, d, dtype=type_of(bf16)), tokens)
    for x, rows, e in ((0, keys, exponent), (1, vals, 0)):
        want = Q.laid_out(*Q.quantise(rows, e), fill=0xA5)
        for got, w in zip(st.bytes(x), want):
            assert np.array_equal(got[7:7 + tokens][..., :w.shape[-1]], w), np.argwhere(got[7:7 + tokens] != w)[:4]
            assert np.all(got[:7] == 0xA5) and np.all(got[7 + tokens:] == 0xA5)
    # and back, in both types
    for to16 in (True, False):
        n = total
        ks, vs = (S.to_device(np.full((n, kv, d), 0x40E0 if to16 else 7.0, np.uint16 if to16 else F)) for _ in range(2))
        S.read_cache4(st.cache, S.make_segments([(7, tokens, 0, 0, 0)]), S.KvCache(ks, vs, kv, d, dtype=type_of(to16)), S.make_segments([(1, tokens, 0, 0, 0)]))
        for buf, rows, e in ((ks, keys, exponent), (vs, vals, 0)):
            got = buf.download(np.uint16 if to16 else F, n * kv * d)
            got = (K.from_bf16(got) if to16 else got).reshape(n, kv, d)
            assert np.array_equal(got[1:1 + tokens], Q.values(*Q.quantise(rows, e), e)) and np.all(got[:1] == 7) and np.all(got[1 + tokens:] == 7)


@pytest.mark.parametrize("bf16", [True, False])
def test_nan_marks_its_block_and_infinities_the_largest_size(bf16):
    d = 64
    x = np.random.default_rng(1).standard_normal((3, 2, d)).astype(F)
    x[0, 1, 20] = np.nan
    x[1, 0, 3], x[1, 0, 5] = np.inf, -np.inf
    x[2, 1, 40:42] = (3e38, -3e38)
    v, raw = K.as_type(x, bf16)
    if bf16:
        raw[0, 1, 20], v[0, 1, 20] = 0xFFC0, np.nan
    st = Stored(3, 2, d)
    S.write_cache4(st.cache, S.make_segments([(0, 3, 0, 3, 0)]), S.KvCache(S.to_device(raw), S.to_device(raw), 2, d, dtype=type_of(bf16)), 3)
    out = S.DeviceBuffer(3 * 2 * d * 4)
    S.read_cache4(st.cache, S.make_segments([(0, 3, 0, 0, 0)]), S.KvCache(out, None, 2, d, dtype=S.F32))
    got = out.download(F, 3 * 2 * d).reshape(3, 2, d)
    assert np.isnan(got[0, 1, 16:32]).all() and np.isfinite(got).sum() == got.size - 16
    assert got[1, 0, 3] == 2688 and got[1, 0, 5] == -2688 and got[2, 1, 40] == 2688 and got[2, 1, 41] == -2688
    want = Q.values(*Q.quantise(np.where(np.isinf(v), np.sign(v) * F(3e38), v), 0), 0)
    assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("on_device", [False, True])
def test_tokens_go_to_their_segments_last_rows(on_device):
    rng = np.random.default_rng(2)
    segs = [(30, 10, 1, 3, 0), (0, 5, 6, 4, 0), (10, 4, 4, 0, 0), (50, 3, 10, 2, 0)]
    counts = np.array([7, 9, 4, 1], np.uint32)
    keys, dk = K.as_type(rng.standard_normal((12, 2, 64)), True)
    vals, dv = K.as_type(rng.standard_normal((12, 2, 64)), True)
    # tokens [head][token] with gaps
    k2 = np.zeros((2, 12, 72), np.uint16)
    k2[:, :, :64] = dk.transpose(1, 0, 2)
    st = Stored(60, 2, 64, rows=S.to_device(counts) if on_device else counts)
    S.write_cache4(st.cache, S.make_segments(segs), S.KvCache(S.to_device(k2), S.to_device(dv), 2, 64, key_row_stride=72, key_head_stride=864), 12)
    for x, rows in ((0, keys), (1, vals)):
        want = Q.laid_out(*Q.quantise(rows, 0))
        got = st.bytes(x)
        written = np.zeros(60, bool)
        for i, (b, n, q0, t, _) in enumerate(segs):
            n = min(n, int(counts[i]))
            ctx = n - min(n, t)
            for j in range(min(t, n - ctx)):
                written[b + ctx + j] = True
                assert all(np.array_equal(g[b + ctx + j], w[q0 + j]) for g, w in zip(got, want))
        assert all(np.all(g[~written] == 0xA5) for g in got)


def test_rows_read_to_other_layouts_from_many_segments_and_counts():
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 40, 80)
    total, kv, d = int(lens.sum()), 3, 96
    codes, scales = rng.integers(0, 16, (total, kv, d)).astype(np.uint8), rng.integers(0, 127, (total, kv, d // 16)).astype(np.uint8)
    a, b = Q.laid_out(codes, scales, fill=0x7F)
    counts = (lens * 3 // 4).astype(np.uint32)
    begins = np.concatenate([[0], np.cumsum(lens)[:-1]])
    for dev in (False, True):
        cache = S.KvCache4(S.to_device(a), S.to_device(a), S.to_device(b), S.to_device(b), kv, d, key_exponent=2, rows=S.to_device(counts) if dev else counts)
        out = S.to_device(np.full((kv, total + 80, d + 4), 7.0, F))
        segs, to = S.make_segments([(int(x), int(n), 0, 0, 0) for x, n in zip(begins, lens)]), S.make_segments([(int(x) + i, int(n) + 1, 0, 0, 0) for i, (x, n) in enumerate(zip(begins, lens))])
        S.read_cache4(cache, segs, S.KvCache(out, None, kv, d, dtype=S.F32, key_row_stride=d + 4, key_head_stride=(total + 80) * (d + 4)), to)
        got = out.download(F, kv * (total + 80) * (d + 4)).reshape(kv, total + 80, d + 4).transpose(1, 0, 2)
        want = np.full(got.shape, 7.0, F)
        full = Q.values(codes, scales, 2)
        for i, (x, c) in enumerate(zip(begins, counts)):
            want[x + i:x + i + c, :, :d] = full[x:x + c]
        assert np.array_equal(got, want)


# --------------------------------------------------------------------------- attention
def make(rng, lens, tokens, kv, group, d, bf16, q_scale=1.5, bases=None, key_exponent=-3, value_exponent=-4, **more):
    total = int(sum(lens))
    raw = []
    vals = []
    for e, x in ((key_exponent, rng.standard_normal((max(total, 1), kv, d)) * np.exp(0.5 * rng.standard_normal(d))), (value_exponent, rng.standard_normal((max(total, 1), kv, d)))):
        codes, scales = Q.quantise(x.astype(F), e)
        vals.append(Q.values(codes, scales, e))
        raw += Q.laid_out(codes, scales, fill=0x7F)
    toks = [tokens] * len(lens) if np.isscalar(tokens) else list(tokens)
    q, dq = K.as_type(q_scale * rng.standard_normal((max(sum(toks), 1), kv * group, d)), bf16)
    segs, at, q0 = [], 0, 0
    for i, (n, t) in enumerate(zip(lens, toks)):
        segs.append((at, int(n), q0, t, 0 if bases is None else bases[i]))
        at += int(n)
        q0 += t
    call = Q.Call4(vals[0], vals[1], q, segs, d ** -0.5, **more)
    call.exponents = key_exponent, value_exponent
    return call, [raw[0], raw[2], raw[1], raw[3], dq]


def on_device(call, raw, bf16):
    up = lambda x, t: None if x is None else S.to_device(np.ascontiguousarray(x, t))  # noqa: E731
    per_head = call.row_pos is not None or call.row_doc is not None
    cache = S.KvCache4(*(S.to_device(x) for x in raw[:4]), call.kv, call.d, dtype=type_of(bf16), key_exponent=call.exponents[0], value_exponent=call.exponents[1],
                       positions=up(call.row_pos, np.uint32), documents=up(call.row_doc, np.uint32), entry_head_stride=call.keys.shape[0] if per_head else 0, rows=call.rows)
    queries = S.CacheQueries(S.to_device(raw[4]), call.q.shape[0], call.heads, call.d, scale=call.scale, softcap=call.softcap, window=call.window, causal=call.causal,
                             slopes=call.slopes, prefix=call.prefix, positions=up(call.q_pos, np.uint32), documents=up(call.q_doc, np.uint32))
    return cache, S.make_segments(call.segs), queries


def results(call, bf16, cache, segs, queries):
    n = call.q.size
    out, lse = S.to_device(np.full(n, 7.0, F) if not bf16 else np.full(n, 0x40E0, np.uint16)), S.to_device(np.full(call.q.shape[:2], 7.0, F))
    if call.parents is not None:
        S.attend_tree4(cache, segs, queries, call.parents, out, lse)
    else:
        S.attend_cache4(cache, segs, queries, out, lse)
    o = out.download(np.uint16 if bf16 else F, n)
    return (K.from_bf16(o) if bf16 else o).reshape(call.q.shape), lse.download(F, call.q.shape[0] * call.heads).reshape(call.q.shape[:2])


def held(got, want, tol):
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


SHAPES = [(2, 4, 1, (1, 63, 64, 65, 128, 129, 700)), (1, 1, 1, (5000,)), (2, 3, 3, (3, 10, 130, 257)), (2, 3, 9, (9, 10, 130, 257)), (1, 8, 37, (37, 300)), (3, 5, 5, (200, 33)),
          (2, 8, 2, (140, 40)), (1, 6, 10, (500, 10))]


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("d", [16, 64, 80, 128, 208, 256])
@pytest.mark.parametrize("kv,group,tokens,lens", SHAPES)
def test_attention_of_every_type_and_width(bf16, d, kv, group, tokens, lens):
    rng = np.random.default_rng(d * 10 + tokens)
    check(*make(rng, lens, tokens, kv, group, d, bf16), bf16)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("tokens", [1, 3, 6, 40, 150])
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
@pytest.mark.parametrize("tokens,group,window", [(1, 1, 0), (7, 4, 0), (33, 1, 0), (7, 2, 20), (100, 3, 0), (256, 1, 0)])
def test_trees_of_drafted_tokens(bf16, tokens, group, window):
    rng = np.random.default_rng(tokens)
    parents = np.concatenate([np.where(rng.random(tokens) < 0.1, K.NONE, (np.arange(tokens) * rng.random(tokens)).astype(np.int64)) for _ in range(3)]).astype(np.uint32)
    check(*make(rng, (tokens, tokens + 70, tokens + 300), tokens, 2, group, 128, bf16, window=window, parents=parents, bases=(0, 5, 100)), bf16)


@pytest.mark.parametrize("bf16", [True, False])
def test_lengths_of_zero_tokens_without_a_row_and_tokens_of_no_segment(bf16):
    rng = np.random.default_rng(3)
    check(*make(rng, (0, 40, 0, 100), (2, 3, 0, 0), 2, 2, 128, bf16), bf16)
    call, raw = make(rng, (40, 90), (2, 30), 2, 2, 64, bf16, row_doc=np.full((2, 130), 5, np.uint32), q_doc=np.full(32, 6, np.uint32))
    o, z = check(call, raw, bf16)
    assert np.all(o == 0) and np.all(z == -np.inf)
    call, raw = make(rng, (70,), (20,), 1, 1, 64, bf16, row_pos=np.full((1, 70), 900, np.uint32), q_pos=np.arange(890, 910, dtype=np.uint32))
    o, z = check(call, raw, bf16)
    assert np.all(o[:10] == 0) and np.all(np.isfinite(z[10:]))
    call, raw = make(rng, (50, 60), (4, 40), 2, 2, 64, bf16)
    call.segs = [(0, 50, 3, 1, 0), (50, 60, 10, 20, 0)]
    check(call, raw, bf16)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("tokens", [1, 2, 6, 100])
def test_rows_that_a_token_does_not_see_may_hold_anything(bf16, tokens):
    rng = np.random.default_rng(tokens)
    lens, kv, group, d = (300, 411), 2, 2, 64
    doc = rng.integers(0, 3, sum(lens)).astype(np.uint32)
    for b, n in ((0, 300), (300, 411)):
        doc[b + n - tokens:b + n] = rng.integers(0, 2, tokens)
    call, raw = make(rng, lens, tokens, kv, group, d, bf16, row_doc=np.stack([doc] * kv), q_doc=np.concatenate([doc[300 - tokens:300], doc[711 - tokens:711]]))
    want = call.attend(bf16)
    for x in range(4):  # no token's document: any bytes, of scales NaN among them
        r = rng.integers(0, 256, raw[x][doc == 2].shape)
        raw[x][doc == 2] = np.where(rng.random(r.shape) < 0.3, 0x7F, r) if x > 1 else r
    got = results(call, bf16, *on_device(call, raw, bf16))
    held(got[1], want[1], want[3])
    held(got[0], want[0], want[2])
    # a NaN block of values that tokens of document 1 see, and those of document 0 do not
    at = int(np.flatnonzero(doc[:300] == 1)[0])
    raw[3][at, :, 1] = 0x7F
    got = results(call, bf16, *on_device(call, raw, bf16))
    sees = np.zeros(call.q.shape[0], bool)
    sees[:tokens] = (call.q_doc[:tokens] == 1) & (at <= 300 - tokens + np.arange(tokens))
    bad = np.zeros(got[0].shape, bool)
    bad[sees, :, 16:32] = True
    assert np.isnan(got[0][bad]).all()
    assert np.all((np.abs(got[0] - want[0]) <= want[2])[~bad])
    held(got[1], want[1], want[3])


@pytest.mark.parametrize("bf16", [True, False])
def test_a_nan_in_a_seen_key_is_in_the_results_of_its_head(bf16):
    rng = np.random.default_rng(9)
    call, raw = make(rng, (200,), 1, 2, 2, 64, bf16)
    want = call.attend(bf16)
    raw[2][50, 1, 0] = 0x7F
    got = results(call, bf16, *on_device(call, raw, bf16))
    assert np.isnan(got[0][:, 2:]).all() and np.isnan(got[1][:, 2:]).all()
    held(got[0][:, :2], want[0][:, :2], want[2][:, :2])


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("tokens", [2, 40])
def test_layouts_strides_and_row_counts(bf16, tokens):
    rng = np.random.default_rng(11)
    kv, group, d, lens = 2, 2, 96, (130, 75)
    call, raw = make(rng, lens, tokens, kv, group, d, bf16)
    call.rows = np.array([100, 900], np.uint32)  # fewer than the table says, and more
    codes, scales = [np.full((kv, 205, 64), 0x7F, np.uint8) for _ in range(2)], [np.full((kv, 205, 16), 0x7F, np.uint8) for _ in range(2)]
    for x in range(2):  # [kv_head][row] with gaps
        codes[x][:, :, :48] = raw[x].transpose(1, 0, 2)
        scales[x][:, :, :8] = raw[2 + x].transpose(1, 0, 2)
    n = 2 * tokens
    q = np.zeros((kv * group, n, d + 8), raw[4].dtype)
    q[:, :, :d] = raw[4].transpose(1, 0, 2)
    want = call.attend(bf16)
    for rows in (call.rows, S.to_device(call.rows)):
        cache = S.KvCache4(*map(S.to_device, codes + scales), kv, d, dtype=type_of(bf16), code_row_stride=64, code_head_stride=205 * 64, scale_row_stride=16, scale_head_stride=205 * 16,
                           key_exponent=-3, value_exponent=-4, rows=rows)
        queries = S.CacheQueries(S.to_device(q), n, kv * group, d, token_stride=d + 8, head_stride=n * (d + 8))
        out = S.to_device(np.zeros((kv * group, n, d + 24), np.uint16 if bf16 else F))
        lse = S.DeviceBuffer(n * kv * group * 4)
        S.attend_cache4(cache, S.make_segments(call.segs), queries, out, lse, out_token_stride=d + 24, out_head_stride=n * (d + 24))
        o = out.download(np.uint16 if bf16 else F, kv * group * n * (d + 24)).reshape(kv * group, n, d + 24)
        assert np.all(o[:, :, d:] == 0)
        o = np.ascontiguousarray(o[:, :, :d].transpose(1, 0, 2))
        held(K.from_bf16(o).reshape(want[0].shape) if bf16 else o, want[0], want[2])


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_queries_of_every_size(bf16, size):
    rng = np.random.default_rng(12)
    call, raw = make(rng, (150,), 2, 2, 2, 64, bf16, q_scale=size)
    call.scale = float(F(0.125 / size))
    check(call, raw, bf16)


def test_weights_of_rows_far_below_the_largest_are_not_lost():
    # one row scores 16 above the others in units of log 2 and 60000 others share what is left
    rng = np.random.default_rng(13)
    call, raw = make(rng, (60001,), 1, 1, 1, 64, True, q_scale=0.0)
    keys = np.zeros((60001, 1, 64), F)
    keys[700, 0, 0] = 4.0
    codes, scales = Q.quantise(keys, -3)
    raw[0], raw[2] = Q.laid_out(codes, scales)
    call.keys = Q.values(codes, scales, -3)
    call.q[:, :, 0] = 16 * np.log(2) / 4 * 8
    call.q, raw[4] = K.as_type(call.q, True)
    check(call, raw, True)


def test_rows_of_a_few_and_of_many_tokens_in_one_call_and_the_same_bits_again():
    rng = np.random.default_rng(13)
    for bf16 in (True, False):
        call, raw = make(rng, (500, 900, 333, 64, 2000, 90), (1, 70, 9, 64, 1, 5), 2, 3, 128, bf16)
        a = check(call, raw, bf16)
        b = results(call, bf16, *on_device(call, raw, bf16))
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_long_tables_and_tables_in_device_memory():
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
    assert lib.slha_b200_attend_cache4(cache.address, dev.data_ptr(), len(segs), queries.address, out.data_ptr(), call.heads * 64, 64, lse.data_ptr()) == 0
    assert np.array_equal(K.from_bf16(out.download(np.uint16, call.q.size)).reshape(call.q.shape), got[0])


def test_a_step_of_a_model_heads_turned_written_attended_and_captured():
    """What a server runs: a prompt's heads are turned and written, then decoded tokens' with the row counts on the device, one graph for every step."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(14)
    seqs, prompt, steps, heads, kv, d, room = 3, 40, 4, 8, 2, 128, 64
    stream = torch.cuda.Stream()
    S.set_stream(stream.cuda_stream)
    try:
        st = Stored(seqs * room, kv, d, key_exponent=-3, value_exponent=-3)
        counts = S.to_device(np.full(seqs, prompt, np.uint32))
        cache = S.KvCache4(*st.arrays, kv, d, key_exponent=-3, value_exponent=-3, rows=counts)
        freq = (10000.0 ** (-np.arange(64) / 64)).astype(F)
        dfreq = S.to_device(freq)
        table = lambda t: S.make_segments([(i * room, room, i * t, t, 0) for i in range(seqs)])  # noqa: E731
        kept_q, kept_k, kept_v = {}, [], []

        def buffers(n):
            return [S.DeviceBuffer(n * (heads + 2 * kv) * d * 2), S.DeviceBuffer(n * heads * d * 2), S.DeviceBuffer(n * kv * d * 2), S.DeviceBuffer(n * kv * d * 2),
                    S.DeviceBuffer(n * heads * d * 2), S.DeviceBuffer(n * heads * 4), S.DeviceBuffer(4 * n)]

        def step(n, t, b):
            rows = S.HeadRows(b[0].data_ptr(), b[0].data_ptr() + heads * d * 2, b[0].data_ptr() + (heads + kv) * d * 2, n, heads, kv, d, token_stride=(heads + 2 * kv) * d, head_stride=d,
                              norm=True)
            fresh = S.KvCache(b[2], b[3], kv, d)
            S.rotate_heads(rows, S.Rotation(dfreq, b[6], d), q_out=b[1], to=fresh)
            S.write_cache4(cache, table(t), fresh, n)
            S.attend_cache4(cache, table(t), S.CacheQueries(b[1], n, heads, d), b[4], b[5])

        def load(n, t, first, b):
            b[0].upload(K.as_type(rng.standard_normal((n, (heads + 2 * kv) * d)), True)[1])
            b[6].upload(np.tile(np.arange(first, first + t), seqs).astype(np.uint32))

        def look(n, t, first, b):
            torch.cuda.synchronize()
            q = K.from_bf16(b[1].download(np.uint16, n * heads * d)).reshape(n, heads, d)
            k, v = (K.from_bf16(x.download(np.uint16, n * kv * d)).reshape(seqs, t, kv, d) for x in b[2:4])
            kept_k.append(Q.values(*Q.quantise(k, -3), -3))
            kept_v.append(Q.values(*Q.quantise(v, -3), -3))
            rows = first + t
            ks, vs = (np.concatenate(x, 1).reshape(seqs * rows, kv, d) for x in (kept_k, kept_v))
            call = Q.Call4(ks, vs, q, [(i * rows, rows, i * t, t, 0) for i in range(seqs)], float(F(d ** -0.5)))
            want = call.attend(True)
            held(K.from_bf16(b[4].download(np.uint16, n * heads * d)).reshape(n, heads, d), want[0], want[2])
            held(b[5].download(F, n * heads).reshape(n, heads), want[1], want[3])

        b = buffers(seqs * prompt)
        load(seqs * prompt, prompt, 0, b)
        step(seqs * prompt, prompt, b)
        look(seqs * prompt, prompt, 0, b)
        b = buffers(seqs)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(seqs, 1, b)
        for at in range(steps):
            load(seqs, 1, prompt + at, b)
            counts.upload(np.full(seqs, prompt + at + 1, np.uint32))
            graph.replay()
            look(seqs, 1, prompt + at, b)
        assert kept_q == {}
    finally:
        S.set_stream(None)
