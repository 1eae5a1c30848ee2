"""Attention by many tokens over rows in 4 bits, whose rows are laid out as bfloat16 first: counts of rows, windows, trees, documents and positions of heads, several batches of segments, other
layouts, and rows that hold anything.  Every test asserts that this path ran; before each call the thread's working memory holds rows of NaN.  The bounds are those of tests/cache4_cases.py."""
import threading

import numpy as np
import pytest

from tests import cache4_cases as Q
from tests import cache_cases as K
from tests import test_gpu_cache4 as T

pytestmark = pytest.mark.gpu
S = pytest.importorskip("slhav2_b200")
F = np.float32


def spoil(kv=8, group=4, d=128, rows=16000, tokens=600):
    """Leaves rows of NaN in the thread's working memory."""
    codes, scales = S.to_device(np.zeros((rows, kv, d // 2), np.uint8)), S.to_device(np.full((rows, kv, Q.scale_bytes(d)), 0x7F, np.uint8))
    out = S.DeviceBuffer(tokens * kv * group * d * 2)
    S.attend_cache4(S.KvCache4(codes, codes, scales, scales, kv, d), S.make_segments([(0, rows, 0, tokens, 0)]), S.CacheQueries(S.to_device(np.zeros(tokens * kv * group * d, np.uint16)), tokens, kv * group, d), out)
    assert S.debug_last_cache_kernels() & S.CACHE_LAID_OUT
    assert np.isnan(K.from_bf16(out.download(np.uint16, tokens * kv * group * d))).all()


def laid_out_results(call, raw, sets=None):
    spoil()
    got = T.results(call, True, *(sets or T.on_device(call, raw, True)))
    assert S.debug_last_cache_kernels() & S.CACHE_LAID_OUT
    return got


def one_head(call, h, tokens=None):
    """The call of KV head h, of some tokens of each segment alone (by their places)."""
    hs = slice(h * call.group, (h + 1) * call.group)
    more = dict(softcap=call.softcap, window=call.window, causal=call.causal, prefix=call.prefix, rows=call.rows, parents=call.parents, slopes=None if call.slopes is None else call.slopes[hs],
                row_pos=None if call.row_pos is None else call.row_pos[h:h + 1], row_doc=None if call.row_doc is None else call.row_doc[h:h + 1], q_pos=call.q_pos, q_doc=call.q_doc)
    picked, segs = [], []
    for i, (b, n, q0, t, base) in enumerate(call.segs):
        of = list(range(t)) if tokens is None else [x for x in tokens if x < t]
        segs.append((b, n, len(picked), len(of), base))
        picked += [q0 + x for x in of]
    if tokens is not None and call.q_pos is None:
        at = np.zeros(call.q.shape[0], np.int64)
        for i, (b, n, q0, t, base) in enumerate(call.segs):
            m = n if call.rows is None else min(n, int(call.rows[i]))
            at[q0:q0 + t] = base + m - min(m, t) + np.arange(t)
        more["q_pos"] = at
    if tokens is not None:
        for name in ("q_pos", "q_doc"):
            more[name] = None if more[name] is None else more[name][picked]
    return Q.Call4(call.keys[:, h:h + 1], call.values[:, h:h + 1], call.q[picked][:, hs], segs, call.scale, **more), picked, hs


def check(call, raw, heads=None, tokens=None, sets=None):
    got = laid_out_results(call, raw, sets)
    for h in (call.kv - 1,) if heads is None else heads:
        one, picked, hs = one_head(call, h, tokens)
        out, lse, out_tol, lse_tol = one.attend(True)
        T.held(got[1][picked][:, hs], lse, lse_tol)
        T.held(got[0][picked][:, hs], out, out_tol)
    return got


@pytest.mark.parametrize("on_device", [False, True])
@pytest.mark.parametrize("window,docs", [(0, False), (300, False), (300, True), (1, False)])
def test_counts_of_rows_with_and_without_a_window(on_device, window, docs):
    rng = np.random.default_rng(window + docs)
    lens, toks, kv = (4000, 3000, 3500), (600, 500, 400), 8
    more = {}
    if docs:
        doc = np.concatenate([np.sort(rng.integers(1, 3, n)) for n in lens]).astype(np.uint32)
        counted = (3900, 2500, 410)
        more = dict(row_doc=np.stack([doc] * kv), q_doc=np.concatenate([doc[b + c - t:b + c] for b, c, t in zip((0, 4000, 7000), counted, toks)]))
    call, raw = T.make(rng, lens, toks, kv, 4, 128, True, window=window, bases=(0, 9, 1 << 20), **more)
    call.rows = np.array([3900, 2500, 410], np.uint32)
    for b, n, c in zip((0, 4000, 7000), lens, call.rows):  # rows behind a segment's last may hold anything
        for x in range(4):
            raw[x][b + c:b + n] = 0x7F
    if window:  # and those that its window leaves behind
        for b, c, t in zip((0, 4000, 7000), call.rows, toks):
            raw[2][b:b + max(0, int(c) - t - window + 1)] = raw[3][b:b + max(0, int(c) - t - window + 1)] = 0x7F
    sets = T.on_device(call, raw, True)
    counts = S.to_device(call.rows)
    if on_device:
        cache = S.KvCache4(*(S.to_device(x) for x in raw[:4]), kv, 128, key_exponent=-3, value_exponent=-4, documents=None if not docs else S.to_device(call.row_doc),
                           entry_head_stride=sum(lens) if docs else 0, rows=counts)
        sets = (cache, *sets[1:])
    a = check(call, raw, sets=sets)
    b = T.results(call, True, *sets)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_a_captured_call_takes_the_counts_that_are_there_when_it_runs():
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(3)
    call, raw = T.make(rng, (4000, 3000), (600, 500), 8, 4, 128, True, window=200)
    counts = S.to_device(np.array([4000, 3000], np.uint32))
    cache = S.KvCache4(*(S.to_device(x) for x in raw[:4]), 8, 128, key_exponent=-3, value_exponent=-4, rows=counts)
    segs = S.make_segments(call.segs)
    queries = S.CacheQueries(S.to_device(raw[4]), call.q.shape[0], call.heads, 128, scale=call.scale, window=200)
    out, lse = S.DeviceBuffer(call.q.size * 2), S.DeviceBuffer(call.q.shape[0] * call.heads * 4)
    stream = torch.cuda.Stream()
    S.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            S.attend_cache4(cache, segs, queries, out, lse)
        assert S.debug_last_cache_kernels() & S.CACHE_LAID_OUT
        for rows in ((4000, 3000), (1500, 2999), (600, 20), (3000, 0)):
            counts.upload(np.array(rows, np.uint32))
            spoil()
            graph.replay()
            torch.cuda.synchronize()
            call.rows = np.array(rows, np.uint32)
            one, picked, hs = one_head(call, 5, (0, 3, 19, 20, 250, 499, 599))
            want = one.attend(True)
            T.held(K.from_bf16(out.download(np.uint16, call.q.size)).reshape(call.q.shape)[picked][:, hs], want[0], want[2])
            T.held(lse.download(F, call.q.shape[0] * call.heads).reshape(call.q.shape[:2])[picked][:, hs], want[1], want[3])
    finally:
        S.set_stream(None)


@pytest.mark.parametrize("window", [0, 150])
@pytest.mark.parametrize("moved", [False, True])
def test_trees_of_many_drafted_tokens(window, moved):
    rng = np.random.default_rng(window)
    tokens, lens, kv = 256, (9000, 8000, 256), 8
    parents = np.concatenate([np.where(rng.random(tokens) < 0.1, K.NONE, (np.arange(tokens) * rng.random(tokens)).astype(np.int64)) for _ in lens]).astype(np.uint32)
    more = {}
    if moved:
        more["row_pos"] = np.stack([np.concatenate([np.sort(rng.permutation(2 * n)[:n]) for n in lens]) for _ in range(kv)]).astype(np.uint32)
        more["q_pos"] = np.concatenate([2 * n + rng.integers(0, 9, tokens) for n in lens]).astype(np.uint32)
    check(*T.make(rng, lens, tokens, kv, 4, 128, True, window=window, parents=parents, bases=(0, 5, 100), **more))


@pytest.mark.parametrize("more", ["", "docs", "moved"])
def test_several_batches_of_segments(more):
    # rows of 8 KV heads of 128 dimensions are 4096 bytes: two of these segments are more than 512 MB, and the short ones share a batch with one
    rng = np.random.default_rng(len(more))
    kv, group, d, lens, toks = 8, 4, 128, (500, 70000, 66000, 900, 0, 64000), (200, 300, 260, 0, 250, 220)
    total = sum(lens)
    raw, vals = [], []
    for _ in range(2):
        codes, scales = rng.integers(0, 256, (total, kv, d // 2), np.uint8), rng.integers(40, 72, (total, kv, 8), np.uint8)
        raw += [codes, scales]
        both = np.empty((total, 1, d), np.uint8)
        both[:, 0, 0::2], both[:, 0, 1::2] = codes[:, kv - 1] & 15, codes[:, kv - 1] >> 4
        vals.append(Q.values(both, scales[:, kv - 1:], -3))
    q, dq = K.as_type(0.3 * rng.standard_normal((sum(toks), kv * group, d)), True)
    starts, q0 = np.cumsum((0,) + lens), np.cumsum((0,) + toks)
    segs = [(int(b), n, int(c), t, 7 * i) for i, (b, n, c, t) in enumerate(zip(starts, lens, q0, toks))]
    kind = {}
    if more == "docs":
        doc = np.concatenate([np.sort(rng.integers(1, 4, n)) for n in lens]).astype(np.uint32)
        kind = dict(row_doc=np.stack([doc] * kv), q_doc=np.concatenate([doc[b + n - t:b + n] if n else np.ones(t, np.uint32) for b, n, t in zip(starts, lens, toks)]))
    if more == "moved":
        kind = dict(row_pos=np.stack([np.concatenate([rng.permutation(2 * n)[:n] for n in lens]) for _ in range(kv)]).astype(np.uint32),
                    q_pos=np.concatenate([2 * n - t + np.arange(t) if n else np.arange(t) for n, t in zip(lens, toks)]).astype(np.uint32), window=9000)
    last = {k: (v[kv - 1:] if k.startswith("row") else v) for k, v in kind.items()}
    call = Q.Call4(vals[0], vals[1], q[:, -group:], segs, float(F(d ** -0.5)), **last)
    up = lambda x: None if x is None else S.to_device(np.ascontiguousarray(x, np.uint32))  # noqa: E731
    cache = S.KvCache4(*(S.to_device(raw[i]) for i in (0, 2, 1, 3)), kv, d, key_exponent=-3, value_exponent=-3, positions=up(kind.get("row_pos")), documents=up(kind.get("row_doc")),
                       entry_head_stride=total if kind else 0)
    queries = S.CacheQueries(S.to_device(dq), sum(toks), kv * group, d, scale=call.scale, window=call.window, positions=up(kind.get("q_pos")), documents=up(kind.get("q_doc")))
    spoil()
    out, lse = S.to_device(np.full(q.size, 0x40E0, np.uint16)), S.DeviceBuffer(q.shape[0] * kv * group * 4)
    S.attend_cache4(cache, S.make_segments(segs), queries, out, lse)
    assert S.debug_last_cache_kernels() & S.CACHE_LAID_OUT
    got = K.from_bf16(out.download(np.uint16, q.size)).reshape(q.shape)[:, -group:], lse.download(F, q.shape[0] * kv * group).reshape(q.shape[:2])[:, -group:]
    one, picked, _ = one_head(call, 0, (0, 1, 100, 199, 219, 259, 299))
    want = one.attend(True)
    T.held(got[1][picked], want[1], want[3])
    T.held(got[0][picked], want[0], want[2])
    assert np.all(got[0][q0[4]:q0[5]] == 0) and np.all(got[1][q0[4]:q0[5]] == -np.inf)  # (the segment without rows)


def test_codes_by_heads_with_gaps():
    rng = np.random.default_rng(5)
    kv, group, d, n, tokens = 8, 4, 96, 5000, 500
    call, raw = T.make(rng, (n,), tokens, kv, group, d, True)
    codes, scales = [np.full((kv, n + 7, 64), 0x7F, np.uint8) for _ in range(2)], [np.full((kv, n + 7, 16), 0x7F, np.uint8) for _ in range(2)]
    for x in range(2):
        codes[x][:, :n, :48], scales[x][:, :n, :8] = raw[x].transpose(1, 0, 2), raw[2 + x].transpose(1, 0, 2)
    cache = S.KvCache4(*map(S.to_device, codes + scales), kv, d, code_row_stride=64, code_head_stride=(n + 7) * 64, scale_row_stride=16, scale_head_stride=(n + 7) * 16, key_exponent=-3, value_exponent=-4)
    check(call, raw, sets=(cache, *T.on_device(call, raw, True)[1:]))


def test_rows_that_hold_anything_and_nan_that_is_seen():
    rng = np.random.default_rng(6)
    kv, group, d, n, tokens = 8, 4, 128, 5000, 500
    doc = rng.integers(0, 3, n).astype(np.uint32)
    doc[n - tokens:] = rng.integers(0, 2, tokens)
    call, raw = T.make(rng, (n,), tokens, kv, group, d, True, row_doc=np.stack([doc] * kv), q_doc=doc[n - tokens:])
    for x in range(4):  # no token's document
        r = rng.integers(0, 256, raw[x][doc == 2].shape)
        raw[x][doc == 2] = np.where(rng.random(r.shape) < 0.3, 0x7F, r) if x > 1 else r
    clean = check(call, raw, heads=(3,))
    at = int(np.flatnonzero(doc == 1)[5])  # every token of document 1 sees it, those of document 0 do not
    raw[3][at, 3, 2] = 0x7F  # values of KV head 3, elements 32 to 47
    raw[2][at, 6, 0] = 0x7F  # keys of KV head 6
    got = laid_out_results(call, raw)
    sees = call.q_doc == 1
    bad = np.zeros(got[0].shape, bool)
    bad[sees, 3 * group:4 * group, 32:48] = True
    bad[sees, 6 * group:7 * group] = True
    assert np.isnan(got[0][bad]).all() and np.array_equal(got[0][~bad], clean[0][~bad])
    assert np.isnan(got[1][sees][:, 6 * group:7 * group]).all()


@pytest.mark.parametrize("sequences", [1, 4])
def test_working_memory_of_rows_and_parts(sequences):
    # 131072 rows laid out are 512 MB, a batch of one segment; 256 tokens are few blocks, so that the rows are split.  A thread keeps what its calls took
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(7)
    kv, group, d, n, tokens = 8, 4, 128, 131072, 256
    codes, scales = S.to_device(rng.integers(0, 256, (n, kv, d // 2), np.uint8)), S.to_device(rng.integers(40, 72, (n, kv, 8), np.uint8))
    cache = S.KvCache4(codes, codes, scales, scales, kv, d, key_exponent=-3, value_exponent=-3)
    q = 0.3 * rng.standard_normal((tokens, kv * group, d))
    queries = S.CacheQueries(S.to_device(np.concatenate([K.as_type(q, True)[1]] * sequences)), sequences * tokens, kv * group, d)
    out = S.DeviceBuffer(sequences * tokens * kv * group * d * 2)
    S.attend_cache4(cache, S.make_segments([(0, 8000, 0, tokens, 0)]), queries, out)  # (the kernels are loaded)
    S.synchronize()
    segs = S.make_segments([(0, n, i * tokens, tokens, 0) for i in range(sequences)])  # (sequences that share their rows)
    taken, got = [], []

    def work():
        before = torch.cuda.mem_get_info()[0]
        for _ in range(3):
            S.attend_cache4(cache, segs, queries, out)
            assert S.debug_last_cache_kernels() & S.CACHE_LAID_OUT
            S.synchronize()
            taken.append(before - torch.cuda.mem_get_info()[0])
            got.append(out.download(np.uint16, sequences * q.size).reshape(sequences, -1))

    t = threading.Thread(target=work)
    t.start()
    t.join()
    # rows, parts (at most 512 MB; here 256 rows of 520 bytes of 8 KV heads for each of 4 blocks and at most 10 runs: 43 MB), a step of the arena of 64 MB
    assert len(taken) == 3 and max(taken) <= 640 << 20, [x >> 20 for x in taken]
    for x in got:  # the same inputs, the same bits, whichever batch
        assert np.array_equal(x, got[0][:1].repeat(sequences, 0)) and np.isfinite(K.from_bf16(x)).all()
