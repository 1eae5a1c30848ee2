"""Attention over rows in 4 bits where it takes one kernel or the other, many columns, far offsets, large scores, streams, graphs and threads; the bounds are those
of tests/cache4_cases.py."""
import threading

import numpy as np
import pytest

from tests import cache4_cases as Q
from tests import cache_cases as K
from tests import test_gpu_cache4 as T

pytestmark = pytest.mark.gpu
S = pytest.importorskip("slhav2_b200")
F = np.float32


@pytest.mark.parametrize("d,group,more", [(64, 4, dict()), (128, 8, dict(window=100)), (80, 3, dict(window=100, softcap=10.0)), (64, 4, dict(prefix=True, window=50)), (80, 3, dict(docs=True)),
                                          (128, 4, dict(moved=True, alibi=True, window=700)), (64, 3, dict(causal=False)), (128, 3, dict(causal=False, window=90)), (48, 4, dict(window=300))])
def test_prompts_whose_rows_are_laid_out(d, group, more):
    rng = np.random.default_rng(d + group)
    lens, kv = (1500, 700, 1650), 8
    toks = (1200, 700, 3)  # and a few tokens in the same call
    total = sum(lens)
    kind = {k: v for k, v in more.items() if k in ("softcap", "window", "causal")}
    if more.get("alibi"):
        kind["slopes"] = (2.0 ** -np.arange(1, kv * group + 1)).astype(F)
    if more.get("prefix"):
        kind["prefix"] = np.array([0, 70, 40], np.uint32)
    if more.get("docs"):
        doc = np.concatenate([np.sort(rng.integers(1, 4, n)) for n in lens]).astype(np.uint32)
        kind["row_doc"] = np.stack([doc] * kv)
        kind["q_doc"] = np.concatenate([doc[e - t:e] for e, t in zip(np.cumsum(lens), toks)])
    if more.get("moved"):
        kind["row_pos"] = np.stack([np.concatenate([rng.permutation(2 * n)[:n] for n in lens]) for _ in range(kv)]).astype(np.uint32)
        kind["q_pos"] = np.concatenate([2 * n - t + np.arange(t) for n, t in zip(lens, toks)]).astype(np.uint32)
    call, raw = T.make(rng, lens, toks, kv, group, d, True, **kind)
    assert total == call.keys.shape[0]
    # (64-bit scores of every head would take minutes: the last KV head's)
    cache, segs, queries = T.on_device(call, raw, True)
    got = T.results(call, True, cache, segs, queries)
    took = S.debug_last_cache_kernels()
    assert took & S.CACHE_LAID_OUT and took & S.CACHE_ATTEND4 and took & S.CACHE_ATTEND_WIDE
    for h in (kv - 1,):
        hs = slice(h * group, (h + 1) * group)
        one = Q.Call4(call.keys[:, h:h + 1], call.values[:, h:h + 1], call.q[:, hs], call.segs, call.scale, **{**kind, **({"slopes": kind["slopes"][hs]} if "slopes" in kind else {}),
                                                                                                            **({"row_pos": kind["row_pos"][h:h + 1]} if "row_pos" in kind else {}),
                                                                                                            **({"row_doc": kind["row_doc"][h:h + 1]} if "row_doc" in kind else {})})
        out, lse, out_tol, lse_tol = one.attend(True)
        T.held(got[1][:, hs], lse, lse_tol)
        T.held(got[0][:, hs], out, out_tol)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("kv,group,tokens,lens", [(1, 16, 2, (900,)), (2, 7, 4, (1000, 300)), (8, 4, 10, (1500, 1400)), (1, 32, 1, (5000,)), (8, 4, 7, (4096,) * 12)])
def test_blocks_of_every_number_of_query_rows(bf16, kv, group, tokens, lens):
    rng = np.random.default_rng(tokens)
    T.check(*T.make(rng, lens, tokens, kv, group, 128, bf16), bf16)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("kv,d", [(40, 128), (33, 80), (300, 16), (9, 256)])
def test_more_columns_than_a_block_has_threads(bf16, kv, d):
    rng = np.random.default_rng(kv)
    keys, dk = T.odd_rows(rng, 21, kv, d, bf16, 0)
    vals, dv = T.odd_rows(rng, 21, kv, d, bf16, 0)
    st = T.Stored(30, kv, d)
    S.write_cache4(st.cache, S.make_segments([(3, 25, 0, 21, 0)]), S.KvCache(S.to_device(dk), S.to_device(dv), kv, d, dtype=T.type_of(bf16)), 21)
    out = [S.to_device(np.full((30, kv, d), 7.0, F)) for _ in range(2)]
    S.read_cache4(st.cache, S.make_segments([(7, 21, 0, 0, 0)]), S.KvCache(*out, kv, d, dtype=S.F32))
    for x, rows in ((0, keys), (1, vals)):
        want = Q.quantise(rows, 0)
        for got, w in zip(st.bytes(x), Q.laid_out(*want, fill=0xA5)):
            assert np.array_equal(got[7:28], w) and np.all(got[:7] == 0xA5) and np.all(got[28:] == 0xA5)
        back = out[x].download(F, 30 * kv * d).reshape(30, kv, d)
        assert np.array_equal(back[7:28], Q.values(*want, 0)) and np.all(back[:7] == 7) and np.all(back[28:] == 7)


@pytest.mark.parametrize("tokens", [1, 60])
def test_rows_beyond_four_gigabytes(tokens):
    rng = np.random.default_rng(5)
    kv, group, d, n, first = 2, 2, 128, 200, 4500
    call, raw = T.make(rng, (n,), tokens, kv, group, d, True)
    step = 1 << 20  # bytes from row to row: row 4500 lies 4.7 GB from the first
    codes, scales = S.DeviceBuffer((first + n) * step), S.DeviceBuffer((first + n) * 64)
    cache = S.KvCache4(codes, codes.view(4096, codes.nbytes - 4096), scales, scales.view(32, scales.nbytes - 32), kv, d, code_row_stride=step, code_head_stride=64, scale_row_stride=64,
                       scale_head_stride=8, key_exponent=-3, value_exponent=-4)
    segs = S.make_segments([(first, n, 0, n, 0)])
    rows = S.KvCache(S.to_device(K.as_type(call.keys, True)[1]), S.to_device(K.as_type(call.values, True)[1]), kv, d)
    S.write_cache4(cache, segs, rows, n)  # (what codes stand for comes out as the same codes)
    back = [S.DeviceBuffer(n * kv * d * 4) for _ in range(2)]
    S.read_cache4(cache, segs, S.KvCache(*back, kv, d, dtype=S.F32), S.make_segments([(0, n, 0, 0, 0)]))
    for b, want in zip(back, (call.keys, call.values)):
        assert np.array_equal(b.download(F, n * kv * d).reshape(n, kv, d), want)
    out, lse = S.DeviceBuffer(call.q.size * 2), S.DeviceBuffer(call.q.shape[0] * 16)
    S.attend_cache4(cache, S.make_segments([(first, n, 0, tokens, 0)]), S.CacheQueries(S.to_device(raw[4]), tokens, kv * group, d), out, lse)
    want = call.attend(True)
    T.held(K.from_bf16(out.download(np.uint16, call.q.size)).reshape(call.q.shape), want[0], want[2])


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0 ** 20])
def test_scales_that_are_negative_zero_or_large(bf16, scale):
    # integers in float32 throughout: scores are exact, and of the large ones the first in each row of 64 is alone at the top
    rng = np.random.default_rng(6)
    call, raw = T.make(rng, (300,), 2, 2, 2, 64, bf16, key_exponent=0, value_exponent=0)
    keys = rng.integers(-3, 4, call.keys.shape).astype(F)
    keys[37] = 6.0
    codes, scales = Q.quantise(keys, 0)
    raw[0], raw[2] = Q.laid_out(codes, scales)
    call.keys = Q.values(codes, scales, 0)
    call.q, raw[4] = K.as_type(np.ones(call.q.shape), bf16)
    call.scale = float(F(scale))
    cache, segs, queries = T.on_device(call, raw, bf16)
    got = T.results(call, bf16, cache, segs, queries)
    if scale < 1:
        want = call.attend(bf16)
        T.held(got[0], want[0], want[2])
        T.held(got[1], want[1], want[3])
    else:
        # scores of 2^20 * 384 = 2^28.6, the next a hundred times 2^20 below: all the weight is row 37's
        assert np.array_equal(got[0], np.broadcast_to(call.values[37].repeat(2, 0), got[0].shape))
        assert np.allclose(got[1], 384 * 2.0 ** 20, rtol=2.0 ** -22)


@pytest.mark.parametrize("bf16", [True, False])
def test_tokens_that_see_nothing_but_nan(bf16):
    rng = np.random.default_rng(7)
    call, raw = T.make(rng, (1, 40), 1, 1, 2, 64, bf16)
    want = call.attend(bf16)
    raw[2][0, 0, 2] = 0x7F  # the only row of the first segment
    got = T.results(call, bf16, *T.on_device(call, raw, bf16))
    assert np.isnan(got[0][0]).all() and np.isnan(got[1][0]).all()
    T.held(got[0][1], want[0][1], want[2][1])


def test_graphs_with_parts_and_rows_laid_out_beside_eager_calls_and_on_other_streams():
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(8)
    calls = [T.make(rng, (20000,), 1, 8, 4, 128, True), T.make(rng, (9000, 12000), 1, 8, 4, 128, True), T.make(rng, (1400, 1500), 1200, 8, 4, 64, True)]
    sets = [T.on_device(c, raw, True) for c, raw in calls]
    want = [T.results(c, True, *s) for (c, _), s in zip(calls, sets)]
    streams = [torch.cuda.Stream() for _ in calls]
    outs = [(S.DeviceBuffer(c.q.size * 2), S.DeviceBuffer(c.q.shape[0] * c.heads * 4)) for c, _ in calls]
    graphs = []
    try:
        for (cache, segs, queries), o, stream in zip(sets, outs, streams):
            S.set_stream(stream.cuda_stream)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                S.attend_cache4(cache, segs, queries, *o)
            graphs.append(g)
        for round_ in range(3):
            for (c, _), o in zip(calls, outs):
                o[0].upload(np.zeros(c.q.size, np.uint16))
            for g, stream in zip(graphs, streams):  # all at once
                with torch.cuda.stream(stream):
                    g.replay()
            S.set_stream(streams[round_].cuda_stream)
            eager = (S.DeviceBuffer(calls[0][0].q.size * 2), S.DeviceBuffer(4 * 32))
            S.attend_cache4(*sets[0], *eager)
            torch.cuda.synchronize()
            for (c, _), o, w in zip(calls, outs, want):
                assert np.array_equal(K.from_bf16(o[0].download(np.uint16, c.q.size)).reshape(c.q.shape), w[0])
                assert np.array_equal(o[1].download(F, c.q.shape[0] * c.heads).reshape(c.q.shape[:2]), w[1])
            assert np.array_equal(K.from_bf16(eager[0].download(np.uint16, calls[0][0].q.size)).reshape(calls[0][0].q.shape), want[0][0])
    finally:
        S.set_stream(None)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("tokens,window,docs", [(1, 1, False), (1, 300, False), (3, 300, True), (40, 1000, False), (40, 5000, True)])
def test_windows_that_leave_most_rows_behind(bf16, tokens, window, docs):
    rng = np.random.default_rng(window)
    lens, kv, group = (4000, 1200, 50), 2, 4
    kind = {}
    if docs:
        doc = np.concatenate([np.sort(rng.integers(1, 4, n)) for n in lens]).astype(np.uint32)
        kind = dict(row_doc=np.stack([doc] * kv), q_doc=np.concatenate([doc[e - tokens:e] for e in np.cumsum(lens)]))
    call, raw = T.make(rng, lens, tokens, kv, group, 64, bf16, window=window, bases=(7, 0, 1 << 31), **kind)
    want = call.attend(bf16)
    for b, n in ((0, 4000), (4000, 1200)):
        behind = max(0, n - tokens - window + 1)
        for x in (2, 3):
            raw[x][b:b + behind] = 0x7F
    got = T.results(call, bf16, *T.on_device(call, raw, bf16))
    T.held(got[1], want[1], want[3])
    T.held(got[0], want[0], want[2])
    call.rows = np.array(lens, np.uint32)  # the same with counts that the host does not look at
    got = T.results(call, bf16, *T.on_device(call, raw, bf16))
    T.held(got[1], want[1], want[3])
    T.held(got[0], want[0], want[2])


def test_many_tokens_of_segments_without_rows():
    rng = np.random.default_rng(11)
    for lens in ((0,), (0, 0, 300)):
        call, raw = T.make(rng, lens, 1200 if len(lens) == 1 else (900, 0, 250), 2, 8, 64, True)
        out, lse = T.results(call, True, *T.on_device(call, raw, True))
        n = 1200 if len(lens) == 1 else 900
        assert np.all(out[:n] == 0) and np.all(lse[:n] == -np.inf)
        if len(lens) > 1:
            want = call.attend(True)
            T.held(out[n:], want[0][n:], want[2][n:])


def test_two_threads_at_once():
    rng = np.random.default_rng(9)
    calls = [T.make(rng, (3000 + 500 * i, 700), (1, 9), 4, 4, 128, True) for i in range(2)]
    sets = [T.on_device(c, raw, True) for c, raw in calls]
    want = [T.results(c, True, *s) for (c, _), s in zip(calls, sets)]
    wrong = []

    def work(i):
        for _ in range(20):
            got = T.results(calls[i][0], True, *sets[i])
            if not (np.array_equal(got[0], want[i][0]) and np.array_equal(got[1], want[i][1])):
                wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_host_arrays_are_refused_under_capture_and_device_arrays_of_the_host():
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(10)
    call, raw = T.make(rng, (100,), 1, 2, 2, 64, True)
    cache, segs, queries = T.on_device(call, raw, True)
    for i in range(4):
        host = [S.to_device(x) for x in raw[:4]]
        host[i] = raw[i]
        with pytest.raises(S.SlhaError) as e:
            S.attend_cache4(S.KvCache4(*host, 2, 64), segs, queries, S.DeviceBuffer(1024), None)
        assert e.value.code == S.ERR_DEVICE and "device memory" in e.value.message
    stream = torch.cuda.Stream()
    S.set_stream(stream.cuda_stream)
    try:
        rows = S.KvCache4(*(S.to_device(x) for x in raw[:4]), 2, 64, rows=np.array([90], np.uint32))
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(Exception):
            with torch.cuda.graph(graph, stream=stream):
                S.attend_cache4(rows, segs, queries, S.DeviceBuffer(1024), None)
    finally:
        S.set_stream(None)
    torch.cuda.synchronize()
    T.check(call, raw, True)
