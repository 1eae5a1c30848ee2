"""The calls on a cache of rows where a caller goes to the edge of what they allow: captured behind calls of any size, arrays that are written again at once, positions
far apart, memory beside a call's own, values that are not finite, long caches.  Plain forms and bounds as in tests/cache_cases.py."""
import ctypes as C

import numpy as np
import pytest

from tests import cache_cases as K
from tests import helpers as H
from tests import test_gpu_cache as T
from tests.test_gpu_streams import Streams

pytestmark = pytest.mark.gpu
S = pytest.importorskip("slhav2_b200")
F = np.float32


def in_a_thread(work):
    """The library's working memory belongs to the thread: a new one begins without any."""
    import threading

    bad = []

    def run():
        try:
            work()
        except BaseException as e:  # noqa: BLE001
            bad.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    if bad:
        raise bad[0]


def chunk_with_large_parts(rng):
    """64 tokens over 20000 rows in parts of more than the 8 MB that a thread's working memory begins with."""
    call, raw = T.make(rng, (20000,), 64, 2, 4, 128, True, causal=True)
    cache, segs, queries = T.on_device(call, raw, True)
    out = S.DeviceBuffer(call.q.size * 2)
    return lambda: S.attend_cache(cache, segs, queries, out)


# ---- graphs
def test_a_call_is_captured_behind_calls_that_chained_working_memory():
    # a small call, one whose parts do not fit beside it, then a capture: nothing is waited for or given back under it
    rng = np.random.default_rng(1)
    call, raw = T.make(rng, (20000,), 1, 2, 4, 128, True)
    handles = T.on_device(call, raw, True)
    out, lse = S.DeviceBuffer(call.q.size * 2), S.DeviceBuffer(call.q.size * 4)
    large = chunk_with_large_parts(rng)
    want = call.attend(True)
    S.synchronize()

    def work():
        with Streams(1) as st:
            rt, graph, exe = st.rt, C.c_void_p(), C.c_void_p()
            S.set_stream(st.all[0].value)
            S.attend_cache(*handles, out, lse)
            large()
            out.upload(np.zeros(call.q.size, np.uint16))
            assert rt.cudaStreamBeginCapture(st.all[0], 0) == 0
            S.attend_cache(*handles, out, lse)
            assert rt.cudaStreamEndCapture(st.all[0], C.byref(graph)) == 0
            assert rt.cudaGraphInstantiate(C.byref(exe), graph, C.c_ulonglong(0)) == 0
            for _ in range(2):
                large()
                assert rt.cudaGraphLaunch(exe, st.all[0]) == 0
            S.synchronize()
            T.held(K.from_bf16(out.download(np.uint16, call.q.size)).reshape(call.q.shape), want[0], want[2])
            rt.cudaGraphExecDestroy(exe)
            rt.cudaGraphDestroy(graph)

    in_a_thread(work)


def test_working_memory_that_a_graph_names_stays():
    # the pool's question is captured with memory of the thread; calls that chain more of it, and put the chain together, come before the graph runs
    rng = np.random.default_rng(2)
    large = chunk_with_large_parts(rng)
    gm = S.Model.from_projection(H.make_model_pair(128, seed=61)[1], 128, 61)
    pools = [S.TilePool(3000, 2**40) for _ in range(2)]
    for p in pools:
        p.append_keys(gm, H.gaussian_keys(65, 3000, 128), S.CODEC_MIXED)
    qc, qs = H.random_queries(1, 12)
    dq, ds = S.to_device(qc), S.to_device(qs)
    S.synchronize()

    def work():
        with Streams(1) as st:
            rt, graph, exe = st.rt, C.c_void_p(), C.c_void_p()
            S.set_stream(st.all[0].value)
            pools[1].observe_query(dq, ds, 3.0)
            assert rt.cudaStreamBeginCapture(st.all[0], 2) == 0
            pools[0].observe_query(dq, ds, 3.0)
            assert rt.cudaStreamEndCapture(st.all[0], C.byref(graph)) == 0
            assert rt.cudaGraphInstantiate(C.byref(exe), graph, C.c_ulonglong(0)) == 0
            for _ in range(2):
                large()
                assert rt.cudaGraphLaunch(exe, st.all[0]) == 0
                pools[1].observe_query(dq, ds, 3.0)
            assert rt.cudaGraphLaunch(exe, st.all[0]) == 0
            S.synchronize()
            rt.cudaGraphExecDestroy(exe)
            rt.cudaGraphDestroy(graph)

    in_a_thread(work)
    assert pools[0].read()[2].tobytes() == pools[1].read()[2].tobytes()



# ---- arrays in host memory
def test_short_arrays_may_be_written_again_once_a_call_has_returned():
    # page-locked ones too, while the call's stream is still busy with what came before
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(3)
    t, lens = 40, (300, 200)
    parents = np.concatenate([T.tree(rng, "random", t) for _ in lens])
    call, raw = T.make(rng, lens, t, 2, 2, 64, True, parents=parents)
    call.rows = np.array([250, 200], np.uint32)
    call.slopes, call.prefix = np.array([0.5, 0.25, 0.125, 0.0], F), np.array([10, 0], np.uint32)
    call.q_pos = rng.integers(150, 260, 2 * t).astype(np.uint32)
    want = call.attend(True)
    pin = lambda x: torch.from_numpy(x.view(np.int32) if x.dtype == np.uint32 else x).pin_memory()  # noqa: E731
    p, rows, slopes, prefix, q_pos = (pin(x) for x in (parents, call.rows, call.slopes, call.prefix, call.q_pos))
    cache = S.KvCache(S.to_device(raw[0]), S.to_device(raw[1]), 2, 64, rows=rows)
    queries = S.CacheQueries(S.to_device(raw[2]), 2 * t, 4, 64, scale=call.scale, slopes=slopes, prefix=prefix, positions=q_pos)
    out, lse = S.DeviceBuffer(call.q.size * 2), S.DeviceBuffer(2 * t * 4 * 4)
    st = torch.cuda.Stream()
    busy = torch.zeros(8192, 8192, device="cuda")
    torch.cuda.synchronize()
    try:
        S.set_stream(st.cuda_stream)
        S.attend_tree(cache, S.make_segments(call.segs), queries, p, out, lse)  # (what a first call does only once)
        with torch.cuda.stream(st):
            for _ in range(20):
                busy @ busy
        S.attend_tree(cache, S.make_segments(call.segs), queries, p, out, lse)
        for x in (p, rows, slopes, prefix, q_pos):
            x.zero_()
        torch.cuda.synchronize()
    finally:
        S.set_stream(None)
    T.held(K.from_bf16(out.download(np.uint16, call.q.size)).reshape(call.q.shape), want[0], want[2])
    T.held(lse.download(F, 2 * t * 4).reshape(2 * t, 4), want[1], want[3])



# ---- positions far apart
@pytest.mark.parametrize("tokens,group,d", [(1, 4, 64), (40, 4, 64), (40, 4, 128), (70, 1, 64), (3, 4, 64)])
@pytest.mark.parametrize("moved", [True, False])
@pytest.mark.parametrize("softcap", [0.0, 8.0])
def test_distances_between_positions_that_are_far_from_the_first_token_s(tokens, group, d, moved, softcap):
    # tokens near 1000 and near 2^31 in one block: a distance is the difference of two positions, however far both are from the block's first token
    rng = np.random.default_rng(tokens + d)
    n, kv, far = 500, 2, 2 ** 31
    if moved:
        row_pos = np.stack([rng.permutation(np.concatenate([np.arange(800, 1050), far - 100 + np.arange(250)])) for _ in range(kv)]).astype(np.uint32)
        base = 0
    else:
        row_pos, base = None, far - 100
    near = 1000 + np.arange((tokens + 1) // 2)
    q_pos = np.concatenate([near, far + 60 + 2 * np.arange(tokens - len(near))]).astype(np.uint32)
    slopes = (0.6 * 2.0 ** -np.arange(kv * group)).astype(F)
    call, raw = T.make(rng, (n,), tokens, kv, group, d, True, bases=[base], row_pos=row_pos, q_pos=q_pos, slopes=slopes, window=300, causal=False, softcap=softcap)
    _, lse = T.check(call, raw, True)
    cache, segs, queries = T.on_device(call, raw, True)
    w = S.to_device(np.zeros((kv, n), F))
    S.observe_cache(cache, segs, queries, S.to_device(lse), w, n)
    want, tol = call.received(lse, np.zeros((kv, n), F), 1.0)
    T.held(w.download(F, kv * n).reshape(kv, n), want, tol)



# ---- memory beside a call's own
@pytest.mark.parametrize("tokens,group,d", [(33, 1, 64), (100, 1, 128), (37, 8, 128), (9, 4, 64), (131, 4, 64)])
@pytest.mark.parametrize("more", [dict(), dict(softcap=6.0), dict(alibi=True), dict(softcap=6.0, alibi=True, window=90)])
def test_equal_inputs_give_equal_bits_whatever_lies_behind_the_queries(tokens, group, d, more):
    rng = np.random.default_rng(tokens)
    kind = {k: v for k, v in more.items() if k != "alibi"}
    if more.get("alibi"):
        kind["slopes"] = (2.0 ** -np.arange(1, 2 * group + 1)).astype(F)
    call, raw = T.make(rng, (700, 10), (tokens, 40), 2, group, d, True, **kind)
    call.segs = call.segs[:1]
    grow = np.linspace(0.1, 2.0, 710)[:, None, None]
    call.keys, raw = K.as_type(call.keys * grow, True)[0], (K.as_type(call.keys * grow, True)[1], raw[1], raw[2].copy())
    before = None
    for other in (0.0, 1.0, 300.0, -3e4, np.nan, np.inf):
        raw[2][tokens:] = K.as_type(np.full(raw[2][tokens:].shape, other), True)[1]
        handles = T.on_device(call, raw, True)
        o, z = T.results(call, True, *handles)
        w = S.to_device(np.zeros((2, 710), F))
        S.observe_cache(handles[0], handles[1], handles[2], S.to_device(z), w, 710)
        now = o[:tokens].tobytes(), z[:tokens].tobytes(), w.download(F, 1420).tobytes()
        assert before in (None, now), other
        before = now



# ---- values that are not finite
def odd_call(rng, lens, tokens, kv, group, d, at, **kind):
    """A call whose values hold infinities and NaN at (row, dimension, value), and its result by the definition: what a token sees counts, nothing else."""
    call, raw = T.make(rng, lens, tokens, kv, group, d, True, **kind)
    for row, dim, x in at:
        raw[1][row, :, dim] = K.as_type(np.full(kv, x), True)[1]
        call.values[row, :, dim] = x
    return call, raw


def held_odd(got, want, tol):
    want = np.where(np.isnan(want), np.nan, want)
    with np.errstate(invalid="ignore"):
        same = (got == want) | (np.abs(got - want) <= tol) | (np.isnan(got) & np.isnan(want))
    assert same.all(), (int((~same).sum()), np.argwhere(~same)[:4], got[~same][:4], want[~same][:4])


@pytest.mark.parametrize("kind", ["causal", "window", "docs", "moved", "tree", "prefix", "split", "strided"])
@pytest.mark.parametrize("tokens,group,d", [(300, 1, 128), (70, 4, 64), (40, 4, 80), (33, 8, 128), (256, 1, 128)])
@pytest.mark.parametrize("softcap", [0.0, 9.0])
def test_values_that_are_not_finite_reach_those_who_see_them_and_nobody_else(kind, tokens, group, d, softcap):
    rng = np.random.default_rng(tokens + len(kind))
    n, kv = 6000 if kind == "split" else 900, 2
    more = dict(softcap=softcap)
    first = n - tokens
    # before all tokens, beside each other in one tile, among the tokens' own rows; one column with both infinities, one with NaN
    at = [(5, 1, np.inf), (first - 3, 2, -np.inf), (first - 2, 2, np.inf), (first + 2, 3, np.inf), (first + tokens // 2, 3, -np.inf), (first + 9, d - 1, np.nan), (n - 1, 4, -np.inf),
          (n - 2, 0, np.inf)]
    if kind == "window":
        more["window"] = 150
    if kind == "prefix":
        more["prefix"], more["window"] = np.array([40], np.uint32), 30
    if kind == "docs":
        doc = rng.integers(0, 3, n).astype(np.uint32)
        doc[first:] = rng.integers(0, 2, tokens)
        more["row_doc"], more["q_doc"] = np.stack([doc] * kv), doc[first:]
        at += [(int(r), 6, np.inf) for r in np.flatnonzero(doc == 2)[::7]]
    if kind == "moved":
        pos = np.stack([rng.permutation(2 * n)[:n] for _ in range(kv)]).astype(np.uint32)
        more["row_pos"], more["q_pos"] = pos, rng.integers(0, 2 * n, tokens).astype(np.uint32)
    if kind == "tree":
        if tokens > 256:
            tokens, first = 256, n - 256
        more["parents"] = T.tree(rng, "random", tokens)
    call, raw = odd_call(rng, (n,), tokens, kv, group, d, at, **more)
    if kind == "strided":  # queries and outputs [head][token]: not in boxes
        heads = kv * group
        q = np.ascontiguousarray(raw[2].transpose(1, 0, 2))
        cache = S.KvCache(S.to_device(raw[0]), S.to_device(raw[1]), kv, d)
        queries = S.CacheQueries(S.to_device(q), tokens, heads, d, softcap=softcap, token_stride=d, head_stride=tokens * d)
        out, dl = S.DeviceBuffer(call.q.size * 2), S.DeviceBuffer(tokens * heads * 4)
        S.attend_cache(cache, S.make_segments(call.segs), queries, out, dl, out_token_stride=d, out_head_stride=tokens * d)
        o = K.from_bf16(out.download(np.uint16, call.q.size)).reshape(heads, tokens, d).transpose(1, 0, 2)
        lse = dl.download(F, tokens * heads).reshape(tokens, heads)
    else:
        o, lse = T.results(call, True, *T.on_device(call, raw, True))
    with np.errstate(invalid="ignore"):
        want = call.attend(True)
    T.held(lse, want[1], want[3])
    held_odd(o, want[0], want[2])
    assert not np.isfinite(want[0]).all() and np.isfinite(want[0]).any()


def test_hidden_rows_of_any_content_cost_little():
    # a hole in every tile of 32768 rows, whose keys and values are NaN: as quick as finite ones but for looking them over
    torch = pytest.importorskip("torch")
    n, kv, group, d, tokens = 32768, 2, 4, 128, 64
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(n, kv, d, device="cuda", generator=g).bfloat16() for _ in range(2))
    q = torch.randn(tokens, kv * group, d, device="cuda", generator=g).bfloat16()
    doc = torch.ones(n, dtype=torch.int32, device="cuda")
    doc[17:n - tokens:64] = 7
    q_doc = torch.ones(tokens, dtype=torch.int32, device="cuda")
    segs = S.make_segments([(0, n, 0, tokens, 0)])
    took, outs = [], []
    for fill in (0.0, float("nan")):
        k[doc == 7] = fill
        v[doc == 7] = fill
        out = torch.empty_like(q)
        cache = S.KvCache(k, v, kv, d, documents=doc)
        queries = S.CacheQueries(q, tokens, kv * group, d, documents=q_doc)
        torch.cuda.synchronize()
        st = torch.cuda.Stream()
        try:
            S.set_stream(st.cuda_stream)
            for _ in range(3):
                S.attend_cache(cache, segs, queries, out)
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record(st)
            for _ in range(5):
                S.attend_cache(cache, segs, queries, out)
            end.record(st)
            torch.cuda.synchronize()
        finally:
            S.set_stream(None)
        took.append(begin.elapsed_time(end) / 5)
        outs.append(out.float().cpu())
    assert took[1] < 8 * took[0] + 0.1, took
    assert torch.equal(outs[0], outs[1])



# ---- long caches
def test_rows_of_more_than_one_run_keep_to_their_working_memory():
    # 140000 rows take two runs a block; 32768 tokens' parts at once would be 1.1 GB
    torch = pytest.importorskip("torch")
    n, kv, group, d, tokens = 140000, 8, 4, 128, 32768
    g = torch.Generator(device="cuda").manual_seed(6)
    k, v = (torch.randn(n, kv, d, device="cuda", generator=g).bfloat16() for _ in range(2))
    q = torch.randn(tokens, kv * group, d, device="cuda", generator=g).bfloat16()
    segs = S.make_segments([(0, n, 0, tokens, 0)])
    cache = S.KvCache(k, v, kv, d)
    outs, lses = [], []
    grown = []
    torch.cuda.synchronize()
    S.attend_cache(cache, S.make_segments([(0, n, 0, 64, 0)]), S.CacheQueries(q, tokens, kv * group, d), torch.empty_like(q), torch.empty(tokens, kv * group, device="cuda"))  # (loads the kernels)

    def work():
        for prefix in (None, torch.zeros(1, dtype=torch.int32, device="cuda")):  # (a prefix of nothing: the same rows are seen, but the runs are made for all)
            out, lse = torch.full_like(q, 7.0), torch.zeros(tokens, kv * group, device="cuda")
            queries = S.CacheQueries(q, tokens, kv * group, d, window=200, prefix=prefix)
            torch.cuda.synchronize()
            before = torch.cuda.mem_get_info()[0]
            S.attend_cache(cache, segs, queries, out, lse)
            grown.append(before - torch.cuda.mem_get_info()[0])
            outs.append(out)
            lses.append(lse)

    in_a_thread(work)
    assert grown[0] <= 16 << 20 and grown[1] <= 600 << 20, grown
    assert float((lses[0] - lses[1]).abs().max()) <= 2e-5
    assert float((outs[0].float() - outs[1].float()).abs().max()) <= 2.0 ** -6 * float(v.float().abs().max())



def test_working_memory_is_given_back_when_its_thread_ends():
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(7)
    large = chunk_with_large_parts(rng)  # (some 14 MB beside the first 8)
    stream = torch.cuda.Stream()

    def work():
        S.set_stream(stream.cuda_stream)
        for _ in range(3):
            large()

    in_a_thread(work)
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    for _ in range(8):
        in_a_thread(work)
    torch.cuda.synchronize()
    assert before - torch.cuda.mem_get_info()[0] <= 32 << 20


# ---- kernels that only long caches reach
@pytest.mark.parametrize("tokens,group,d,lens,name", [(16, 4, 128, (10000,), "MID"), (40, 4, 128, (10000,), "MID"), (64, 4, 128, (9990,), "MID"), (100, 4, 128, (10000,), "MANY"),
                                                      (64, 8, 80, (9000, 700), "MANY"), (1, 4, 128, (20000, 77), "MID"), (8, 4, 128, (19990, 130), "MID"), (16, 4, 80, (10000,), "MID"),
                                                      (1, 4, 128, (9000, 4100, 7000, 2900, 5200, 3300), "FEW"), (4, 4, 80, (9000, 4100, 7000, 2900, 5200, 3300), "FEW"),
                                                      (12, 4, 64, (10000,), "MID"), (128, 4, 64, (10000,), "MANY"), (1, 4, 64, (9000, 4100, 7000, 2900, 5200, 3300), "FEW")])
@pytest.mark.parametrize("more", [dict(), dict(softcap=5.0, alibi=True), dict(docs=True), dict(window=3000)])
def test_weights_of_rows_by_every_kernel_in_runs_longer_than_its_ring(tokens, group, d, lens, name, more):
    rng = np.random.default_rng(tokens * 7 + group + d)
    kv, total = 8, sum(lens)
    kind = {k: v for k, v in more.items() if k in ("softcap", "window")}
    if more.get("alibi"):
        kind["slopes"] = (2.0 ** -np.arange(1, kv * group + 1) / 64).astype(F)
    if more.get("docs"):
        doc = np.sort(rng.integers(1, 4, total)).astype(np.uint32)
        kind["row_doc"] = np.stack([doc] * kv)
        kind["q_doc"] = rng.integers(1, 5, tokens * len(lens)).astype(np.uint32)
    call, raw = T.make(rng, lens, tokens, kv, group, d, True, **kind)
    cache, segs, queries = T.on_device(call, raw, True)
    _, lse = T.results(call, True, cache, segs, queries)
    before = rng.random((kv, total)).astype(F)
    w = S.to_device(before)
    S.observe_cache(cache, segs, queries, S.to_device(lse), w, total, weights_in=w, decay=0.5)
    assert S.debug_last_cache_kernels() == getattr(S, "CACHE_OBSERVE_" + name)
    want, tol = call.received(lse, before, 0.5)
    T.held(w.download(F, kv * total).reshape(kv, total), want, tol)


@pytest.mark.parametrize("n_kv,n,budget,ctas", [(3, 20001, 20000, 4), (2, 16384, 90, 4), (13, 70000, 600, 4), (25, 16500, 500, 2), (1, 65536, 65535, 8), (3, 131072, 70000, 8), (1, 500000, 3000, 8), (40, 9000, 100, 1)])
@pytest.mark.parametrize("recent", [0, 700])
def test_removal_by_clusters_from_rows_that_have_moved(n_kv, n, budget, ctas, recent):
    # each head's newest row lies in another CTA's share; the second segment's rows begin elsewhere
    rng = np.random.default_rng(n)
    lens, total = (n, n // 3), n + n // 3
    pos = np.zeros((n_kv, total), np.uint32)
    w = rng.integers(0, 50, (n_kv, total)).astype(F)
    for h in range(n_kv):
        b = 0
        for m in lens:
            p = rng.permutation(2 * m)[:m]
            top = int(p.argmax())
            to = (h * 2 + 1) * m // (2 * n_kv)
            p[top], p[to] = p[to], p[top]
            pos[h, b:b + m] = p
            b += m
    k = rng.integers(0, 65536, (total, n_kv, 8)).astype(np.uint16)
    cache = S.KvCache(S.to_device(k), S.to_device(k), n_kv, 8, positions=S.to_device(pos), entry_head_stride=total)
    src = S.DeviceBuffer(2 * 4 * n_kv * budget)
    keep = S.KvCache(S.DeviceBuffer(2 * budget * n_kv * 16), S.DeviceBuffer(2 * budget * n_kv * 16), n_kv, 8)
    S.evict_cache(cache, S.make_segments([(0, n, 0, 0, 0), (n, n // 3, 0, 0, 0)]), S.to_device(w), total, budget, sink_window=9, recent_window=recent, source_out=src, to=keep,
                  to_segments=S.make_segments([(0, budget, 0, 0, 0), (budget, budget, 0, 0, 0)]))
    assert S.debug_last_cache_kernels() == S.CACHE_SELECT * ctas
    got = src.download(np.uint32, 2 * n_kv * budget).reshape(2, n_kv, budget)
    for h in range(0, n_kv, max(1, n_kv // 4)):
        for i, (b, m) in enumerate(((0, n), (n, n // 3))):
            want = K.evict(w[h, b:b + m], pos[h, b:b + m], budget, 9, recent)
            assert np.array_equal(got[i, h, :len(want)], want)


# ---- sums that the tensor cores cut off
@pytest.mark.parametrize("tokens,d", [(1, 256), (24, 200), (600, 128)])
def test_scores_of_observed_rows_are_not_cut_off_step_by_step(tokens, d):
    # All products are positive, so that a sum taken on the tensor cores loses half a step of 2^-23 of itself with every 16 elements: (1 + .. + 16) / 16 halves of a score of 20 for 256
    # dimensions, 2.5 where four steps are taken at a time and added to the nearest: 20 * 2.5 * 2^-24 = 3.0e-6 of a weight, here with half as much again.
    rng = np.random.default_rng(d)
    n = 1000
    keys, dk = K.as_type(2.0 ** rng.uniform(-5.0, 0.0, (n, 1, d)), True)  # (of several sizes: sums of equally large ones would be exact)
    q, dq = K.as_type(2.0 ** rng.uniform(-5.0, 0.0, (tokens, 1, d)), True)
    scale = float(F(20.0 / np.einsum("tgd,rgd->tr", q, keys).mean()))
    call = K.Call(keys, keys, q, [(0, n, 0, tokens, 0)], scale, causal=False)
    want_lse = call.attend(True)[1].astype(F)
    cache, queries = S.KvCache(S.to_device(dk), None, 1, d), S.CacheQueries(S.to_device(dq), tokens, 1, d, scale=scale, causal=False)
    w = S.to_device(np.zeros(n, F))
    S.observe_cache(cache, S.make_segments(call.segs), queries, S.to_device(want_lse), w, n)
    assert S.debug_last_cache_kernels() == S.CACHE_OBSERVE
    want, _ = call.received(want_lse, np.zeros((1, n), F), 1.0)
    off = w.download(F, n) / want[0] - 1.0
    print(off.mean(), off.std())
    assert abs(off.mean()) <= 20 * 1.5 * 2.5 * 2.0 ** -24


# ---- shapes that fill no box
@pytest.mark.parametrize("tokens,group,kv", [(3, 48, 1), (1, 128, 2), (5, 128, 1), (40, 12, 2), (70, 7, 1)])
@pytest.mark.parametrize("d", [8, 40, 72, 120, 128])
@pytest.mark.parametrize("more", [dict(), dict(softcap=7.0, window=333)])
def test_wide_blocks_of_any_group_and_width(tokens, group, kv, d, more):
    rng = np.random.default_rng(tokens * group + d)
    call, raw = T.make(rng, (900, 77), tokens, kv, group, d, True, **more)
    _, lse = T.check(call, raw, True)
    assert S.debug_last_cache_kernels() == S.CACHE_ATTEND_WIDE
    cache, segs, queries = T.on_device(call, raw, True)
    w = S.to_device(np.zeros((kv, 977), F))
    S.observe_cache(cache, segs, queries, S.to_device(lse), w, 977)
    want, tol = call.received(lse, np.zeros((kv, 977), F), 1.0)
    T.held(w.download(F, kv * 977).reshape(kv, 977), want, tol)


def test_several_sequences_read_the_same_rows():
    # a shared prompt: attention reads it for each; each sequence's tokens see what their own positions allow
    rng = np.random.default_rng(9)
    call, raw = T.make(rng, (600,), 3 * 50, 2, 4, 64, True)
    call.segs = [(0, 600, 0, 50, 0), (0, 600, 50, 50, 0), (100, 400, 100, 50, 100)]
    T.check(call, raw, True)


def test_a_graph_of_a_step_with_large_parts_beside_eager_ones():
    # the graph's working memory is its own: replays on one stream while the thread's next calls run on another
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(10)
    call, raw = T.make(rng, (9000,), 64, 2, 4, 128, True)
    handles = T.on_device(call, raw, True)
    want = call.attend(True)
    a, b = (torch.cuda.Stream() for _ in range(2))
    outs = [torch.empty(call.q.shape, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    S.synchronize()
    torch.cuda.synchronize()
    try:
        S.set_stream(a.cuda_stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=a):
            S.attend_cache(*handles, outs[0])
        S.set_stream(b.cuda_stream)
        for _ in range(10):
            with torch.cuda.stream(a):
                g.replay()
            S.attend_cache(*handles, outs[1])
        torch.cuda.synchronize()
    finally:
        S.set_stream(None)
    for o in outs:
        T.held(o.float().cpu().numpy(), want[0], want[2])
