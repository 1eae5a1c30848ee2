"""A cache in 4 bits that lies [sequence][head][row]: what sequences' tokens write, what is read back and attended to."""
import numpy as np
import pytest

from tests import cache4_cases as Q
from tests import cache_cases as K
from tests import test_gpu_cache4 as T

pytestmark = pytest.mark.gpu
S = pytest.importorskip("slhav2_b200")
F = np.float32


@pytest.mark.parametrize("counted", ["no", "host", "device"])
@pytest.mark.parametrize("tokens", [1, 7])
def test_sequences_that_lie_head_by_head(counted, tokens):
    rng = np.random.default_rng(tokens)
    seqs, kv, group, room, d = 5, 4, 3, 40, 64
    lens = np.array([40, 9, 31, 40, 12]) if counted != "no" else np.full(seqs, room)
    total = seqs * kv * room
    codes = [[rng.integers(0, most, (seqs, kv, room, n)).astype(np.uint8) for n, most in ((d // 2, 256), (4, 80))] for _ in range(2)]
    arrays = [S.to_device(codes[0][0]), S.to_device(codes[1][0]), S.to_device(codes[0][1]), S.to_device(codes[1][1])]
    rows = None if counted == "no" else lens.astype(np.uint32)
    cache = S.KvCache4(*arrays, kv, d, code_row_stride=d // 2, code_head_stride=room * d // 2, scale_row_stride=4, scale_head_stride=room * 4, key_exponent=-3, value_exponent=-3,
                       rows=S.to_device(rows) if counted == "device" else rows)
    segs = S.make_segments([(i * kv * room, room, i * tokens, tokens, 0) for i in range(seqs)])
    k, dk = K.as_type(rng.standard_normal((seqs * tokens, kv, d)), True)
    v, dv = K.as_type(rng.standard_normal((seqs * tokens, kv, d)), True)
    S.write_cache4(cache, segs, S.KvCache(S.to_device(dk), S.to_device(dv), kv, d), seqs * tokens)
    held = []  # [sequence][head][row][d], what the cache should hold now
    for x, new in ((0, k), (1, v)):
        a, b = codes[x][0].copy(), codes[x][1].copy()
        na, nb = Q.laid_out(*Q.quantise(new, -3))
        for i in range(seqs):
            at = slice(int(lens[i]) - tokens, int(lens[i]))
            a[i][:, at], b[i][:, at] = na[i * tokens:(i + 1) * tokens].transpose(1, 0, 2), nb[i * tokens:(i + 1) * tokens].transpose(1, 0, 2)
        assert np.array_equal(arrays[x].download(np.uint8, a.size).reshape(a.shape), a) and np.array_equal(arrays[2 + x].download(np.uint8, b.size).reshape(b.shape), b)
        both = np.stack([a & 15, a >> 4], -1).reshape(seqs, kv, room, d)
        held.append(Q.values(both, b, -3))
    out = [S.to_device(np.full((seqs, kv, room, d), 7.0, F)) for _ in range(2)]
    to = S.KvCache(*out, kv, d, dtype=S.F32, key_row_stride=d, key_head_stride=room * d, value_row_stride=d, value_head_stride=room * d)
    S.read_cache4(cache, segs, to)
    for o, h in zip(out, held):
        got = o.download(F, total * d).reshape(h.shape)
        there = np.arange(room)[None] < lens[:, None]
        assert np.array_equal(got.transpose(0, 2, 1, 3)[there], h.transpose(0, 2, 1, 3)[there]) and np.all(got.transpose(0, 2, 1, 3)[~there] == 7)
    q, dq = K.as_type(rng.standard_normal((seqs * tokens, kv * group, d)), True)
    res = S.DeviceBuffer(q.size * 2)
    S.attend_cache4(cache, segs, S.CacheQueries(S.to_device(dq), seqs * tokens, kv * group, d), res)
    flat = [h.transpose(0, 2, 1, 3).reshape(seqs * room, kv, d) for h in held]
    want = Q.Call4(flat[0], flat[1], q, [(i * room, int(lens[i]), i * tokens, tokens, 0) for i in range(seqs)], float(F(d ** -0.5))).attend(True)
    T.held(K.from_bf16(res.download(np.uint16, q.size)).reshape(q.shape), want[0], want[2])
    # and heads turned into rows that lie so
    key, val = (S.to_device(np.full((seqs, kv, room, d), 0x40E0, np.uint16)) for _ in range(2))
    S.rotate_heads(S.HeadRows(None, S.to_device(dk), S.to_device(dv), seqs * tokens, kv, kv, d), to=S.KvCache(key, val, kv, d, key_row_stride=d, key_head_stride=room * d, value_row_stride=d,
                                                                                                               value_head_stride=room * d, rows=cache.kept[-1]), segments=segs)
    for buf, new in ((key, k), (val, v)):
        got = K.from_bf16(buf.download(np.uint16, total * d)).reshape(seqs, kv, room, d)
        for i in range(seqs):
            at = slice(int(lens[i]) - tokens, int(lens[i]))
            assert np.array_equal(got[i][:, at].transpose(1, 0, 2), new[i * tokens:(i + 1) * tokens])
            got[i][:, at] = 7
        assert np.all(got == 7)
