"""Norms and rotation of heads on their way into a cache (slha_b200_rotate_heads) against a plain form in 64 bits; the bounds are those of tests/cache4_cases.py."""
import numpy as np
import pytest

from tests import cache4_cases as Q
from tests import cache_cases as K

pytestmark = pytest.mark.gpu
S = pytest.importorskip("slhav2_b200")
F = np.float32


class Heads:
    """Tokens' heads in one array [token][n_heads + 2 n_kv][d], as a projection leaves them, and what is asked for."""

    def __init__(self, seed, n, heads, kv, d, bf16, norm=True, weights=True, rotary=None, interleaved=False, axes=1, far=0, magnitude=1.0, eps=1e-6, gap=0):
        rng = np.random.default_rng(seed)
        self.n, self.heads, self.kv, self.d, self.bf16, self.norm, self.eps, self.interleaved, self.magnitude, self.axes = n, heads, kv, d, bf16, norm, eps, interleaved, magnitude, axes
        self.width = (heads + 2 * kv) * d + gap
        self.x, self.raw = K.as_type(rng.standard_normal((n, self.width)) * np.exp(rng.standard_normal(self.width)), bf16)
        at = lambda a, b: self.x[:, a * d:b * d].reshape(n, b - a, d)  # noqa: E731
        self.q, self.k, self.v = at(0, heads), at(heads, heads + kv), at(heads + kv, heads + 2 * kv)
        self.qw, self.kw = ((1 + 0.3 * rng.standard_normal(d)).astype(F) if norm and weights else None for _ in range(2))
        self.rotary = d if rotary is None else rotary
        self.freq = (10000.0 ** (-np.arange(self.rotary // 2) / max(1, self.rotary // 2))).astype(F)
        self.pos = (far + rng.integers(0, 5000, (axes, n))).astype(np.uint32)
        self.of_pair = rng.integers(0, axes, self.rotary // 2).astype(np.uint8) if axes > 1 else None
        self.dtype = S.BF16 if bf16 else S.F32
        self.dev = S.to_device(self.raw)
        self.np = np.uint16 if bf16 else F

    def rows(self, parts="qkv", dev=None):
        dev, e = dev or self.dev, 2 if self.bf16 else 4
        at = {p: dev.data_ptr() + o * self.d * e for p, o in zip("qkv", (0, self.heads, self.heads + self.kv))}
        return S.HeadRows(*(at[p] if p in parts else None for p in "qkv"), self.n, self.heads, self.kv, self.d, dtype=self.dtype, token_stride=self.width, head_stride=self.d,
                          norm=self.norm, eps=self.eps, q_weight=self.qw, k_weight=self.kw)

    def rotation(self):
        return S.Rotation(self.freq, self.pos, self.rotary, n_axes=self.axes, axes=self.of_pair, interleaved=self.interleaved, magnitude=self.magnitude) if self.rotary else None

    def want(self):
        of = lambda x, w: Q.rotate(x, self.norm, w, self.eps, self.freq, self.pos, self.of_pair, self.rotary, self.interleaved, float(F(self.magnitude)), self.bf16)  # noqa: E731
        return of(self.q, self.qw), of(self.k, self.kw)

    def filled(self, *shape):
        return S.to_device(np.full(shape, 0x40E0 if self.bf16 else 7.0, self.np))

    def values(self, dev, *shape):
        x = dev.download(self.np, int(np.prod(shape)))
        return (K.from_bf16(x) if self.bf16 else x).reshape(shape)


def near(got, want):
    y, tol = want
    bad = ~(np.abs(got - y) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3], got[bad][:3], y[bad][:3], tol[bad][:3])


def run_rows(h, total=None):
    """Without segments: queries, keys and values [token]."""
    out, keys, vals = h.filled(h.n, h.heads, h.d), h.filled(h.n, h.kv, h.d), h.filled(h.n, h.kv, h.d)
    S.rotate_heads(h.rows(), h.rotation(), q_out=out, to=S.KvCache(keys, vals, h.kv, h.d, dtype=h.dtype))
    return h.values(out, h.n, h.heads, h.d), h.values(keys, h.n, h.kv, h.d), h.values(vals, h.n, h.kv, h.d)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("d,rotary", [(8, 8), (16, 8), (64, 64), (72, 40), (80, 80), (96, 64), (128, 128), (128, 32), (136, 136), (256, 256), (256, 64), (64, 0)])
@pytest.mark.parametrize("interleaved,norm", [(False, True), (True, False), (True, True)])
def test_heads_of_every_type_and_width(bf16, d, rotary, interleaved, norm):
    h = Heads(d + rotary, 5, 6, 2, d, bf16, norm=norm, rotary=rotary, interleaved=interleaved)
    q, k, v = run_rows(h)
    wq, wk = h.want()
    near(q, wq)
    near(k, wk)
    assert np.array_equal(v, h.v)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("heads,kv,n", [(1, 1, 1), (32, 8, 1), (7, 1, 33), (40, 8, 130), (3, 3, 1000)])
def test_numbers_of_heads_and_tokens(bf16, heads, kv, n):
    h = Heads(heads * n, n, heads, kv, 64, bf16, gap=16)
    q, k, v = run_rows(h)
    wq, wk = h.want()
    near(q, wq)
    near(k, wk)
    assert np.array_equal(v, h.v)


@pytest.mark.parametrize("axes", [2, 3, 4, 7])
@pytest.mark.parametrize("far", [0, 1 << 20, (1 << 32) - 5000])
def test_axes_and_far_positions(axes, far):
    h = Heads(axes, 9, 4, 2, 128, False, axes=axes, far=far, magnitude=1.25, weights=False, eps=1e-2)
    q, k, _ = run_rows(h)
    wq, wk = h.want()
    near(q, wq)
    near(k, wk)


def test_the_rotation_turns_as_its_inverse_and_its_differences_say():
    # scores of turned heads depend on the distance of their positions alone
    h = Heads(3, 2, 1, 1, 64, False, norm=False)
    h.x[:] = h.x[:1]
    h.dev, h.q, h.k = S.to_device(h.x), h.x[:, :64].reshape(2, 1, 64), h.x[:, 64:128].reshape(2, 1, 64)
    got = []
    for p in (5, 1005, 4000000):
        h.pos = np.array([[p, p + 17]], np.uint32)
        q, k, _ = run_rows(h)
        got.append(float(q[1, 0].astype(np.float64) @ k[0, 0]))
    # each element is off by (|a| + |b|) (2 pi 2^-24 + 8 2^-24), a head by sqrt(2) of that of its length; two heads, two scores
    size = float(np.linalg.norm(h.q[0, 0].astype(np.float64)) * np.linalg.norm(h.k[0, 0].astype(np.float64)))
    assert max(got) - min(got) <= 6 * size * (2 * np.pi * 2.0 ** -24 + 8 * K.EPS_F32) and size > 0


@pytest.mark.parametrize("bf16", [True, False])
def test_tokens_go_to_their_segments_rows_and_nothing_else_is_written(bf16):
    h = Heads(4, 12, 4, 2, 64, bf16)
    segs = [(30, 10, 1, 3, 0), (0, 5, 6, 4, 0), (10, 4, 4, 0, 0), (50, 3, 10, 2, 0)]  # tokens 0, 4 and 5 belong to none
    counts = np.array([7, 9, 4, 1], np.uint32)  # fewer rows than the table says, more, fewer than tokens
    for rows in (None, counts, S.to_device(counts)):
        total = 60
        out, keys, vals = h.filled(12, 4, 64), h.filled(total, 2, 64), h.filled(total, 2, 64)
        S.rotate_heads(h.rows(), h.rotation(), q_out=out, to=S.KvCache(keys, vals, 2, 64, dtype=h.dtype, rows=rows), segments=S.make_segments(segs))
        wq, wk = h.want()
        q, k, v = h.values(out, 12, 4, 64), h.values(keys, total, 2, 64), h.values(vals, total, 2, 64)
        written, tokens = np.zeros(total, bool), np.zeros(12, bool)
        for i, (b, n, q0, t, _) in enumerate(segs):
            n = n if rows is None else min(n, int(counts[i]))
            ctx = n - min(n, t)
            for j in range(t):
                tokens[q0 + j] = True
                near(q[q0 + j], (wq[0][q0 + j], wq[1][q0 + j]))
                if ctx + j < n:
                    written[b + ctx + j] = True
                    near(k[b + ctx + j], (wk[0][q0 + j], wk[1][q0 + j]))
                    assert np.array_equal(v[b + ctx + j], h.v[q0 + j])
        assert np.all(q[~tokens] == 7) and np.all(k[~written] == 7) and np.all(v[~written] == 7)


@pytest.mark.parametrize("bf16", [True, False])
def test_layouts_parts_and_heads_turned_in_place(bf16):
    h = Heads(5, 10, 4, 2, 96, bf16)
    wq, wk = h.want()
    # queries alone, [head][token] with a gap
    out = h.filled(4, 10, 96 + 8)
    S.rotate_heads(h.rows("q"), h.rotation(), q_out=out, q_out_token_stride=104, q_out_head_stride=1040)
    got = h.values(out, 4, 10, 104)
    assert np.all(got[:, :, 96:] == 7)
    near(got[:, :, :96].transpose(1, 0, 2), wq)
    # keys alone, [kv_head][row]
    keys = h.filled(2, 10, 96)
    S.rotate_heads(h.rows("k"), h.rotation(), to=S.KvCache(keys, None, 2, 96, dtype=h.dtype, key_row_stride=96, key_head_stride=960))
    near(h.values(keys, 2, 10, 96).transpose(1, 0, 2), wk)
    # values alone
    vals = h.filled(10, 2, 96)
    S.rotate_heads(h.rows("v"), h.rotation(), to=S.KvCache(None, vals, 2, 96, dtype=h.dtype))
    assert np.array_equal(h.values(vals, 10, 2, 96), h.v)
    # in place
    dev = S.to_device(h.raw)
    rows, e = h.rows("qk", dev), 2 if bf16 else 4
    S.rotate_heads(rows, h.rotation(), q_out=dev.data_ptr(), q_out_token_stride=h.width, q_out_head_stride=96,
                   to=S.KvCache(dev.data_ptr() + 4 * 96 * e, None, 2, 96, dtype=h.dtype, key_row_stride=h.width, key_head_stride=96))
    got = h.values(dev, 10, h.width)
    near(got[:, :4 * 96].reshape(10, 4, 96), wq)
    near(got[:, 4 * 96:6 * 96].reshape(10, 2, 96), wk)
    assert np.array_equal(got[:, 6 * 96:], h.x[:, 6 * 96:])


def test_infinities_and_nan_stay_in_their_heads_and_values_keep_their_bits():
    h = Heads(6, 4, 4, 2, 64, True)
    raw = h.raw.reshape(4, -1).copy()
    raw[1, 64 * 2 + 5] = 0x7FC0  # a NaN in query head 2 of token 1
    raw[2, 64 * 6 + 1:64 * 6 + 4] = (0x7F80, 0xFF81, 0x8000)  # an infinity, a NaN and -0 in value head 0 of token 2
    raw[3, :64] = 0  # a head of zeros
    h.dev = S.to_device(raw)
    out, keys, vals = h.filled(4, 4, 64), h.filled(4, 2, 64), S.DeviceBuffer(4 * 128 * 2)
    S.rotate_heads(h.rows(), h.rotation(), q_out=out, to=S.KvCache(keys, vals, 2, 64, dtype=S.BF16))
    q = h.values(out, 4, 4, 64)
    assert np.isnan(q[1, 2]).all() and np.all(q[3, 0] == 0)
    keep = np.ones((4, 4), bool)
    keep[1, 2] = keep[3, 0] = False
    wq, _ = h.want()
    near(q[keep], (wq[0][keep], wq[1][keep]))
    assert np.array_equal(vals.download(np.uint16, 512).reshape(4, 128), raw[:, 64 * 6:])


def test_many_segments_and_tables_in_device_memory():
    h = Heads(7, 90, 4, 2, 64, True)
    segs = S.make_segments([(3 * i, 3, i, 1, 0) for i in range(90)])
    wq, wk = h.want()
    lib = S.load_library()
    for seg in (segs.ctypes.data, S.to_device(segs)):
        out, keys, vals = h.filled(90, 4, 64), h.filled(270, 2, 64), h.filled(270, 2, 64)
        cache = S.KvCache(keys, vals, 2, 64)
        assert lib.slha_b200_rotate_heads(h.rows().address, h.rotation().address, seg if isinstance(seg, int) else seg.data_ptr(), 90, out.data_ptr(), 256, 64, cache.address) == 0
        near(h.values(out, 90, 4, 64), wq)
        k = h.values(keys, 270, 2, 64).reshape(90, 3, 2, 64)
        near(k[:, 2], wk)
        assert np.all(k[:, :2] == 7)


def test_positions_in_device_memory_on_a_stream_and_captured():
    torch = pytest.importorskip("torch")
    h = Heads(8, 6, 8, 2, 128, True)
    stream = torch.cuda.Stream()
    S.set_stream(stream.cuda_stream)
    try:
        dev = [S.to_device(x) for x in (h.freq, h.pos, h.qw, h.kw)]
        rows = S.HeadRows(h.dev.data_ptr(), h.dev.data_ptr() + 8 * 256, h.dev.data_ptr() + 10 * 256, 6, 8, 2, 128, token_stride=h.width, head_stride=128, norm=True,
                          q_weight=dev[2], k_weight=dev[3])
        turn = S.Rotation(dev[0], dev[1], 128)
        out, keys, vals = h.filled(6, 8, 128), h.filled(6, 2, 128), h.filled(6, 2, 128)
        to, segs = S.KvCache(keys, vals, 2, 128), S.make_segments([(0, 6, 0, 6, 0)])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            S.rotate_heads(rows, turn, q_out=out, to=to, segments=segs)
        for x in (out, keys, vals):
            x.upload(np.full(x.nbytes // 2, 0x40E0, np.uint16))
        graph.replay()
        torch.cuda.synchronize()
        wq, wk = h.want()
        near(h.values(out, 6, 8, 128), wq)
        near(h.values(keys, 6, 2, 128), wk)
        assert np.array_equal(h.values(vals, 6, 2, 128), h.v)
    finally:
        S.set_stream(None)
