"""Attention over rows in 4 bits where scores are so large that their last places count: each query row's largest score grows between the tiles that a warp takes, by steps that
float32 just holds."""
import numpy as np
import pytest

from tests import cache4_cases as Q
from tests import cache_cases as K
from tests import test_gpu_cache4 as T

pytestmark = pytest.mark.gpu
S = pytest.importorskip("slhav2_b200")
F = np.float32
TILE = 128


def with_log2(power):
    """The float32 that times log2(e), in float32, is a power of two: scores in units of log 2 are then exact."""
    log2e, want = F(1.4426950408889634), F(2.0 ** power)
    x = F(want / log2e)
    for y in (x, np.nextafter(x, F(0)), np.nextafter(x, F(np.inf))):
        if F(y * log2e) == want:
            return y
    raise AssertionError("no float32 does")


STEPS = (0, 1, 2, 3, 4, 6)  # what a code holds
PAIRS = [(a, b) for a in STEPS for b in STEPS if a < b] + [(4, 0)]


def rows_of_steps(rng, kv, d, steps, exponent):
    """Codes and scales of rows [row][kv] whose element 0 is 1024 and whose element 16 is steps[row][kv]; values are random."""
    n = len(steps)
    codes, scales = np.zeros((n, kv, d), np.uint8), np.zeros((n, kv, d // 16), np.uint8)
    codes[:, :, 0], scales[:, :, 0] = 6, 120  # 4 times 256
    codes[:, :, 16], scales[:, :, 1] = np.searchsorted(Q.E2M1, steps), 56  # times 1
    held = Q.values(codes, scales, 0)
    assert np.array_equal(held[:, :, 16], steps) and np.all(held[:, :, 0] == 1024)
    v_codes, v_scales = Q.quantise(rng.standard_normal((n, kv, d)).astype(F), exponent)
    return (codes, scales), (v_codes, v_scales)


def expected(weights, values, bf16):
    """Results and bounds for weights [row][kv] (the exact ones) and values [row][kv][d]."""
    w = weights / weights.sum(0)
    v = values.astype(np.float64)
    out, mag = np.einsum("rk,rkd->kd", w, v), np.einsum("rk,rkd->kd", w, np.abs(v))
    # the factor is 2^-23 of a score's distance from the largest off, and beyond 2^7 units of log 2 of that nothing is left of a weight; the sums of n terms; weights as one float16 number
    # (bfloat16) or two, below 2^-22 of the largest in steps of 2^-33 of it
    tol = (2.0 ** -16 * np.log(2) + (len(w) / 8 + 48) * K.EPS_F32 + 2.0 ** -20) * mag + 2.0 ** -33 * np.abs(v).sum(0) + 1e-30
    if bf16:
        tol = tol + 2.0 ** -11 * mag + 2.0 ** -8 * (np.abs(out) + tol + 2.0 ** -11 * mag)
    return out, tol


def attend(keys, vals, q, segs, kv, group, d, bf16, exponent, **more):
    a = [Q.laid_out(*x) for x in (keys, vals)]
    at = more.pop("row_pos", None)  # [kv_head][row]
    cache = S.KvCache4(S.to_device(a[0][0]), S.to_device(a[1][0]), S.to_device(a[0][1]), S.to_device(a[1][1]), kv, d, dtype=T.type_of(bf16), value_exponent=exponent,
                       positions=None if at is None else S.to_device(np.ascontiguousarray(at)), entry_head_stride=0 if at is None else at.shape[1])
    n = len(segs)
    out, lse = S.DeviceBuffer(q.size * (2 if bf16 else 4)), S.DeviceBuffer(n * kv * group * 4)
    S.attend_cache4(cache, S.make_segments(segs), S.CacheQueries(S.to_device(q), n, kv * group, d, **more), out, lse)
    assert S.debug_last_cache_kernels() == S.CACHE_ATTEND4
    o = out.download(np.uint16 if bf16 else F, q.size)
    return (K.from_bf16(o) if bf16 else o).reshape(n, kv, group, d), lse.download(F, n * kv * group).reshape(n, kv, group)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("power", [-1, 0, 1, 2, 3, 4, 5])
def test_largest_scores_that_grow_by_their_last_places_from_tile_to_tile(bf16, sign, power):
    # scores of (1.5 2^23 + step) 2^power, or less that: float32's steps there are 2^power; a head for each pair of steps, so many sequences on the same rows that each warp takes several tiles
    rng = np.random.default_rng(power + 10)
    kv, group, d, seqs, n = len(PAIRS), 2, 64, 48, 3 * TILE
    steps = np.zeros((n, kv), F)
    for h, (a, b) in enumerate(PAIRS):
        first, second = (a, b) if sign > 0 else (b, a)  # (the score falls with the step where it is negative)
        steps[:TILE, h], steps[TILE:2 * TILE, h], steps[2 * TILE:, h] = first, second, min(a, b) if sign > 0 else max(a, b)
    keys, vals = rows_of_steps(rng, kv, d, steps, -4)
    x = np.zeros((seqs, kv, group, d), F)
    x[..., 0], x[..., 16] = sign * 12288.0, sign
    q = K.as_type(x, bf16)[1]
    scale = with_log2(power)
    got, lse = attend(keys, vals, q, [(0, n, i, 1, 0) for i in range(seqs)], kv, group, d, bf16, -4, scale=scale, causal=False)
    score = sign * (12288.0 * 1024 + steps.astype(np.float64)) * float(scale)
    weights = np.exp(score - score.max(0))
    want, tol = expected(weights, Q.values(*vals, -4), bf16)
    T.held(got, np.broadcast_to(want[None, :, None], got.shape), tol[None, :, None])
    z = score.max(0) + np.log(weights.sum(0))
    # the factor's, the sum's and the last product's roundings: five halves of a step
    T.held(lse, np.broadcast_to(z[None, :, None], lse.shape), 2.0 ** -22 * np.abs(z)[None, :, None])


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("power", [0, 1, 2, 3, 4, 5])
def test_far_rows_whose_biases_grow_by_their_last_places_weigh_nothing_beside_near_ones(bf16, power):
    # a slope of 1 in units of log 2: the score of a row at distance x is -x.  All rows but the last two are (1.5 2^23 - step) 2^power away, steps by tile
    rng = np.random.default_rng(power)
    kv, group, d, seqs, n, at = len(PAIRS), 2, 64, 48, 4 * TILE, (1 << 31) + 5
    steps = np.zeros((n, kv), np.int64)
    for h, (a, b) in enumerate(PAIRS):
        steps[:TILE, h], steps[TILE:2 * TILE, h] = a, b
    away = (12288 * 1024 - steps) << power
    away[-2:] = [[1], [0]]
    keys, vals = rows_of_steps(rng, kv, d, np.zeros((n, kv), F), -4)
    q = K.as_type(np.zeros((seqs, kv, group, d)), bf16)[1]
    got, lse = attend(keys, vals, q, [(0, n, i, 1, 0) for i in range(seqs)], kv, group, d, bf16, -4, scale=1.0, slopes=np.full(kv * group, with_log2(0), F),
                      row_pos=(at - away).T.astype(np.uint32), positions=np.full(seqs, at, np.uint32))
    want, tol = expected(np.exp2(-away.astype(np.float64)), Q.values(*vals, -4), bf16)
    T.held(got, np.broadcast_to(want[None, :, None], got.shape), tol[None, :, None])
    T.held(lse, np.full(lse.shape, np.log(1.5)), 2.0 ** -20)
