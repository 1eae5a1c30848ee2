"""Norms of heads whose squares leave the range of float32, on either side, against the plain form in 64 bits; the bounds are those of tests/cache4_cases.py."""
import numpy as np
import pytest

from tests import cache_cases as K
from tests import test_gpu_rotate as R

pytestmark = pytest.mark.gpu
S = pytest.importorskip("slhav2_b200")
F = np.float32


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("d,rotary,heads,kv,n", [(64, 64, 6, 2, 5), (128, 0, 3, 1, 33), (256, 256, 2, 2, 4), (72, 40, 5, 1, 7)])
@pytest.mark.parametrize("power,eps", [(60, 1e-6), (100, 1e-6), (120, 1e-6), (-50, 0.0), (-90, 0.0), (-115, 0.0), (-60, 1e-36), (-50, 1e-30), (-100, 1e-44)])
def test_norms_of_very_large_and_very_small_heads(bf16, d, rotary, heads, kv, n, power, eps):
    h = R.Heads(abs(d + power), n, heads, kv, d, bf16, rotary=rotary, eps=eps)
    # every other head of its usual size, beside one in the same warp that is not
    size = np.where(np.arange((heads + 2 * kv) * n).reshape(n, -1) % 2 == 1, 2.0 ** power, 1.0).repeat(d, -1)
    h.x, h.raw = K.as_type(h.x / np.abs(h.x).max() * 2 * size, bf16)
    at = lambda a, b: h.x[:, a * d:b * d].reshape(n, b - a, d)  # noqa: E731
    h.q, h.k, h.v = at(0, heads), at(heads, heads + kv), at(heads + kv, heads + 2 * kv)
    h.dev = S.to_device(h.raw)
    q, k, v = R.run_rows(h)
    wq, wk = h.want()
    R.near(q, wq)
    R.near(k, wk)
    assert np.array_equal(v, h.v)


def test_infinities_still_take_their_heads_with_them():
    h = R.Heads(9, 3, 2, 1, 64, False, rotary=0, weights=False)
    h.x[1, 5], h.x[2, 64:128] = np.inf, 0.0
    h.dev = S.to_device(h.x)
    q, k, v = R.run_rows(h)
    assert np.isnan(q[1, 0, 5]) and np.all(np.delete(q[1, 0], 5) == 0) and np.all(q[2, 1] == 0)
    h.q = h.x[:, :128].reshape(3, 2, 64)
    wq, _ = h.want()
    R.near(q[0], (wq[0][0], wq[1][0]))
