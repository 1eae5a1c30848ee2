"""Norm weights that lie at any word: slices of packed arrays, on the device and on the host."""
import numpy as np
import pytest

from tests import test_gpu_rotate as R

pytestmark = pytest.mark.gpu
S = pytest.importorskip("slhav2_b200")
F = np.float32


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("on_device", [True, False])
@pytest.mark.parametrize("first", [1, 2, 3, 5])
def test_weights_that_begin_at_any_word(bf16, on_device, first):
    h = R.Heads(first, 7, 4, 2, 72, bf16)
    packed = np.concatenate([np.full(first, np.nan, F), h.qw, h.kw, np.full(3, np.nan, F)])
    qw, kw = packed[first:first + 72], packed[first + 72:first + 144]
    if on_device:
        dev = S.to_device(packed)
        h.qw, h.kw = dev.data_ptr() + 4 * first, dev.data_ptr() + 4 * (first + 72)
    else:
        h.qw, h.kw = qw, kw
    q, k, v = R.run_rows(h)
    h.qw, h.kw = qw, kw
    wq, wk = h.want()
    R.near(q, wq)
    R.near(k, wk)
    assert np.array_equal(v, h.v)


def test_weights_within_a_word_are_refused():
    h = R.Heads(1, 3, 2, 1, 64, True)
    dev = S.to_device(np.ones(80, F))
    for name in ("qw", "kw"):
        h.qw, h.kw = None, None
        setattr(h, name, dev.data_ptr() + 2)
        with pytest.raises(S.SlhaError) as e:
            R.run_rows(h)
        assert e.value.code == S.ERR_DIMENSION and "weights" in e.value.message
