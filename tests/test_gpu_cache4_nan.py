"""A NaN among the values in 4 bits that a token sees is in its results, however little its row weighs and whoever else sees the row."""
import numpy as np
import pytest

from tests import cache_cases as K
from tests import test_gpu_cache4 as T

pytestmark = pytest.mark.gpu
S = pytest.importorskip("slhav2_b200")
F = np.float32


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("tokens,lens", [(1, (100, 400)), (3, (100, 2000)), (9, (130, 700)), (1, (20000,))])
def test_a_seen_nan_whose_weight_underflows(bf16, d, tokens, lens):
    # a slope of 40: the weight of row 3 is 2^-2000 and less.  Its tile is seen as a whole, or in part (the segment's last, or one whose other rows are another document's)
    rng = np.random.default_rng(d + tokens)
    kv, group = 2, 2
    total = sum(lens)
    doc = np.full(total, 5, np.uint32)
    for split in (False, True):
        if split:
            doc[np.cumsum((0,) + lens[:-1]) + 10] = 6  # a row that nobody sees
        call, raw = T.make(rng, lens, tokens, kv, group, d, bf16, slopes=np.full(kv * group, 40.0, F), row_doc=np.stack([doc] * kv), q_doc=np.full(tokens * len(lens), 5, np.uint32))
        want = call.attend(bf16)
        for b in np.cumsum((0,) + lens[:-1]):
            raw[3][b + 3, 1, 1] = 0x7F  # KV head 1, elements 16 to 31
            raw[3][b + 10, :, 0] = 0x7F if split else raw[3][b + 10, :, 0]  # (not seen)
        got = T.results(call, bf16, *T.on_device(call, raw, bf16))
        T.held(got[1], want[1], want[3])
        bad = np.zeros(got[0].shape, bool)
        bad[:, group:, 16:32] = True
        assert np.isnan(got[0][bad]).all(), int(np.isfinite(got[0][bad]).sum())
        T.held(got[0][~bad], want[0][~bad], want[2][~bad])


@pytest.mark.parametrize("bf16", [True, False])
def test_drafted_tokens_see_the_nan_of_their_own_branch_alone(bf16):
    # two branches behind one root; the second branch's first row holds a NaN that its last token sees with no weight left
    rng = np.random.default_rng(4)
    tokens, n = 40, 90
    parents = np.array([K.NONE] + [0, 0] + list(range(1, 38)), np.uint32)  # rows 1, 3, 5 .. and 2, 4, 6 ..
    call, raw = T.make(rng, (n,), tokens, 1, 2, 64, bf16, slopes=np.full(2, 40.0, F), parents=parents)
    want = call.attend(bf16)
    raw[3][n - tokens + 2, 0, 0] = 0x7F
    got = T.results(call, bf16, *T.on_device(call, raw, bf16))
    sees = K.family(parents)[0][:, 2]
    assert np.isnan(got[0][sees][:, :, :16]).all()
    T.held(got[0][~sees], want[0][~sees], want[2][~sees])
    T.held(got[0][sees][:, :, 16:], want[0][sees][:, :, 16:], want[2][sees][:, :, 16:])
