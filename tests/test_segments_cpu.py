"""A table of segments is a numpy array like any other: what is taken from it has numpy's own types, and the address that it knows is where it lies."""
import copy
import pickle

import numpy as np
import pytest

import slhav2_b200 as S
from slhav2_b200 import api

ROWS = [(0, 5, 0, 1, 0), (5, 7, 1, 1, 9)]


def plain():
    a = np.zeros(2, S.SEGMENT_DTYPE)
    for i, r in enumerate(ROWS):
        a[i] = r
    return a


@pytest.mark.parametrize("take", [lambda s: s["n_tiles"], lambda s: s["n_tiles"].sum(), lambda s: s["n_tiles"].max(), lambda s: s["tile_begin"] + 1, lambda s: s[0], lambda s: s[1]["n_tiles"],
                                  lambda s: s[:1], lambda s: s[::2], lambda s: s[np.array([1, 0])], lambda s: s[["n_tiles", "index_base"]], lambda s: np.cumsum(s["n_queries"]), lambda s: s == s,
                                  lambda s: s["n_tiles"].astype(np.int64), lambda s: np.concatenate([s, s]), lambda s: s.tolist(), lambda s: s.tobytes(), lambda s: s.dtype, lambda s: len(s),
                                  lambda s: repr(s), lambda s: str(s), lambda s: list(s["n_tiles"]), lambda s: {int(x): 1 for x in s["n_tiles"]}, lambda s: hash(s["n_tiles"].max()),
                                  lambda s: np.sort(s["n_tiles"])[::-1], lambda s: s[-1:]["tile_begin"].item()])
def test_what_is_taken_from_a_table(take):
    got, want = take(S.make_segments(ROWS)), take(plain())
    assert type(got) is type(want)
    assert np.array_equal(got, want) if isinstance(want, np.ndarray) else got == want


def address_of(segments):
    address, n, kept = api._table(segments)
    of = kept if kept is not None else segments
    assert address == np.asarray(of).ctypes.data and n == len(of)
    return np.array(of)


def test_a_table_s_address_is_where_it_lies():
    s = S.make_segments(ROWS)
    assert np.array_equal(address_of(s), plain())
    s["n_tiles"][1] = 6
    assert address_of(s)[1]["n_tiles"] == 6
    for other in (s.copy(), s[1:], s[::-1], copy.copy(s), copy.deepcopy(s), pickle.loads(pickle.dumps(s)), s.view(), s.reshape(2), s.view(np.ndarray), s.tolist(), plain()):
        assert np.array_equal(address_of(other), np.array(other, S.SEGMENT_DTYPE))


def test_a_table_that_grows():
    s, p = S.make_segments(ROWS), plain()
    s.resize(5000, refcheck=False)
    p.resize(5000, refcheck=False)
    assert np.array_equal(address_of(s), p)
    assert np.array_equal(np.resize(S.make_segments(ROWS), 3), np.resize(plain(), 3))
    assert len(S.make_segments([])) == 0 and address_of(S.make_segments([])).shape == (0,)
