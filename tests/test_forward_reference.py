"""tests/forward_reference.py against oracle/forward.py, entry by entry."""
import numpy as np
import pytest

from oracle import forward as ofw
from oracle import oracle as orc
from tests import forward_reference as ref


@pytest.mark.parametrize("F", [orc.FrField, orc.GlField])
@pytest.mark.parametrize("weighted", [True, False])
@pytest.mark.parametrize("full_range", [True, False])
def test_row_sums(F, weighted, full_range):
    rng = np.random.default_rng(1)
    for n, n_keys, width, per, m in ((1, 1, 1, 1, 1), (7, 3, 2, 2, -5), (40, 9, 3, 1, 2**40), (12, 70, 5, 3, -2**63)):
        lim = 2**63 if full_range else 2**13
        rows = rng.integers(-lim, lim - 1, size=(-(-n // per), width), endpoint=True)
        rows[0, 0], rows[-1, -1] = -lim, lim - 1
        keys = rng.integers(0, n_keys, size=n)
        t = F.random_ext_table(rng, n) if F is orc.GlField else F.random_table(rng, n)
        scal = orc.array_to_scalars(F, t) if weighted else None
        for r in (rows, None):
            want = orc.scalars_to_array(F, ofw.row_sums(F, keys, n_keys, scal, r, per, m))
            got = ref.row_sums(F, keys, n_keys, np.asarray(t, dtype=np.uint64) if weighted else None, r, per, m)
            assert np.array_equal(got, want.reshape(got.shape))


def test_lookup_and_product():
    rng = np.random.default_rng(2)
    E, tokens = rng.integers(-2048, 2048, size=(9, 5)), rng.integers(0, 9, size=6)
    for m, s, padded in ((1, 0, False), (-37, 3, True), (27713, 10, False)):
        assert np.array_equal(ref.lookup(E, tokens, m, s, padded), ofw.embedding_lookup(E, tokens, m, s, padded))
    x, w, keys = rng.integers(-2**14, 2**14, size=(4, 33)), rng.integers(-2**14, 2**14, size=(3, 33, 6)), rng.integers(0, 3, size=8)
    assert np.array_equal(ref.product(x, keys, w, 2), ofw.grouped_product(x, keys, w, 2))
