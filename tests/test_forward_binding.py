"""What the forward operators' Python face refuses by itself, without a GPU: the library is replaced by a fake that has
tables on no device and must not be reached by a refused call."""
import importlib

import numpy as np
import pytest


class FakeTable:
    """A table of the fake library: what the binding may ask about it."""

    def __init__(self, dtype, n):
        self.dtype, self.len, self.ptr = dtype, n, 4096


@pytest.fixture
def fw(dpb, monkeypatch):
    mod = importlib.import_module("deep_prove_b200.forward")

    class Lib:
        reached = None

        def dpb_mle_len(self, t):
            return t.len

        def dpb_mle_dtype(self, t):
            return t.dtype

        def dpb_mle_device_ptr(self, t):
            return t.ptr

        def __getattr__(self, name):
            def call(*args):
                Lib.reached = (name, args)
                return 0
            return call

    monkeypatch.setattr(dpb, "lib", Lib())
    monkeypatch.setattr(mod, "lib", dpb.lib)
    monkeypatch.setattr(mod, "Fake", Lib, raising=False)
    return mod


class Ctx:
    h = object()


def groups_of(fw, n, n_keys=4):
    g = fw.RowGroups.__new__(fw.RowGroups)
    g.ctx, g.h, g.n, g.n_keys = Ctx(), object(), n, n_keys
    return g


def calls(dpb, fw, device):
    """Every call that takes a device tensor, with `device` as that tensor; its shape decides what the others are."""
    table = dpb.Mle(Ctx(), FakeTable(dpb.FR_I32, 64))
    shape = device[1]
    out = [lambda: fw.embedding_lookup(Ctx(), table, 8, 8, None, device_tokens=device),
           lambda: fw.RowGroups(Ctx(), None, 8, device_keys=device)]
    if len(shape) == 2:
        w = fw.ExpertWeights.__new__(fw.ExpertWeights)
        w.h, w.n_experts, w.inner, w.cols = object(), 4, shape[1], 5
        out += [lambda: groups_of(fw, shape[0]).sums(dpb.FR, device_rows=device),
                lambda: fw.grouped_product(Ctx(), groups_of(fw, shape[0]), None, 8, w, device_x=device)]
    if len(shape) == 3:
        out += [lambda: fw.ExpertWeights(Ctx(), None, 8, device_weights=device)]
    return out


@pytest.mark.parametrize("shape", [(17,), (3, 6), (2, 3, 3), (2**40, 2**30)])
def test_a_table_shorter_than_the_shape(dpb, fw, shape):
    for dtype in (dpb.GL_BASE, dpb.FR_I64, dpb.GL_I64):
        device = (dpb.Mle(Ctx(), FakeTable(dtype, 16)), shape)
        for call in calls(dpb, fw, device):
            fw.Fake.reached = None
            with pytest.raises(ValueError, match="in a table of 16 entries"):
                call()
            assert fw.Fake.reached is None


@pytest.mark.parametrize("shape", [(8,), (2, 4), (2, 2, 2)])
def test_a_table_of_other_entries_or_freed(dpb, fw, shape):
    for dtype in (dpb.GL_EXT, dpb.FR, dpb.GL_I32, dpb.FR_I32):
        for call in calls(dpb, fw, (dpb.Mle(Ctx(), FakeTable(dtype, 16)), shape)):
            with pytest.raises(ValueError, match="8-byte entries"):
                call()
    mle = dpb.Mle(Ctx(), FakeTable(dpb.FR_I64, 16))
    for call in calls(dpb, fw, (mle, shape)):
        call()  # asked once, and then freed
    mle.free()
    for call in calls(dpb, fw, (mle, shape)):
        fw.Fake.reached = None
        with pytest.raises(ValueError, match="freed"):
            call()
        assert fw.Fake.reached is None


def test_freed_weights_are_not_ones(dpb, fw):
    """The library takes no weights for ones."""
    w = dpb.Mle(Ctx(), FakeTable(dpb.FR, 8))
    groups_of(fw, 5).sums(dpb.FR, weights=w)
    w.free()
    for rows in (None, np.ones((5, 2), np.int64)):
        fw.Fake.reached = None
        with pytest.raises(ValueError, match="freed"):
            groups_of(fw, 5).sums(dpb.FR, weights=w, rows=rows)
        assert fw.Fake.reached is None


def test_integers_that_the_arguments_cannot_hold(dpb, fw):
    """2^32 + 1 rows per token would arrive as 1 row, 2^63 times as -2^63 times."""
    table, tokens, x = dpb.Mle(Ctx(), FakeTable(dpb.FR_I32, 64)), np.zeros(3, np.int64), np.ones((3, 2), np.int64)
    w = fw.ExpertWeights(Ctx(), np.ones((4, 2, 5), np.int64), 8)
    lookup = lambda **kw: fw.embedding_lookup(Ctx(), table, **{**dict(vocab=8, width=8, tokens=tokens), **kw})
    for call in (lambda: lookup(multiplier=2**63), lambda: lookup(multiplier=-2**63 - 1), lambda: lookup(right_shift=2**32),
                 lambda: lookup(right_shift=-1), lambda: lookup(vocab=2**64 + 1), lambda: lookup(row_stride=2**64 + 8),
                 lambda: lookup(width=-8), lambda: fw.RowGroups(Ctx(), tokens, 2**64 + 4),
                 lambda: groups_of(fw, 3).sums(dpb.FR, rows=x, rows_per_token=2**32 + 1),
                 lambda: groups_of(fw, 3).sums(dpb.FR, multiplier=2**63),
                 lambda: fw.ExpertWeights(Ctx(), np.ones((4, 2, 5), np.int64), 2**32 + 8),
                 lambda: fw.grouped_product(Ctx(), groups_of(fw, 3), x, 2**32 + 8, w)):
        fw.Fake.reached = None
        with pytest.raises(ValueError, match="does not fit"):
            call()
        assert fw.Fake.reached is None
    # the library itself refuses none per token, with rows as well
    for kw in (dict(), dict(rows=x)):
        groups_of(fw, 3).sums(dpb.FR, rows_per_token=0, **kw)
        assert fw.Fake.reached[0] == "dpb_row_groups_sum" and fw.Fake.reached[1][7] == 0
    lookup(multiplier=-2**63, right_shift=62)
    assert fw.Fake.reached[1][8:10] == (-2**63, 62)


@pytest.mark.parametrize("shape,dtype,freed", [((3, 6), "GL_BASE", False), ((2, 4), "FR", False), ((2, 4), "FR_I64", True)])
def test_the_calls_that_take_such_results(dpb, fw, shape, dtype, freed):
    """The einsum and lookup calls' device tensors are held to the same."""
    prover = importlib.import_module("deep_prove_b200.prover")
    mle = dpb.Mle(Ctx(), FakeTable(getattr(dpb, dtype), 16))
    if freed:
        mle.free()
    ctx = dpb.Context.__new__(dpb.Context)
    ctx.h = None
    kinds, info, x = (dpb.AXIS_OUTER, dpb.AXIS_CONTRACTED), dpb.ChunkingInfo(), np.zeros((2, 2), np.int64)
    for call in (lambda: ctx.einsum_fix_axes(dpb.FR, None, kinds, [None, None], device_tensor=(mle, shape)),
                 lambda: prover.EinsumOperand(None, kinds, [None, None], device_tensor=(mle, shape)),
                 lambda: dpb.lookup_witness(ctx, dpb.FR, info, 1, 0, None, None, 1, device_tensor=(mle, shape)),
                 lambda: dpb.lookup_witness(ctx, dpb.FR, info, 1, 0, x, None, 2, device_table=(mle, shape))):
        fw.Fake.reached = None
        with pytest.raises(ValueError, match="device tensor"):
            call()
        assert fw.Fake.reached is None


def test_extents_that_numpy_would_cut(dpb, fw):
    """2^40 * 2^24 = 2^64 is 0 in 64 bits."""
    shape = (np.int64(2**40), np.int64(2**24))
    for call in calls(dpb, fw, (dpb.Mle(Ctx(), FakeTable(dpb.FR_I64, 16)), shape))[1:2]:
        with pytest.raises(ValueError, match="in a table of 16"):
            call()


def test_negative_extents(dpb, fw):
    for call in calls(dpb, fw, (dpb.Mle(Ctx(), FakeTable(dpb.FR_I64, 16)), (-2, -3))):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("shape", [(16,), (4, 4), (2, 2, 4), (0,)])
def test_what_fits_is_handed_on(dpb, fw, shape):
    for call in calls(dpb, fw, (dpb.Mle(Ctx(), FakeTable(dpb.GL_BASE, 16)), shape)):
        fw.Fake.reached = None
        call()
        assert 4096 in fw.Fake.reached[1]
