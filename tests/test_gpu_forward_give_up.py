"""What follows when a forward kernel's wait ran out: the result is not valid, and every call that hands values to the host
or takes forward work says so until dpb_sync has.  The word such a kernel leaves is set from the host here, so that no
kernel has to fail."""
import ctypes
import importlib

import numpy as np
import pytest

from oracle import oracle as orc
from tests.helpers import family_dtype

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def give_up(dpb):
    f = dpb.lib.dpb_forward_give_up  # not part of the interface
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_void_p]
    return lambda c: dpb.check(f(c.h))


@pytest.mark.parametrize("F", [orc.FrField, orc.GlField])
def test_every_call_says_so_until_a_sync(dpb, give_up, F):
    fw = importlib.import_module("deep_prove_b200.forward")
    fam = family_dtype(dpb, F)
    ctx = dpb.Context(0)
    try:
        rng = np.random.default_rng(3)
        ints = rng.integers(-50, 50, size=64)
        tab = ctx.upload_ints(ints, dpb.FR_I64 if F is orc.FrField else dpb.GL_I64)
        one = ctx.upload_ints(ints[:1], dpb.FR_I64 if F is orc.FrField else dpb.GL_I64)
        point = orc.scalars_to_array(F, [F.random_scalar(rng) for _ in range(6)])
        terms = dpb.make_terms([(F.one, [0, 1])], F.to_native)
        groups = fw.RowGroups(ctx, np.array([0, 1, 1]), 2)
        weights = fw.ExpertWeights(ctx, np.ones((2, 3, 4), np.int64), 8)
        counts = dpb.LookupCounts(ctx, 4)
        tree = ctx.logup(dpb.LOGUP_LOOKUP, [tab], point[:1], point[1:2])
        x = np.ones((3, 3), np.int64)
        info = dpb.ChunkingInfo.new(9, 8, dpb.SIGN_MIXED, 20)

        def rounds():
            s = ctx.sumcheck(6, [tab, tab], terms)
            try:
                s.round()
            finally:
                s.free()

        calls = {
            "download": lambda: tab.to_host(),
            "evaluate": lambda: ctx.evaluate(tab, point),
            "evaluate a constant": lambda: ctx.evaluate(one, point[:0]),
            "evaluate many": lambda: dpb.evaluate_many(ctx, [tab, tab], point),
            "a sumcheck's round": rounds,
            "logup outputs": lambda: tree.outputs(),
            "lookup counters": lambda: counts.to_host(),
            "lookup witness": lambda: dpb.lookup_witness(ctx, fam, info, 1, 0, ints.reshape(8, 8), None, 1),
            "lookup": lambda: fw.embedding_lookup(ctx, tab, 8, 8, np.array([1])),
            "groups": lambda: fw.RowGroups(ctx, np.array([0]), 2),
            "weights": lambda: fw.ExpertWeights(ctx, np.ones((2, 3, 4), np.int64), 8),
            "sums": lambda: groups.sums(fam),
            "product": lambda: fw.grouped_product(ctx, groups, x, 8, weights),
        }
        for f in calls.values():  # nothing is wrong yet
            f()
        ctx.sync()
        sc = ctx.sumcheck(6, [tab, tab], terms)
        first = sc.round()
        give_up(ctx)
        with pytest.raises(dpb.DpbError, match="gave up waiting"):
            sc.round(point[:1])
        sc.free()
        for name, f in list(calls.items()) * 2:  # and it stays said
            with pytest.raises(dpb.DpbError, match="gave up waiting") as e:
                f()
            assert e.value.code == dpb.ETIMEOUT, name
        with pytest.raises(dpb.DpbError, match="gave up waiting"):
            ctx.sync()
        ctx.sync()  # told once
        for f in calls.values():
            f()
        y, shape = fw.grouped_product(ctx, groups, x, 8, weights)
        assert (y.to_host(n=12) == 3).all()
        again = ctx.sumcheck(6, [tab, tab], terms)
        assert np.array_equal(again.round(), first)
        again.free()
    finally:
        ctx.close()


def test_a_prover_and_a_commitment_say_so(dpb, give_up):
    """Whole-protocol calls, whose values come out of the calls above, and the commitments."""
    prover, pcs = (importlib.import_module("deep_prove_b200." + m) for m in ("prover", "pcs"))
    F = orc.FrField
    ctx = dpb.Context(0)
    try:
        rng = np.random.default_rng(4)
        tab = ctx.upload_ints(rng.integers(-50, 50, size=64), dpb.FR_I32)
        bases = pcs.G1Bases.synthetic(ctx, 64)
        point = orc.scalars_to_array(F, [F.random_scalar(rng) for _ in range(6)])
        prove = lambda: prover.hadamard_prove(ctx, prover.Blake3Transcript(dpb.FR), point, tab, tab)
        commit = lambda: pcs.batch_commit(ctx, bases, [tab, tab])
        proof, points = prove(), commit()
        give_up(ctx)
        for f in (prove, commit, prove):
            with pytest.raises(dpb.DpbError, match="gave up waiting"):
                f()
        with pytest.raises(dpb.DpbError, match="gave up waiting"):
            ctx.sync()
        assert np.array_equal(np.asarray(commit()), np.asarray(points))
        prove()
    finally:
        ctx.close()


@pytest.mark.parametrize("num_vars", [3, 6, 14])
@pytest.mark.parametrize("at", [0, 1, 2])
def test_a_sumcheck_that_was_told_goes_no_further(dpb, give_up, num_vars, at):
    """Its rounds have gone on when the call fails: nothing but freeing it is left, also after the sync."""
    F = orc.FrField
    ctx = dpb.Context(0)
    try:
        rng = np.random.default_rng(5)
        tabs = [ctx.upload_ints(rng.integers(-50, 50, size=1 << num_vars), dpb.FR_I32) for _ in range(2)]
        r = orc.scalars_to_array(F, [F.random_scalar(rng)])
        sc = ctx.sumcheck(num_vars, tabs, dpb.make_terms([(F.one, [0, 1])], F.to_native))
        for i in range(at):
            sc.round(r if i else None)
        give_up(ctx)
        with pytest.raises(dpb.DpbError, match="gave up waiting"):
            sc.round(r if at else None)
        with pytest.raises(dpb.DpbError, match="gave up waiting"):
            ctx.sync()
        for _ in range(num_vars + 2):
            for call in (lambda: sc.round(r if at else None), lambda: sc.round(r), lambda: sc.finish(r)):
                with pytest.raises(dpb.DpbError) as e:
                    call()
                assert e.value.code == dpb.ESTATE
        sc.free()
        # and at its end
        sc = ctx.sumcheck(num_vars, tabs, dpb.make_terms([(F.one, [0, 1])], F.to_native))
        for i in range(num_vars):
            sc.round(r if i else None)
        give_up(ctx)
        with pytest.raises(dpb.DpbError, match="gave up waiting"):
            sc.finish(r)
        with pytest.raises(dpb.DpbError, match="gave up waiting"):
            ctx.sync()
        with pytest.raises(dpb.DpbError) as e:
            sc.finish(r)
        assert e.value.code == dpb.ESTATE
        sc.free()
        assert tabs[0].to_host(n=1).size == 1
    finally:
        ctx.close()


def test_other_contexts_are_not_concerned(dpb, ctx, give_up):
    other = dpb.Context(0)
    try:
        give_up(other)
        tab = ctx.upload_ints(np.arange(4), dpb.FR_I32)
        assert tab.to_host().tolist() == [0, 1, 2, 3]
        ctx.sync()
    finally:
        other.close()  # with the word still set
