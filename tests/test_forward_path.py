"""The forward operators together, as a proving program uses them: tokens are looked up, the embeddings feed an einsum,
routed feed-forward layers run as grouped products, and each result's claim at a point is proven by the sumcheck over
tables that the sums by token and by expert make.  CPU part: the formulas (oracle/forward.py) and the walk on the CPU
restatement, whose sumchecks must start from the claims.  GPU part: the same walk on the library, payload by payload."""
import importlib

import numpy as np
import pytest

from oracle import forward as ofw
from oracle import oracle as orc
from oracle.path_backend import OracleBackend
from tests.test_path_workload import load_workloads_without_gpu

FIELDS = {"fr": orc.FrField, "gl": orc.GlField}


def scalars_of(F, payload):
    return orc.array_to_scalars(F, np.frombuffer(payload, dtype=np.uint64).reshape(-1, F.elem_words))


@pytest.mark.parametrize("field", ["fr", "gl"])
def test_walk_on_the_cpu_backend(field):
    wl = load_workloads_without_gpu()
    F = FIELDS[field]
    rec, timer = wl.transformer_path(OracleBackend(field), wl.TINY_EXPERTS, seed=3)
    kinds = [r[1] for r in rec]
    assert kinds.count("experts") == 2 and kinds.count("embeddings") == 1 and kinds.count("einsum") == 5
    assert {"embedding_lookup", "grouped_product", "experts", "embeddings"} <= set(timer.by_kind)
    for name, kind, payload in rec:
        if kind in ("experts", "embeddings"):
            # the claim (the result's value at the row and column point) is what the first round's message adds up to
            claim, at0, at1 = scalars_of(F, payload)[:3]
            assert F.add(at0, at1) == claim, name


@pytest.mark.parametrize("F", FIELDS.values())
def test_bound_rows_prove_a_grouped_product(F):
    """sum_{e,k} X[e,k] W[e,k] over the bound tables = the product's value at the points, with ragged sizes, an expert
    without rows, several rows per token."""
    rng = np.random.default_rng(1)
    tokens, per, experts, inner, cols = 5, 3, 4, 6, 5
    x, w = rng.integers(-50, 50, size=(tokens, inner)), rng.integers(-50, 50, size=(experts, inner, cols))
    keys = np.array([0, 3, 1] * tokens)
    y = ofw.grouped_product(x, keys, w, per)
    row_point, col_point = [F.random_scalar(rng) for _ in range(4)], [F.random_scalar(rng) for _ in range(3)]
    eq_r, eq_c = (orc.array_to_scalars(F, np.asarray(orc.eq_evals(F, p))) for p in (row_point, col_point))
    want = F.from_int(0)
    for i in range(len(keys)):
        for c in range(cols):
            want = F.add(want, F.mul(F.mul(eq_r[i], eq_c[c]), F.from_int(int(y[i, c]))))
    bound = ofw.row_sums(F, keys, experts, eq_r, x, per)
    got = F.from_int(0)
    for e in range(experts):
        for k in range(inner):
            wk = F.from_int(0)
            for c in range(cols):
                wk = F.add(wk, F.mul(eq_c[c], F.from_int(int(w[e, k, c]))))
            got = F.add(got, F.mul(bound[e * 8 + k], wk))
    assert got == want


def test_lookup_and_its_transpose():
    """<u, lookup(E)> = <transpose(u), E> for integer rows, with the scale on both sides and repeated tokens."""
    rng = np.random.default_rng(2)
    F = orc.FrField
    E, tokens, u = rng.integers(-99, 99, size=(7, 3)), np.array([2, 2, 6, 0, 2]), rng.integers(-99, 99, size=(5, 3))
    y = ofw.embedding_lookup(E, tokens, 13)
    t = ofw.row_sums(F, tokens, 7, rows=u, multiplier=13)
    right = sum(int(E[k, c]) * t[k * 4 + c] for k in range(7) for c in range(3)) % orc.FR_MOD
    assert F.from_int(int((u * y).sum())) == right


@pytest.mark.gpu
@pytest.mark.parametrize("field", ["fr", "gl"])
@pytest.mark.parametrize("seed", [7, 8])
def test_gpu_walk_equals_the_cpu_walk(dpb, ctx, field, seed):
    wl, prover = (importlib.import_module("deep_prove_b200." + m) for m in ("workloads", "prover"))
    want, _ = wl.transformer_path(OracleBackend(field), wl.TINY_EXPERTS, seed=seed)
    got = wl.run_transformer_path(dpb, prover, ctx, wl.TINY_EXPERTS, field=field, seed=seed)
    assert [r[:2] for r in got["records"]] == [r[:2] for r in want]
    for (name, kind, g), (_, _, w) in zip(got["records"], want):
        assert g == w, f"{name} ({kind}) differs from the CPU restatement"


@pytest.mark.gpu
@pytest.mark.parametrize("F", FIELDS.values())
def test_operators_back_to_back(dpb, ctx, F):
    """One program's calls queued one after the other without waiting: embeddings of a prompt, their requantisation
    witness, the routed product of the embeddings, its rows bound, and the handles freed while work is still queued."""
    fw = importlib.import_module("deep_prove_b200.forward")
    rng = np.random.default_rng(11)
    vocab, width, n, experts, cols, per = 500, 96, 130, 6, 70, 2
    E = rng.integers(-2048, 2048, size=(vocab, width))
    W = rng.integers(-2048, 2048, size=(experts, width, cols))
    flat = np.zeros(1 << 16, np.int64)
    flat[:E.size] = E.reshape(-1)
    table = ctx.upload_ints(flat, dpb.FR_I32 if F is orc.FrField else dpb.GL_I32)
    family = dpb.FR if F is orc.FrField else dpb.GL_EXT
    laid_out = fw.ExpertWeights(ctx, W, 12)
    point = [F.random_scalar(rng) for _ in range(9)]
    for _ in range(3):
        tokens = rng.integers(0, vocab, size=n)
        keys = np.stack([rng.permutation(experts)[:per] for _ in range(n)]).reshape(-1)
        rows = fw.embedding_lookup(ctx, table, vocab, width, tokens, multiplier=3, right_shift=1)
        info = dpb.ChunkingInfo.new(9, 8, dpb.SIGN_MIXED, 20)
        owner, ins, outs = dpb.lookup_witness(ctx, family, info, 1, 0, None, None, 1, device_tensor=rows)
        groups = fw.RowGroups(ctx, None, experts, device_keys=ctx.upload_tensor_i64(keys))
        y, shape = fw.grouped_product(ctx, groups, None, 14, laid_out, per, device_x=rows)
        bound = groups.sums(family, weights=ctx.eq_table(family, orc.scalars_to_array(F, point)), device_rows=rows,
                            rows_per_token=per)
        rows[0].free()
        groups.free()
        x = ofw.embedding_lookup(E, tokens, 3, 1)
        assert np.array_equal(y.to_host(n=int(np.prod(shape))).reshape(shape), ofw.grouped_product(x, keys, W, per))
        want = ofw.row_sums(F, keys, experts, orc.array_to_scalars(F, np.asarray(orc.eq_evals(F, point))), x, per)
        assert np.array_equal(bound.to_host().reshape(len(want), -1), orc.scalars_to_array(F, want).reshape(len(want), -1))
        for h in (y, bound, owner):
            h.free()


@pytest.mark.gpu
def test_two_contexts_and_another_stream(dpb, ctx):
    """Another context of the GPU works next to the first one, and refuses its handles; inputs written on a torch stream
    are read after the context's stream was told to wait for it."""
    import torch
    fw = importlib.import_module("deep_prove_b200.forward")
    other = dpb.Context(0)
    try:
        rng = np.random.default_rng(5)
        keys = rng.integers(0, 50, size=4000)
        a, b = fw.RowGroups(ctx, keys, 50), fw.RowGroups(other, keys[::-1].copy(), 50)
        assert np.array_equal(a.sums(dpb.FR).to_host(), b.sums(dpb.FR).to_host())
        out = dpb.ctypes.c_void_p()
        with pytest.raises(dpb.DpbError, match="another context"):
            dpb.check(dpb.lib.dpb_row_groups_sum(ctx.h, b.h, dpb.FR, None, None, 0, 1, 1, 1, dpb.ctypes.byref(out)))
        w = fw.ExpertWeights(other, np.ones((50, 3, 2), np.int64), 8)
        with pytest.raises(dpb.DpbError, match="another context"):
            fw.grouped_product(ctx, a, np.ones((4000, 3), np.int64), 8, w)
        table = other.upload_ints(np.arange(64), dpb.FR_I32)
        with pytest.raises(dpb.DpbError, match="another context"):
            fw.embedding_lookup(ctx, table, 8, 8, np.array([0]))
        stream = torch.cuda.Stream()
        library = torch.cuda.ExternalStream(other.stream)
        with torch.cuda.stream(stream):
            tokens = torch.zeros(1 << 20, dtype=torch.int64, device="cuda")
            for _ in range(20):
                tokens = tokens + 1  # 20 once everything has run; out of the table before the last steps is no matter
            tokens = tokens % 7
        library.wait_stream(stream)
        rows, shape = fw.embedding_lookup(other, table, 8, 8, None,
                                          device_tokens=(other.wrap_device(tokens.data_ptr(), dpb.GL_BASE, 1 << 20), (1 << 20,)))
        assert np.array_equal(rows.to_host(n=64).reshape(8, 8), np.tile(np.arange(8) + 8 * (20 % 7), (8, 1)))
        other.sync()
    finally:
        other.close()


@pytest.mark.gpu
def test_two_threads_with_a_context_each(dpb, ctx):
    """Two host threads work at the same time, each on a context of its own: products and sums of both share the GPU."""
    import threading
    fw = importlib.import_module("deep_prove_b200.forward")
    failures = []

    def work(seed):
        try:
            c = dpb.Context(0)
            rng = np.random.default_rng(seed)
            W = rng.integers(-2048, 2048, size=(5, 300, 260))
            laid_out = fw.ExpertWeights(c, W, 12)
            for _ in range(15):
                n = int(rng.integers(1, 400))
                keys, x = rng.integers(0, 5, size=n), rng.integers(-8192, 8192, size=(n, 300))
                g = fw.RowGroups(c, None, 5, device_keys=c.upload_tensor_i64(keys))
                y, shape = fw.grouped_product(c, g, x, 14, laid_out)
                s = g.sums(dpb.GL_EXT, rows=x)
                want = np.zeros((8, 512), dtype=object)
                for k in range(5):
                    want[k, :300] = x[keys == k].sum(axis=0)
                got = s.to_host().reshape(8, 512, 2)
                if not np.array_equal(y.to_host(n=n * 260).reshape(shape), ofw.grouped_product(x, keys, W)):
                    failures.append((seed, "product"))
                if (got[:, :, 0].astype(object) != want % orc.GL_MOD).any() or got[:, :, 1].any():
                    failures.append((seed, "sums"))
                for h in (y, s, g):
                    h.free()
            laid_out.free()
            c.close()
        except Exception as e:  # a thread's exception must not pass unseen
            failures.append((seed, repr(e)))

    threads = [threading.Thread(target=work, args=(s,)) for s in (1, 2, 3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
