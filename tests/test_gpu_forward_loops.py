"""The forward kernels at sizes where their loops go round: blocks of a grouped product that go on to further work items
(their ring of stages and their accumulators carried over), lookups whose threads make several groups of steps, sums of
rows whose slices hold several batches and many runs."""
import importlib

import numpy as np
import pytest

from oracle import oracle as orc
from tests import forward_reference as ref
from tests.helpers import family_dtype

pytestmark = pytest.mark.gpu
FIELDS = [orc.FrField, orc.GlField]


@pytest.fixture(scope="module")
def fw(dpb):
    return importlib.import_module("deep_prove_b200.forward")


# ------------------------------------------------------------------------------------------------ grouped products
def draw_ints(rng, bits, shape):
    """Values of so many bits, with whole stretches at either end of the range."""
    half = 1 << (bits - 1)
    v = rng.integers(-half, half, size=shape)
    flat = v.reshape(-1)
    flat[:flat.size // 7] = -half
    flat[flat.size // 7:flat.size // 5] = half - 1
    return v


# rows per tile as the average number of rows per expert picks it; columns for more work items (213 and more) than blocks (148)
@pytest.mark.parametrize("tile,n,experts,cols", [(16, 30, 5, 128 * 70 + 3), (32, 60, 4, 128 * 70 + 64), (64, 200, 4, 128 * 60),
                                                 (128, 700, 4, 128 * 45 + 1), (160, 1300, 4, 128 * 33 + 100)])
@pytest.mark.parametrize("xb,wb", [(15, 15), (14, 8), (8, 12), (8, 8)])
@pytest.mark.parametrize("inner", [130, 700])
def test_products_of_many_items(ctx, fw, tile, n, experts, cols, xb, wb, inner):
    rng = np.random.default_rng(n + inner + xb)
    x, w = draw_ints(rng, xb, (n, inner)), draw_ints(rng, wb, (experts, inner, cols))
    keys = rng.permutation(np.repeat(np.arange(experts), n // experts))
    check_product(ctx, fw, x, keys, w, xb, wb)


@pytest.mark.parametrize("counts", [[690, 1, 9, 0], [0, 0, 1, 699], [129, 127, 128, 316], [161, 320, 159, 660]])
def test_products_of_skewed_routes(ctx, fw, counts):
    rng = np.random.default_rng(sum(counts))
    keys = rng.permutation(np.repeat(np.arange(len(counts)), counts))
    x, w = draw_ints(rng, 15, (len(keys), 300)), draw_ints(rng, 12, (len(counts), 300, 128 * 30 + 5))
    check_product(ctx, fw, x, keys, w, 15, 12)


@pytest.mark.parametrize("n,cols", [(40, 128 * 45 + 1), (700, 128 * 20 + 1)])
def test_products_of_many_items_that_add_up(ctx, fw, n, cols):
    """An inner dimension cut into several work items, more items than blocks: results are added to the output."""
    rng = np.random.default_rng(n)
    x, w = draw_ints(rng, 15, (n, 2100)), draw_ints(rng, 15, (2, 2100, cols))
    check_product(ctx, fw, x, rng.integers(0, 2, size=n), w, 15, 15)


def check_product(ctx, fw, x, keys, w, xb, wb):
    g, laid_out, dev = fw.RowGroups(ctx, keys, w.shape[0]), fw.ExpertWeights(ctx, w, wb), ctx.upload_tensor_i64(x)
    got, shape = fw.grouped_product(ctx, g, None, xb, laid_out, device_x=dev)
    assert np.array_equal(got.to_host(n=len(keys) * w.shape[2]).reshape(shape), ref.product(x, keys, w))
    for h in (got, dev[0], laid_out, g):
        h.free()


# ------------------------------------------------------------------------------------------------ embedding lookups
# the grid has at most 4 blocks of 256 threads on each of 148 SMs, of four steps each: over 606208 steps go round
@pytest.mark.parametrize("dtype", ["FR_I32", "GL_I64"])
@pytest.mark.parametrize("n,width,stride", [(5000, 1000, 1024), (2500, 999, 1001), (5003, 1002, 1002)])
@pytest.mark.parametrize("padded", [False, True])
def test_lookups_that_go_round(dpb, ctx, fw, dtype, n, width, stride, padded):
    rng = np.random.default_rng(n)
    vocab = 1500
    E, tokens = rng.integers(-2048, 2048, size=(vocab, width)), rng.integers(0, vocab, size=n)
    flat = np.full(ref.pow2(vocab * stride), 77777, dtype=np.int64)
    flat[:vocab * stride].reshape(vocab, stride)[:, :width] = E
    tab, dev = ctx.upload_ints(flat, getattr(dpb, dtype)), ctx.upload_tensor_i64(tokens)
    for m, s in ((-27713, 10), (2**33 + 5, 3)):  # the second: every product is checked, whatever the entries
        got, shape = fw.embedding_lookup(ctx, tab, vocab, width, None, m, s, stride, padded, device_tokens=dev)
        assert np.array_equal(got.to_host(n=shape[0] * shape[1]).reshape(shape), ref.lookup(E, tokens, m, s, padded))
        got.free()
        for at in (0, n // 2, n - 1):
            bad = tokens.copy()
            bad[at] = vocab
            with pytest.raises(dpb.DpbError, match="outside the table"):
                fw.embedding_lookup(ctx, tab, vocab, width, bad, m, s, stride, padded)
    big = E.copy()
    big[tokens[n - 1], width - 1] = 2**31 - 1
    flat[:vocab * stride].reshape(vocab, stride)[:, :width] = big
    tab2 = ctx.upload_ints(flat, getattr(dpb, dtype))
    with pytest.raises(dpb.DpbError, match="does not fit 64 bits"):  # the last entry's product alone
        fw.embedding_lookup(ctx, tab2, vocab, width, tokens, 2**33, 0, stride, padded)
    for h in (tab, tab2, dev[0]):
        h.free()


def test_lookup_of_more_than_2_to_the_31_entries(dpb, fw):
    """Steps and places beyond 32 bits (17 GB of result), compared on the device a stretch of rows at a time."""
    import torch
    n, vocab, width = 2**20 + 24, 1000, 2049
    ctx = dpb.Context(0)
    try:
        gen = torch.Generator(device="cuda")
        gen.manual_seed(3)
        E = torch.zeros(1 << 21, dtype=torch.int32, device="cuda")
        E[:vocab * width] = torch.randint(-2048, 2048, (vocab * width,), generator=gen, device="cuda", dtype=torch.int32)
        tokens = torch.zeros(1 << 21, dtype=torch.int64, device="cuda")
        tokens[:n] = torch.randint(0, vocab, (n,), generator=gen, device="cuda")
        tokens[n - 1] = vocab - 1
        torch.cuda.synchronize()
        table = ctx.wrap_device(E.data_ptr(), dpb.FR_I32, 1 << 21)
        ids = (ctx.wrap_device(tokens.data_ptr(), dpb.GL_BASE, 1 << 21), (n,))
        out, shape = fw.embedding_lookup(ctx, table, vocab, width, None, 77, 3, device_tokens=ids)
        ctx.sync()

        class Words:
            __cuda_array_interface__ = {"shape": shape, "typestr": "<i8", "data": (out.device_ptr, False), "version": 3}

        got, rows = torch.as_tensor(Words(), device="cuda"), E[:vocab * width].view(vocab, width)
        for i in range(0, n, 1 << 16):
            want = (rows[tokens[i:min(i + (1 << 16), n)]].long() * 77 + 4) >> 3
            assert torch.equal(got[i:i + want.shape[0]], want), i
        torch.cuda.synchronize()
        del got
        out.free()
    finally:
        ctx.close()


# ------------------------------------------------------------------------------------------------ sums of rows
def check_sums(dpb, ctx, fw, F, keys, n_keys, rows, per=1, m=1, seed=0):
    rng = np.random.default_rng(seed)
    n = len(keys)
    words = rng.integers(0, 2**64, size=(n, 4 if F is orc.FrField else 2), dtype=np.uint64)
    words[:, -1] &= np.uint64(2**60 - 1)
    if F is orc.GlField:
        words[:, 0] >>= np.uint64(1)  # below the modulus
    table = np.zeros((ref.pow2(n), words.shape[1]), np.uint64)
    table[:n] = words
    fam = family_dtype(dpb, F)
    w, dev = ctx.upload(table, fam), ctx.upload_tensor_i64(rows) if rows is not None else None
    g = fw.RowGroups(ctx, keys, n_keys)
    for weights, mle in ((words, w), (None, None)):
        got = g.sums(fam, weights=mle, device_rows=dev, rows_per_token=per, multiplier=m)
        assert np.array_equal(got.to_host().reshape(-1, words.shape[1]), ref.row_sums(F, keys, n_keys, weights, rows, per, m))
        got.free()
    for h in (g, w) + ((dev[0],) if dev else ()):
        h.free()


def ragged_keys(rng, n, n_keys):
    """Runs of one row and of hundreds, one key with a third of all rows, keys without rows."""
    keys = rng.integers(0, n_keys, size=n)
    keys[rng.random(n) < 0.3] = n_keys // 2
    few = rng.integers(0, n_keys, size=max(1, n_keys // 4))
    keys[np.isin(keys, few) & (rng.random(n) < 0.98)] = n_keys // 3
    keys[keys == n_keys - 1] = 0
    return keys


# narrow: one block of columns, so that the rows are cut into slices of 136 and more (85 without weights), each several
# batches of 128 (64) rows; the odd width is read entry by entry, the even one in pairs
@pytest.mark.parametrize("F", FIELDS)
@pytest.mark.parametrize("width", [1, 3, 4])
@pytest.mark.parametrize("n_keys", [300, 3000])
def test_sums_of_several_batches(dpb, ctx, fw, F, width, n_keys):
    rng = np.random.default_rng(width * n_keys)
    n = 100003
    check_sums(dpb, ctx, fw, F, ragged_keys(rng, n, n_keys), n_keys, rng.integers(-2**15, 2**15, size=(n, width)), m=7)


@pytest.mark.parametrize("F", FIELDS)
def test_sums_of_several_batches_with_wide_entries(dpb, ctx, fw, F):
    """Some entries have more than 16 bits, in any batch, run and column."""
    rng = np.random.default_rng(5)
    n = 100003
    rows = rng.integers(-2**15, 2**15, size=(n, 2))
    at = rng.random((n, 2)) < 0.01
    rows[at] = rng.integers(-2**63, 2**63 - 1, size=int(at.sum()))
    rows[::5003] = [[-2**63, 2**63 - 1]]
    check_sums(dpb, ctx, fw, F, ragged_keys(rng, n, 50), 50, rows)


@pytest.mark.parametrize("F", FIELDS)
@pytest.mark.parametrize("width,per", [(600, 4), (601, 3), (257, 1)])
def test_sums_of_several_batches_and_columns(dpb, ctx, fw, F, width, per):
    rng = np.random.default_rng(width)
    n = 48000
    check_sums(dpb, ctx, fw, F, ragged_keys(rng, n, 12), 12, rng.integers(-2**15, 2**15, size=(n // per, width)), per)


@pytest.mark.parametrize("F", FIELDS)
def test_sums_of_weights_over_many_slices(dpb, ctx, fw, F):
    rng = np.random.default_rng(6)
    for n, n_keys in ((100003, 300), (60000, 40000)):
        check_sums(dpb, ctx, fw, F, ragged_keys(rng, n, n_keys), n_keys, None, m=-11)
