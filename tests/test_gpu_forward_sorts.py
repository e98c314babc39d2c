"""Rows sorted by key, by each of the three forms and around their borders, with keys that are all valid: sums of weights,
sums of weighted rows and grouped products are compared, whose results are wrong when a row's place, its key's first place
or a tile's prefix sum is.  Forms: counted by comparisons up to 4096 rows; one block up to 16384 rows of up to 256 keys; the
counting sort, whose counters are scanned in tiles of 4096, for all others.  First places are kept up to 1024 keys."""
import importlib

import numpy as np
import pytest

from oracle import oracle as orc
from tests import forward_reference as ref
from tests.helpers import family_dtype

pytestmark = pytest.mark.gpu

COMPARISONS = [(4095, 5000), (4096, 1), (4096, 8), (4096, 256), (4096, 1024), (4096, 1025)]
ONE_BLOCK = [(4097, 1), (4097, 8), (4097, 255), (4097, 256), (5121, 60), (8192, 256), (16383, 7), (16384, 1), (16384, 8), (16384, 256)]
COUNTING = [(4097, 257), (5000, 1023), (5000, 1024), (5000, 1025), (5000, 4094), (5000, 4095), (5000, 4096), (5000, 4097),
            (5000, 50000), (16385, 1), (16385, 5), (16385, 256), (20000, 257), (20000, 1024), (33333, 12289), (70001, 262144)]
SIZES = [pytest.param(*c, id=f"{name}-{c[0]}-{c[1]}") for name, cs in
         (("comparisons", COMPARISONS), ("one_block", ONE_BLOCK), ("counting", COUNTING)) for c in cs]


def draw_keys(rng, n, n_keys):
    """A few keys with most of the rows, neighbouring equal keys, keys without rows (the first or the last among them)."""
    keys = np.minimum((rng.random(n) ** 3 * n_keys).astype(np.int64), n_keys - 1)
    run = rng.integers(0, n - 100)
    keys[run:run + 100] = keys[run]
    if n_keys > 4:
        empty = rng.integers(0, n_keys, size=max(1, n_keys // 5))
        keys[np.isin(keys, empty)] = (empty[0] + 1) % n_keys
        if rng.random() < 0.5:
            keys[keys == n_keys - 1] = n_keys - 2
    return keys


def groups(ctx, fw, keys, n_keys, on_device):
    return fw.RowGroups(ctx, None if on_device else keys, n_keys, device_keys=ctx.upload_tensor_i64(keys) if on_device else None)


@pytest.mark.parametrize("F", [orc.FrField, orc.GlField])
@pytest.mark.parametrize("n,n_keys", SIZES)
def test_sums(dpb, ctx, F, n, n_keys):
    fw = importlib.import_module("deep_prove_b200.forward")
    rng = np.random.default_rng(n * 7 + n_keys)
    keys = draw_keys(rng, n, n_keys)
    t = F.random_ext_table(rng, n) if F is orc.GlField else F.random_table(rng, n)
    words = np.asarray(t, dtype=np.uint64)
    table = np.zeros((ref.pow2(n), words.shape[1]), np.uint64)
    table[:n] = words
    fam = family_dtype(dpb, F)
    w = ctx.upload(table, fam)
    per = (1, 2, 3)[n_keys % 3]
    rows = rng.integers(-8192, 8192, size=(-(-n // per), 3))
    for on_device in (False, True):
        g = groups(ctx, fw, keys, n_keys, on_device)
        for kw, want in ((dict(weights=w), dict(weights=words)), (dict(), dict()),
                         (dict(weights=w, rows=rows, rows_per_token=per, multiplier=-3), dict(weights=words, rows=rows, per=per, multiplier=-3)),
                         (dict(rows=rows, rows_per_token=per), dict(rows=rows, per=per))):
            got = g.sums(fam, **kw)
            assert np.array_equal(got.to_host().reshape(-1, words.shape[1]), ref.row_sums(F, keys, n_keys, **want)), kw.keys()
            got.free()
        g.free()
    w.free()


@pytest.mark.parametrize("n,n_keys", [p for p in SIZES if p.values[1] <= 1024])
def test_products(ctx, n, n_keys):
    fw = importlib.import_module("deep_prove_b200.forward")
    rng = np.random.default_rng(n * 5 + n_keys)
    per = max(p for p in (1, 2, 3) if n % p == 0)
    keys = draw_keys(rng, n, n_keys)
    x, w = rng.integers(-8192, 8192, size=(n // per, 20)), rng.integers(-2048, 2048, size=(n_keys, 20, 9))
    laid_out = fw.ExpertWeights(ctx, w, 12)
    want = ref.product(x, keys, w, per)
    for on_device in (False, True):
        g = groups(ctx, fw, keys, n_keys, on_device)
        got, shape = fw.grouped_product(ctx, g, x, 14, laid_out, per)
        assert np.array_equal(got.to_host(n=want.size).reshape(shape), want)
        got.free()
        g.free()
    laid_out.free()
