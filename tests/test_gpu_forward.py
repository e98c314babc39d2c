"""Forward operators (include/dpb_forward.h) on the GPU against their formulas in 64-bit and Python integers
(oracle/forward.py).  Results are integers and field elements: every comparison is for equality."""
import importlib

import numpy as np
import pytest

from oracle import forward as ofw
from oracle import oracle as orc
from tests.helpers import family_dtype

pytestmark = pytest.mark.gpu
FIELDS = [orc.FrField, orc.GlField]


@pytest.fixture(scope="module")
def fw(dpb):
    return importlib.import_module("deep_prove_b200.forward")


def pow2(n):
    return ofw.pow2(n)


def upload_table(dpb, ctx, table, stride, dtype):
    """An integer table with its rows `stride` apart; what lies between rows must never be read as data."""
    flat = np.full(pow2(max(table.shape[0] * stride, 2)), 77777, dtype=np.int64)
    v = flat[:table.shape[0] * stride].reshape(table.shape[0], stride)
    v[:, :table.shape[1]] = table
    return ctx.upload_ints(flat, dtype)


def read(mle, shape):
    return mle.to_host(n=int(np.prod(shape))).reshape(shape) if np.prod(shape) else np.zeros(shape, np.int64)


# ------------------------------------------------------------------------------------------------ embedding lookup
@pytest.mark.parametrize("dtype", ["FR_I32", "FR_I64", "GL_I32", "GL_I64"])
@pytest.mark.parametrize("n,vocab,width,stride", [(1, 1, 1, 1), (1, 300, 48, 64), (5, 7, 3, 3), (33, 200, 48, 48),
                                                  (130, 50, 130, 256), (17, 1000, 129, 131), (3000, 97, 20, 32)])
@pytest.mark.parametrize("padded", [False, True])
def test_lookup(dpb, ctx, fw, dtype, n, vocab, width, stride, padded):
    rng = np.random.default_rng(n * 1000 + width)
    table = rng.integers(-2048, 2048, size=(vocab, width))
    tokens = rng.integers(0, vocab, size=n)
    tokens[0], tokens[-1] = vocab - 1, 0
    dt = getattr(dpb, dtype)
    tab = upload_table(dpb, ctx, table, stride, dt)
    for m, s in ((1, 0), (-37, 0), (27713, 10), (-3, 1), (0, 5)):
        want = ofw.embedding_lookup(table, tokens, m, s, padded)
        for dev in (None, ctx.upload_tensor_i64(tokens)):
            got, shape = fw.embedding_lookup(ctx, tab, vocab, width, tokens, m, s, stride, padded, device_tokens=dev)
            assert shape == want.shape and got.dtype == (dpb.FR_I64 if dtype.startswith("FR") else dpb.GL_I64)
            assert got.len == want.size
            assert np.array_equal(read(got, shape), want)
            got.free()
            if dev:
                dev[0].free()
    tab.free()


def test_lookup_no_tokens(dpb, ctx, fw):
    tab = ctx.upload_ints(np.arange(64), dpb.FR_I32)
    got, shape = fw.embedding_lookup(ctx, tab, 8, 8, np.zeros(0, np.int64))
    assert shape == (0, 8) and got.len == 0
    pad, shape = fw.embedding_lookup(ctx, tab, 8, 8, np.zeros(0, np.int64), padded=True)
    assert shape == (1, 8) and not pad.to_host().any()


def test_lookup_extremes(dpb, ctx, fw):
    """The ends of the integer ranges, exact products next to 2^63, and the ones beyond it refused."""
    lo32, hi32 = -2**31, 2**31 - 1
    tab = ctx.upload_ints(np.array([lo32, hi32, -1, 0] * 2), dpb.FR_I32)
    table = np.array([[lo32, hi32, -1, 0]])
    for m, s in ((2**31 - 1, 0), (-(2**31 - 1), 62), (2**31 - 1, 62), (-1, 31), (1, 1), (-2**31, 0), (2**32 - 1, 0)):
        got, shape = fw.embedding_lookup(ctx, tab, 1, 4, np.array([0]), m, s)
        assert np.array_equal(read(got, shape), ofw.embedding_lookup(table, [0], m, s)), (m, s)
    with pytest.raises(dpb.DpbError, match="does not fit 64 bits"):
        fw.embedding_lookup(ctx, tab, 1, 4, np.array([0]), 2**33, 0)  # 2^31 * 2^33
    wide = np.array([[-2**62, 2**62 - 1]])
    t64 = ctx.upload_ints(wide.reshape(-1), dpb.GL_I64)
    got, shape = fw.embedding_lookup(ctx, t64, 1, 2, np.array([0, 0]), 2, 0)
    assert np.array_equal(read(got, shape), ofw.embedding_lookup(wide, [0, 0], 2, 0))
    for m, s in ((3, 0), (-3, 4), (2, 62)):  # the last: 2^63 - 2 + 2^61 before the shift
        with pytest.raises(dpb.DpbError, match="does not fit 64 bits"):
            fw.embedding_lookup(ctx, t64, 1, 2, np.array([0]), m, s)


def test_lookup_refusals(dpb, ctx, fw):
    tab = ctx.upload_ints(np.arange(64), dpb.FR_I32)
    ok = np.array([0, 1])
    for bad in (np.array([8]), np.array([-1]), np.array([0] * 999 + [2**40]), np.array([0] * 5000 + [8])):
        with pytest.raises(dpb.DpbError, match="outside the table"):
            fw.embedding_lookup(ctx, tab, 8, 8, bad)
    for kw in (dict(vocab=9), dict(width=65), dict(row_stride=7), dict(vocab=0), dict(width=0), dict(right_shift=63),
               dict(vocab=2**63, width=8, row_stride=2**62)):
        with pytest.raises(dpb.DpbError) as e:
            fw.embedding_lookup(ctx, tab, **{**dict(vocab=8, width=8, tokens=ok), **kw})
        assert e.value.code == dpb.EINVAL
    field = ctx.upload(np.arange(64, dtype=np.uint64), dpb.GL_BASE)
    with pytest.raises(dpb.DpbError, match="integer table"):
        fw.embedding_lookup(ctx, field, 8, 8, ok)
    got, shape = fw.embedding_lookup(ctx, tab, 8, 8, ok)  # the context works on after refusals
    assert np.array_equal(read(got, shape), np.arange(16).reshape(2, 8))


def test_a_tensor_is_no_table(dpb, ctx, fw):
    """The unpadded result's handle is refused where a table's variables count, unless its length is a power of two."""
    tab = ctx.upload_ints(np.arange(64), dpb.GL_I32)
    tensor, shape = fw.embedding_lookup(ctx, tab, 8, 8, np.array([3, 1, 7]))
    point = np.ones((2, 2), np.uint64)
    terms = dpb.make_terms([(0, [0])], lambda c: dpb.one_bytes(dpb.GL_EXT))
    for call in (lambda: ctx.sumcheck(5, [tensor], terms), lambda: ctx.fix_low(tensor, point), lambda: ctx.fix_high(tensor, point),
                 lambda: ctx.logup(dpb.LOGUP_LOOKUP, [tensor], point[:1], point[:1])):
        with pytest.raises(dpb.DpbError, match="power of two"):
            call()
    tensor, shape = fw.embedding_lookup(ctx, tab, 8, 8, np.array([3, 1]))
    assert ctx.fix_low(tensor, point).len == 4


# ------------------------------------------------------------------------------------------------ sums by key
def random_weights(F, rng, n):
    t = F.random_ext_table(rng, n) if F is orc.GlField else F.random_table(rng, n)
    return orc.array_to_scalars(F, t), t


def check_sums(dpb, ctx, fw, F, keys, n_keys, weights=True, rows=None, per=1, m=1, seed=0):
    rng = np.random.default_rng(seed)
    n = len(keys)
    scal, tab = random_weights(F, rng, pow2(n)) if weights else (None, None)
    wm = ctx.upload(np.ascontiguousarray(tab), family_dtype(dpb, F)) if weights else None
    want = orc.scalars_to_array(F, ofw.row_sums(F, keys, n_keys, scal, rows, per, m))
    g = fw.RowGroups(ctx, np.asarray(keys, dtype=np.int64), n_keys)
    for dev in (None, ctx.upload_tensor_i64(rows)) if rows is not None and rows.size else (None,):
        got = g.sums(family_dtype(dpb, F), weights=wm, rows=rows if dev is None else None, rows_per_token=per, multiplier=m,
                     device_rows=dev)
        assert got.len == want.shape[0] and got.dtype == family_dtype(dpb, F)
        assert np.array_equal(got.to_host().reshape(want.shape), want)
        got.free()
    g.free()


@pytest.mark.parametrize("F", FIELDS)
@pytest.mark.parametrize("n,n_keys", [(1, 1), (1, 300), (16, 1), (17, 1), (18, 2), (512, 3), (513, 1), (1024, 1), (1500, 700),
                                      (2048, 5000), (2049, 5), (2500, 4095), (2600, 4096), (3000, 9000)])
def test_weight_sums(dpb, ctx, fw, F, n, n_keys):
    """Weights alone: few and many rows per key, runs across slices of 512, both sorts."""
    rng = np.random.default_rng(n + n_keys)
    check_sums(dpb, ctx, fw, F, rng.integers(0, n_keys, size=n), n_keys, m=1 if n % 2 else -29)


@pytest.mark.parametrize("F", FIELDS)
@pytest.mark.parametrize("counts", [[511, 2, 511], [512, 512], [500, 17, 16, 491, 600, 1, 15], [0, 2100, 0, 1], [16, 480, 17, 503, 16, 9]])
def test_weight_sums_runs_across_slices(dpb, ctx, fw, F, counts):
    keys = np.repeat(np.arange(len(counts)), counts)
    np.random.default_rng(1).shuffle(keys)
    check_sums(dpb, ctx, fw, F, keys, len(counts))


@pytest.mark.parametrize("F", FIELDS)
def test_row_counts(dpb, ctx, fw, F):
    """No weights and no rows: how many rows a key has."""
    keys = np.random.default_rng(2).integers(0, 37, size=3000)
    keys[:900] = 5
    check_sums(dpb, ctx, fw, F, keys, 40, weights=False)


@pytest.mark.parametrize("F", FIELDS)
@pytest.mark.parametrize("weights", [True, False])
@pytest.mark.parametrize("n,n_keys,width,per", [(1, 1, 1, 1), (1, 5, 3, 1), (6, 4, 130, 2), (64, 3, 20, 4), (65, 1, 9, 1),
                                               (200, 300, 17, 1), (387, 6, 5, 3), (2100, 3, 2, 2)])
def test_row_sums(dpb, ctx, fw, F, weights, n, n_keys, width, per):
    rng = np.random.default_rng(n * 7 + width)
    rows = rng.integers(-8192, 8192, size=(-(-n // per), width))
    keys = rng.integers(0, n_keys, size=n)
    if n_keys == 6:
        keys[keys == 2] = 3  # a key without rows between others
    check_sums(dpb, ctx, fw, F, keys, n_keys, weights, rows, per, m=1 if n % 2 else 1001)


@pytest.mark.parametrize("F", FIELDS)
@pytest.mark.parametrize("weights", [True, False])
def test_row_sums_full_range(dpb, ctx, fw, F, weights):
    """Entries over the whole 64 bits: sums beyond 64 bits stay exact."""
    rng = np.random.default_rng(3)
    rows = rng.integers(-2**63, 2**63 - 1, size=(150, 4))
    rows[:60, 0], rows[:60, 1], rows[:60, 2] = -2**63, 2**63 - 1, -1
    keys = np.array([0] * 60 + [1] * 90)
    check_sums(dpb, ctx, fw, F, keys, 2, weights, rows, m=-2**63)


def test_row_sums_of_a_long_run(dpb, ctx, fw):
    """One key with 70000 rows that all name the same wide row, entries and words of the weights at their largest: more
    than 2^63 in a word's sum, unless the run is cut."""
    n, width = 70000, 160000
    limbs = np.array([2**64 - 1, 2**64 - 1, 2**64 - 1, 0x2fffffffffffffff], dtype=np.uint64)
    table = np.zeros((1 << 17, 4), np.uint64)
    table[:n] = limbs
    weights = ctx.upload(table, dpb.FR)
    x = np.full((1, width), -32768)
    x[0, 1::2] = 32767
    g = fw.RowGroups(ctx, np.zeros(n, np.int64), 1)
    got = g.sums(dpb.FR, weights=weights, rows=x, rows_per_token=n).to_host(n=width)
    w = sum(int(v) << (64 * i) for i, v in enumerate(limbs))
    for c in (0, 1, width - 2, width - 1):
        want = w * n * int(x[0, c]) % orc.FR_MOD
        assert sum(int(v) << (64 * i) for i, v in enumerate(got[c])) == want
    assert (got[0::2] == got[0]).all() and (got[1::2] == got[1]).all()


@pytest.mark.parametrize("F", FIELDS)
def test_no_rows_at_all(dpb, ctx, fw, F):
    g = fw.RowGroups(ctx, np.zeros(0, np.int64), 5)
    for kw in (dict(), dict(rows=np.zeros((0, 3), np.int64))):
        got = g.sums(family_dtype(dpb, F), **kw)
        assert got.len == (8 if not kw else 32) and not got.to_host().any()


def test_groups_refusals(dpb, ctx, fw):
    for bad in ([5], [-1], [0] * 3000 + [5], [2**33], [0] * 3000 + [-2**62]):
        with pytest.raises(dpb.DpbError, match="key lies outside"):
            fw.RowGroups(ctx, np.array(bad), 5)
    for n_keys in (0, 2**22 + 1):
        with pytest.raises(dpb.DpbError) as e:
            fw.RowGroups(ctx, np.array([0]), n_keys)
        assert e.value.code == dpb.EINVAL
    g = fw.RowGroups(ctx, np.array([0, 1, 1]), 2)
    short = ctx.upload(np.zeros((2, 4), np.uint64), dpb.FR)
    with pytest.raises(dpb.DpbError, match="2 weights for 3 rows"):
        g.sums(dpb.FR, weights=short)
    four = ctx.upload(np.zeros((4, 4), np.uint64), dpb.FR)
    with pytest.raises(dpb.DpbError, match="challenge elements"):
        g.sums(dpb.GL_EXT, weights=four)
    with pytest.raises(dpb.DpbError, match="at least 1"):
        dpb.check(dpb.lib.dpb_row_groups_sum(ctx.h, g.h, dpb.FR, None, None, 0, 1, 0, 1, dpb.ctypes.byref(dpb.ctypes.c_void_p())))
    with pytest.raises(dpb.DpbError, match="one column"):
        dpb.check(dpb.lib.dpb_row_groups_sum(ctx.h, g.h, dpb.FR, None, None, 0, 2, 1, 1, dpb.ctypes.byref(dpb.ctypes.c_void_p())))
    with pytest.raises(ValueError):
        g.sums(dpb.FR, rows=np.zeros((2, 4), np.int64))


def test_row_sums_refuse_what_no_device_holds(dpb, ctx, fw):
    """Sizes whose bytes would pass 64 bits further up are refused by their number, before anything is read or made."""
    g = fw.RowGroups(ctx, np.zeros(512, np.int64), 1)
    few = np.zeros(4, np.int64)
    out = dpb.ctypes.c_void_p()
    for width, per, match in ((2**32, 1, "rows of more than 2.40"), (2**32 + 1, 1, "1..2.32"), (2**31 + 1, 1, "rows of more than 2.40")):
        with pytest.raises(dpb.DpbError, match=match) as e:
            dpb.check(dpb.lib.dpb_row_groups_sum(ctx.h, g.h, dpb.FR, None, dpb.ctypes.c_void_p(few.ctypes.data), 0, width, per, 1,
                                                 dpb.ctypes.byref(out)))
        assert e.value.code == dpb.EINVAL
    many = fw.RowGroups(ctx, np.zeros(3, np.int64), 2**22)
    with pytest.raises(dpb.DpbError, match="result of more than 2.36"):
        dpb.check(dpb.lib.dpb_row_groups_sum(ctx.h, many.h, dpb.FR, None, dpb.ctypes.c_void_p(few.ctypes.data), 0, 2**15, 1, 1,
                                             dpb.ctypes.byref(out)))
    assert g.sums(dpb.GL_EXT).to_host().reshape(-1).tolist() == [512, 0]  # the context works on


@pytest.mark.parametrize("n_keys", [4, 5, 2048])
@pytest.mark.parametrize("n,bad", [(3, [2]), (3000, range(0, 3000, 7)), (700, range(600)), (6000, [5999]), (5000, range(5000))])
def test_bad_device_keys(dpb, ctx, fw, n_keys, n, bad):
    """Keys on the device are refused by the call that uses them, in every form, and nothing outside the result is
    written: tables made before keep their entries."""
    rng = np.random.default_rng(n)
    keys = rng.integers(0, n_keys, size=n)
    keys[list(bad)] = [n_keys, -1, 2**40][n % 3]
    neighbours = [ctx.upload(rng.integers(0, 2**60, size=(4096, 4), dtype=np.uint64), dpb.FR) for _ in range(4)]
    before = [t.to_host() for t in neighbours]
    dev = ctx.upload_tensor_i64(keys)
    w = ctx.upload(np.ones((pow2(n), 4), np.uint64), dpb.FR)
    rows = np.ones((n, 3), np.int64)
    for kw in (dict(weights=w), dict(), dict(rows=rows), dict(rows=rows, weights=w)):
        g = fw.RowGroups(ctx, None, n_keys, device_keys=dev)
        for _ in range(2):  # and again, once it is known
            with pytest.raises(dpb.DpbError, match="key lies outside"):
                g.sums(dpb.FR, **kw)
        g.free()
    if n_keys <= 5:
        wt = fw.ExpertWeights(ctx, np.ones((n_keys, 3, 4), np.int64), 8)
        g = fw.RowGroups(ctx, None, n_keys, device_keys=dev)
        with pytest.raises(dpb.DpbError, match="key lies outside"):
            fw.grouped_product(ctx, g, rows, 8, wt)
    for t, b in zip(neighbours, before):
        assert np.array_equal(t.to_host(), b)


def test_many_unused_groups(dpb, ctx, fw):
    """More handles whose check nobody waited for than the context has places for."""
    keys = [ctx.upload_tensor_i64(np.array([i % 3, 0, 2])) for i in range(100)]
    gs = [fw.RowGroups(ctx, None, 3, device_keys=k) for k in keys]
    for i in (99, 0, 70, 63, 64):
        got = gs[i].sums(dpb.GL_EXT).to_host()
        assert got[:, 0].tolist() == np.bincount([i % 3, 0, 2], minlength=4).tolist()
    for g in gs[::-1]:
        g.free()
    g = fw.RowGroups(ctx, None, 3, device_keys=keys[1])
    assert g.sums(dpb.GL_EXT).to_host()[:, 0].tolist() == [1, 1, 1, 0]


# ------------------------------------------------------------------------------------------------ grouped products
def check_product(ctx, fw, keys, x, w, xb, wb, per=1):
    want = ofw.grouped_product(x, keys, w, per)
    g = fw.RowGroups(ctx, np.asarray(keys, dtype=np.int64), w.shape[0])
    wt = fw.ExpertWeights(ctx, w, wb)
    for dev in (None, ctx.upload_tensor_i64(x)) if x.size else (None,):
        got, shape = fw.grouped_product(ctx, g, x if dev is None else None, xb, wt, per, device_x=dev)
        assert shape == want.shape
        assert np.array_equal(read(got, shape), want)
        got.free()
    wt.free()
    g.free()


@pytest.mark.parametrize("xb,wb", [(14, 12), (8, 12), (15, 8), (8, 8), (2, 2), (15, 15)])
@pytest.mark.parametrize("n,experts,inner,cols", [(1, 1, 1, 1), (3, 2, 128, 128), (16, 1, 130, 129), (40, 3, 257, 100),
                                                  (100, 2, 64, 300), (300, 2, 384, 65), (700, 4, 1100, 130), (999, 2, 150, 200)])
def test_product(ctx, fw, xb, wb, n, experts, inner, cols):
    rng = np.random.default_rng(n + inner)
    x = rng.integers(-2**(xb - 1), 2**(xb - 1), size=(n, inner))
    w = rng.integers(-2**(wb - 1), 2**(wb - 1), size=(experts, inner, cols))
    check_product(ctx, fw, rng.integers(0, experts, size=n), x, w, xb, wb)


@pytest.mark.parametrize("value", ["low", "high", "mixed"])
def test_product_extremes(ctx, fw, value):
    """Every digit product at its largest, all of one sign, over a long inner dimension."""
    inner, lo, hi = 9000, -2**14, 2**14 - 1
    x = np.full((2, inner), lo if value != "high" else hi)
    w = np.full((1, inner, 3), lo if value == "low" else hi)
    check_product(ctx, fw, [0, 0], x, w, 15, 15)


def test_product_inner_beyond_one_item(ctx, fw):
    """More than 2^15 inner entries: several work items per tile, whose 32-bit sums each stay in range."""
    rng = np.random.default_rng(4)
    inner = 2**15 * 2 + 77
    x = np.full((3, inner), -2**14)
    x[1] = rng.integers(-2**14, 2**14, size=inner)
    w = np.full((2, inner, 4), -2**14)
    w[1] = rng.integers(-2**14, 2**14, size=(inner, 4))
    check_product(ctx, fw, [0, 1, 0], x, w, 15, 15)


@pytest.mark.parametrize("per", [2, 4])
def test_product_routed(ctx, fw, per):
    """Several experts per token, experts without rows, one expert with nearly all."""
    rng = np.random.default_rng(5)
    tokens, experts = 150, 9
    keys = np.array([rng.choice([0, 2, 3, 5, 7], size=per, replace=False) for _ in range(tokens)]).reshape(-1)
    keys[:tokens] = 3
    x = rng.integers(-2**13, 2**13, size=(tokens, 200))
    w = rng.integers(-2**11, 2**11, size=(experts, 200, 140))
    check_product(ctx, fw, keys, x, w, 14, 12, per)


def test_product_no_rows(ctx, fw):
    check_product(ctx, fw, [], np.zeros((0, 20), np.int64), np.ones((2, 20, 30), np.int64), 8, 8)


def test_product_refusals(dpb, ctx, fw):
    x, w = np.zeros((3, 20), np.int64), np.zeros((2, 20, 30), np.int64)
    g, wt = fw.RowGroups(ctx, np.array([0, 1, 1]), 2), fw.ExpertWeights(ctx, w, 12)
    for bits in (1, 16):
        with pytest.raises(dpb.DpbError, match="bits"):
            fw.ExpertWeights(ctx, w, bits)
        with pytest.raises(dpb.DpbError, match="bits"):
            fw.grouped_product(ctx, g, x, bits, wt)
    for v, bits in ((128, 8), (-129, 8), (2**11, 12), (2**40, 15), (-2**63, 15)):
        bad = x.copy()
        bad[2, 19] = v
        with pytest.raises(dpb.DpbError, match="does not fit"):
            fw.grouped_product(ctx, g, bad, bits, wt)
        bad = w.copy()
        bad[1, 19, 29] = v
        with pytest.raises(dpb.DpbError, match="does not fit"):
            fw.ExpertWeights(ctx, bad, bits)
    other = fw.RowGroups(ctx, np.array([0, 1, 1]), 3)
    with pytest.raises(dpb.DpbError, match="routed to 3 experts"):
        fw.grouped_product(ctx, other, x, 8, wt)
    with pytest.raises(dpb.DpbError, match="multiple"):
        dpb.check(dpb.lib.dpb_grouped_product(ctx.h, dpb.FR, g.h, dpb.ctypes.c_void_p(x.ctypes.data), 0, 8, 2, wt.h,
                                              dpb.ctypes.byref(dpb.ctypes.c_void_p())))
    with pytest.raises(ValueError):
        fw.grouped_product(ctx, g, x[:2], 8, wt)
    got, shape = fw.grouped_product(ctx, g, x, 8, wt)
    assert not read(got, shape).any()
