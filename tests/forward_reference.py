"""The forward operators' formulas over whole arrays, for sizes at which oracle/forward.py's entry-by-entry form takes too
long: integer sums as float64 products that stay below 2^53, field elements from 16-bit digits in Python integers."""
import numpy as np

from oracle import oracle as orc


def pow2(n):
    return 1 << (max(int(n), 1) - 1).bit_length()


def lookup(table, tokens, multiplier=1, right_shift=0, padded=False):
    """For products within 64 bits."""
    y = table[tokens].astype(np.int64) * np.int64(multiplier)
    if right_shift:
        y = (y + np.int64(1 << (right_shift - 1))) >> np.int64(right_shift)
    if padded:
        y = np.pad(y, ((0, pow2(len(tokens)) - len(tokens)), (0, pow2(table.shape[1]) - table.shape[1])))
    return y


def product(x, keys, weights, per=1):
    """|x|, |w| <= 2^14 and fewer than 2^25 inner entries: every sum is a whole number below 2^53."""
    out = np.zeros((len(keys), weights.shape[2]), dtype=np.int64)
    for k in np.unique(keys):
        r = np.flatnonzero(keys == k)
        out[r] = (x[r // per].astype(np.float64) @ weights[k].astype(np.float64)).astype(np.int64)
    return out


def _digits(words):
    """uint64 [n, m] -> float64 [n, 4 m], 16 bits each"""
    shifts = np.arange(0, 64, 16, dtype=np.uint64)
    return ((words[:, :, None] >> shifts) & np.uint64(0xFFFF)).reshape(len(words), -1).astype(np.float64)


def _signed_parts(x):
    """int64 -> signed 16-bit parts, lowest first: x = sum of part_i 2^(16 i)"""
    parts = []
    while True:
        lo = (x & 0xFFFF).astype(np.int64)
        lo = np.where(lo >= 0x8000, lo - 0x10000, lo)
        parts.append(lo.astype(np.float64))
        x = (x >> 16) + ((x >> 15) & 1)
        if not x.any():
            return parts


def row_sums(F, keys, n_keys, weights=None, rows=None, per=1, multiplier=1):
    """weights: the table's words, uint64 [n or more, words].  Returns the result table's words."""
    fr = F is orc.FrField
    p, n_words = (orc.FR_MOD, 4) if fr else (orc.GL_MOD, 2)
    comps, per_comp = (1, 16) if fr else (2, 4)  # components, 16-bit digits of each
    width = 1 if rows is None else rows.shape[1]
    out = np.zeros((pow2(n_keys), pow2(width), n_words), dtype=np.uint64)
    digits = None if weights is None else _digits(weights[:len(keys)])
    one = (1 << 256) % p if fr else 1  # the integer 1 in the table's form
    order = np.argsort(keys, kind="stable")
    cuts = np.flatnonzero(np.diff(keys[order])) + 1
    for r in np.split(order, cuts):
        if not len(r):
            continue
        parts = [np.ones((len(r), 1))] if rows is None else _signed_parts(rows[r // per])
        totals = [np.zeros(width, dtype=object) for _ in range(comps)]
        for i, part in enumerate(parts):
            if digits is None:  # only the first component of an integer is there
                totals[0] += (part.sum(axis=0).astype(np.int64).astype(object) << (16 * i)) * one
                continue
            prod = (digits[r].T @ part).astype(np.int64).astype(object)  # 2^16 * 2^15 * rows
            for j in range(comps):
                for d in range(per_comp):
                    totals[j] += prod[j * per_comp + d] << (16 * (d + i))
        k = int(keys[r[0]])
        for j, t in enumerate(totals):
            raw = b"".join((int(v) * multiplier % p).to_bytes(8 * n_words // comps, "little") for v in t)
            out[k, :width, j * n_words // comps:(j + 1) * n_words // comps] = np.frombuffer(raw, dtype=np.uint64).reshape(width, -1)
    return out.reshape(-1, n_words)
