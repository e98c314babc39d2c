"""CPU restatement of the forward operators (include/dpb_forward.h) from their formulas, in 64-bit integers and Python
integers.  TEST INFRASTRUCTURE ONLY, like the rest of oracle/."""
import numpy as np


def pow2(n):
    return 1 << (max(int(n), 1) - 1).bit_length()


def embedding_lookup(table, tokens, multiplier=1, right_shift=0, padded=False):
    """table: int64 [vocab, width]; the rescaling is the lookup witness's: add half a unit, shift towards -infinity."""
    y = [[int(x) * multiplier for x in table[t]] for t in tokens]
    half = 1 << (right_shift - 1) if right_shift else 0
    out = np.array([[(v + half) >> right_shift for v in r] for r in y], dtype=np.int64).reshape(len(tokens), table.shape[1])
    if padded:
        full = np.zeros((pow2(len(tokens)), pow2(table.shape[1])), dtype=np.int64)
        full[:out.shape[0], :out.shape[1]] = out
        return full
    return out


def row_sums(F, keys, n_keys, weights=None, rows=None, rows_per_token=1, multiplier=1):
    """multiplier * sum over rows i with key k of weights[i] * rows[i // rows_per_token, c] -> the table's entries
    (scalars of F) as a list of pow2(n_keys) * pow2(width)."""
    width = 1 if rows is None else rows.shape[1]
    zero = F.from_int(0)
    pk, pw = pow2(n_keys), pow2(width)
    out = [zero] * (pk * pw)
    for i, k in enumerate(keys):
        w = F.one if weights is None else weights[i]
        for c in range(width):
            x = 1 if rows is None else int(rows[i // rows_per_token, c])
            j = int(k) * pw + c
            out[j] = F.add(out[j], F.mul(w, F.from_int(x)))
    if multiplier != 1:
        m = F.from_int(multiplier)
        out = [F.mul(m, v) for v in out]
    return out


def grouped_product(x, keys, weights, rows_per_token=1):
    """int64 x[i // rows_per_token] @ weights[keys[i]]"""
    out = np.zeros((len(keys), weights.shape[2]), dtype=np.int64)
    for i, k in enumerate(keys):
        out[i] = x[i // rows_per_token].astype(np.int64) @ weights[k].astype(np.int64)
    return out
