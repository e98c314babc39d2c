"""Python face of include/dpb_forward.h: the forward operators that make the integer tensors the provers take, and their
transposes.  Device tensors are (table, shape) pairs, as Context.upload_tensor_i64 returns them; results of that form can
be handed to the einsum and lookup calls' device_tensor arguments.  A pair whose table was freed, has entries of another
size than 8 bytes or fewer of them than the shape is a ValueError."""
import ctypes
import math

import numpy as np

from . import FR_I64, Mle, _buf, _int, _pp, _u32, _u64, _vp, check, lib

_i64 = ctypes.c_int64
FORWARD_SIGNATURES = {
    "dpb_embedding_lookup": (_int, [_vp, _vp, _u64, _u64, _u64, _vp, _int, _u64, _i64, _u32, _int, _pp]),
    "dpb_row_groups_new": (_int, [_vp, _vp, _int, _u64, _u64, _pp]),
    "dpb_row_groups_len": (_u64, [_vp]),
    "dpb_row_groups_free": (None, [_vp]),
    "dpb_row_groups_sum": (_int, [_vp, _vp, _int, _vp, _vp, _int, _u64, _u32, _i64, _pp]),
    "dpb_expert_weights_new": (_int, [_vp, _vp, _int, _u32, _u64, _u64, _u32, _pp]),
    "dpb_expert_weights_free": (None, [_vp]),
    "dpb_grouped_product": (_int, [_vp, _int, _vp, _vp, _int, _u32, _u32, _vp, _pp]),
}
for _name, (_res, _args) in FORWARD_SIGNATURES.items():
    _fn = getattr(lib, _name)
    _fn.restype = _res
    _fn.argtypes = _args


def _source(array, device):
    """(pointer, 1 when on the device, shape, what must stay alive) of an int64 tensor given either way."""
    if device is not None:
        mle, shape = device
        return mle.tensor_ptr(shape), 1, shape, mle
    a = np.ascontiguousarray(array, dtype=np.int64)
    return _buf(a), 0, a.shape, a


# The library's integer arguments have fixed widths, and ctypes would cut what does not fit.  Compared in line: a call of
# one token takes 17 us, and a function with named arguments one of them.
_U32, _U64, _I63 = 1 << 32, 1 << 64, 1 << 63


def _unfit(**values):
    return ValueError(", ".join(f"{k} {v}" for k, v in values.items()) + ": one does not fit its argument's bits")


def _pow2(n):
    return 1 << (max(int(n), 1) - 1).bit_length()


def embedding_lookup(ctx, table, vocab, width, tokens, multiplier=1, right_shift=0, row_stride=None, padded=False,
                     device_tokens=None):
    """dpb_embedding_lookup: the rows of `tokens`, rescaled.  `table`: an integer table of vocab rows, row_stride
    (default: width) entries apart.  Returns (table, shape): the [n, width] tensor, or with padded=True the table of
    the padded shape."""
    row_stride = width if row_stride is None else row_stride
    if not (0 <= vocab < _U64 and 0 <= width < _U64 and 0 <= row_stride < _U64 and 0 <= right_shift < _U32
            and -_I63 <= multiplier < _I63):
        raise _unfit(vocab=vocab, width=width, row_stride=row_stride, right_shift=right_shift, multiplier=multiplier)
    ptr, on_device, shape, _keep = _source(tokens, device_tokens)
    n = math.prod(shape)
    h = ctypes.c_void_p()
    check(lib.dpb_embedding_lookup(ctx.h, table.h, vocab, width, row_stride, ptr, on_device, n,
                                   multiplier, right_shift, 1 if padded else 0, ctypes.byref(h)))
    return Mle(ctx, h), (_pow2(n), _pow2(width)) if padded else (n, width)


class RowGroups:
    """dpb_row_groups: rows sorted by key (tokens, or the expert of every routed row).  A key outside 0..n_keys-1 raises
    here for keys on the host, in the first call that uses the rows for device_keys."""

    def __init__(self, ctx, keys, n_keys, device_keys=None):
        self.ctx, self.h = ctx, None
        if not 0 <= n_keys < _U64:
            raise _unfit(n_keys=n_keys)
        ptr, on_device, shape, _keep = _source(keys, device_keys)
        self.n, self.n_keys = math.prod(shape), int(n_keys)
        h = ctypes.c_void_p()
        check(lib.dpb_row_groups_new(ctx.h, ptr, on_device, self.n, n_keys, ctypes.byref(h)))
        self.h = h

    def sums(self, family_dtype, weights=None, rows=None, rows_per_token=1, multiplier=1, device_rows=None):
        """dpb_row_groups_sum: out[k, c] = multiplier * sum over rows i with key k of weights[i] * rows[i //
        rows_per_token, c], a table of the padded shape over the family's challenge elements."""
        if not (0 <= rows_per_token < _U32 and -_I63 <= multiplier < _I63):
            raise _unfit(rows_per_token=rows_per_token, multiplier=multiplier)
        if rows is None and device_rows is None:
            ptr, on_device, width = None, 0, 1
        else:
            ptr, on_device, shape, _keep = _source(rows, device_rows)
            if len(shape) != 2 or shape[0] < -(-self.n // max(rows_per_token, 1)):
                raise ValueError(f"rows of shape {shape} for {self.n} keys, {rows_per_token} per token")
            width = shape[1]
        if weights is not None and not weights.h:
            raise ValueError("weights that were freed")
        h = ctypes.c_void_p()
        check(lib.dpb_row_groups_sum(self.ctx.h, self.h, family_dtype, weights.h if weights is not None else None, ptr, on_device,
                                     width, rows_per_token, multiplier, ctypes.byref(h)))
        return Mle(self.ctx, h)

    def free(self):
        if self.h:
            lib.dpb_row_groups_free(self.h)
            self.h = None


class ExpertWeights:
    """dpb_expert_weights: [expert, in, out] integers of at most `bits` bits, laid out for grouped_product."""

    def __init__(self, ctx, weights, bits, device_weights=None):
        self.ctx, self.h = ctx, None
        if not 0 <= bits < _U32:
            raise _unfit(bits=bits)
        ptr, on_device, shape, _keep = _source(weights, device_weights)
        if len(shape) != 3:
            raise ValueError(f"weights of shape {shape}: [expert, in, out] expected")
        self.n_experts, self.inner, self.cols = (int(d) for d in shape)
        h = ctypes.c_void_p()
        check(lib.dpb_expert_weights_new(ctx.h, ptr, on_device, self.n_experts, self.inner, self.cols, bits, ctypes.byref(h)))
        self.h = h

    def free(self):
        if self.h:
            lib.dpb_expert_weights_free(self.h)
            self.h = None


def grouped_product(ctx, groups, x, x_bits, weights, rows_per_token=1, device_x=None, family_dtype=FR_I64):
    """dpb_grouped_product: row i of x[i // rows_per_token] times its expert's matrix, exact.  Returns (table, shape) of
    the [rows, out] tensor, rows in the order of the groups' keys."""
    if not (0 <= x_bits < _U32 and 0 <= rows_per_token < _U32):
        raise _unfit(x_bits=x_bits, rows_per_token=rows_per_token)
    ptr, on_device, shape, _keep = _source(x, device_x)
    if len(shape) != 2 or shape[1] != weights.inner or shape[0] * rows_per_token != groups.n:
        raise ValueError(f"x of shape {shape} for {groups.n} routed rows, {rows_per_token} per token, of {weights.inner} entries")
    h = ctypes.c_void_p()
    check(lib.dpb_grouped_product(ctx.h, family_dtype, groups.h, ptr, on_device, x_bits, rows_per_token, weights.h, ctypes.byref(h)))
    return Mle(ctx, h), (groups.n, weights.cols)
