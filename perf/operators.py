"""Forward operators of quantised models and their transposes, as a proving program calls them: embedding lookups with a
fixed-point scale, sums of rows by sorted key (the lookup's transpose: tokens or experts as keys, field elements or
integers as rows), and integer matrix products grouped by expert.

Every output is a whole number or a field element in the library's layout (BN254: four 64-bit Montgomery limbs;
Goldilocks extension: two canonical words), compared for equality.  The plain form works on 16-bit digits of field
elements in 64-bit integers, and on float64 products whose sums stay below 2^53 for the matrix products.
"""
import importlib
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FR_P = 21888242871839275222246405745257275088548364400416034343698204186575808495617
GL_P = 2**64 - 2**32 + 1


def _package():
    # the package's directory name is not an identifier: it is loaded by path, as its own tests and benchmark do
    name = "deep_prove_b200"
    if name not in sys.modules:
        pkg = os.path.join(ROOT, "deep-prove_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(pkg, "__init__.py"),
                                                      submodule_search_locations=[pkg])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name], importlib.import_module(name + ".forward")


_CTX = []


def _context():
    # one context per process and GPU, as a prover process keeps it
    if not _CTX:
        _CTX.append(_package()[0].Context(torch.cuda.current_device()))
    return _CTX[0]


def lg(x):
    return max(int(x) - 1, 0).bit_length()


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one generated token's row of a large vocabulary: all latency
        dict(name="lookup_one_token", kind="lookup", tokens=1, vocab=262144, width=1152, bits=12, entry=4, mult=34, shift=0, padded=False),
        # a prompt of the GPT-2-small shape, rescaled to the activations' bits, as the padded table a sumcheck takes
        dict(name="lookup_prompt_padded", kind="lookup", tokens=509, vocab=50257, width=768, bits=12, entry=4, mult=27713, shift=10, padded=True),
        # a batch of long prompts over 64-bit entries
        dict(name="lookup_batch_i64", kind="lookup", tokens=16384, vocab=32000, width=4096, bits=12, entry=8, mult=64, shift=0, padded=False),
        # the embedding claim of a 512-token proof over a large vocabulary: eq weights summed by token
        dict(name="token_sums_fr_prompt", kind="sums", field="fr", keys="tokens", rows=512, n_keys=262144, width=0, weights=True, top=1, mult=34),
        # the same for a long batch, ragged, over Goldilocks
        dict(name="token_sums_gl_batch", kind="sums", field="gl", keys="tokens", rows=200003, n_keys=50257, width=0, weights=True, top=1, mult=1),
        # the lookup's integer gradient over a reduced vocabulary (the bounded CPU sample's sizes)
        dict(name="row_sums_fr_tokens", kind="sums", field="fr", keys="tokens", rows=2048, n_keys=4000, width=192, weights=False, top=1, mult=1),
        # the routed rows of a grouped product bound by the row point, one table row per expert
        dict(name="row_sums_fr_experts", kind="sums", field="fr", keys="experts", rows=8192, n_keys=8, width=4096, weights=True, top=2, mult=1),
        dict(name="row_sums_gl_experts_ragged", kind="sums", field="gl", keys="experts", rows=1996, n_keys=60, width=1152, weights=True, top=4, mult=1),
        # one generated token through its two experts (Llama-2-7B-style feed-forward sizes): the weights' bytes count
        dict(name="experts_one_token", kind="experts", tokens=1, top=2, n_experts=8, inner=4096, cols=11008, x_bits=14, w_bits=12),
        # a prompt through Gemma-3-1B-style feed-forward sizes
        dict(name="experts_prompt", kind="experts", tokens=512, top=2, n_experts=8, inner=1152, cols=6912, x_bits=14, w_bits=12),
        # many small experts, 8-bit operands, ragged sizes everywhere
        dict(name="experts_ragged_8bit", kind="experts", tokens=777, top=4, n_experts=60, inner=769, cols=1003, x_bits=8, w_bits=8),
        # a batch of long prompts: bound by the multiplications
        dict(name="experts_batch", kind="experts", tokens=8192, top=2, n_experts=8, inner=4096, cols=11008, x_bits=14, w_bits=12),
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["lookup", "sums", "sums", "experts"])
    if kind == "lookup":
        width = log_int(16, 4096)
        return dict(kind=kind, tokens=log_int(1, min(16384, 2**26 // width)), vocab=log_int(100, 262144 if width <= 1152 else 32000),
                    width=width, bits=rng.choice([8, 10, 12]), entry=rng.choice([4, 4, 8]), mult=log_int(1, 2**20),
                    shift=rng.choice([0, 0, rng.randint(1, 20)]), padded=rng.random() < 0.4)
    if kind == "sums":
        field, form = rng.choice(["fr", "gl"]), rng.choice(["claim", "claim", "gradient", "experts", "experts"])
        if form == "claim":
            return dict(kind=kind, field=field, keys="tokens", rows=log_int(1, 200003), n_keys=log_int(100, 262144), width=0,
                        weights=True, top=1, mult=rng.choice([1, log_int(2, 2**20)]))
        if form == "gradient":
            return dict(kind=kind, field=field, keys="tokens", rows=log_int(1, 4096), n_keys=log_int(100, 4000),
                        width=log_int(16, 768), weights=False, top=1, mult=rng.choice([1, log_int(2, 2**20)]))
        top = rng.choice([1, 2, 4])
        return dict(kind=kind, field=field, keys="experts", rows=top * log_int(1, 2048), n_keys=log_int(4, 128),
                    width=log_int(16, 4096), weights=True, top=top, mult=1)
    wide = rng.random() < 0.6
    n_experts = log_int(4, 64)
    inner = log_int(64, 4096)
    cols = log_int(64, min(11008, 2**28 // (inner * n_experts)))
    return dict(kind=kind, tokens=log_int(1, 2048), top=rng.choice([1, 2, 4]), n_experts=n_experts, inner=inner, cols=cols,
                x_bits=14 if wide else 8, w_bits=rng.choice([12, 8]) if wide else 8)


# ------------------------------------------------------------------------------------------------ inputs
class State:
    """What the program keeps: integer tensors and field tables on the device, library handles over them."""

    def __init__(self, case, seed):
        self.case = case
        self.own = own
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)
        self.keep, self.handles, self.last = [], [], []
        if self.own:
            self.dpb, self.fwd = _package()
            self.ctx = _context()
            # The program's torch work runs on the library's stream from here on: the calls return before their results
            # are written, and what they free may still be read by work that is queued.
            torch.cuda.set_stream(torch.cuda.ExternalStream(self.ctx.stream))

    def __del__(self):
        try:
            for h in self.last + self.handles[::-1]:
                h.free()
        except Exception:
            pass  # interpreter shutdown

    def ints(self, bits, shape, dtype=torch.int64):
        half = 1 << (bits - 1)
        return torch.randint(-half, half, shape, generator=self.gen, device="cuda", dtype=dtype)

    def wrap(self, t, dtype):
        """A library handle over a tensor's memory, padded to a power of two entries as its tables are."""
        n = t.numel() // (2 if dtype == self.dpb.GL_EXT else 4 if dtype == self.dpb.FR else 1)
        if n & (n - 1):
            raise ValueError("pad the tensor first")
        self.keep.append(t)
        h = self.ctx.wrap_device(t.data_ptr(), dtype, n)
        self.handles.append(h)
        return h

    def tensor(self, t):
        """An int64 tensor in the device form the library's calls take: (handle, shape)."""
        flat = torch.zeros(1 << lg(max(t.numel(), 2)), dtype=torch.int64, device="cuda")
        flat[:t.numel()] = t.reshape(-1)
        return self.wrap(flat, self.dpb.GL_BASE), tuple(t.shape)


def _tokens(s, n, vocab):
    # text: a few tokens are frequent, most are rare
    u = torch.rand(n, generator=s.gen, device="cuda", dtype=torch.float64)
    ranks = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp_(0, vocab - 1)
    return (ranks * 2654435761) % vocab


def _routes(s, tokens, top, n_experts):
    # a router's choice of `top` different experts per token; some experts are preferred, some may get no row
    bias = torch.randn(n_experts, generator=s.gen, device="cuda") * 0.7
    gumbel = -torch.log(-torch.log(torch.rand(tokens, n_experts, generator=s.gen, device="cuda").clamp(1e-6, 1 - 1e-6)))
    return (bias + gumbel).topk(min(top, n_experts), dim=1).indices.reshape(-1).contiguous()


def _field(s, field, n):
    """n uniform field elements in the library's layout, as the entries of an eq table are."""
    t = torch.randint(-2**63, 2**63 - 1, (n, 4 if field == "fr" else 2), generator=s.gen, device="cuda", dtype=torch.int64)
    if field == "fr":
        t[:, 3] &= (1 << 60) - 1
        return t
    return torch.where((t < 0) & (t >= -(2**32) + 1), t & (2**62 - 1), t)  # below the modulus


def prepare(case, seed):
    s = State(case, seed)
    kind = case["kind"]
    if kind == "lookup":
        v, w = case["vocab"], case["width"]
        ps = 1 << lg(w)
        table = torch.zeros((1 << lg(v), ps), dtype=torch.int32 if case["entry"] == 4 else torch.int64, device="cuda")
        table[:v, :w] = s.ints(case["bits"], (v, w), torch.int32)
        tokens = _tokens(s, case["tokens"], v)
        if s.own:
            s.table = s.wrap(table.reshape(-1), s.dpb.FR_I32 if case["entry"] == 4 else s.dpb.FR_I64)
            s.tokens = s.tensor(tokens)
        else:
            s.table, s.tokens = table, tokens
    elif kind == "sums":
        n, k = case["rows"], case["n_keys"]
        keys = _tokens(s, n, k) if case["keys"] == "tokens" else _routes(s, n // case["top"], case["top"], k)
        n = keys.numel()
        weights = _field(s, case["field"], 1 << lg(n)) if case["weights"] else None
        rows = s.ints(14, (n // case["top"], case["width"])) if case["width"] else None
        if s.own:
            s.family = s.dpb.FR if case["field"] == "fr" else s.dpb.GL_EXT
            s.keys = s.tensor(keys)
            s.weights = s.wrap(weights.reshape(-1), s.family) if weights is not None else None
            s.rows = s.tensor(rows) if rows is not None else None
        else:
            s.keys, s.weights, s.rows = keys, weights, rows
    else:
        g, k, c = case["n_experts"], case["inner"], case["cols"]
        keys = _routes(s, case["tokens"], case["top"], g)
        x = s.ints(case["x_bits"], (case["tokens"], k))
        w = s.ints(case["w_bits"], (g, k, c), torch.int16)
        if s.own:
            s.keys, s.x = s.tensor(keys), s.tensor(x)
            raw, shape = s.tensor(w)
            torch.cuda.synchronize()
            s.weights = s.fwd.ExpertWeights(s.ctx, None, case["w_bits"], device_weights=(raw, shape))
            s.ctx.sync()  # the integers are laid out for the products: the program keeps that form only
            s.handles.remove(raw)
            raw.free()
            s.keep.pop()
            s.handles.append(s.weights)
        else:
            s.keys, s.x, s.w = keys, x, w
    torch.cuda.synchronize()  # the library's stream reads what torch's stream wrote
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _digits(words, n_words):
    """[..., n_words] 64-bit words (as int64) -> [..., 4 n_words] 16-bit digits."""
    sh = torch.arange(0, 64, 16, device=words.device)
    return ((words.unsqueeze(-1) >> sh) & 0xFFFF).reshape(*words.shape[:-1], 4 * n_words)


def _const_digits(value, n, device):
    return torch.tensor([(value >> (16 * i)) & 0xFFFF for i in range(n)], dtype=torch.int64, device=device)


def _carry(d, n):
    """Digits of any size and sign -> n digits in 0..2^16 and one more, signed, with all that is above them."""
    d = list(d.unbind(-1))
    c = torch.zeros_like(d[0])
    for i in range(n):
        v = d[i] + c
        d[i] = v & 0xFFFF
        c = v >> 16
    return torch.stack(d[:n] + [d[n] + c if len(d) > n else c], dim=-1)


def _mod(d, p, n):
    """A number in n signed digits -> its residue mod p in n digits of 16 bits."""
    pd = _const_digits(p, n, d.device)
    fold = _const_digits(pow(2, 16 * n, p), n, d.device)
    for _ in range(4):  # what stands above digit n - 1 comes down as a multiple of 2^(16 n) mod p
        d = _carry(d, n)
        d = d[..., :n] + d[..., n:] * fold
    d = _carry(d, n)
    value = sum(d[..., i].double() * 2.0 ** (16 * i) for i in range(n - 4, n + 1))
    q = torch.floor(value / float(p)).long()
    d = _carry(torch.cat([d[..., :n] - q.unsqueeze(-1) * pd, d[..., n:]], dim=-1), n)
    for _ in range(2):  # the estimate is off by one at most, either way
        d = _carry(torch.cat([d[..., :n] + (d[..., n:] < 0) * pd, d[..., n:]], dim=-1), n)
        less = _carry(torch.cat([d[..., :n] - pd, d[..., n:]], dim=-1), n)
        d = torch.where(less[..., n:] >= 0, less, d)
    return d[..., :n]


def _words(digits):
    """[..., 4 m] digits -> [..., m] words as int64."""
    d = digits.reshape(*digits.shape[:-1], -1, 4)
    return d[..., 0] | (d[..., 1] << 16) | (d[..., 2] << 32) | (d[..., 3] << 48)


def _by_key(keys, n_keys, values):
    """values [n, c] int64 summed by key -> [n_keys, c]"""
    return torch.zeros((n_keys, values.shape[1]), dtype=torch.int64, device=values.device).index_add_(0, keys, values)


def _plain_lookup(s):
    c = s.case
    y = s.table[s.tokens, :c["width"]].long() * c["mult"]
    if c["shift"]:
        y = (y + (1 << (c["shift"] - 1))) >> c["shift"]
    if not c["padded"]:
        return y
    out = torch.zeros((1 << lg(c["tokens"]), 1 << lg(c["width"])), dtype=torch.int64, device="cuda")
    out[:c["tokens"], :c["width"]] = y
    return out


def _plain_sums(s):
    c = s.case
    p, comps, n_dig = (FR_P, 1, 16) if c["field"] == "fr" else (GL_P, 2, 4)
    n, k, width = s.keys.numel(), c["n_keys"], max(c["width"], 1)
    out = torch.zeros((1 << lg(k), 1 << lg(width), comps * n_dig // 4), dtype=torch.int64, device="cuda")

    def finish(d):  # [..., comps, digits of the sum] -> words, times the multiplier
        d = _mod(_mod(d, p, n_dig) * c["mult"], p, n_dig)
        return _words(d).reshape(*d.shape[:-2], -1)

    if s.weights is not None:
        wd = _digits(s.weights[:n], comps * n_dig // 4).reshape(n, comps, n_dig)
    if s.rows is None:
        sums = _by_key(s.keys, k, wd.reshape(n, -1)).reshape(k, comps, n_dig)
        out[:k, 0] = finish(sums)
    elif s.weights is None:
        total = _by_key(s.keys, k, s.rows)  # integers: |sum| < 2^13 * 2^17
        one = (1 << 256) % p if c["field"] == "fr" else 1
        d = torch.zeros((k, width, comps, n_dig), dtype=torch.int64, device="cuda")
        d[:, :, 0] = total.unsqueeze(-1) * _const_digits(one, n_dig, "cuda")
        out[:k, :width] = finish(d)
    else:
        x = s.rows.double()
        wd = wd.reshape(n, -1).double()
        prod = torch.empty((k, width, comps, n_dig), dtype=torch.int64, device="cuda")
        for e in range(k):
            r = (s.keys == e).nonzero().reshape(-1)
            # 2^16 * 2^13 * rows: exact in float64
            prod[e] = (x[r // c["top"]].t() @ wd[r]).long().reshape(width, comps, n_dig)
        out[:k, :width] = finish(prod)
    return out


def _plain_experts(s):
    c = s.case
    out = torch.empty((s.keys.numel(), c["cols"]), dtype=torch.int64, device="cuda")
    for e in range(c["n_experts"]):
        r = (s.keys == e).nonzero().reshape(-1)
        # 2^13 * 2^11 * inner: exact in float64
        out[r] = (s.x[r // (s.keys.numel() // c["tokens"])].double() @ s.w[e].double()).long()
    return out


# ------------------------------------------------------------------------------------------------ one pass
class _DeviceWords:
    def __init__(self, mle, words):
        self.__cuda_array_interface__ = {"shape": (words,), "typestr": "<i8", "data": (mle.device_ptr, False), "version": 3}


def _view(mle, shape):
    """A device table's 64-bit words as a torch tensor, without a copy."""
    return torch.as_tensor(_DeviceWords(mle, math.prod(shape)), device="cuda").view(shape)


def run(s):
    c = s.case
    kind = c["kind"]
    if not s.own:
        return _plain_lookup(s) if kind == "lookup" else _plain_sums(s) if kind == "sums" else _plain_experts(s)
    for h in s.last:
        h.free()
    if kind == "lookup":
        out, shape = s.fwd.embedding_lookup(s.ctx, s.table, c["vocab"], c["width"], None, multiplier=c["mult"],
                                            right_shift=c["shift"], row_stride=1 << lg(c["width"]), padded=c["padded"],
                                            device_tokens=s.tokens)
        s.last = [out]
        return _view(out, shape)
    if kind == "sums":
        groups = s.fwd.RowGroups(s.ctx, None, c["n_keys"], device_keys=s.keys)
        out = groups.sums(s.family, weights=s.weights, device_rows=s.rows, rows_per_token=c["top"], multiplier=c["mult"])
        s.last = [out, groups]
        return _view(out, (1 << lg(c["n_keys"]), 1 << lg(max(c["width"], 1)), 4 if c["field"] == "fr" else 2))
    groups = s.fwd.RowGroups(s.ctx, None, c["n_experts"], device_keys=s.keys)
    out, shape = s.fwd.grouped_product(s.ctx, groups, None, c["x_bits"], s.weights,
                                       rows_per_token=groups.n // c["tokens"], device_x=s.x)
    s.last = [out, groups]
    return _view(out, shape)


def work(case):
    kind = case["kind"]
    if kind == "lookup":
        n, w = case["tokens"], case["width"]
        rows = min(n, case["vocab"])  # a row that several tokens name is read once
        written = (1 << lg(n)) * (1 << lg(w)) if case["padded"] else n * w
        return {"bytes": rows * w * case["entry"] + 8 * n + 8 * written, "flops": 2 * n * w}
    es = 32 if case.get("field") == "fr" else 16
    if kind == "sums":
        n, w = case["rows"], max(case["width"], 1)
        out = (1 << lg(case["n_keys"])) * (1 << lg(w)) * es
        rows = n // case["top"] * w * 8 if case["width"] else 0
        # a 14-bit integer times a field element: one multiplication per 32-bit word of the element
        return {"bytes": 8 * n + (n * es if case["weights"] else 0) + rows + out,
                "flops": 2 * n * w * (es // 4 if case["weights"] else 1)}
    n, k, c = case["tokens"] * min(case["top"], case["n_experts"]), case["inner"], case["cols"]
    used = min(case["n_experts"], n)
    weight_bytes = 1 if case["w_bits"] <= 8 else 2
    return {"bytes": case["tokens"] * k * 8 + used * k * c * weight_bytes + n * c * 8 + 8 * n, "flops": 2 * n * k * c}


# ------------------------------------------------------------------------------------------------ the definition
def exact(case, seed):
    """The operators in Python integers or 64-bit integers on the host, on the inputs that `prepare` makes."""
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    kind = case["kind"]
    if kind == "lookup":
        w = case["width"]
        if case["tokens"] * w > 2**24:
            return None
        t = s.tokens.cpu().numpy()
        rows = np.stack([s.table[int(i), :w].cpu().numpy() for i in np.unique(t)]).astype(np.int64)
        y = rows[np.searchsorted(np.unique(t), t)] * np.int64(case["mult"])
        if case["shift"]:
            y = np.floor_divide(y + np.int64(1 << (case["shift"] - 1)), np.int64(1 << case["shift"]))
        if case["padded"]:
            y = np.pad(y, ((0, (1 << lg(case["tokens"])) - case["tokens"]), (0, (1 << lg(w)) - w)))
        return y
    if kind == "sums":
        fr = case["field"] == "fr"
        n_words, p = (4, FR_P) if fr else (2, GL_P)
        n, k, width = s.keys.numel(), case["n_keys"], max(case["width"], 1)
        if n * width > 2**22:
            return None
        keys = s.keys.cpu().numpy()
        if s.weights is not None:
            wb = s.weights[:n].cpu().numpy().astype("<i8").tobytes()
            size = 32 if fr else 8
            elems = [int.from_bytes(wb[i:i + size], "little") for i in range(0, len(wb), size)]
            elems = [[e] for e in elems] if fr else [elems[2 * i:2 * i + 2] for i in range(n)]
        else:
            one = (1 << 256) % p if fr else 1  # integers as field elements (BN254: in Montgomery form)
            elems = [[one] if fr else [one, 0]] * n
        comps = len(elems[0])
        acc = {}
        rows = s.rows.cpu().numpy() if s.rows is not None else None
        for i in range(n):
            a = acc.setdefault(int(keys[i]), np.zeros((width, comps), dtype=object))
            x = rows[i // case["top"]].astype(object) if rows is not None else np.ones(1, dtype=object)
            for j in range(comps):
                a[:, j] += x * elems[i][j]
        out = np.zeros((1 << lg(k), 1 << lg(width), n_words), dtype=np.int64)
        for key, a in acc.items():
            for c in range(width):
                raw = b"".join(int(v * case["mult"] % p).to_bytes(32 if fr else 8, "little") for v in a[c])
                out[key, c] = np.frombuffer(raw, dtype="<i8")
        return out
    g, k, c = case["n_experts"], case["inner"], case["cols"]
    n = s.keys.numel()
    if n * k * c > 2**36 or min(g, n) * k * c > 2**28:
        return None
    keys, x, out = s.keys.cpu().numpy(), s.x.cpu().numpy(), np.zeros((n, c), dtype=np.int64)
    for e in range(g):
        r = np.flatnonzero(keys == e)
        if r.size:
            w = s.w[e].cpu().numpy()
            # two 7-bit halves of the rows: every product and sum is a whole number below 2^53
            hi, lo = np.divmod(x[r // (n // case["tokens"])], 128)
            wf = w.astype(np.float64)
            out[r] = (hi.astype(np.float64) @ wf).astype(np.int64) * 128 + (lo.astype(np.float64) @ wf).astype(np.int64)
    return out
