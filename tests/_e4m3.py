"""The e4m3 cache in 64 bits: codec, block scales, append and attention, as
the header states them (tge_kv_append_rows, tge_attention_rows)."""
import ctypes as C
import math

import numpy as np

import synth
import tge_kv as tk

HALF_STEP = {tk.ROWS_F32: 2.0 ** -24, tk.ROWS_F16: 2.0 ** -11, tk.ROWS_BF16: 2.0 ** -8}
MIN_EXP, MAX_EXP = -15, 7


def _positive():
    c = np.arange(127)
    e, m = c >> 3, c & 7
    return np.where(e > 0, (8.0 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)


POSITIVE = _positive()  # value of codes 0..126 (127: NaN)


def decode(codes):
    codes = np.asarray(codes, np.uint8)
    mag = np.append(POSITIVE, np.nan)[codes & 127]
    return np.where(codes > 127, -mag, mag)


def encode(x):
    """Nearest code, ties to the even one; out of range the largest; NaN: 0."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.where(np.isnan(x), 0.0, np.abs(x)), 448.0)
    i = np.clip(np.searchsorted(POSITIVE, a, side="right") - 1, 0, 125)
    lo, hi = a - POSITIVE[i], POSITIVE[i + 1] - a
    code = np.where((hi < lo) | ((hi == lo) & (i % 2 == 1)), i + 1, i)
    return (code + np.where(np.signbit(x) & ~np.isnan(x), 128, 0)).astype(np.uint8)


def exponent(most):
    """The smallest e with most <= 448 * 2^e, clamped."""
    e = MIN_EXP
    while e < MAX_EXP and most > 448.0 * 2.0 ** e:
        e += 1
    return e


def f32(x):
    return np.asarray(x, np.float32)


def round_bf16(x):
    u = f32(x).view(np.uint32).astype(np.uint64)
    u = (u + 0x7FFF + ((u >> 16) & 1)) >> 16
    return (u.astype(np.uint32) << 16).view(np.float32)


def as_type(x, row_type):
    """fp32 values that the row type holds."""
    if row_type == tk.ROWS_F16:
        return f32(x).astype(np.float16).astype(np.float32)
    return round_bf16(x) if row_type == tk.ROWS_BF16 else f32(x)


def to_bytes(x, row_type):
    x = np.ascontiguousarray(f32(x))
    if row_type == tk.ROWS_F16:
        return x.astype(np.float16)
    return (x.view(np.uint32) >> 16).astype(np.uint16) if row_type == tk.ROWS_BF16 else x


def from_bytes(x, row_type):
    if row_type == tk.ROWS_F16:
        return x.view(np.float16).astype(np.float32)
    if row_type == tk.ROWS_BF16:
        return (x.view(np.uint16).astype(np.uint32) << 16).view(np.float32)
    return x.view(np.float32)


def np_type(row_type):
    return np.float32 if row_type == tk.ROWS_F32 else np.uint16


def rotate(x, bias, cos, sin, hd, fma=True):
    """x + bias, then the halves of every head turned: l c - h s, l s + h c in
    fp32, the second product rounded, then one rounding (fma) or two."""
    with np.errstate(invalid="ignore", over="ignore"):
        y = f32(f32(x) + f32(bias)).reshape(x.shape[0], -1, hd)
        lo, hi = y[..., : hd // 2], y[..., hd // 2:]
        c, s = f32(cos)[:, None], f32(sin)[:, None]

        def one(a, ca, b, cb):
            t = f32(b * cb)
            if fma:
                return f32(a.astype(np.float64) * ca + t)
            return f32(f32(a * ca) + t)
        return np.concatenate([one(lo, c, hi, -s), one(lo, s, hi, c)], -1).reshape(x.shape[0], -1)


class Cache:
    """One session's cache: codes [rows][kvh][hd] and exponents [pages][kvh] of K and V."""

    def __init__(self, kvh, hd):
        self.kvh, self.hd = kvh, hd
        self.codes = [np.zeros((0, kvh, hd), np.uint8) for _ in range(2)]
        self.exps = [np.zeros((0, kvh), np.int64) for _ in range(2)]

    def append(self, ctx, k, v):
        for part, x in enumerate((k, v)):
            x = np.asarray(x, np.float64).reshape(-1, self.kvh, self.hd)
            codes, exps = list(self.codes[part][:ctx]), list(self.exps[part][: -(-ctx // 16)])
            pos = ctx
            while pos < ctx + len(x):
                slot = pos % 16
                n = min(16 - slot, ctx + len(x) - pos)
                rows = x[pos - ctx: pos - ctx + n]
                with np.errstate(invalid="ignore"):
                    need = [exponent(np.max(np.where(np.isnan(r), 0.0, np.abs(r)))) for r in rows.transpose(1, 0, 2)]
                if slot == 0:
                    exps.append(np.array(need))
                else:
                    had = exps[-1]
                    exps[-1] = np.maximum(had, need)
                    for i in range(pos - slot, pos):
                        codes[i] = encode(decode(codes[i]) * 2.0 ** (had - exps[-1])[:, None])
                for r in rows:
                    codes.append(encode(r * 2.0 ** -exps[-1].astype(np.float64)[:, None]))
                pos += n
            self.codes[part], self.exps[part] = np.array(codes), np.array(exps)
        return self

    def values(self, part):
        e = np.repeat(self.exps[part], 16, 0)[: len(self.codes[part])]
        return decode(self.codes[part]) * 2.0 ** e.astype(np.float64)[..., None]


def attend(cache, ctx, q, qh, scale=None):
    """(out, bound) [n][qh*hd] in 64 bits: what the kernel's roundings may
    change at most, apart from the output's own.

    q is rounded to f16 after scaling (half a step 2^-11 of each value, so a
    score moves by at most d_j = (2^-11 + (hd + 2) 2^-24) sum|q k_j| scale, the
    fp32 sum of hd products and the scaling included; a value below f16's
    normal range by 2^-25), weights are rounded to f16 (2^-11, and 2^-25 of the
    largest for subnormals; exp2 itself 2^-22), sums of L terms are fp32. With
    every weight off by a factor within exp(+-d) (1 +- u),
    |out' - out| <= (exp(2d) (1 + 2u) - 1) * sum w |v| + L 2^-24 (2 sum w|v|).
    """
    n, kvh, hd = q.shape[0], cache.kvh, cache.hd
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    k, v = cache.values(0), cache.values(1)
    q = np.asarray(q, np.float64).reshape(n, qh, hd)
    out, bound = np.zeros((n, qh, hd)), np.zeros((n, qh, hd))
    for h in range(qh):
        kh, vh = k[:, h // (qh // kvh)], v[:, h // (qh // kvh)]
        for i in range(n):
            length = ctx + i + 1
            s = kh[:length] @ q[i, h] * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            reach = np.abs(kh[:length]) @ np.abs(q[i, h]) * scale
            lost = 2.0 ** -25 * np.abs(kh[:length]).sum(1)  # q below f16's normal range (log2 domain)
            d = np.max((2.0 ** -11 + (hd + 2) * 2.0 ** -24) * reach + lost)
            u = 2.0 ** -11 + 2.0 ** -22
            absv = w @ np.abs(vh[:length])
            sub = length * 2.0 ** -24 * np.abs(vh[:length]).max(0)  # subnormal weights, twice 2^-25
            out[i, h] = w @ vh[:length]
            bound[i, h] = (math.exp(2 * d) * (1 + 2 * u) - 1) * absv + 2 * length * 2.0 ** -24 * absv + sub
    return out.reshape(n, -1), bound.reshape(n, -1)


# Steps whose attention items read more pages than the kernel holds block
# numbers for at a time (1024): (query heads, KV heads, head_dim, ctx, new
# tokens, sessions over the same pages) -> rows of a tile / 32.
LONG_ITEMS = {(4, 1, 64, 17000, 1, 900): 1, (40, 1, 128, 17000, 1, 600): 2, (8, 1, 256, 17000, 1, 300): 1,
              (64, 1, 256, 17000, 1, 300): 2, (64, 1, 64, 17000, 2000, 1): 4, (128, 1, 128, 17000, 1100, 1): 2,
              (128, 1, 128, 17000, 2300, 1): 4}


class Rows:
    """Device rows of a type, `gap` elements between them, the gaps (and the
    rows behind the last) filled with a pattern that must stay."""

    def __init__(self, x, row_type, gap=0, spare=0):
        x = np.asarray(x, np.float32)
        self.n, self.len, self.type, self.stride = x.shape[0], x.shape[1], row_type, x.shape[1] + gap
        buf = np.full((self.n + spare, self.stride), 0x4242 if row_type else np.float32(77.0), np_type(row_type))
        buf[: self.n, : self.len] = to_bytes(x, row_type).view(np_type(row_type))
        self.before, self.dev = buf, tk.DeviceArray.from_numpy(buf)
        self.ptr = self.dev.ptr

    def read(self):
        """The rows; asserts that nothing around them changed."""
        got = self.dev.numpy()
        assert np.array_equal(got[:, self.len:], self.before[:, self.len:]), "gaps between the rows changed"
        assert np.array_equal(got[self.n:], self.before[self.n:]), "rows behind the last one changed"
        return from_bytes(np.ascontiguousarray(got[: self.n, : self.len]), self.type)


class Case:
    """Sessions on one e4m3 pool: (ctx, n_new) each, contexts stored first."""

    def __init__(self, qh, kvh, hd, sessions, seed=0, layers=1, loud=True):
        self.qh, self.kvh, self.hd, self.sessions, self.layers = qh, kvh, hd, list(sessions), layers
        self.rng = np.random.default_rng(seed)
        need = sum(-(-(c + n) // 16) for c, n in self.sessions)
        self.table = synth.fragmented_table(need + 5, seed + 1)
        self.pool = tk.KvPool(layers, need + 5, kvh, hd, tk.KV_E4M3)
        self.pages = [[self.table.allocate() for _ in range(-(-(c + n) // 16))] for c, n in self.sessions]
        self.gain = np.ones(kvh * hd)
        if loud:
            self.gain[self.rng.permutation(kvh * hd)[: max(1, kvh * hd // 100)]] = 8.0
        self.cache = [Cache(kvh, hd) for _ in self.sessions]

    def rows(self, n, row_type):
        k = as_type(self.rng.standard_normal((n, self.kvh * self.hd)) * self.gain, row_type)
        return k, as_type(self.rng.standard_normal((n, self.kvh * self.hd)), row_type)

    def plan(self, which=None):
        ss = [tk.Session(c, n, p) for (c, n), p in zip(self.sessions, self.pages)] if which is None else which
        return tk.Batch().plan(self.pool, ss, self.qh)

    def fill(self, row_type=tk.ROWS_F32, layer=0, chunk=None):
        """Store the contexts, whole or in calls of `chunk` tokens."""
        for (c, _), p, cache in zip(self.sessions, self.pages, self.cache):
            at = 0
            while at < c:
                n = min(chunk or c, c - at)
                k, v = self.rows(n, row_type)
                self.plan([tk.Session(at, n, p)]).append_rows(
                    self.pool, layer, tk.append_rows_args(row_type, *(self._keep(Rows(x, row_type)) for x in (k, v))))
                tk.hip().sync()
                cache.append(at, k, v)
                at += n
        return self

    def _keep(self, x):
        self.kept = getattr(self, "kept", [])[-8:] + [x]
        return x

    def step_rows(self, row_type, nan=False):
        return [self.rows(n, row_type) for _, n in self.sessions]

    def check_pool(self, batch, layer=0):
        """The gathered cache equals the model's, codes and scales, bit for bit."""
        for s, ((c, n), cache) in enumerate(zip(self.sessions, self.cache)):
            count = len(cache.codes[0])
            got = batch.gather(self.pool, layer, s, count)
            for part in range(2):
                want_e = ((cache.exps[part] + 127) << 7).astype(np.uint16)
                assert np.array_equal(got[2 + part], want_e), (s, part, "scales")
                same = got[part].reshape(count, self.kvh, self.hd) == cache.codes[part]
                assert same.all(), (s, part, "codes", np.argwhere(~same)[:5])

    def close(self):
        self.pool.close()


def raw_layer(pool, layer=0):
    """The layer's blocks [pages][kvh][2][16 W] and scales [pages][kvh][2] (bf16 bits)."""
    view = pool.layer(layer)
    n = pool.pages * pool.kv_heads
    codes = np.empty((n, view.block_bytes), np.uint8)
    scales = np.empty((n, 2), np.uint16)
    tk.hip().sync()
    tk.hip().ok(tk.hip().h.hipMemcpy(codes.ctypes.data_as(C.c_void_p), C.c_void_p(view.k), codes.nbytes, 2), "D2H")
    tk.hip().ok(tk.hip().h.hipMemcpy(scales.ctypes.data_as(C.c_void_p), C.c_void_p(view.k_scales), scales.nbytes, 2),
                "D2H")
    return codes.reshape(pool.pages, pool.kv_heads, 2, -1), scales.reshape(pool.pages, pool.kv_heads, 2)
