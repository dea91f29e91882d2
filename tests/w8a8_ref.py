"""Plain forms of the W8A8 and scoring operators in 64 bits, and device helpers for their tests."""
import numpy as np

from llm170_amd import ffi, ops

TYPES = {ffi.F32: np.float32, ffi.F16: np.float16}


def to_bf16(v):
    """f32 -> bf16 bits, to nearest even (finite values)."""
    b = np.ascontiguousarray(v, np.float32).view(np.uint32).astype(np.uint64)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(bits):
    return (np.ascontiguousarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def narrow(v, kind):
    """(bits or values to put on the device, the f32 values they stand for)"""
    if kind == ffi.BF16:
        b = to_bf16(v)
        return b, from_bf16(b)
    a = np.ascontiguousarray(v, np.float32).astype(TYPES[kind])
    return a, a.astype(np.float32)


def quantised(x):
    """x f32 values [t][k] -> (q int8, s f32): quotients of f32 numbers in 64 bits keep their side of every half."""
    x = x.astype(np.float32)
    finite = np.isfinite(x).all(1)
    big = np.where(np.isfinite(x), np.abs(x), 0).max(1)
    s = (big.astype(np.float64) / 127).astype(np.float32)
    s[s < np.float32(2.0**-126)] = 0
    div = np.where(s == 0, 1, s).astype(np.float64)[:, None]
    with np.errstate(invalid="ignore"):
        q = np.rint(x.astype(np.float64) / div)
    q = np.where((s == 0)[:, None] | ~finite[:, None], 0, q)
    return q.astype(np.int8), np.where(finite, s, np.nan).astype(np.float32)


def product(q, s, w, ws):
    """f32 [t][n], rounded as the header says: whole sum, times s, times ws."""
    acc = (q.astype(np.float64) @ w.astype(np.float64).T).astype(np.float32)  # whole numbers below 2^53: exact, then one rounding
    return (acc * s[:, None].astype(np.float32)).astype(np.float32) * ws[None, :].astype(np.float32)


def as_type(v, kind):
    """Bits of v (f32) in a result type."""
    return v.view(np.uint32) if kind == ffi.F32 else to_bf16(v) if kind == ffi.BF16 else v.astype(np.float16).view(np.uint16)


def bits_type(kind):
    return np.uint32 if kind == ffi.F32 else np.uint16


def weights(seed, n, k, s_kind=ffi.F32):
    r = np.random.default_rng(seed)
    w = r.integers(-128, 128, (n, k), dtype=np.int8)
    s = (r.random(n) * 0.02 + 0.001).astype(np.float32)
    bits, val = narrow(s, s_kind)
    return w, bits, val


class Buffers:
    """Device buffers of one test, freed at its end."""

    def __init__(self, cc):
        self.cc, self.held = cc, []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for p in self.held:
            self.cc.free(p)

    def put(self, a, offset=0):
        """a on the device, `offset` bytes behind a 256-byte boundary"""
        a = np.ascontiguousarray(a)
        p = self.cc.alloc(a.nbytes + offset + 64)
        self.held.append(p)
        if a.nbytes:
            self.cc.h2d(p + offset, a)
        return p + offset

    def filled(self, nbytes, byte=0xA5, offset=0):
        return self.put(np.full(nbytes, byte, np.uint8), offset)


def scores(z, targets, top):
    """z f32 values [t][v] -> (logp, entropy, idx, top_logp) in 64 bits, rows of infinities and NaN as documented."""
    z = z.astype(np.float64)
    t, v = z.shape
    logp, ent = np.zeros(t), np.zeros(t)
    idx, lp = np.zeros((t, top), np.int32), np.zeros((t, top))
    for r in range(t):
        row = z[r] + 0.0
        with np.errstate(all="ignore"):
            if np.isnan(row).any() or (row == np.inf).any():
                all_lp, ent[r] = np.full(v, np.nan), np.nan
            elif (row == -np.inf).all():
                all_lp, ent[r] = np.full(v, -np.inf), 0.0
            else:
                m = row.max()
                e = np.exp(row - m)
                all_lp = row - m - np.log(e.sum())
                p = e / e.sum()
                ent[r] = -(p[p > 0] * all_lp[p > 0]).sum()
        order = np.argsort(np.where(np.isnan(row), -np.inf, -row) if np.isnan(row).any() else -row, kind="stable")
        if np.isnan(row).any():  # NaN first, by index, then the rest
            order = np.concatenate([np.flatnonzero(np.isnan(row)), [i for i in np.argsort(-row, kind="stable") if not np.isnan(row[i])]])
        idx[r] = order[:top]
        lp[r] = all_lp[idx[r]]
        g = targets[r]
        logp[r] = 0.0 if g < 0 else np.nan if g >= v else all_lp[g]
    return logp, ent, idx, lp
