"""numpy restatement of the 8-bit Adam step whose first moment is rounded against thresholds (adam8_step(first_moment="threshold"), what HipAdam(state_bits=8) takes), on top of
adam8_ref (whose first moment is rounded to nearest): fp32 arithmetic, one IEEE rounding per operation, so that the device's results can be compared bit for bit."""
import numpy as np

import adam8_ref as A8
from helpers import drop_u16

F = np.float32
M_STREAM = 0x6D38
ROOT = A8.ROOT.copy()
ROOT[254] = np.inf              # the root of a second moment beyond fp32's range


def m_thresholds(n, step, first=0):
    """16 uniform bits per element and step (`first`: the flat index of the first one), as 20 bits with the middle of the interval: odd multiples of 2^-17"""
    i = np.arange(first, first + n, dtype=np.int64)
    return drop_u16(int(step) & 0xFFFFFFFF, M_STREAM, i >> 26, i & ((1 << 26) - 1)).astype(np.uint32) * np.uint32(16) + np.uint32(8)


def encode_e4m3(x, u):
    """magnitude rounded up or down by the threshold u (20 bits), sign kept; NaN and infinities -> 0x7f"""
    bits = x.astype(F).view(np.uint32)
    a = bits & np.uint32(0x7FFFFFFF)
    with np.errstate(invalid="ignore", over="ignore"):
        large = ((a.astype(np.int64) + u) >> 20) - 960
        small = np.floor(np.nan_to_num(a.view(F) * F(512), posinf=0) + u.astype(F) * F(2.0 ** -20)).astype(np.int64)
    code = np.where(a >= 0x3C800000, large, small) + ((bits >> 24) & 0x80)
    return np.where(np.isfinite(x), code, 0x7F).astype(np.uint8)


def encode(m, r, step, first=0):
    n = m.size
    from_zero = A8.thresholds
    try:
        if first:
            A8.thresholds = lambda count, t: (
                (np.arange(first, first + count, dtype=np.uint64) * np.uint64(0xC13FA9A9) + np.uint64((t * 0x91E10DA5) & 0xFFFFFFFF)) & np.uint64(0xFFFFFFFF)).astype(np.uint32)
        cm, cr, ex = A8.encode(m, r, step)
    finally:
        A8.thresholds = from_zero
    pad = -n % A8.BLOCK
    x = np.concatenate([m.reshape(-1), np.zeros(pad, F)]).astype(F).reshape(-1, A8.BLOCK)
    with np.errstate(invalid="ignore", over="ignore"):
        y = (x * (F(2) ** (-ex[:, 0].astype(np.int64)).astype(F))[:, None]).reshape(-1)
    return encode_e4m3(y, m_thresholds(y.size, step, first))[:n], overflowed(cr, m, r), ex


def overflowed(cr, m, r):
    """root codes: infinity where the root is infinite and the first moment is not"""
    return np.where(np.isposinf(r) & np.isfinite(m), 254, cr).astype(np.uint8)


def step(p, g, codes, t, lr, b1, b2, eps, wd=0.0, decoupled=False, first=0):
    """fp32 p (flat; a bf16 parameter is rounded by the caller), new codes"""
    kept = {}

    def keep(m, r, t, nearest=False):
        kept["m"], kept["r"] = m, r
        return None
    before, A8.encode, A8.ROOT = (A8.encode, A8.ROOT), keep, ROOT
    try:
        p, _ = A8.step(p, g, codes, t, lr, b1, b2, eps, wd, decoupled)
    finally:
        A8.encode, A8.ROOT = before
    return p, encode(kept["m"], kept["r"], t, first)
