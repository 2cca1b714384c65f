"""numpy restatement of the 8-bit Adam step (formats and operation order of csrc/mtl_optim8.hip): fp32 arithmetic, one IEEE rounding per operation, so that the device's results
can be compared bit for bit. `nearest=True` rounds the root to nearest instead of against the running threshold (to show what that would do)."""
import numpy as np

F = np.float32
BLOCK = 64


def e4m3_values():
    c = np.arange(256)
    s, e, f = c >> 7, (c >> 3) & 15, c & 7
    v = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e.astype(float) - 10))
    v[(c & 0x7F) == 0x7F] = np.nan
    return np.where(s == 1, -v, v).astype(F)


def root_values():
    c = np.arange(256)
    e, f = c >> 4, c & 15
    v = np.where(e == 0, f, (16 + f) * 2.0 ** (np.maximum(e, 1) - 1)).astype(F)
    v[255] = np.nan
    return v


E4M3, ROOT = e4m3_values(), root_values()


def encode_e4m3(x):
    """nearest even; |x| < 464, NaN and infinities -> 0x7f"""
    a = np.abs(x).astype(np.float64)
    fin = np.isfinite(a)
    a = np.where(fin, a, 0.0)
    e = np.maximum(np.floor(np.log2(np.maximum(a, 2.0 ** -40))), -6)
    q = np.rint(a / 2.0 ** (e - 3))                       # 8 .. 16 (normal), 0 .. 8 (e = -6): the code is continuous over the binades
    code = ((e + 6) * 8 + q).astype(np.int64)
    return np.where(fin, code + np.where(np.signbit(x), 128, 0), 0x7F).astype(np.uint8)


def thresholds(n, step):
    return ((np.arange(n, dtype=np.uint64) * np.uint64(0xC13FA9A9) + np.uint64((step * 0x91E10DA5) & 0xFFFFFFFF)) & np.uint64(0xFFFFFFFF)).astype(np.uint32)


def exponents(x, below):
    a = np.abs(x)
    top = np.where(np.isfinite(a), a, F(0)).reshape(-1, BLOCK).max(1).astype(F)
    return np.maximum((top.view(np.uint32) >> 23).astype(np.int64) - 127 - below, -126)


def encode(m, r, step, nearest=False):
    n = m.size
    pad = -n % BLOCK
    m, r = (np.concatenate([t.reshape(-1), np.zeros(pad, F)]) for t in (m, r))
    em, er = exponents(m, 7), exponents(r, 17)
    with np.errstate(invalid="ignore", over="ignore"):
        cm = encode_e4m3((m.reshape(-1, BLOCK) * (F(2) ** (-em).astype(F))[:, None]).reshape(-1))
        y = (r.reshape(-1, BLOCK) * (F(2) ** (-er).astype(F))[:, None]).reshape(-1).astype(F)
        u = np.full(y.size, 1 << 31, np.uint32) if nearest else thresholds(y.size, step)
        large = ((y.view(np.uint32).astype(np.int64) + (u >> 13)) >> 19) - 2080
        small = np.floor(np.nan_to_num(y, posinf=0) + (u >> 8).astype(F) * F(2.0 ** -24)).astype(np.int64)
    cr = np.where(y >= 16, large, small)
    cr = np.where((r > 0) & (cr < 1), 1, cr)
    cr = np.where(np.isfinite(r), cr, 255)
    return cm[:n], cr[:n].astype(np.uint8), np.stack([em, er], 1).astype(np.int8)


def decode(cm, cr, ex):
    at = np.arange(cm.size) // BLOCK
    with np.errstate(invalid="ignore"):
        return E4M3[cm.reshape(-1)] * (F(2) ** ex[:, 0].astype(F))[at], ROOT[cr.reshape(-1)] * (F(2) ** ex[:, 1].astype(F))[at]


def step(p, g, codes, t, lr, b1, b2, eps, wd=0.0, decoupled=False, nearest=False):
    """fp32 p (flat; a bf16 parameter is rounded by the caller), new codes"""
    m, r = decode(*codes)
    p, g = p.reshape(-1).astype(F), g.reshape(-1).astype(F)
    with np.errstate(all="ignore"):
        v = r * r
        if wd and decoupled:
            p = p * F(1.0 - lr * wd)
        elif wd:
            g = g + p * F(wd)
        m = m + (g - m) * F(1.0 - b1)
        v = v * F(b2) + (g * g) * F(1.0 - b2)
        r = np.sqrt(v)
        denom = r * F(1.0 / np.sqrt(1.0 - b2 ** t)) + F(eps)
        p = p - (m / denom) * F(lr / (1.0 - b1 ** t))
    return p, encode(m, r, t, nearest)
