"""The 8-bit moments of AdamW in numpy, written from their description (pin_adamw.hip): values, not bits."""
import numpy as np

BLOCK = 256
K1, K2, K3 = 0x9E3779B1, 0x6A09E667, 0xBB67AE85


def mix(x):
    x = np.asarray(x, dtype=np.uint64) & np.uint64(0xFFFFFFFF)
    for shift, k in ((16, K1), (15, K2)):
        x = x ^ (x >> np.uint64(shift))
        x = (x * np.uint64(k)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def dither(place, step, seed, group):
    """Two whole numbers below 2^17 for each element's place in the group's flat state."""
    salt = (seed * K1 + group * K3 + step * K2) & 0xFFFFFFFF
    place = (np.asarray(place, dtype=np.uint64) & np.uint64(0xFFFFFFFF)) * np.uint64(K3)
    h = mix(mix(np.uint64(salt)) + place)
    return (h & np.uint64(0x1FFFF)).astype(np.float64), (h >> np.uint64(15)).astype(np.float64)


def _per_block(x, fill=0.0):
    pad = -x.size % BLOCK
    return np.concatenate([x, np.full(pad, fill)]).reshape(-1, BLOCK)


def exponent(x):
    """floor(log2) of each block's largest finite value."""
    a = np.abs(_per_block(x))
    a = np.where(np.isfinite(a), a, 0.0).max(1)
    return np.where(a > 0, np.maximum(np.frexp(a)[1] - 1, -900), -900)


def spread(e, n):
    return np.repeat(e, BLOCK)[:n]


def encode(m, v, dm, dv):
    em, ev = exponent(m), exponent(v)
    n = m.size
    # first moment: units of 2^(e-3), e the value's exponent, at least that of 2^(E-13)
    a, E = np.abs(np.where(np.isfinite(m), m, 0.0)), spread(em, n)
    e = np.maximum(np.where(a > 0, np.frexp(a)[1] - 1, -2000), E - 13)
    q = np.floor(np.ldexp(a, 3 - e) + dm / 2 ** 17).astype(np.int64)      # 0..16 units
    cm = np.where(q < 8, q, ((e - E + 14) << 3) + (q - 8))
    cm = np.where(np.isfinite(m), cm | (np.signbit(m).astype(np.int64) << 7), 0x7F)
    # second moment: the same without underflow, at least code 1 for what is positive
    b, E = np.where(np.isfinite(v), v, 0.0), spread(ev, n)
    e = np.where(b > 0, np.frexp(b)[1] - 1, 0)
    q = np.floor(np.ldexp(b, 3 - e) + dv / 2 ** 17).astype(np.int64)
    cv = np.where(b > 0, np.maximum(((e - E + 30) << 3) + (q - 8), 1), 0)
    cv = np.where(np.isfinite(v), cv, 0xFF)
    return cm.astype(np.uint8), cv.astype(np.uint8), np.stack((em, ev), 1).astype(np.int16)


def decode(cm, cv, exps):
    n = cm.size
    cm, cv = cm.astype(np.int64), cv.astype(np.int64)
    em, ev = (spread(exps[:, i].astype(np.int64), n) for i in (0, 1))
    e, f = (cm >> 3) & 15, cm & 7
    m = np.where(e == 0, np.ldexp(f.astype(float), em - 16), np.ldexp((8.0 + f), e + em - 17))
    m = np.where(cm & 0x7F == 0x7F, np.nan, np.where(cm & 0x80, -m, m))
    v = np.where(cv == 0, 0.0, np.ldexp(8.0 + (cv & 7), (cv >> 3) - 33 + ev))
    return m, np.where(cv == 0xFF, np.nan, v)
