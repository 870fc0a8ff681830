"""AdamW with a global-norm clip in 64 bits, one tensor at a time, with moments in 32 bits or as 8-bit codes.

Every value comes with a bound on how far fp32 arithmetic may take it: `u` = 2^-24 is half a step of fp32, each elementary
operation adds one, and a sum of terms that may cancel is bounded by the terms, not by the sum.
"""
import numpy as np

U = 2.0 ** -24
BLOCK = 256


def norm(grads):
    return float(np.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in grads)))


def clip_coef(total, max_norm):
    c = max_norm / (total + 1e-6)
    return c if not c > 1.0 else 1.0


def step(p, g, m, v, t, lr, b1, b2, eps, wd, factor=1.0, factor_err=0.0, half=0.0, tiny=0.0):
    """Moments and parameter after step number t (v the second moment before it); returns values and their bounds.
    factor_err: relative error of the factor on the gradient; half: half a step of the parameter's own type, relative,
    and tiny its smallest normal number."""
    p, g, m, v = (np.asarray(x, dtype=np.float64) for x in (p, g, m, v))
    with np.errstate(all='ignore'):
        g = g * factor
        ge = np.abs(g) * (U + factor_err)
        m2 = b1 * m + (1 - b1) * g
        # two rounded constants, two products, one sum
        me = 3 * U * (b1 * np.abs(m) + (1 - b1) * np.abs(g)) + (1 - b1) * ge + U * np.abs(m2) + 2.0 ** -149
        v2 = b2 * v + (1 - b2) * g * g
        ve = 4 * U * v2 + 2 * (1 - b2) * np.abs(g) * ge + 2.0 ** -148
        root = np.sqrt(v2)
        re = np.where(v2 > 0, np.minimum(ve / np.maximum(root, 1e-300), np.sqrt(ve)), np.sqrt(ve)) + U * root
        bc1, bc2 = 1 - b1 ** t, np.sqrt(1 - b2 ** t)
        denom = root / bc2 + eps
        upd = lr / bc1 * m2 / denom
        p2 = p * (1 - lr * wd) - upd
        # the denominator's bound: the root's, the rounded correction, eps's rounding and the sum's
        de = re / bc2 + 3 * U * denom
        pe = np.abs(upd) * (4 * U + 2 * de / denom) + lr / bc1 * me / denom + 3 * U * np.abs(p) + (U + half) * (np.abs(p2)) \
            + half * tiny
    return dict(p=p2, m=m2, v=v2, r=root, pe=pe, me=me, ve=ve, re=re)


# ---- 8-bit codes
def mix(h):
    """The 32-bit MurmurHash3's finalizer."""
    h = np.asarray(h, dtype=np.uint64) & 0xFFFFFFFF
    h = ((h ^ (h >> np.uint64(16))) * np.uint64(0x85EBCA6B)) & np.uint64(0xFFFFFFFF)
    h = ((h ^ (h >> np.uint64(13))) * np.uint64(0xC2B2AE35)) & np.uint64(0xFFFFFFFF)
    return h ^ (h >> np.uint64(16))


def fractions(n, t, seed, first=0):
    """(for m, for the root): the number in [0, 1) that each element's code is rounded by."""
    key = mix((int(t) * 0x9E3779B9 + int(seed)) & 0xFFFFFFFF)
    i = np.arange(first, first + n, dtype=np.uint64)
    h = mix((i & np.uint64(0xFFFFFFFF)) ^ (i >> np.uint64(32)) ^ key)
    return [(x.astype(np.float64) + 0.5) / 65536 for x in (h & np.uint64(0xFFFF), h >> np.uint64(16))]


def scale_exponent(x):
    """The smallest k >= -127 with every finite |value| of a block <= 448 * 2^k, per block."""
    n = len(x)
    b = np.zeros(-(-n // BLOCK) * BLOCK)
    b[:n] = np.where(np.isfinite(x), np.abs(x), 0.0)
    top = b.reshape(-1, BLOCK).max(1)
    frac, power = np.frexp(top)
    return np.where(top > 0, np.maximum(power - 9 + (frac > 0.875), -127), -127).astype(int)


def round_code(y, fraction, positive):
    """|y| <= 448 to the e4m3 grid: down by what `fraction` does not carry over the next point."""
    a = np.abs(y)
    _, power = np.frexp(a)
    ulp = np.exp2(np.maximum(power - 4, -9).astype(float))
    q = np.floor(a / ulp + fraction) * ulp
    if positive:
        q = np.where(a > 0, np.maximum(q, 2.0 ** -9), q)
    return np.sign(y) * q


def code_range(x, err, k, fraction, positive):
    """Lowest and highest code (as the value it stands for, over 2^k) that x +- err may round to."""
    s = np.exp2(-np.repeat(k, BLOCK)[:len(x)].astype(float))
    lo, hi = (np.clip((x + e) * s, -448, 448) for e in (-err, err))
    a, b = round_code(lo, fraction, positive), round_code(hi, fraction, positive)
    return np.minimum(a, b), np.maximum(a, b)
