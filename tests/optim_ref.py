"""The optimizer step of include/hydra_optim.h in 64 bits (numpy), and in fp32 operation by
operation: what the optimizer tests compare the kernels with.  Plain loops and whole-array
arithmetic; nothing here is shared with hydra_amd."""
import numpy as np

BLOCK = 256
U32 = 2.0 ** -24  # half a step of fp32, relative
M32 = 0xFFFFFFFF


def fmix(h):
    h = np.asarray(h, np.uint64)
    h = h ^ (h >> np.uint64(16))
    h = (h * np.uint64(0x85EBCA6B)) & np.uint64(M32)
    h = h ^ (h >> np.uint64(13))
    h = (h * np.uint64(0xC2B2AE35)) & np.uint64(M32)
    return h ^ (h >> np.uint64(16))


def random_words(seed, t, tensor, index):
    """The 32 random bits of the elements `index` of the plan's tensor number `tensor` at step t."""
    k = 0
    for part in (seed & M32, seed >> 32, t & M32, t >> 32, tensor):
        k = int(fmix(k ^ part))
    i = np.asarray(index, np.uint64)
    lo = ((i & np.uint64(M32)) * np.uint64(0x9E3779B1)) & np.uint64(M32)
    hi = ((i >> np.uint64(32)) * np.uint64(0x85EBCA6B)) & np.uint64(M32)
    return fmix(lo ^ hi ^ np.uint64(k))


def step64(p, g, m, v, *, lr, t, mult=1.0, b1=0.9, b2=0.999, eps=1e-8, wd=0.0):
    """One step in fp64 and how far fp32 arithmetic may be from it: (p, m, v), (ep, em, ev).

    Roundings counted (each at most U32 relative to its value):
      g'  = g * mult: mult's own and the product's                                   2
      m   : b1, product on one term; 1-b1, g' (2), product on the other; the sum
      v   : b2, product; 1-b2, g' twice (4), two products = 7; the sum: <= 8 in all (all terms >= 0)
      p   : lr' (2), wd, product, 1 - . on the decay: 4 lr wd + 1; product 1
      U = m / (sqrt(v) * c2 + eps) * size: sqrt 8/2 + 1, c2, product, eps, sum, division,
          size = lr' (2) * c1 (1) + 1, product: 4 + 1 + 1 + 1 + 1 + 1 + 1 + 4 + 1 = 15, and m's error
      the difference: 1"""
    p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
    g = g * mult
    a, b = b1 * m, (1 - b1) * g
    m1 = a + b
    em = U32 * (2 * np.abs(a) + 4 * np.abs(b) + np.abs(m1)) + 2.0 ** -149
    v1 = b2 * v + (1 - b2) * g * g
    ev = U32 * 9 * v1 + 2.0 ** -148
    c1, c2 = 1 / (1 - b1 ** t), 1 / np.sqrt(1 - b2 ** t)
    with np.errstate(invalid="ignore", divide="ignore"):
        denom = np.sqrt(v1) * c2 + eps
        u = m1 / denom * (lr * c1)
        # a v below 2^-126 is held in steps of 2^-149: three roundings (two products, the sum) of half
        # a step, and its old value's; half of their share in v is the root's
        coarse = np.where(v1 > 0, np.minimum(2.0 ** -148 / (2 * v1), 1.0), 0.0) * np.sqrt(v1) * c2 / denom
        eu = em / denom * (lr * c1) + np.abs(u) * np.where(denom > 0, coarse, 0.0)
    p1 = p * (1 - lr * wd) - u
    ep = U32 * (np.abs(p) * (2 + 5 * abs(lr * wd)) + 16 * np.abs(u) + np.abs(p1)) + 2 * eu + 2.0 ** -149
    return (p1, m1, v1), (ep, em, ev)


def step32(p, g, m, v, *, lr, t, mult=1.0, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, lr_scale=1.0):
    """The same in fp32, each operation rounded in the documented order: the kernels' own bits."""
    f = np.float32
    p, g, m, v = (np.asarray(x, f) for x in (p, g, m, v))
    lr = f(lr) * f(lr_scale)
    with np.errstate(all="ignore"):
        g = g * f(mult)
        m = m * f(b1) + g * f(1 - b1)
        v = v * f(b2) + (g * f(1 - b2)) * g
        denom = np.sqrt(v) * f(1 / np.sqrt(1 - b2 ** t)) + f(eps)
        p = p * (f(1) - lr * f(wd)) - (m / denom) * (lr * f(1 / (1 - b1 ** t)))
    return p, m, v


# ---- 8-bit moments ---------------------------------------------------------------------------------
def values8(codes, scales, bits):
    """What the bytes stand for, in fp64: m (bits 3), or sqrt(v) (bits 4)."""
    c = codes.astype(np.int64)
    s = np.repeat(scales.astype(np.float64), BLOCK)[: c.size]
    k = c & 127 if bits == 3 else c
    f = np.where(k < (1 << bits), k * 2.0 ** -(14 + bits),
                 2.0 ** ((k >> bits) - 15.0) * (1 + (k % (1 << bits)) / 2.0 ** bits))
    with np.errstate(invalid="ignore"):
        x = f * s
    if bits == 3:
        x = np.where(c == 0x80, np.nan, np.where(c > 0x80, -x, x))
    else:
        x = np.where(c == 255, np.inf, x)
    return x


def scales64(x):
    """The scales of a moment's blocks, from values in fp64 (not finite ones left out)."""
    a = np.abs(np.asarray(x, np.float64))
    a = np.where(np.isfinite(a), a, 0.0)
    a = np.append(a, np.zeros(-a.size % BLOCK)).reshape(-1, BLOCK)
    top = a.max(1)
    return np.where(top < 2.0 ** -100, 0.0, top / 1.875)


def check_codes(x, ex, codes, scales, bits, noise, where="", loose=1e-3):
    """x: a moment (sqrt of v for bits 4) in fp64, ex: how far fp32 may be from it, codes and scales:
    the kernel's.  Every byte must be floor(|x| / s in units of its spacing + noise), where |x| / s
    may be off by what fp32 may be off: ex, the scale's two roundings and the block's largest value's
    error, the quotient's three (1 / s, the product, the rebasing below the smallest power).  At most
    `loose` of the bytes may lie so near a border that two are allowed (values without a grid of their
    own come within 2^-17 of one, the widest interval, with a probability below 2^-15)."""
    n = x.size
    s64 = scales64(x)
    exb = np.append(np.where(np.isfinite(x), ex, 0), np.zeros(-n % BLOCK)).reshape(-1, BLOCK).max(1)
    assert (np.abs(scales - s64) <= exb / 1.875 + 3 * U32 * s64 + 2.0 ** -149).all(), where
    fin = np.isfinite(x)
    c = codes.astype(np.int64)
    bad = 0x80 if bits == 3 else 255
    assert (c[~fin] == bad).all(), where
    assert not (c[fin] == bad).any(), where
    s = np.repeat(scales.astype(np.float64), BLOCK)[:n]
    on = fin & (s > 0)
    assert (c[fin & (s == 0)] <= 1).all(), where  # 1: a v above zero in a block of nothing
    if bits == 3:
        neg = c > 0x80
        assert (x[neg & on] < 0).all(), where
        assert (~neg & on & (x < 0) & (c != 0)).sum() == 0, where
        c = c & 127
    a, e = np.abs(x[on]) / s[on], ex[on] / s[on]
    exp = np.maximum(np.frexp(a)[1] - 1, -14)
    spacing = np.ldexp(1.0, exp - bits)
    y = a / spacing + noise[on]
    d = e / spacing + 6 * U32 * a / spacing + 2.0 ** -20
    got = np.abs(values8(c[on], np.ones(-(-on.sum() // BLOCK)), bits)) / spacing
    top = 1.875 / spacing
    lo, hi = np.minimum(np.floor(y - d), top), np.minimum(np.floor(y + d), top)
    if bits == 4:
        least = np.where(x[on] > 0, 2.0 ** -18 / spacing, 0.0)
        lo, hi = np.maximum(lo, least), np.maximum(hi, least)
    wrong = (got < lo) | (got > hi)
    assert not wrong.any(), (where, int(wrong.sum()), a[wrong][:4], got[wrong][:4], lo[wrong][:4], hi[wrong][:4])
    # the intervals are narrow: almost every byte is pinned to one value (counted where fp32 has the
    # value to 2^-19: what comes from a v below 2^-126, held in steps of 2^-149, has a wide one)
    sure = e <= 2.0 ** -19 * a
    assert sure.sum() < 1000 or (lo != hi)[sure].mean() < loose, where


def encode32(m, v, r):
    """Bytes and scales of both moments from fp32 ones, operation by operation: (m codes, m scales, v
    codes, v scales, which bytes are above the gradual underflow).  All values finite."""
    f = np.float32

    def one(x, bits, top, r16):
        n = x.size
        rows = np.append(x, np.zeros(-n % BLOCK, f)).astype(f).reshape(-1, BLOCK)
        amax = rows.max(1)
        s = np.where(amax < f(2.0 ** -100), f(0), amax * f(1 / 1.875)).astype(f)
        with np.errstate(divide="ignore"):
            inv = np.where(s > 0, f(1) / s, f(0)).astype(f)
        t = (rows * inv[:, None]).reshape(-1)[:n]
        u = (t * f(2.0 ** -112)).astype(f).view(np.uint32).astype(np.uint64)
        drop = np.uint64(23 - bits)
        c = (u + (r16.astype(np.uint64) << np.uint64(7 - bits))) >> drop
        return np.minimum(c, top), s, t >= 2.0 ** -14

    cm, sm, am = one(np.abs(m), 3, 127, r & np.uint64(0xFFFF))
    root = np.sqrt(v)
    cv, sv, av = one(root, 4, 254, r >> np.uint64(16))
    cm = np.where((m < 0) & (cm > 0), cm + 128, cm)
    cv = np.where(root > 0, np.maximum(cv, 1), 0)
    return cm.astype(np.uint8), sm, cv.astype(np.uint8), sv, am & av


# ---- the norm ------------------------------------------------------------------------------------------
def norm64(grads, grad_scale, max_norm):
    total = sum(float((np.asarray(g, np.float64) ** 2).sum()) for g in grads)
    norm = abs(grad_scale) * np.sqrt(total)
    clip = min(1.0, max_norm / (norm + 1e-6)) if max_norm > 0 else 1.0
    return norm, grad_scale * clip
