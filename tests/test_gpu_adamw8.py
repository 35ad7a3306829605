"""GPU tests of the 8-bit step where fp32 itself runs out (include/hydra_optim.h has the formulas)."""
import numpy as np
import pytest

import optim_ref as R
from hydra_amd import optim

pytestmark = pytest.mark.gpu

F = np.float32


def step(gpu, g, *, lr=1e-3, t=1, eps=1e-8, b2=0.999, seed=0):
    """One step of zeroed weights and moments: (p, m bytes, m scales, v bytes, v scales), and m and v as
    the documented fp32 operations give them."""
    import torch

    n, rows = g.size, optim.moment_scales(g.size)
    p = torch.zeros(n, device=gpu)
    m8, v8 = (torch.zeros(n, dtype=torch.uint8, device=gpu) for _ in "mv")
    ms, vs = (torch.zeros(rows, device=gpu) for _ in "mv")
    plan = optim.AdamW([p], [torch.from_numpy(g).to(gpu)], [m8], [v8], m_scale=[ms], v_scale=[vs], betas=(0.9, b2),
                       eps=eps, weight_decay=0.0)
    plan.step_(lr=lr, step=t, seed=seed)
    zero = np.zeros(n, F)
    _, m, v = R.step32(zero, g, zero, zero, lr=lr, t=t, b2=b2, eps=eps)
    return [x.cpu().numpy() for x in (p, m8, ms, v8, vs)], m, v


def squares(rng, blocks, b2, low, high):
    """Gradients whose v spread from 2^low to 2^high under a block's largest just above 2^-86."""
    g = np.exp2((rng.uniform(low, high, (blocks, 256)) - np.log2(1 - b2)) / 2) * rng.choice([-1, 1], (blocks, 256))
    g[:, 0] = np.exp2((-86 - np.log2(1 - b2)) / 2) * rng.uniform(1.01, 2, blocks)
    return g.astype(F).reshape(-1)


def weights(p, m, v, *, lr, t, eps, b2, roundings):
    """p, that was zero, is -m / (sqrt(v) * c2 + eps) * (lr * c1) to so many half steps of fp32."""
    c2, size = F(1 / np.sqrt(1 - b2 ** t)), F(lr) * F(1 / (1 - 0.9 ** t))
    u = m.astype(np.float64) / (np.sqrt(v.astype(np.float64)) * np.float64(c2) + np.float64(F(eps))) * np.float64(size)
    off = np.abs(p + u) - (roundings * 1.001 * R.U32 * np.abs(u) + 2.0 ** -149)
    assert (off <= 0).all(), (int((off > 0).sum()), off.max(), np.abs((p + u) / u).max() / R.U32)


@pytest.mark.parametrize("b2", [0.999, 0.9999])
@pytest.mark.parametrize("eps", [2.0 ** -40, 1e-11])
@pytest.mark.parametrize("low,high", [(-148, -126), (-126, -98), (-98, -88)])
def test_weights_of_small_squares(gpu, low, high, eps, b2):
    """The update where v is denormal or near it and eps small: the root is fp32's (1 half step), the
    denominator one rounding, the reciprocal 1 ulp (2), its product with m, the product with the rate
    joined to the difference with p (1): 6 half steps."""
    g = squares(np.random.default_rng(3), 64, b2, low, high)
    (p, *_), m, v = step(gpu, g, eps=eps, b2=b2)
    weights(p, m, v, lr=1e-3, t=1, eps=eps, b2=b2, roundings=6)


@pytest.mark.parametrize("lr", [1e-12, 1e-3, 1e3])
@pytest.mark.parametrize("size", [2.0 ** -97, 2.0 ** -60, 1.0])
def test_weights_of_small_updates(gpu, size, lr):
    """The quotient comes before its product with the rate, as documented: m times a small rate alone
    would be denormal."""
    g = (np.random.default_rng(5).normal(0, 1, 4096) * size).astype(F)
    (p, *_), m, v = step(gpu, g, lr=lr)
    weights(p, m, v, lr=lr, t=1, eps=1e-8, b2=0.999, roundings=6)


def exact_bytes(x, bits, r16):
    """Bytes and scales of fp32 magnitudes (sqrt of v for bits 4) as documented: x / s from one product
    with fp32's 1 / s, rounded to fp32 or, below 2^-14, to a multiple of 2^-37; then floor(. + r16 / 2^16)
    in units of the byte's step.  Not finite: 128 or 255."""
    fin = np.isfinite(x)
    a = np.append(np.where(fin, np.abs(x), 0), np.zeros(-x.size % R.BLOCK)).astype(F).reshape(-1, R.BLOCK)
    top = a.max(1)
    s = np.where(top < F(2.0 ** -100), F(0), top * F(1 / 1.875)).astype(F)
    with np.errstate(divide="ignore"):
        inv = np.where(s > 0, F(1) / s, F(0)).astype(F)
    exact = (a.astype(np.float64) * inv[:, None].astype(np.float64)).reshape(-1)[: x.size]  # 48 bits
    q = np.where(exact < 2.0 ** -14, np.rint(exact * 2.0 ** 37) * 2.0 ** -37, exact.astype(F).astype(np.float64))
    e = np.maximum(np.frexp(q)[1] - 1, -14)
    n = np.floor(np.ldexp(q, bits - e) + r16 / 65536.0).astype(np.int64)  # of the step 2^(e - bits)
    c = np.minimum(n + (e + 14) * 2 ** bits, 2 ** (bits + 4) - (1 if bits == 3 else 2))
    return np.where(fin, c, 128 if bits == 3 else 255), s


def both_bytes(m, root, r):
    cm, sm = exact_bytes(m, 3, (r & np.uint64(0xFFFF)).astype(np.float64))
    cm = np.where((m < 0) & (cm > 0) & (cm < 128), cm + 128, cm)
    cv, sv = exact_bytes(root, 4, (r >> np.uint64(16)).astype(np.float64))
    return cm.astype(np.uint8), sm, np.where(root > 0, np.maximum(cv, 1), cv).astype(np.uint8), sv


def at_borders(rng, blocks, top, bits, low):
    """Magnitudes around the borders between bytes from 2^low of their block's largest on, where one
    rounding more or less, or the root's last bit, makes another byte (to nearest)."""
    tops = (top * rng.uniform(1, 2, blocks)).astype(F)
    s = (tops * F(1 / 1.875)).astype(np.float64)
    code = rng.integers((low + 15) << bits if low > -15 else 0, 3 << bits, (blocks, 256))
    k = np.where(code < 1 << bits, 0, (code >> bits) - 1)  # the step 2^(k - 14 - bits)
    x = (np.where(k == 0, code, code % (1 << bits) + (1 << bits)) + 0.5) * np.exp2(k - 14.0 - bits) * s[:, None]
    x = (x.astype(F).view(np.int32) + rng.integers(-4, 5, x.shape).astype(np.int32)).view(F)
    x[:, 0] = tops
    return x.reshape(-1)


@pytest.mark.parametrize("bad", [None, float("nan"), float("inf")])
@pytest.mark.parametrize("top", [2.0 ** -30, 1.0, 2.0 ** 13.5, 2.0 ** 20, 2.0 ** 60])
def test_bytes_of_conversions_at_borders(gpu, top, bad):
    """Every byte of an encoding, whatever else its block holds."""
    import torch

    rng = np.random.default_rng(6)
    m = at_borders(rng, 400, top, 3, -15) * rng.choice([-1, 1], 400 * 256).astype(F)
    v = np.square(at_borders(rng, 400, top, 4, -15), dtype=F)
    if bad is not None:
        m[256 * 7 + 5::512], v[5::512] = bad, bad
    n = m.size
    m8, v8 = (torch.zeros(n, dtype=torch.uint8, device=gpu) for _ in "mv")
    ms, vs = (torch.zeros(n // 256, device=gpu) for _ in "mv")
    optim.moments8_encode_(m8, ms, v8, vs, torch.from_numpy(m).to(gpu), torch.from_numpy(v).to(gpu))
    cm, sm, cv, sv = both_bytes(m, np.sqrt(v), np.full(n, 0x80008000, np.uint64))
    for got, want in ((ms, sm), (vs, sv), (m8, cm), (v8, cv)):
        got = got.cpu().numpy()
        assert np.array_equal(got, want), ((got != want).sum(), np.flatnonzero(got != want)[:8])


@pytest.mark.parametrize("seed", [0, 12345])
@pytest.mark.parametrize("eps", [1e-8, 1e-20])
@pytest.mark.parametrize("top", [2.0 ** -42.9, 2.0 ** -30, 1.0, 2.0 ** 20])
def test_bytes_of_steps_at_borders(gpu, top, eps, seed):
    """Every byte of a step, by the short path and by the other one (eps 1e-20; a large top)."""
    rng = np.random.default_rng(8)
    omb1, omb2 = F(1 - 0.9), F(1 - 0.999)
    roots = at_borders(rng, 500, top, 4, -15)
    g = np.concatenate([(at_borders(rng, 500, top, 3, -15) / omb1), (roots.astype(np.float64) / np.sqrt(np.float64(omb2))).astype(F)])
    (_, cm, sm, cv, sv), m, v = step(gpu, g, eps=eps, seed=seed)
    r = R.random_words(seed, 1, 0, np.arange(g.size)) if seed else np.full(g.size, 0x80008000, np.uint64)
    for got, want in zip((cm, sm, cv, sv), both_bytes(m, np.sqrt(v), r)):
        assert np.array_equal(got, want), ((got != want).sum(), np.flatnonzero(got != want)[:8])
