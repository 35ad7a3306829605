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
