"""GPU tests of the optimizer step (hydra_amd/optim.py, include/hydra_optim.h) against the 64-bit
reference of optim_ref.py.

fp32 results may differ from the 64-bit ones by the roundings that optim_ref.step64 counts; fp32
moments and weights are also compared bit for bit with the documented order of fp32 operations.
8-bit moments: every byte has to be the one that the definition gives, but where fp32 may see the
other side of a border (optim_ref.check_codes).  16-bit weights: half a step of their type more."""
import numpy as np
import pytest

import optim_ref as R
from hydra_amd import _lib, optim

pytestmark = pytest.mark.gpu

HALF = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
KINDS = [("f32", False), ("bf16", False), ("f16", False), ("bf16", True), ("f16", True)]
GRADS = ["f32", "bf16", "f16"]
B1, B2, EPS = 0.9, 0.999, 1e-8


def dt(name):
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def f64(t):
    return t.detach().double().cpu().numpy()


def f32(t):
    return t.detach().float().cpu().numpy()


class Flat:
    """Tensors of the given lengths as views of one buffer, `pad` guard elements before, between and
    after them; check() fails if a guard changed."""

    def __init__(self, torch, gpu, sizes, dtype, fill, pad=3, guard=1):
        total = sum(sizes) + pad * (len(sizes) + 1)
        self.buf = torch.full((total,), guard, dtype=dtype, device=gpu)
        self.views, at = [], pad
        for n, x in zip(sizes, fill):
            v = self.buf[at:at + n]
            v.copy_(x)
            self.views.append(v)
            at += n + pad
        self.inside = torch.zeros(total, dtype=torch.bool, device=gpu)
        at = pad
        for n in sizes:
            self.inside[at:at + n] = True
            at += n + pad
        self.guard = guard

    def check(self, what):
        assert (self.buf[~self.inside] == self.guard).all(), f"guard elements of {what} changed"


class Setup:
    """A plan over tensors of `sizes` with random contents, every buffer guarded, at odd offsets."""

    def __init__(self, gpu, sizes, param="f32", master=False, grad="f32", eight=False, seed=0, pad=3,
                 wd=None, lr_scale=1.0, cold=False, bucket=False, eps=EPS):
        import torch

        self.torch, self.gpu, self.sizes, self.eight, self.param, self.master = torch, gpu, sizes, eight, param, master
        gen = torch.Generator(device=gpu)
        gen.manual_seed(seed)

        def normal(n, scale=1.0):
            return torch.randn(n, generator=gen, device=gpu) * scale

        def flat(fill, dtype, sz=sizes, guard=1):
            return Flat(torch, gpu, sz, dtype, fill, pad, guard)

        def level(n):  # gradients spread over orders of magnitude within a tensor
            return torch.exp2(torch.randint(-8, 4, (n,), generator=gen, device=gpu).float())

        zero = 0.0 if cold else 1.0
        p = [normal(n, 0.05) for n in sizes]
        self.p = flat(p, dt(param))
        self.pm = flat(p, torch.float32) if master else None
        self.g = flat([normal(n, 0.01) * level(n) for n in sizes], dt(grad))
        m = [normal(n, 0.002 * zero) * level(n) for n in sizes]
        v = [(normal(n, 0.01 * zero) * level(n)) ** 2 for n in sizes]
        kw = {}
        if eight:
            rows = [optim.moment_scales(n) for n in sizes]
            self.m, self.v = (flat([torch.zeros(n, dtype=torch.uint8, device=gpu) for n in sizes], torch.uint8, guard=77) for _ in "mv")
            self.ms, self.vs = (flat([torch.zeros(r, device=gpu) for r in rows], torch.float32, rows) for _ in "mv")
            for i, n in enumerate(sizes):
                if n:
                    optim.moments8_encode_(self.m.views[i], self.ms.views[i], self.v.views[i], self.vs.views[i], m[i], v[i])
            kw = dict(m_scale=self.ms.views, v_scale=self.vs.views)
        else:
            self.m, self.v = flat(m, torch.float32), flat(v, torch.float32)
        self.wd = wd if wd is not None else [0.1 if i % 3 else 0.0 for i in range(len(sizes))]
        self.ls = [lr_scale * (1 + i % 2) for i in range(len(sizes))]
        self.plan = optim.AdamW(self.p.views, self.g.views, self.m.views, self.v.views,
                                master=self.pm.views if master else None, betas=(B1, B2), eps=eps,
                                weight_decay=self.wd, lr_scale=self.ls,
                                bucket=self.g.buf if bucket else None, **kw)
        self.eps = eps

    def state(self):
        """Everything a step reads or writes, in fp64 on the host: a list by tensor."""
        self.torch.cuda.synchronize()
        out = []
        for i, n in enumerate(self.sizes):
            s = {"p": f64((self.pm if self.master else self.p).views[i]), "p16": f64(self.p.views[i]), "g": f64(self.g.views[i])}
            if self.eight:
                s.update(mc=self.m.views[i].cpu().numpy(), vc=self.v.views[i].cpu().numpy(),
                         ms=self.ms.views[i].cpu().numpy(), vs=self.vs.views[i].cpu().numpy())
                s["m"] = R.values8(s["mc"], s["ms"], 3)
                s["v"] = R.values8(s["vc"], s["vs"], 4) ** 2
            else:
                s.update(m=f64(self.m.views[i]), v=f64(self.v.views[i]))
            out.append(s)
        return out

    def guards(self):
        for what in ("p", "pm", "g", "m", "v", "ms", "vs"):
            x = getattr(self, what, None)
            if x is not None:
                x.check(what)

    def compare(self, before, after, *, lr, t, mult=1.0, seed=0):
        """after = one step from before, within the derived bounds."""
        for i, (a, b) in enumerate(zip(before, after)):
            n = self.sizes[i]
            where = f"tensor {i} of {n}"
            assert np.array_equal(a["g"], b["g"], equal_nan=True), where
            if not n:
                continue
            (p, m, v), (ep, em, ev) = R.step64(a["p"], a["g"], a["m"], a["v"], lr=lr * self.ls[i], t=t, mult=mult,
                                               b1=B1, b2=B2, eps=self.eps, wd=self.wd[i])
            if self.eight:
                # the old values in fp32: their two products' roundings, once more for the square
                em = em + 2 * R.U32 * B1 * np.abs(a["m"])
                ev = ev + 5 * R.U32 * B2 * a["v"]
                ep = ep + lr * self.ls[i] / (1 - B1 ** t) * (2 * R.U32 * B1 * np.abs(a["m"])) / (np.sqrt(v / (1 - B2 ** t)) + self.eps) \
                    + 5 * R.U32 * np.abs(p - a["p"] * (1 - lr * self.ls[i] * self.wd[i]))
                r = R.random_words(seed, t, i, np.arange(n)) if seed else np.full(n, 0x80008000, np.uint64)
                root = np.sqrt(v)
                R.check_codes(m, em, b["mc"], b["ms"], 3, (r & np.uint64(0xFFFF)) / 65536.0, where + " m")
                with np.errstate(divide="ignore", invalid="ignore"):
                    er = np.where(root > 0, ev / (2 * root), 0) + R.U32 * root
                R.check_codes(root, er, b["vc"], b["vs"], 4, (r >> np.uint64(16)) / 65536.0, where + " v")
            else:
                assert (np.abs(b["m"] - m) <= em).all(), where
                assert (np.abs(b["v"] - v) <= ev).all(), where
            tol = ep if self.master else ep + HALF[self.param] * (np.abs(p) + ep) + (2.0 ** -25 if self.param == "f16" else 0)
            assert (np.abs(b["p"] - p) <= tol).all(), (where, np.abs(b["p"] - p).max())
            if self.master:  # the 16-bit copy is exactly the rounded master
                want = self.torch.from_numpy(b["p"]).float().to(dt(self.param)).double().numpy()
                assert np.array_equal(want, b["p16"]), where


RAGGED = [1, 0, 2, 3, 63, 64, 65, 255, 256, 257, 1000, 4095, 4096, 4097, 8191, 12289]


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("grad", GRADS)
@pytest.mark.parametrize("param,master", KINDS)
def test_step_types(gpu, param, master, grad, eight):
    """Every type of weights, gradients and moments over ragged lengths at odd offsets."""
    s = Setup(gpu, RAGGED, param, master, grad, eight, seed=1)
    before = s.state()
    s.plan.step_(lr=1e-3, step=7, grad_scale=0.5, seed=99 if eight else 0)
    after = s.state()
    s.compare(before, after, lr=1e-3, t=7, mult=0.5, seed=99)
    s.guards()


@pytest.mark.parametrize("pad", [0, 1, 2, 4, 5, 8, 16])
@pytest.mark.parametrize("eight", [False, True])
def test_step_offsets(gpu, eight, pad):
    """Buffers of different types at offsets that leave them differently aligned."""
    s = Setup(gpu, [5000, 1, 771, 4096], "bf16", True, "f16", eight, seed=pad, pad=pad)
    before = s.state()
    s.plan.step_(lr=1e-3, step=3, seed=5)
    s.compare(before, s.state(), lr=1e-3, t=3, seed=5)
    s.guards()


def test_step_fp32_bits(gpu):
    """fp32 weights and moments: the documented operations in the documented order, bit for bit."""
    s = Setup(gpu, [4097, 70001], seed=4)
    a = [{k: s_[k].astype(np.float32) for k in "pgmv"} for s_ in s.state()]
    for t in (1, 2, 3):
        s.plan.step_(lr=3e-4, step=t, grad_scale=0.25)
        b = s.state()
        for i in range(2):
            p, m, v = R.step32(a[i]["p"], a[i]["g"], a[i]["m"], a[i]["v"], lr=3e-4, t=t, mult=0.25, wd=s.wd[i],
                               lr_scale=s.ls[i])
            for name, want in (("p", p), ("m", m), ("v", v)):
                assert np.array_equal(b[i][name].astype(np.float32).view(np.uint32), want.view(np.uint32)), (t, i, name)
            a[i].update(p=p, m=m, v=v)


@pytest.mark.parametrize("eight", [False, True])
def test_steps_from_nothing(gpu, eight):
    """Several steps from zeroed moments, the first among them (its correction divides by 1 - beta2)."""
    s = Setup(gpu, [300, 1, 5000], "bf16", True, "bf16", eight, seed=6, cold=True)
    for t in (1, 2, 3, 4):
        before = s.state()
        s.plan.step_(lr=1e-3, step=t, seed=123456789012345)
        s.compare(before, s.state(), lr=1e-3, t=t, seed=123456789012345)
    s.guards()


@pytest.mark.parametrize("seed,t", [(0, 1), (1, 1), ((1 << 64) - 1, 5), (77, (1 << 33) + 1)])
def test_moments_seeds(gpu, seed, t):
    """8-bit rounding with no, small and full-width seeds, and a step number beyond 32 bits."""
    s = Setup(gpu, [70000, 333], eight=True, seed=8)
    before = s.state()
    s.plan.step_(lr=1e-3, step=t, seed=seed)
    s.compare(before, s.state(), lr=1e-3, t=t, seed=seed)


@pytest.mark.parametrize("seed", [0, 1234567])
@pytest.mark.parametrize("size", [2.0 ** -30, 1.0, 2.0 ** 10])
def test_bytes_are_those_of_fp32(gpu, size, seed):
    """The bytes and scales are those of the documented fp32 operations, exactly (in the gradual
    underflow, below 2^-14 of a block's largest, the order of two products is open: see check_codes)."""
    s = Setup(gpu, [70001, 300, 256], eight=True, seed=18)
    for v in s.g.views:
        v.mul_(size)
    for t in (1, 2, 3):
        a = s.state()
        s.plan.step_(lr=1e-3, step=t, grad_scale=0.5, seed=seed)
        b = s.state()
        for i, n in enumerate(s.sizes):
            # the old values: one product for m, one and its square for v
            m0 = R.values8(a[i]["mc"], a[i]["ms"], 3).astype(np.float32)
            r0 = R.values8(a[i]["vc"], a[i]["vs"], 4).astype(np.float32)
            _, m, v = R.step32(a[i]["p"], a[i]["g"], m0, r0 * r0, lr=1e-3, t=t, mult=0.5)
            r = R.random_words(seed, t, i, np.arange(n)) if seed else np.full(n, 0x80008000, np.uint64)
            cm, sm, cv, sv, above = R.encode32(m, v, r)
            assert np.array_equal(sm, b[i]["ms"]) and np.array_equal(sv, b[i]["vs"]), (t, i)
            assert np.array_equal(cm[above], b[i]["mc"][above]) and np.array_equal(cv[above], b[i]["vc"][above]), (t, i)


@pytest.mark.parametrize("eps", [0.0, 1e-16, 1e-8, 1e20])
@pytest.mark.parametrize("size", [1e-18, 1e-12, 1e-7, 1e6, 1e17])
def test_moments_of_every_size(gpu, size, eps):
    """8-bit moments whose blocks lie outside the short path in one way or another: tiny and huge
    gradients, every kind of eps, blocks with nothing in them beside others."""
    s = Setup(gpu, [256 * 5 + 40, 3], "f32", False, "f32", True, seed=19, eps=eps, wd=[0.1, 0.0])
    g = s.g.views[0]
    g.mul_(size)
    g[256:512] = 0.0
    for x in (s.m.views[0], s.v.views[0]):
        x[256:512] = 0
        x[700:720] = 0
    g[700:720] = size  # so that no quotient is 0 / 0 with eps 0 there
    if eps == 0.0:
        g[256:512] = size * 1e-3
    for t in (1, 2):
        before = s.state()
        s.plan.step_(lr=1e-3, step=t, seed=77)
        s.compare(before, s.state(), lr=1e-3, t=t, seed=77)
    s.guards()


def test_stochastic_rounding_keeps_the_mean(gpu):
    """v drifting by 0.1 % a step: rounded to nearest it stands still, by the seed its mean follows.
    The largest element holds its block's scale, so the others' bytes have to move by themselves."""
    import torch

    n = 256 * 64
    v0 = torch.full((n,), 0.01, device=gpu) ** 2
    v0[::256] = 1.0
    g = torch.full((n,), 0.02, device=gpu)
    g[::256] = 1.0
    means = {}
    for seed in (0, 5):
        codes = [torch.zeros(n, dtype=torch.uint8, device=gpu) for _ in range(2)]
        scales = [torch.zeros(64, device=gpu) for _ in range(2)]
        optim.moments8_encode_(codes[0], scales[0], codes[1], scales[1], torch.zeros(n, device=gpu), v0)
        plan = optim.AdamW(torch.zeros(n, device=gpu), g, codes[0], codes[1], m_scale=scales[0], v_scale=scales[1])
        out = torch.empty(n, device=gpu)
        optim.moments8_decode_(None, out, None, None, codes[1], scales[1])
        start = out.view(64, 256)[:, 1:].sqrt().mean().item()
        for t in range(1, 401):
            plan.step_(lr=0.0, step=t, seed=seed)
        optim.moments8_decode_(None, out, None, None, codes[1], scales[1])
        means[seed] = (start, out.view(64, 256)[:, 1:].sqrt().mean().item())
    assert means[0][0] == means[0][1]  # nearest: not one byte moved in 400 steps
    # exact: v_t = g^2 + (v_0 - g^2) beta2^t; each step adds noise to the root of at most half a byte's
    # step (2^-4 relative) of mean 0: over 400 steps and 16320 elements the mean's deviation is below
    # 0.5 * 2^-4 * 0.02 * sqrt(400 / 16320) = 1e-4; the mean of roots lies below the root of the mean
    # by var / 2 (relative (2^-4)^2 * 400 * 0.0005 / 2 = 4e-4 at most): 5 deviations
    want = np.sqrt(0.02 ** 2 + (means[5][0] ** 2 - 0.02 ** 2) * 0.999 ** 400)
    assert abs(means[5][1] - want) < 5e-4 + 4e-4 * want * 10, (means, want)


def test_not_finite_without_control(gpu):
    """Gradients that are not finite poison their own elements alone, in both forms."""
    import torch

    n = 1024
    bad = {3: float("nan"), 300: float("inf"), 301: -float("inf"), 511: 3e38, 1023: float("nan")}
    for eight in (False, True):
        s = Setup(gpu, [n], eight=eight, seed=11)
        for i, x in bad.items():
            s.g.views[0][i] = x
        before = s.state()[0]
        s.plan.step_(lr=1e-3, step=2, seed=0)
        after = s.state()[0]
        fine = np.ones(n, bool)
        fine[list(bad)] = False
        (p, m, v), (ep, em, ev) = R.step64(before["p"], before["g"], before["m"], before["v"], lr=1e-3 * s.ls[0], t=2, wd=s.wd[0])
        assert (np.abs(after["p"] - p) <= ep * 3 + 1e-9)[fine].all()
        for i in (3, 300, 301, 1023):
            assert np.isnan(after["p"][i]) and not np.isfinite(after["m"][i]), (eight, i)
            assert not np.isfinite(after["v"][i]), (eight, i)
        assert np.isfinite(after["m"][511]) and np.isinf(after["v"][511]) and np.isfinite(after["p"][511])
        assert np.isfinite(after["m"][fine]).all() and np.isfinite(after["v"][fine]).all()
        if eight:
            m[~fine & (np.arange(n) != 511)] = np.nan
            root = np.sqrt(v)
            root[~fine] = np.inf
            half = np.full(n, 0.5)
            R.check_codes(m, em + 2 * R.U32 * np.abs(before["m"]), after["mc"], after["ms"], 3, half)
            R.check_codes(root, 8 * R.U32 * np.where(fine, root, 0), after["vc"], after["vs"], 4, half)


def test_eps_zero_and_all_zero(gpu):
    """Zero gradients and moments: nothing moves but by the decay; with eps 0 the formula's 0 / 0."""
    import torch

    for eight in (False, True):
        for eps in (1e-8, 0.0):
            s = Setup(gpu, [700], eight=eight, seed=3, cold=True, eps=eps, wd=[0.1])
            s.g.views[0].zero_()
            before = s.state()[0]
            s.plan.step_(lr=0.01, step=1, seed=9)
            after = s.state()[0]
            assert (after["m"] == 0).all() and (after["v"] == 0).all()
            if eps:
                assert (np.abs(after["p"] - before["p"] * (1 - 0.01 * 0.1)) <= 4 * R.U32 * np.abs(before["p"])).all()
            else:
                assert np.isnan(after["p"]).all()


# ---- the norm -------------------------------------------------------------------------------------
@pytest.mark.parametrize("grad", GRADS)
@pytest.mark.parametrize("sizes", [[1], [4096], [4097, 1, 0, 255], [84 * 1024], [85 * 1024], [70, 0, 500, 1025, 3, 2000],
                                   [9] * 7 + [0], [9] * 8, [1 << 20, 3, 5_000_001], RAGGED * 8])
def test_norm(gpu, grad, sizes):
    """Norm, clip factor, step number and corrections; the same bits every time."""
    import torch

    gen = torch.Generator(device=gpu)
    gen.manual_seed(2)
    flat = Flat(torch, gpu, sizes, dt(grad), [torch.randn(n, generator=gen, device=gpu) for n in sizes])
    plan = optim.AdamW(None, flat.views, betas=(B1, B2))
    for scale, max_norm in ((1.0, 0.0), (-0.5, 0.25), (0.125, 1e9)):
        ctrl = optim.Control(gpu, lr=0.5, step=9)
        plan.grad_norm_(ctrl, max_norm=max_norm, grad_scale=scale)
        norm, mult = R.norm64([f64(x) for x in flat.views], scale, max_norm)
        # fp64 sums of at most 2^24 squares: 2^-28 at worst; then one rounding to fp32
        assert abs(ctrl.norm.item() - norm) <= norm * (R.U32 + 2.0 ** -28)
        assert abs(ctrl.mult.item() - mult) <= abs(mult) * (R.U32 + 2.0 ** -28)
        assert (ctrl.step.item(), ctrl.skip.item(), ctrl.skipped.item(), ctrl.lr.item()) == (10, 0, 0, 0.5)
        c = ctrl.buffer.view(torch.float32)[8:10].cpu().numpy()
        assert np.allclose(c, [1 / (1 - B1 ** 10), 1 / np.sqrt(1 - B2 ** 10)], rtol=R.U32 * 1.01, atol=0)
        again = optim.Control(gpu, lr=0.5, step=9)
        plan.grad_norm_(again, max_norm=max_norm, grad_scale=scale)
        assert torch.equal(ctrl.buffer, again.buffer)
    flat.check("grads")


def test_norm_of_huge_and_tiny(gpu):
    """Squares beyond fp32's range in both directions."""
    import torch

    for x in (3e38, 1e-40):
        plan = optim.AdamW(None, [torch.full((1000,), x, device=gpu)])
        ctrl = optim.Control(gpu)
        plan.grad_norm_(ctrl, max_norm=1.0, grad_scale=1e-3)
        want = 1e-3 * float(np.float32(x)) * np.sqrt(1000)
        assert abs(ctrl.norm.item() - want) <= 2 * R.U32 * want + 2.0 ** -149 and ctrl.skip.item() == 0


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_skip(gpu, bad, eight):
    """One gradient that is not finite, anywhere: the step writes nothing and does not count."""
    import torch

    s = Setup(gpu, [100, 9000, 5], "bf16", True, "bf16", eight, seed=5)
    ctrl = optim.Control(gpu, lr=1e-3, step=4)
    keep = s.g.views[1][8999].clone()
    s.g.views[1][8999] = bad
    bufs = [x.buf for x in (s.p, s.pm, s.m, s.v)] + ([s.ms.buf, s.vs.buf] if eight else [])
    before = [x.clone() for x in bufs]
    s.plan.grad_norm_(ctrl, max_norm=1.0)
    s.plan.step_(ctrl=ctrl, seed=3)
    assert (ctrl.skip.item(), ctrl.skipped.item(), ctrl.step.item()) == (1, 1, 4)
    assert all(torch.equal(a, b) for a, b in zip(before, bufs))
    s.g.views[1][8999] = keep  # and the next one counts again
    state = s.state()
    s.plan.grad_norm_(ctrl, max_norm=0.05)
    s.plan.step_(ctrl=ctrl, seed=3)
    assert (ctrl.skip.item(), ctrl.skipped.item(), ctrl.step.item()) == (0, 1, 5)
    s.compare(state, s.state(), lr=float(np.float32(1e-3)), t=5, mult=ctrl.mult.item(), seed=3)


def test_control_equals_arguments(gpu):
    """The same step through ctrl and through arguments: the same bits."""
    import torch

    for eight in (False, True):
        a, b = (Setup(gpu, RAGGED, eight=eight, seed=12) for _ in range(2))
        ctrl = optim.Control(gpu, lr=2e-3, step=41)
        a.plan.grad_norm_(ctrl, grad_scale=0.5)
        a.plan.step_(ctrl=ctrl, seed=8)
        b.plan.step_(lr=2e-3, step=42, grad_scale=0.5, seed=8)
        for x, y in ((a.p, b.p), (a.m, b.m), (a.v, b.v)):
            assert torch.equal(x.buf, y.buf)


# ---- how a program calls it -------------------------------------------------------------------------
def test_graph_replays(gpu):
    """grad_norm + step captured once: every replay is the next step, lr and gradients as they are by
    then, with eager work between; the results are those of eager calls."""
    import torch

    for eight in (False, True):
        a, b = (Setup(gpu, [4097, 300, 1], "bf16", True, "f32", eight, seed=21) for _ in range(2))
        ca, cb = (optim.Control(gpu, lr=1e-3) for _ in range(2))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        values = torch.empty(4097, device=gpu)
        dropped = [Setup(gpu, [10])]
        with torch.cuda.graph(graph, stream=side):
            a.plan.grad_norm_(ca, max_norm=0.1)
            dropped.clear()  # a plan that goes during a capture does not end it
            a.plan.step_(ctrl=ca, seed=4)
            if eight:
                optim.moments8_decode_(values, None, a.m.views[0], a.ms.views[0], None, None)
        gen = torch.Generator(device=gpu)
        for k in range(6):
            gen.manual_seed(k)
            for s in (a, b):
                gen.manual_seed(k)
                for v in s.g.views:
                    v.copy_(torch.randn(v.numel(), generator=gen, device=gpu) * 0.01)
            if k == 3:  # an overflow in the middle
                a.g.views[0][7] = b.g.views[0][7] = float("inf")
            for c in (ca, cb):
                c.lr.fill_(1e-3 / (k + 1))
            graph.replay()
            b.plan.grad_norm_(cb, max_norm=0.1)
            b.plan.step_(ctrl=cb, seed=4)
            torch.cuda.synchronize()
            for x, y in ((a.p, b.p), (a.pm, b.pm), (a.m, b.m), (a.v, b.v)):
                assert torch.equal(x.buf, y.buf), k
            assert torch.equal(ca.buffer, cb.buffer), k
            if eight:
                want = R.values8(b.m.views[0].cpu().numpy(), b.ms.views[0].cpu().numpy(), 3)
                assert (np.abs(f64(values) - want) <= R.U32 * np.abs(want)).all(), k
        assert ca.step.item() == 5 and ca.skipped.item() == 1
        del graph


def test_two_graphs_of_one_plan(gpu):
    """Two graphs that hold the same plan, replayed in turn on one stream: each has its own workspace."""
    import torch

    a, b = (Setup(gpu, RAGGED, seed=31) for _ in range(2))
    ca, cb = (optim.Control(gpu, lr=1e-3) for _ in range(2))
    graphs = []
    for norm in (0.1, 0.01):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            a.plan.grad_norm_(ca, max_norm=norm)
            a.plan.step_(ctrl=ca)
    for k in range(4):
        graphs[k % 2].replay()
        b.plan.grad_norm_(cb, max_norm=(0.1, 0.01)[k % 2])
        b.plan.step_(ctrl=cb)
        assert torch.equal(a.p.buf, b.p.buf) and torch.equal(ca.buffer, cb.buffer)


def test_graph_of_a_bucket(gpu):
    """A captured step that names its bucket: checked at the capture, replayed without the host."""
    import torch

    a, b = (Setup(gpu, RAGGED, grad="bf16", seed=33, bucket=True) for _ in range(2))
    other = a.g.buf.clone()
    ca, cb = (optim.Control(gpu, lr=1e-3) for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.plan.grad_norm_(ca, max_norm=0.1, bucket=other)
        a.plan.step_(ctrl=ca, bucket=other)
    for k in range(3):
        other.mul_(-0.5)
        graph.replay()
        b.plan.grad_norm_(cb, max_norm=0.1, bucket=other)
        b.plan.step_(ctrl=cb, bucket=other)
        torch.cuda.synchronize()
        assert torch.equal(a.p.buf, b.p.buf) and torch.equal(ca.buffer, cb.buffer), k


def test_thousands_of_tensors(gpu):
    """A long list of tiny tensors: one launch, every tensor with its own decay and rate."""
    s = Setup(gpu, [1 + i % 37 for i in range(5000)], "f32", False, "f32", False, seed=3, pad=1)
    before = s.state()
    ctrl = optim.Control(gpu, lr=1e-3)
    s.plan.grad_norm_(ctrl)
    s.plan.step_(ctrl=ctrl)
    norm, _ = R.norm64([x["g"] for x in before], 1.0, 0.0)
    assert abs(ctrl.norm.item() - norm) <= 2 * R.U32 * norm
    s.compare(before, s.state(), lr=float(np.float32(1e-3)), t=1)
    s.guards()


def test_threads_share_a_plan(gpu):
    """Two threads, each with its stream, its ctrl and its bucket, over one plan of gradients."""
    import threading

    import torch

    gen = torch.Generator(device=gpu)
    gen.manual_seed(1)
    bucket = torch.randn(200000, generator=gen, device=gpu)
    plan = optim.AdamW(None, [bucket[:70000], bucket[70001:200000]], bucket=bucket)
    others = [torch.randn(200000, generator=gen, device=gpu) for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        side = torch.cuda.Stream()
        ctrl = optim.Control(gpu)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(50):
                plan.grad_norm_(ctrl, bucket=others[i])
        side.synchronize()
        got[i] = (ctrl.norm.item(), ctrl.step.item())

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for i in range(2):
        x = f64(others[i])
        norm, _ = R.norm64([x[:70000], x[70001:200000]], 1.0, 0.0)
        assert got[i][1] == 50 and abs(got[i][0] - norm) <= 2 * R.U32 * norm


def test_other_stream(gpu):
    """Calls on a side stream, by torch's context and by handle."""
    import torch

    a, b = (Setup(gpu, [50000], eight=True, seed=14) for _ in range(2))
    ctrl = [optim.Control(gpu, lr=1e-3) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.plan.grad_norm_(ctrl[0], max_norm=0.5)
        a.plan.step_(ctrl=ctrl[0], seed=2)
    torch.cuda.current_stream().wait_stream(side)
    side.wait_stream(torch.cuda.current_stream())
    b.plan.grad_norm_(ctrl[1], max_norm=0.5, stream=side.cuda_stream)
    b.plan.step_(ctrl=ctrl[1], seed=2, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(a.p.buf, b.p.buf) and torch.equal(a.m.buf, b.m.buf) and torch.equal(a.vs.buf, b.vs.buf)


def test_bucket_in_turn(gpu):
    """Gradients as views of a bucket, another bucket of the same layout in the next call."""
    import torch

    a = Setup(gpu, RAGGED, grad="bf16", seed=15, bucket=True)
    other = torch.randn(a.g.buf.numel() + 10, device=gpu).to(torch.bfloat16)
    ctrl = optim.Control(gpu, lr=1e-3)
    a.plan.grad_norm_(ctrl)
    first = ctrl.norm.item()
    a.plan.grad_norm_(ctrl, bucket=other)
    assert first != ctrl.norm.item()
    before = a.state()
    a.plan.step_(lr=1e-3, step=2, bucket=other)
    kept = a.g.buf.clone()
    a.g.buf.copy_(other[: a.g.buf.numel()])
    for s, v in zip(before, a.g.views):
        s["g"] = f64(v)
    a.compare(before, a.state(), lr=1e-3, t=2)
    a.g.buf.copy_(kept)
    with pytest.raises(_lib.HydraError, match="shorter"):
        a.plan.step_(lr=1e-3, step=3, bucket=other[:100])
    with pytest.raises(_lib.HydraError, match="like the grads"):
        a.plan.step_(lr=1e-3, step=3, bucket=other.float())
    with pytest.raises(_lib.HydraError, match="without a bucket"):
        Setup(gpu, [10]).plan.step_(lr=1e-3, step=3, bucket=other)


def test_allreduce_then_step(gpu):
    """As a data-parallel program runs it: P ranks' buckets reduced by the framework's own ring (every
    rank on this GPU), then norm, clip and step on each rank: all ranks end with the same bits, and
    those are the 64-bit reference's step on the mean gradient."""
    import torch

    from hydra_amd import ring, synth

    P, sizes = 3, [5000, 1, 777, 4096]
    total = sum(sizes) + 3 * (len(sizes) + 1)
    ranks = [Setup(gpu, sizes, "bf16", True, "f32", True, seed=40, bucket=True) for _ in range(P)]
    for r, s in enumerate(ranks):
        s.g.buf.copy_(torch.from_numpy(synth.uniform_f32(total, 100 + r)) * 0.01)
    ctrls = [optim.Control(gpu, lr=1e-3) for _ in range(P)]
    for k in range(2):
        for r, s in enumerate(ranks):
            s.g.buf.copy_(torch.from_numpy(synth.uniform_f32(total, 100 + 10 * k + r)) * 0.01)
        ring.simulate([s.g.buf for s in ranks], algo="ring")
        before = ranks[0].state()
        for s, c in zip(ranks, ctrls):
            s.plan.grad_norm_(c, max_norm=0.2, grad_scale=1.0 / P)
            s.plan.step_(ctrl=c, seed=17)
        after = ranks[0].state()
        norm, mult = R.norm64([x["g"] for x in before], float(1.0 / P), 0.2)
        assert abs(ctrls[0].norm.item() - norm) <= 2 * R.U32 * norm
        ranks[0].compare(before, after, lr=float(np.float32(1e-3)), t=k + 1, mult=ctrls[0].mult.item(), seed=17)
        for s, c in zip(ranks[1:], ctrls[1:]):
            for name in ("p", "pm", "m", "v", "ms", "vs"):
                assert torch.equal(getattr(s, name).buf, getattr(ranks[0], name).buf), (k, name)
            assert torch.equal(c.buffer, ctrls[0].buffer)


def test_refusals(gpu):
    """What the Python face and the device checks refuse."""
    import ctypes

    import torch

    def new(n=64, dtype=torch.float32):
        return torch.zeros(n, dtype=dtype, device=gpu)

    bad = [
        (dict(grads=[torch.zeros(64)]), "one GPU"), (dict(params=[new(65)]), "elements"), (dict(m=[new(), new()]), "2 m for 1"),
        (dict(params=[new(128)[::2]]), "contiguous"), (dict(m=[new(dtype=torch.bfloat16)]), "float32 or both uint8"),
        (dict(m=[new(dtype=torch.uint8)], v=[new(dtype=torch.uint8)]), "m_scale and v_scale"),
        (dict(m_scale=[new(1)], v_scale=[new(1)]), "m_scale and v_scale"), (dict(master=[new()]), "master"),
        (dict(weight_decay=[0.1, 0.2]), "weight_decay"), (dict(betas=(1.0, 0.9)), "betas"),
        (dict(params=[new(dtype=torch.float64)]), "unsupported"), (dict(bucket=new(200)), "view of the bucket"),
    ]
    for kw, word in bad:
        args = dict(params=[new()], grads=[new()], m=[new()], v=[new()])
        args.update(kw)
        with pytest.raises(_lib.HydraError, match=word):
            optim.AdamW(**args)
    x = new()
    with pytest.raises(_lib.HydraError, match="overlap"):
        optim.AdamW([x], [new()], [x], [new()])
    with pytest.raises(_lib.HydraError, match="overlaps"):
        optim.AdamW([x], [x], [new()], [new()])
    norm = optim.AdamW(None, [x])
    with pytest.raises(_lib.HydraError, match="gradients alone"):
        norm.step_(lr=1e-3, step=1)
    plan = optim.AdamW([new()], [new()], [new()], [new()])
    ctrl = optim.Control(gpu)
    for call, word in ((lambda: plan.step_(lr=1e-3, step=0), "from 1"), (lambda: plan.step_(lr=float("nan"), step=1), "finite"),
                       (lambda: plan.step_(lr=1e39, step=1), "finite"), (lambda: plan.step_(), "lr and step"),
                       (lambda: plan.step_(lr=1.0, ctrl=ctrl), "come from ctrl"),
                       (lambda: plan.grad_norm_(ctrl, max_norm=-1.0), "max_norm"),
                       (lambda: plan.grad_norm_(ctrl, grad_scale=float("inf")), "grad_scale")):
        with pytest.raises(_lib.HydraError, match=word):
            call()
    # host memory in a C caller's list
    host = np.zeros(64, np.float32)
    t = _lib.AdamWTensor(x.data_ptr(), None, host.ctypes.data, new().data_ptr(), new().data_ptr(), None, None, 64, 1.0, 0.0)
    m, v = new(), new()
    t.m, t.v = m.data_ptr(), v.data_ptr()
    cfg = _lib.AdamWConfig(_lib.FLOAT32, _lib.FLOAT32, _lib.FLOAT32, 0, 0.9, 0.999, 1e-8)
    h = ctypes.c_void_p()
    L = _lib.lib()
    assert L.hydra_adamw_create(0, ctypes.byref(cfg), (_lib.AdamWTensor * 1)(t), 1, ctypes.byref(h)) == _lib.ERR_INVALID
    assert b"not memory of the plan's device" in L.hydra_last_error()
    assert L.hydra_adamw_create(999, ctypes.byref(cfg), (_lib.AdamWTensor * 1)(t), 1, ctypes.byref(h)) == 4
    # a workspace that is too small
    ws = torch.empty(8, dtype=torch.uint8, device=gpu)
    big = optim.AdamW(None, [new(100000)])
    assert L.hydra_adamw_grad_norm(big._h, None, 1.0, 0.0, ctrl.buffer.data_ptr(), ws.data_ptr(), 0, None) == _lib.ERR_INVALID
    plan.close()
    with pytest.raises(_lib.HydraError, match="closed"):
        plan.step_(lr=1e-3, step=1)


def test_empty_plans(gpu):
    """No elements at all: nothing to do, a norm of zero."""
    import torch

    e = [torch.zeros(0, device=gpu) for _ in range(4)]
    plan = optim.AdamW([e[0]], [e[1]], [e[2]], [e[3]])
    ctrl = optim.Control(gpu, lr=1.0)
    plan.grad_norm_(ctrl, max_norm=1.0)
    plan.step_(ctrl=ctrl)
    plan.step_(lr=1.0, step=1)
    assert (ctrl.norm.item(), ctrl.mult.item(), ctrl.step.item(), ctrl.skip.item()) == (0.0, 1.0, 1, 0)


# ---- 8-bit moments ------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 3, 255, 256, 257, 1024, 70001])
def test_moments8(gpu, n, kind):
    """Encode against the definition, decode against the bytes' values; the lengths around a block."""
    import torch

    gen = torch.Generator(device=gpu)
    gen.manual_seed(n)
    level = torch.exp2(torch.randint(-24, 4, (n,), generator=gen, device=gpu).float())
    m = Flat(torch, gpu, [n], dt(kind), [torch.randn(n, generator=gen, device=gpu) * level])
    v = Flat(torch, gpu, [n], dt(kind), [(torch.randn(n, generator=gen, device=gpu) * level) ** 2])
    if n > 700:
        m.views[0][:256] = 0
        v.views[0][256:512] = 0
        m.views[0][600], m.views[0][601], v.views[0][602] = float("nan"), float("-inf"), float("inf")
    rows = optim.moment_scales(n)
    m8, v8 = (Flat(torch, gpu, [n], torch.uint8, [torch.full((n,), 9, device=gpu)], guard=77) for _ in "mv")
    ms, vs = (Flat(torch, gpu, [rows], torch.float32, [torch.full((rows,), 9.0, device=gpu)]) for _ in "mv")
    optim.moments8_encode_(m8.views[0], ms.views[0], v8.views[0], vs.views[0], m.views[0], v.views[0])
    x, root = f64(m.views[0]), np.sqrt(f64(v.views[0]))
    half = np.full(n, 0.5)
    cm, cv, sm, sv = (t.views[0].cpu().numpy() for t in (m8, v8, ms, vs))
    # bf16 values X * 2^a (X of 8 bits) over a scale 8/15 A * 2^b (A of 8 bits): 15 X / A * 2^c is a
    # half-integer in [8, 16), a tie to nearest, for every X = 8 mod 16 where A = 240: 1/16 of them
    # at worst, and twice that for the draw
    loose = 1e-3 if kind == "f32" else 1 / 8
    R.check_codes(x, np.zeros(n), cm, sm, 3, half, "m", loose)
    R.check_codes(root, np.where(np.isfinite(root), R.U32 * root, 0), cv, sv, 4, half, "v", loose)
    for out in ("f32", "bf16"):
        mo, vo = (Flat(torch, gpu, [n], dt(out), [torch.zeros(n, device=gpu)]) for _ in "mv")
        optim.moments8_decode_(mo.views[0], vo.views[0], m8.views[0], ms.views[0], v8.views[0], vs.views[0])
        want = R.values8(cm, sm, 3), R.values8(cv, sv, 4) ** 2
        for got, w, k in ((mo, want[0], 1), (vo, want[1], 3)):  # one product; the same, doubled by the square, and it
            got = f64(got.views[0])
            fin = np.isfinite(w)
            assert np.array_equal(np.isnan(got), np.isnan(w)) and np.array_equal(np.isinf(got), np.isinf(w))
            tol = np.abs(w[fin]) * (k * R.U32 + HALF[out]) * 1.01 + 2.0 ** -133
            assert (np.abs(got[fin] - w[fin]) <= tol).all()
        mo.check("m out"), vo.check("v out")
    # one moment at a time gives the same
    m8b, msb = torch.zeros_like(m8.views[0]), torch.zeros_like(ms.views[0])
    optim.moments8_encode_(m8b, msb, None, None, m.views[0], None)
    assert torch.equal(m8b, m8.views[0]) and torch.equal(msb, ms.views[0])
    v8b, vsb = torch.zeros_like(v8.views[0]), torch.zeros_like(vs.views[0])
    optim.moments8_encode_(None, None, v8b, vsb, None, v.views[0])
    assert torch.equal(v8b, v8.views[0]) and torch.equal(vsb, vs.views[0])
    for t, what in ((m8, "m8"), (v8, "v8"), (ms, "ms"), (vs, "vs"), (m, "m"), (v, "v")):
        t.check(what)


def test_moments8_extremes(gpu):
    """Blocks at both ends of fp32's range, and a block too small to store."""
    import torch

    for x in (3e38, 1e30, 1e-20, 2.0 ** -99, 2.0 ** -101, 1e-40):
        m = torch.linspace(-1, 1, 256, device=gpu, dtype=torch.float64).mul(x).float()
        v = torch.linspace(0, 1, 256, device=gpu, dtype=torch.float64).mul(min(x, 1e38)).float()
        m8, v8 = (torch.zeros(256, dtype=torch.uint8, device=gpu) for _ in "mv")
        ms, vs = (torch.zeros(1, device=gpu) for _ in "mv")
        optim.moments8_encode_(m8, ms, v8, vs, m, v)
        R.check_codes(f64(m), np.zeros(256), m8.cpu().numpy(), ms.cpu().numpy(), 3, np.full(256, 0.5), x)
        root = np.sqrt(f64(v))
        R.check_codes(root, R.U32 * root, v8.cpu().numpy(), vs.cpu().numpy(), 4, np.full(256, 0.5), x)


def test_beyond_32_bits(gpu):
    """Tensors of more than 2^32 elements: offsets, blocks and random words beyond 32 bits."""
    import torch

    n = (1 << 32) + 4096 * 3 + 77
    bf = torch.bfloat16
    p, g = torch.zeros(n, dtype=bf, device=gpu), torch.empty(n, dtype=bf, device=gpu)
    pattern = (torch.randn(1 << 20, device=gpu) * 0.01).to(bf)
    for at in range(0, n, 1 << 28):  # the same values in every stretch
        part = g[at:at + (1 << 28)]
        part.copy_(pattern.repeat(-(-part.numel() // (1 << 20)))[: part.numel()])
    m8, v8 = (torch.zeros(n, dtype=torch.uint8, device=gpu) for _ in "mv")
    ms, vs = (torch.zeros(optim.moment_scales(n), device=gpu) for _ in "mv")
    plan = optim.AdamW([p], [g], [m8], [v8], m_scale=[ms], v_scale=[vs], weight_decay=0.0)
    ctrl = optim.Control(gpu, lr=0.5)
    plan.grad_norm_(ctrl)
    total = float((f64(pattern) ** 2).sum()) * 4096 + float((f64(g[1 << 32:]) ** 2).sum())
    assert abs(ctrl.norm.item() - np.sqrt(total)) <= np.sqrt(total) * (R.U32 + 2.0 ** -30)
    plan.step_(ctrl=ctrl, seed=7)
    for at in (0, (1 << 31) - 512, 1 << 32, n // 256 * 256 - 2560):
        end = min(n, at + 5120)
        x = f64(g[at:end])
        zero = np.zeros(x.size)
        (want, m, v), (ep, em, ev) = R.step64(zero, x, zero, zero, lr=0.5, t=1)
        r = R.random_words(7, 1, 0, np.arange(at, end))
        rows = slice(at // 256, -(-end // 256))
        root = np.sqrt(v)
        R.check_codes(m, em, m8[at:end].cpu().numpy(), ms[rows].cpu().numpy(), 3, (r & np.uint64(0xFFFF)) / 65536.0, at)
        er = np.where(root > 0, ev / np.maximum(2 * root, 1e-300), 0) + R.U32 * root
        R.check_codes(root, er, v8[at:end].cpu().numpy(), vs[rows].cpu().numpy(), 4, (r >> np.uint64(16)) / 65536.0, at)
        assert (np.abs(f64(p[at:end]) - want) <= ep + 2.0 ** -8 * (np.abs(want) + ep)).all()
