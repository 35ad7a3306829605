"""The optimizer step's boundary without a GPU: exports, layouts, and every refusal that comes before
HIP is touched."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

import optim_ref as R
from hydra_amd import _lib, optim

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, BF16, F16, U8 = _lib.FLOAT32, _lib.BFLOAT16, _lib.FLOAT16, _lib.UINT8


def test_header_symbols_exported():
    txt = open(os.path.join(ROOT, "include", "hydra_optim.h")).read()
    declared = set(re.findall(r"\b(hydra_[a-z0-9_]+)\s*\(", re.sub(r"/\*.*?\*/", "", txt, flags=re.S)))
    assert declared == set(_lib.OPTIM_EXPORTS)
    out = subprocess.check_output(["nm", "-D", "--defined-only", _lib.LIB_PATH], text=True)
    assert declared <= {ln.split()[-1] for ln in out.splitlines() if " T " in ln}


def test_header_is_plain_c(tmp_path):
    """The header compiles as C11, and its structs have the layout the ctypes face assumes."""
    src = tmp_path / "t.c"
    src.write_text('#include "hydra_optim.h"\n#include <stdio.h>\nint main(void) {'
                   'printf("%zu %zu %zu %zu\\n", sizeof(hydra_adamw_tensor_t), '
                   'sizeof(hydra_adamw_config_t), sizeof(hydra_adamw_ctrl_t), '
                   '__builtin_offsetof(hydra_adamw_ctrl_t, skip)); return 0; }')
    exe = tmp_path / "t"
    subprocess.check_call(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"),
                           str(src), "-o", str(exe)])
    got = [int(x) for x in subprocess.check_output([str(exe)], text=True).split()]
    assert got == [ctypes.sizeof(_lib.AdamWTensor), ctypes.sizeof(_lib.AdamWConfig), 64, 28]


def config(**kw):
    c = dict(param_dtype=F32, grad_dtype=F32, state_dtype=F32, flags=0, beta1=0.9, beta2=0.999, eps=1e-8)
    c.update(kw)
    return _lib.AdamWConfig(*(c[f] for f, _ in _lib.AdamWConfig._fields_))


BASE = 1 << 20  # addresses never touched: every refusal here comes before HIP


def tensor(**kw):
    n = kw.pop("n", 1000)
    t = dict(param=BASE, master=None, grad=BASE + 0x10000, m=BASE + 0x20000, v=BASE + 0x30000,
             m_scale=None, v_scale=None, n=n, lr_scale=1.0, weight_decay=0.0)
    t.update(kw)
    return _lib.AdamWTensor(*(t[f] for f, _ in _lib.AdamWTensor._fields_))


def create(cfg, *ts, count=None):
    arr = (_lib.AdamWTensor * max(1, len(ts)))(*ts)
    h = ctypes.c_void_p()
    rc = _lib.lib().hydra_adamw_create(0, ctypes.byref(cfg), arr, len(ts) if count is None else count,
                                       ctypes.byref(h))
    if rc == 0:
        _lib.lib().hydra_adamw_destroy(h)
    assert rc == 0 or not h
    return rc, _lib.lib().hydra_last_error().decode()


@pytest.mark.parametrize("cfg,word", [
    (dict(grad_dtype=_lib.INT32), "gradients"), (dict(grad_dtype=_lib.FLOAT64), "gradients"),
    (dict(param_dtype=_lib.FLOAT64), "params"), (dict(state_dtype=BF16), "moments"),
    (dict(flags=8), "flags"), (dict(beta1=1.0), "betas"), (dict(beta2=-0.1), "betas"),
    (dict(beta2=float("nan")), "betas"), (dict(beta2=1 - 2.0 ** -40), "fp32"),
    (dict(eps=-1e-8), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(flags=_lib.ADAMW_MASTER), "master"),
])
def test_bad_configs(cfg, word):
    rc, msg = create(config(**cfg), tensor())
    assert rc == _lib.ERR_INVALID and word in msg, (rc, msg)


@pytest.mark.parametrize("cfg,t,word", [
    ({}, dict(param=None), "null param"), ({}, dict(grad=None), "null gradient"),
    ({}, dict(m=None), "null m"), ({}, dict(v=None), "null v"),
    ({}, dict(param=BASE + 2), "aligned"), ({}, dict(grad=BASE + 0x10002), "aligned"),
    ({}, dict(m=BASE + 0x20001), "aligned"), ({}, dict(master=BASE + 0x40000), "master given"),
    ({}, dict(m_scale=BASE + 0x40000), "m_scale given"), ({}, dict(n=(1 << 40) + 1), "2^40"),
    ({}, dict(lr_scale=float("nan")), "finite"), ({}, dict(weight_decay=float("inf")), "finite"),
    ({}, dict(m=BASE + 0x20000, v=BASE + 0x20000 + 3996), "overlap"),
    ({}, dict(grad=BASE + 3996), "gradient overlaps"),
    (dict(param_dtype=BF16, flags=_lib.ADAMW_MASTER), {}, "null master"),
    (dict(state_dtype=U8), {}, "null m_scale"),
    (dict(state_dtype=U8), dict(m_scale=BASE + 0x40000), "null v_scale"),
    (dict(state_dtype=U8), dict(m_scale=BASE + 0x40000, v_scale=BASE + 0x4000c), "overlap"),
    (dict(flags=_lib.ADAMW_BUCKET), dict(grad=2), "aligned"),
    (dict(flags=_lib.ADAMW_BUCKET), dict(grad=1 << 60), "offset"),
])
def test_bad_tensors(cfg, t, word):
    rc, msg = create(config(**cfg), tensor(**t))
    assert rc == _lib.ERR_INVALID and word in msg, (rc, msg)


def test_the_same_tensor_twice_is_refused():
    rc, msg = create(config(), tensor(), tensor())
    assert rc == _lib.ERR_INVALID and "overlap" in msg
    rc, msg = create(config(), tensor(), tensor(param=BASE + 0x100000, m=BASE + 0x110000, v=BASE + 0x20000 + 3996))
    assert rc == _lib.ERR_INVALID and "overlap" in msg


def test_a_plan_beyond_one_launch_is_refused():
    rc, msg = create(config(), tensor(n=1 << 37))
    assert rc == _lib.ERR_INVALID and "split" in msg


def test_null_handles_and_scalars():
    L = _lib.lib()
    size = ctypes.c_size_t()
    assert L.hydra_adamw_destroy(None) == 0
    assert L.hydra_adamw_workspace(None, ctypes.byref(size)) == _lib.ERR_INVALID
    assert L.hydra_adamw_step(None, None, 1e-3, 1, 1.0, 0, None) == _lib.ERR_INVALID
    assert L.hydra_adamw_step_ctrl(None, None, None, 0, None) == _lib.ERR_INVALID
    assert L.hydra_adamw_grad_norm(None, None, 1.0, 0.0, None, None, 0, None) == _lib.ERR_INVALID
    assert L.hydra_adamw_create(0, None, None, 0, None) == _lib.ERR_INVALID
    h = ctypes.c_void_p()
    assert L.hydra_adamw_create(0, None, None, 0, ctypes.byref(h)) == _lib.ERR_INVALID
    c = config()
    assert L.hydra_adamw_create(0, ctypes.byref(c), None, 2, ctypes.byref(h)) == _lib.ERR_INVALID
    assert b"null tensor list" in L.hydra_last_error()


@pytest.mark.parametrize("name", ["hydra_moments8_encode", "hydra_moments8_decode"])
def test_bad_conversions(name):
    L = _lib.lib()
    enc = name.endswith("encode")
    good = dict(m8=BASE, ms=BASE + 0x10000, v8=BASE + 0x20000, vs=BASE + 0x30000, m=BASE + 0x40000,
                v=BASE + 0x50000, dtype=F32, n=1000)

    def call(**kw):
        a = dict(good, **kw)
        if enc:
            rc = L.hydra_moments8_encode(a["m8"], a["ms"], a["v8"], a["vs"], a["m"], a["v"], a["dtype"], a["n"], None)
        else:
            rc = L.hydra_moments8_decode(a["m"], a["v"], a["dtype"], a["m8"], a["ms"], a["v8"], a["vs"], a["n"], None)
        return rc, L.hydra_last_error().decode()

    none = dict(m=None, m8=None, ms=None)
    for kw, word in [(dict(dtype=F16), "fp32 or bf16"), (dict(dtype=99), "fp32 or bf16"), (dict(m=None), "null pointer"),
                     (dict(vs=None), "null pointer"), (dict(none, v=None, v8=None, vs=None), "neither"),
                     (dict(m=BASE + 0x40002), "aligned"), (dict(ms=BASE + 0x10001), "aligned"),
                     (dict(n=(1 << 40) + 1), "2^40"), (dict(m=BASE + 0x50000 - 3996), "overlap" if not enc else ""),
                     (dict(m8=BASE + 0x20000 - 999), "overlap" if enc else ""), (dict(m8=BASE + 0x40000 + 3999), "overlap")]:
        if word:
            rc, msg = call(**kw)
            assert rc == _lib.ERR_INVALID and word in msg, (kw, rc, msg)
    assert call(n=0)[0] == 0  # nothing to do, HIP untouched


def test_python_face_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    g = [torch.zeros(8)]
    with pytest.raises(_lib.HydraError, match="GPU"):
        optim.AdamW([torch.zeros(8)], g, [torch.zeros(8)], [torch.zeros(8)])
    with pytest.raises(_lib.HydraError, match="no tensors"):
        optim.AdamW([], [], [], [])
    with pytest.raises(_lib.HydraError, match="m and v"):
        optim.AdamW([torch.zeros(8)], g)
    with pytest.raises(_lib.HydraError, match="GPU"):
        optim.Control("cpu")
    with pytest.raises(_lib.HydraError, match="one GPU"):
        optim.moments8_decode_(torch.zeros(8), None, torch.zeros(8, dtype=torch.uint8), torch.zeros(1), None, None)
    with pytest.raises(_lib.HydraError, match="neither"):
        optim.moments8_encode_(None, None, None, None, None, None)
    assert [optim.moment_scales(n) for n in (0, 1, 256, 257)] == [0, 1, 1, 2]


# ---- the reference itself: the tests' own oracle is held to the definition ---------------------------
def test_reference_fp32_within_its_own_bounds():
    """step32 lies within step64's derived bounds: mistakes in either would show here, without a GPU."""
    rng = np.random.default_rng(1)
    n = 20000
    p, g = rng.normal(0, 0.05, n).astype(np.float32), (rng.normal(0, 1, n) * 2.0 ** rng.integers(-20, 6, n)).astype(np.float32)
    m, v = (rng.normal(0, 0.1, n)).astype(np.float32), (rng.normal(0, 0.2, n) ** 2).astype(np.float32)
    for t in (1, 2, 1000, 10 ** 6):
        kw = dict(lr=1e-3, t=t, mult=0.3, wd=0.1)
        want, tol = R.step64(p, g, m, v, **kw)
        for a, b, e in zip(R.step32(p, g, m, v, **kw), want, tol):
            assert (np.abs(a - b) <= e).all()


def test_reference_gradient_direction_by_differences():
    """At t = 1 with no decay and eps far above the gradient, the step is lr * g / eps: descending on
    a quadratic follows its gradient, taken by central differences."""
    rng = np.random.default_rng(2)
    a, x = rng.uniform(0.5, 2, 16), rng.normal(0, 1, 16)

    def f(y):
        return 0.5 * (a * y * y).sum()

    h = 1e-6
    grad = np.array([(f(x + h * e) - f(x - h * e)) / (2 * h) for e in np.eye(16)])
    (p, _, _), _ = R.step64(x, grad, np.zeros(16), np.zeros(16), lr=1.0, t=1, eps=1e6)
    assert np.allclose((x - p) * 1e6, a * x, rtol=1e-4)


def test_reference_bytes_round_trip():
    """Every byte reads as a value that encodes, to nearest, to the same byte."""
    for bits, codes in ((3, np.arange(128)), (4, np.arange(255))):
        f = R.values8(codes.astype(np.uint8), np.ones(1), bits)
        assert f.max() == 1.875 and (np.diff(f) > 0).all()
        R.check_codes(f, np.zeros(f.size), codes.astype(np.uint8), np.ones(1), bits, np.full(f.size, 0.5))


def test_reference_check_sees_wrong_bytes():
    """check_codes refuses a byte that is one off."""
    rng = np.random.default_rng(3)
    x = rng.normal(0, 1, 256)
    s = np.float32(np.abs(x).max() / 1.875)
    f = R.values8(np.arange(128, dtype=np.uint8), np.ones(1), 3)
    c = np.array([np.abs(f - abs(y) / s).argmin() for y in x])
    codes = np.where(x < 0, c + 128, c).astype(np.uint8)
    R.check_codes(x, np.abs(x) * R.U32, codes, np.array([s]), 3, np.full(256, 0.5))
    codes[7] ^= 1
    with pytest.raises(AssertionError):
        R.check_codes(x, np.abs(x) * R.U32, codes, np.array([s]), 3, np.full(256, 0.5))


def test_reference_fp32_bytes_are_the_definitions():
    """encode32, the fp32 form operation by operation, passes check_codes, the definition in 64 bits."""
    rng = np.random.default_rng(4)
    n = 256 * 40 + 17
    m = (rng.normal(0, 1, n) * 2.0 ** rng.integers(-12, 3, n)).astype(np.float32)
    v = ((rng.normal(0, 1, n) * 2.0 ** rng.integers(-12, 3, n)) ** 2).astype(np.float32)
    for r in (R.random_words(9, 4, 2, np.arange(n)), np.full(n, 0x80008000, np.uint64)):
        cm, sm, cv, sv, _ = R.encode32(m, v, r)
        R.check_codes(m.astype(np.float64), np.zeros(n), cm, sm, 3, (r & np.uint64(0xFFFF)) / 65536.0)
        root = np.sqrt(v.astype(np.float64))
        R.check_codes(root, R.U32 * root, cv, sv, 4, (r >> np.uint64(16)) / 65536.0)
