"""The optimizer step on a reduced gradient bucket: cases to measure and to compare.

What follows an allreduce of a gradient bucket: the norm of all gradients with its clip factor, the
AdamW step over many tensors with states in 32 or in 8 bits, and the conversion of 8-bit moments
from and to values.  With `own` false, run() computes each in its plain form, elementary torch
operations on whole buffers; with `own` true it makes the calls of hydra_amd.optim.

The buffers are flat, as a bucket is: every tensor is a view at its own offset, odd offsets among
them; the 8-bit form starts every tensor on a block of 256 elements.  The sizes are those of the
framework's own buckets and sweeps (4 Ki, 64 Mi, 256 Mi elements) and ragged ones between them.
"""
import math
import random

import torch

own = False

BLOCK = 256          # elements that share one scale of an 8-bit moment
BETAS, EPS, LR, DECAY = (0.9, 0.999), 1e-8, 3e-5, 0.1
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
M32 = 0xFFFFFFFF


def listed():
    return [
        # the norm: one small bucket, where the launch is all; the 64 Mi fp32 bucket; a model's many
        # bf16 gradients, packed without gaps
        {"name": "norm 4Ki f32", "op": "norm", "tensors": 1, "elements": 4096, "grad": "f32", "mix": 0},
        {"name": "norm 64Mi f32", "op": "norm", "tensors": 1, "elements": 64 << 20, "grad": "f32", "mix": 0},
        {"name": "norm 397 ragged bf16", "op": "norm", "tensors": 397, "elements": 100_000_007, "grad": "bf16", "mix": 1},
        # 32-bit states: the smallest bucket; a small model's tensors with fp16 gradients, clipped;
        # the 64 Mi fp32 bucket; the 256 Mi mixed-precision bucket (bf16 weights and gradients, fp32 master)
        {"name": "adamw 4Ki f32", "op": "adamw", "tensors": 1, "elements": 4096, "param": "f32", "grad": "f32", "clip": False, "mix": 0},
        {"name": "adamw 291 ragged clip", "op": "adamw", "tensors": 291, "elements": 24_000_001, "param": "f32", "grad": "f16", "clip": True, "mix": 2},
        {"name": "adamw 64Mi f32", "op": "adamw", "tensors": 1, "elements": 64 << 20, "param": "f32", "grad": "f32", "clip": False, "mix": 0},
        {"name": "adamw 256Mi master bf16", "op": "adamw", "tensors": 1, "elements": 256 << 20, "param": "master_bf16", "grad": "bf16", "clip": False, "mix": 0},
        # 8-bit states: an adapter's few small tensors; a model's ragged ones, clipped; the large bucket
        {"name": "adamw8 12 small f32", "op": "adamw8", "tensors": 12, "elements": 65_536, "param": "f32", "grad": "f32", "clip": False, "mix": 3},
        {"name": "adamw8 397 ragged clip", "op": "adamw8", "tensors": 397, "elements": 100_000_007, "param": "master_bf16", "grad": "bf16", "clip": True, "mix": 1},
        {"name": "adamw8 64Mi f32", "op": "adamw8", "tensors": 1, "elements": 64 << 20, "param": "f32", "grad": "f32", "clip": False, "mix": 0},
        # moments into 8 bits and back as bf16 values: one layer's, and the large bucket's
        {"name": "moments8 300001", "op": "moments8", "elements": 300_001},
        {"name": "moments8 64Mi", "op": "moments8", "elements": 64 << 20},
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(2 ** rng.uniform(math.log2(lo), math.log2(hi)))) | rng.randint(0, 1)

    op = rng.choice(["norm", "adamw", "adamw", "adamw8", "adamw8", "moments8"])
    if op == "moments8":
        return {"op": op, "elements": size(256, 64 << 20)}
    case = {"op": op, "tensors": rng.choice([1, size(2, 400)]), "elements": size(4096, 64 << 20)}
    case["grad"] = rng.choice(["f32", "bf16", "f16"])
    case["mix"] = rng.randint(1, 1 << 20)
    if op != "norm":
        case["param"] = rng.choice(["f32", "bf16", "f16", "master_bf16", "master_f16"])
        case["clip"] = rng.random() < 0.5
    return case


# ---- sizes and layout --------------------------------------------------------------------------
def sizes_of(case):
    """The tensors' lengths: they span three orders of magnitude, a length of zero among them at times."""
    k, n = case.get("tensors", 1), case["elements"]
    r = random.Random(case.get("mix", 0))
    w = [2.0 ** r.uniform(0, 12) for _ in range(k)]
    total, at, cuts = sum(w), 0.0, [0]
    for x in w:
        at += x
        cuts.append(min(n, int(n * (at / total))))
    cuts[-1] = n
    return [b - a for a, b in zip(cuts, cuts[1:])]


def offsets_of(case, sizes):
    """Every tensor's place in the flat buffers and their whole length."""
    step = BLOCK if case["op"] in ("adamw8", "moments8") else 1
    at, offs = 0, []
    for n in sizes:
        offs.append(at)
        at += -(-n // step) * step
    return offs, at


def decay_of(case):
    """Weight decay by tensor: every fourth has none, as biases and norms have."""
    return [0.0 if i % 4 == 3 else DECAY for i in range(case.get("tensors", 1))]


def split_types(case):
    """(type of the weights, whether an fp32 master stands beside them)"""
    p = case["param"]
    return (TYPES[p[7:]], True) if p.startswith("master_") else (TYPES[p], False)


def _clipping(case, seed):
    """The factor that makes a sum over 8 ranks their mean, where the bucket holds 16 bits, and the norm to clip to:
    the inputs of every other seed exceed it."""
    scale = 1.0 if case["grad"] == "f32" else 0.125
    return scale, scale * math.sqrt(case["elements"]) * (0.02 if seed % 2 else 0.2)


# ---- inputs --------------------------------------------------------------------------------------
def _values(case, seed):
    """fp32 weights, gradients and moments on the flat buffers, zero in the gaps between tensors.
    Gradients vary by 2^+-3 between stretches of 4 Ki elements, as layers' do."""
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed * 2654435761 % (1 << 62))
    sizes = sizes_of(case)
    offs, total = offsets_of(case, sizes)

    def normal():
        return torch.randn(total, generator=gen, device=dev)

    rows = -(-total // 4096)
    level = torch.exp2(6 * torch.rand(rows, generator=gen, device=dev) - 3).mul_(1e-2)

    def by_level(x, power):
        full = total // 4096 * 4096
        x[:full].view(-1, 4096).mul_(level[: full // 4096, None] ** power)
        x[full:].mul_(level[-1] ** power)
        return x

    g = by_level(normal(), 1)
    m = v = p = None
    if case["op"] != "norm":
        m = by_level(normal().mul_(0.2), 1)
        v = by_level(normal().abs_().add_(0.3).square_(), 2)
    if case["op"] in ("adamw", "adamw8"):
        p = normal().mul_(0.05)
    if total != sum(sizes):
        gap = torch.ones(total, dtype=torch.bool, device=dev)
        for o, n in zip(offs, sizes):
            gap[o:o + n] = False
        for x in (g, m, v, p):
            if x is not None:
                x.masked_fill_(gap, 0.0)
    return sizes, offs, total, p, g, m, v


def prepare(case, seed):
    sizes, offs, total, p, g, m, v = _values(case, seed)
    s = {"case": case, "sizes": sizes, "offs": offs, "total": total, "step": 1000, "seed": (seed << 20) | 0x5EED}
    views = lambda x: [x[o:o + n] for o, n in zip(offs, sizes)]  # noqa: E731
    dev = g.device
    if case["op"] == "moments8":
        blocks = total // BLOCK
        s.update(m=m, v=v, m8=torch.zeros(total, dtype=torch.uint8, device=dev), v8=torch.zeros(total, dtype=torch.uint8, device=dev),
                 ms=torch.empty(blocks, device=dev), vs=torch.empty(blocks, device=dev),
                 m_out=torch.empty(total, dtype=torch.bfloat16, device=dev), v_out=torch.empty(total, dtype=torch.bfloat16, device=dev))
        if own:
            from hydra_amd import optim

            s["api"] = optim
        return s
    s["g"] = g.to(TYPES[case["grad"]])
    del g
    s["scale"], s["max_norm"] = _clipping(case, seed)
    if case["op"] != "norm":
        kind, master = split_types(case)
        s["wd"] = decay_of(case)
        s["master"] = p if master else None
        s["p"] = p.to(kind)
        if case["op"] == "adamw":
            s["m"], s["v"] = m, v
        else:
            s["m8"], s["ms"], s["v8"], s["vs"] = _encode(m, v, None)
            s["m_out"] = torch.empty(total, dtype=torch.bfloat16, device=dev)
            s["v_out"] = torch.empty(total, dtype=torch.bfloat16, device=dev)
    if own:
        from hydra_amd import optim

        s["api"] = optim
        grads = views(s["g"])
        if case["op"] == "norm":
            s["plan"] = optim.AdamW(None, grads, betas=BETAS)
        else:
            more = {"master": views(s["master"])} if s["master"] is not None else {}
            if case["op"] == "adamw8":
                scales = lambda x: [x[o // BLOCK:o // BLOCK + -(-n // BLOCK)] for o, n in zip(offs, sizes)]  # noqa: E731
                more.update(m_scale=scales(s["ms"]), v_scale=scales(s["vs"]))
            pair = ("m", "v") if case["op"] == "adamw" else ("m8", "v8")
            s["plan"] = optim.AdamW(views(s["p"]), grads, views(s[pair[0]]), views(s[pair[1]]), betas=BETAS, eps=EPS, weight_decay=s["wd"], **more)
        s["ctrl"] = optim.Control(dev, lr=LR, step=1000)
    elif case["op"] != "norm" and case["tensors"] > 1:
        spans = torch.tensor([b - a for a, b in zip(offs, offs[1:] + [total])], device=dev)
        s["which"] = torch.repeat_interleave(torch.arange(len(sizes), device=dev), spans)
        s["starts"] = torch.tensor(offs, device=dev)
        s["wd_t"] = torch.tensor(s["wd"], device=dev)
    return s


# ---- the plain forms -------------------------------------------------------------------------------
def _norm(g, scale, max_norm):
    total = g.double().square().sum()
    norm = abs(scale) * total.sqrt()
    clip = torch.clamp(max_norm / (norm + 1e-6), max=1.0)
    return norm.float(), (scale * clip).float(), (~torch.isfinite(total)).to(torch.int32)


def _fmix(h):
    h = h ^ (h >> 16)
    h = (h * 0x85EBCA6B) & M32
    h = h ^ (h >> 13)
    h = (h * 0xC2B2AE35) & M32
    return h ^ (h >> 16)


def _random(s, step):
    """32 random bits for each element: a hash of seed, step, tensor and the element's index in it."""
    i = torch.arange(s["total"], device=s["g"].device)
    which = s.get("which", 0)
    if "which" in s:
        i = i - s["starts"][which]
    k = torch.zeros((), dtype=torch.int64, device=s["g"].device)
    k = _fmix(k + (s["seed"] & M32))
    k = _fmix(k ^ (s["seed"] >> 32))
    k = _fmix(k ^ (step & M32))
    k = _fmix(k ^ (step >> 32))
    k = _fmix(k ^ which)
    return _fmix(((i & M32) * 0x9E3779B1 & M32) ^ k)


def _code(t, bits, r):
    """The 8-bit float of t in [0, 1.875 (1 + 2^-22)]: exponents 2^-14 .. 1, `bits` of mantissa, gradual underflow;
    r: 16 random bits, or None for the nearest."""
    drop = 23 - bits
    r = 0x8000 if r is None else r
    up = ((t.view(torch.int32) + (r << (drop - 16))) >> drop) - (112 << bits)
    low = torch.floor(t * 2.0 ** (14 + bits) + r / 65536.0).int()
    return torch.where(t < 2.0 ** -14, low, up)


def _decoded(c, bits):
    c = c.int()
    high = ((c + (112 << bits)) << (23 - bits)).view(torch.float32)
    return torch.where(c < (1 << bits), c.float() * 2.0 ** -(14 + bits), high)


def _blocks(x):
    pad = -x.numel() % BLOCK
    x = torch.cat([x, x.new_zeros(pad)]) if pad else x
    return x.view(-1, BLOCK)


def _encode(m, v, r):
    """Both moments in 8 bits: codes and scale of m (a sign and e4m3), codes and scale of v (its root, e4m4 without a sign)."""
    m, root = _blocks(m), _blocks(v).sqrt()
    low = high = None
    if r is not None:
        low, high = _blocks((r & 0xFFFF).int()), _blocks((r >> 16).int())
    ms, vs = m.abs().amax(1) * (1 / 1.875), root.amax(1) * (1 / 1.875)
    per = lambda s: torch.where(s > 0, 1.0 / s, s)[:, None]  # noqa: E731
    c = _code(m.abs() * per(ms), 3, low).clamp_(max=127)
    c = torch.where((m < 0) & (c > 0), c + 128, c)
    k = _code(root * per(vs), 4, high).clamp_(max=254)
    k = torch.where(root > 0, k.clamp(min=1), k)
    return c.to(torch.uint8).view(-1), ms, k.to(torch.uint8).view(-1), vs


def _values8(m8, ms, v8, vs):
    m = _decoded(m8.view(-1, BLOCK) & 127, 3) * ms[:, None]
    m = torch.where(m8.view(-1, BLOCK) >= 128, -m, m)
    return m.view(-1), (_decoded(v8.view(-1, BLOCK), 4) * vs[:, None]).square().view(-1)


def _adamw(p, g, m, v, step, mult, wd):
    """One step on fp32 weights and moments, in place; wd: a number, or one for each element."""
    b1, b2 = BETAS
    g = g.float() * mult
    m.mul_(b1).add_(g * (1 - b1))
    v.mul_(b2).add_((g * (1 - b2)) * g)
    denom = v.sqrt() * (1 / math.sqrt(1 - b2 ** step)) + EPS
    p.mul_(1 - LR * wd).sub_((m / denom) * (LR / (1 - b1 ** step)))


def _plain(s):
    case, out = s["case"], {}
    if case["op"] == "moments8":
        s["m8"], s["ms"], s["v8"], s["vs"] = _encode(s["m"], s["v"], None)
        m, v = _values8(s["m8"], s["ms"], s["v8"], s["vs"])
        return {"m": m.bfloat16(), "v": v.bfloat16(), "m_scale": s["ms"], "v_scale": s["vs"]}
    if case["op"] == "norm":
        norm, mult, skip = _norm(s["g"], s["scale"], s["max_norm"])
        return {"norm": norm, "mult": mult, "skip": skip}
    s["step"] += 1
    mult = s["scale"]
    if case["clip"]:
        norm, mult, _ = _norm(s["g"], s["scale"], s["max_norm"])
        out["norm"] = norm
    wd = s["wd_t"][s["which"]] if "which" in s else s["wd"][0]
    p = s["master"] if s["master"] is not None else s["p"].float()
    if case["op"] == "adamw":
        m, v = s["m"], s["v"]
        _adamw(p, s["g"], m, v, s["step"], mult, wd)
    else:
        m, v = _values8(s["m8"], s["ms"], s["v8"], s["vs"])
        _adamw(p, s["g"], m, v, s["step"], mult, wd)
        s["m8"], s["ms"], s["v8"], s["vs"] = _encode(m, v, _random(s, s["step"]))
        m, v = (x.bfloat16() for x in _values8(s["m8"], s["ms"], s["v8"], s["vs"]))
        out.update(m_scale=s["ms"], v_scale=s["vs"])
    s["p"] = p.to(s["p"].dtype)
    out.update(p=s["p"], m=m, v=v)
    if s["master"] is not None:
        out["master"] = p
    return out


# ---- the framework's calls -----------------------------------------------------------------------
def _own(s):
    case, api, out = s["case"], s["api"], {}
    if case["op"] == "moments8":
        n = case["elements"]
        api.moments8_encode_(s["m8"][:n], s["ms"], s["v8"][:n], s["vs"], s["m"][:n], s["v"][:n])
        api.moments8_decode_(s["m_out"], s["v_out"], s["m8"], s["ms"], s["v8"], s["vs"])
        return {"m": s["m_out"], "v": s["v_out"], "m_scale": s["ms"], "v_scale": s["vs"]}
    plan, ctrl = s["plan"], s["ctrl"]
    if case["op"] == "norm":
        plan.grad_norm_(ctrl, max_norm=s["max_norm"], grad_scale=s["scale"])
        return {"norm": ctrl.norm, "mult": ctrl.mult, "skip": ctrl.skip}
    if case["clip"]:
        plan.grad_norm_(ctrl, max_norm=s["max_norm"], grad_scale=s["scale"])
        out["norm"] = ctrl.norm
        plan.step_(ctrl=ctrl, seed=s["seed"])
    else:
        s["step"] += 1
        plan.step_(lr=LR, step=s["step"], grad_scale=s["scale"], seed=s["seed"])
    if case["op"] == "adamw":
        out.update(m=s["m"], v=s["v"])
    else:
        api.moments8_decode_(s["m_out"], s["v_out"], s["m8"], s["ms"], s["v8"], s["vs"])
        out.update(m=s["m_out"], v=s["v_out"], m_scale=s["ms"], v_scale=s["vs"])
    out["p"] = s["p"]
    if s["master"] is not None:
        out["master"] = s["master"]
    return out


def run(s):
    return _own(s) if own else _plain(s)


# ---- what a pass cannot do without -----------------------------------------------------------------
def work(case):
    n = case["elements"]
    if case["op"] == "moments8":  # fp32 moments in; codes, scales and bf16 values out
        return {"bytes": n * (8 + 2 + 4) + n // BLOCK * 8, "flops": 24 * n}
    grad = TYPES[case["grad"]].itemsize
    if case["op"] == "norm":
        return {"bytes": n * grad, "flops": 2 * n}
    kind, master = split_types(case)
    weights = 8 + kind.itemsize if master else 2 * kind.itemsize
    if case["op"] == "adamw":
        return {"bytes": n * (weights + grad + 16), "flops": 16 * n}
    # codes in and out, and the values that they stand for
    return {"bytes": n * (weights + grad + 4 + 4) + n // BLOCK * 16, "flops": 60 * n}


# ---- the definition, in 64 bits -----------------------------------------------------------------
def _mix64(h):
    for shift, factor in ((16, 0x85EBCA6B), (13, 0xC2B2AE35)):
        h = ((h ^ (h >> shift)) * factor) % (1 << 32)
    return h ^ (h >> 16)


def _round8(x, mantissa, top, noise):
    """x in [0, 1.875] to the float grid of spacing 2^(e - mantissa), e >= -14: down, or up where the noise carries it."""
    _, e = torch.frexp(x)
    spacing = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-14) - mantissa)
    return torch.minimum(torch.floor(x / spacing + noise) * spacing, torch.full_like(x, top))


def _through8(x, mantissa, noise, floor):
    """x >= 0 by blocks of 256: what its 8-bit form stands for, and the scales."""
    n = x.numel()
    rows = torch.nn.functional.pad(x, (0, -n % BLOCK)).view(-1, BLOCK)
    if torch.is_tensor(noise):
        noise = torch.nn.functional.pad(noise, (0, -n % BLOCK)).view(-1, BLOCK)
    scale = rows.amax(1) / 1.875
    unit = torch.where(scale > 0, scale, torch.ones_like(scale))[:, None]
    q = _round8(rows / unit, mantissa, 1.875, noise)
    if floor:
        q = torch.where(rows > 0, q.clamp(min=2.0 ** -18), q)
    return (q * unit).view(-1), scale


def _stored(m, v, noise):
    """The values of both moments after 8 bits, laid out in whole blocks, and their scales."""
    low, high = (0.5, 0.5) if noise is None else ((noise % 65536) / 65536.0, (noise // 65536) / 65536.0)
    size, ms = _through8(m.abs(), 3, low, False)
    sign = torch.sign(torch.nn.functional.pad(m, (0, -m.numel() % BLOCK)))
    root, vs = _through8(v.sqrt(), 4, high, True)
    return size * sign, root * root, ms, vs


def exact(case, seed):
    sizes, offs, total, p0, g0, m0, v0 = _values(case, seed)
    d = lambda x: x.double()  # noqa: E731
    if case["op"] == "moments8":
        m, v, ms, vs = _stored(d(m0), d(v0), None)
        return {"m": m, "v": v, "m_scale": ms, "v_scale": vs}
    scale, max_norm = _clipping(case, seed)
    g = d(g0.to(TYPES[case["grad"]]))
    norm = scale * torch.linalg.vector_norm(g)
    clipped = scale * min(1.0, max_norm / (float(norm) + 1e-6))
    if case["op"] == "norm":
        return {"norm": norm, "mult": torch.tensor(clipped, dtype=torch.float64), "skip": None}
    kind, master = split_types(case)
    mult, t = clipped if case["clip"] else scale, 1001
    b1, b2 = BETAS
    if case["op"] == "adamw8":
        m8 = _encode(m0, v0, None)
        m0, v0 = (d(x) for x in _values8(*m8))
    word = (seed << 20) | 0x5EED
    p_all = d(p0 if master else p0.to(kind))
    m_all, v_all = torch.zeros_like(p_all), torch.zeros_like(p_all)
    ms_all, vs_all = (torch.zeros(-(-total // BLOCK), dtype=torch.float64, device=g.device) for _ in range(2))
    for i, (o, n) in enumerate(zip(offs, sizes)):
        if not n:
            continue
        at = slice(o, o + n)
        gi = g[at] * mult
        m = b1 * d(m0[at]) + (1 - b1) * gi
        v = b2 * d(v0[at]) + (1 - b2) * gi * gi
        ahead = (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + EPS)
        p_all[at] = p_all[at] - LR * (ahead + (0.0 if i % 4 == 3 else DECAY) * p_all[at])
        if case["op"] == "adamw":
            m_all[at], v_all[at] = m, v
            continue
        key = 0
        for part in (word % (1 << 32), word >> 32, t, 0, i):
            key = _mix64(key ^ part)
        noise = _mix64(torch.arange(n, device=g.device) * 0x9E3779B1 % (1 << 32) ^ key)
        full, row = -(-n // BLOCK) * BLOCK, o // BLOCK
        m_all[o:o + full], v_all[o:o + full], ms_all[row:row + full // BLOCK], vs_all[row:row + full // BLOCK] = _stored(m, v, noise)
    out = {"p": p_all, "m": m_all, "v": v_all}
    if master:
        out["master"] = p_all
    if case["clip"]:
        out["norm"] = norm
    if case["op"] == "adamw8":
        out.update(m_scale=ms_all, v_scale=vs_all)
    return out
