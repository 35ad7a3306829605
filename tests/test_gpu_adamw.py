"""GPU tests of how a program calls the optimizer step: streams, captures, threads, alignments and
sizes beyond one launch's or 32 bits (hydra_amd/optim.py); the operators' values are tested in
test_gpu_optim.py."""
import numpy as np
import pytest

import optim_ref as R
from hydra_amd import optim
from test_gpu_optim import Setup, dt, f64

pytestmark = pytest.mark.gpu


def test_norm_on_a_stream_beside_pending_work(gpu):
    """A norm of two launches on a stream that is ordered behind its inputs, while the current stream
    still has work queued on a block of the workspace's size that it has already freed: both keep
    their results."""
    import torch

    gen = torch.Generator(device=gpu)
    gen.manual_seed(5)
    grads = [torch.randn(n, generator=gen, device=gpu) for n in (200_000, 77_777)]
    plan, ctrl = optim.AdamW(None, grads), optim.Control(gpu)
    assert plan._workspace > 0
    norm, _ = R.norm64([f64(g) for g in grads], 1.0, 0.0)
    a = torch.randn(4096, 4096, generator=gen, device=gpu)
    side, ready = torch.cuda.Stream(), torch.cuda.Event()
    kept = []
    for k in range(3):
        ready.record()
        side.wait_event(ready)
        b = a
        for _ in range(8):  # several ms of work that the side stream does not wait for
            b = (a @ b) * 0.01
        blocks = [torch.empty(size, dtype=torch.uint8, device=gpu) for size in (plan._workspace, 16384, 16448)]
        for x in blocks:
            x.fill_(3 + k)
        b = a @ b
        kept.append([x.clone() for x in blocks])
        del blocks, x
        plan.grad_norm_(ctrl, stream=side.cuda_stream)
    torch.cuda.synchronize()
    assert ctrl.step.item() == 3 and abs(ctrl.norm.item() - norm) <= 2 * R.U32 * norm
    for k, xs in enumerate(kept):
        assert all((x == 3 + k).all() for x in xs)


def test_capture_of_a_stream_that_is_not_current(gpu):
    """Calls by handle on a stream that is being captured while the current one is not: what the graph
    holds stays its own, whatever is allocated between its replays."""
    import torch

    a, b = (Setup(gpu, [70_000, 50_001], "bf16", True, "bf16", seed=6) for _ in range(2))
    ca, cb = (optim.Control(gpu, lr=1e-3) for _ in range(2))
    assert a.plan._workspace > 0
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.capture_begin()
    a.plan.grad_norm_(ca, max_norm=0.1, stream=side.cuda_stream)
    a.plan.step_(ctrl=ca, stream=side.cuda_stream)
    with torch.cuda.stream(side):
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    for k in range(4):
        junk = [torch.full((16384 + 64 * i,), 255, dtype=torch.uint8, device=gpu) for i in range(40)]
        graph.replay()
        b.plan.grad_norm_(cb, max_norm=0.1)
        b.plan.step_(ctrl=cb)
        torch.cuda.synchronize()
        assert torch.equal(a.p.buf, b.p.buf) and torch.equal(a.pm.buf, b.pm.buf) and torch.equal(ca.buffer, cb.buffer), k
        assert all((x == 255).all() for x in junk)


def at_a_border(rng, n, kind):
    """n gradients of type `kind` (in fp64) whose norm lies half way between two fp32 numbers to less than
    a step of fp64: sums of their squares in different orders round to different norms."""
    import torch

    def toward_zero(x):
        y = torch.tensor(x, dtype=torch.float64).to(dt(kind)).double().item()
        if y <= x:
            return y
        return torch.nextafter(torch.tensor(y).to(dt(kind)), torch.zeros((), dtype=dt(kind))).double().item()

    ends = 6 if kind == "f32" else 16  # each leaves at most 2^-9 of the rest
    g = torch.from_numpy(rng.normal(0, 1, n)).to(dt(kind)).double().numpy()
    g[-ends:] = 0.0
    total = (g.astype(np.longdouble) ** 2).sum()
    step = float(np.spacing(np.float32(np.sqrt(float(total)))))
    border = np.longdouble(float(np.float32(np.sqrt(float(total)))) + 2.5 * step)
    rest = border * border - total
    for i in range(ends):
        g[n - ends + i] = toward_zero(float(np.sqrt(rest)))
        rest -= np.longdouble(g[n - ends + i]) ** 2
        assert rest >= 0
    assert rest < border * border * 2.0 ** -54
    return g


@pytest.mark.parametrize("grad", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("sizes", [[5000], [200_003], [20_001, 70, 0, 1025, 66_000], [1, 1087, 3, 2049]])
def test_norm_bits_at_any_address(gpu, sizes, grad):
    """The same gradients at other addresses, in plans whose weights and moments lie elsewhere, in other
    buckets, and in a plan of gradients alone: the same bits."""
    import torch

    total, gaps = sum(sizes), (0, 1, 2, 3, 5, 8, 31)

    def views(at, gap, dtype):
        out, buf = [], torch.zeros(total + 64 + gap * len(sizes), dtype=dtype, device=gpu)
        for n in sizes:
            out.append(buf[at:at + n])
            at += n + gap
        return out

    layouts = []
    for gap in gaps:
        grads = views(gap, gap, dt(grad))
        layouts.append((optim.AdamW(None, grads), grads, None))
        p, m, v = (views(gap + i * 7, (gap + i) % 5, torch.float32) for i in range(3))
        grads = views(31 - gap, gap, dt(grad))
        layouts.append((optim.AdamW(p, grads, m, v), grads, None))
    bucket = torch.zeros(total, dtype=dt(grad), device=gpu)
    grads, at = [], 0
    for n in sizes:
        grads.append(bucket[at:at + n])
        at += n
    in_bucket = optim.AdamW(None, grads, bucket=bucket)
    for gap in gaps:
        layouts.append((in_bucket, None, torch.zeros(total + 64, dtype=dt(grad), device=gpu)[gap:gap + total]))
    rng = np.random.default_rng(7)
    ctrl = optim.Control(gpu)
    for draw in range(24):
        g = at_a_border(rng, total, grad)
        values = torch.from_numpy(g).to(dt(grad)).to(gpu)
        got = set()
        for plan, grads, other in layouts:
            if other is not None:
                other.copy_(values)
            else:
                for x, y in zip(grads, values.split(sizes)):
                    x.copy_(y)
            plan.grad_norm_(ctrl, bucket=other)
            got.add(ctrl.norm.item())
        norm, _ = R.norm64([g], 1.0, 0.0)
        assert abs(got.pop() - norm) <= (R.U32 + 2.0 ** -28) * norm and not got, (draw, got)


@pytest.mark.parametrize("sizes,launches", [([80 * 1024], 1), ([80 * 1024 + 1], 2), ([9] * 9 + [0], 1), ([9] * 10, 2),
                                            ([4096] * 7, 1), ([4096] * 8, 2), ([], 1)])
def test_norm_in_one_launch_or_two(gpu, sizes, launches):
    """Both sides of the border: the same definition."""
    import torch

    sizes = sizes or [0]
    gen = torch.Generator(device=gpu)
    gen.manual_seed(9)
    grads = [torch.randn(n, generator=gen, device=gpu) for n in sizes]
    plan, ctrl = optim.AdamW(None, grads), optim.Control(gpu, step=5)
    assert (plan._workspace == 0) == (launches == 1)
    for k in range(3):
        plan.grad_norm_(ctrl, max_norm=0.5, grad_scale=0.25)
        norm, mult = R.norm64([f64(x) for x in grads], 0.25, 0.5)
        assert abs(ctrl.norm.item() - norm) <= (R.U32 + 2.0 ** -28) * norm
        assert abs(ctrl.mult.item() - mult) <= (R.U32 + 2.0 ** -28) * mult
        assert (ctrl.step.item(), ctrl.skip.item()) == (6 + k, 0)


@pytest.mark.parametrize("gap", [0, 1, 2, 3, 5, 8, 16, 31])
def test_step_of_heads_and_last_tiles(gpu, gap):
    """Lengths a little above whole tiles, at offsets whose heads leave the last tile without elements."""
    sizes = [1025, 1026, 2049, 1024 + 31, 1024 + 32, 1024 + 63, 4096 + 64, 1024, 2048, 31, 63, 64]
    s = Setup(gpu, sizes, "bf16", True, "bf16", seed=gap, pad=gap)
    t = Setup(gpu, sizes, seed=gap, pad=gap)
    for x in (s, t):
        before = x.state()
        x.plan.step_(lr=1e-3, step=3)
        x.compare(before, x.state(), lr=1e-3, t=3)
        x.guards()


def test_a_plan_dropped_while_another_thread_captures(gpu):
    """The capture lives on, and the graph does what eager calls do."""
    import threading

    import torch

    a, b = (Setup(gpu, [70_000, 3], seed=41) for _ in range(2))
    ca, cb = (optim.Control(gpu, lr=1e-3) for _ in range(2))
    dropped, graph, side = [Setup(gpu, [10], seed=1)], torch.cuda.CUDAGraph(), torch.cuda.Stream()
    begun, gone, errors = threading.Event(), threading.Event(), []

    def capture():
        try:
            with torch.cuda.graph(graph, stream=side):
                a.plan.grad_norm_(ca, max_norm=0.1)
                begun.set()
                gone.wait(30)
                a.plan.step_(ctrl=ca)
        except Exception as e:
            errors.append(e)
            begun.set()

    t = threading.Thread(target=capture)
    t.start()
    begun.wait(30)
    dropped.clear()
    gone.set()
    t.join()
    assert not errors, errors
    for k in range(3):
        graph.replay()
        b.plan.grad_norm_(cb, max_norm=0.1)
        b.plan.step_(ctrl=cb)
        torch.cuda.synchronize()
        assert torch.equal(a.p.buf, b.p.buf) and torch.equal(ca.buffer, cb.buffer), k
    assert len(optim._left) > 0
    optim.AdamW(None, [b.g.views[0]]).close()
    assert len(optim._left) == 0


def repeated(x, n):
    """n elements that repeat x."""
    import torch

    out = torch.empty(n, dtype=x.dtype, device=x.device)
    for at in range(0, n, 1 << 28):
        part = out[at:at + (1 << 28)]
        part.copy_(x.repeat(-(-part.numel() // x.numel()))[: part.numel()])
    return out


def test_conversions_beyond_one_launch(gpu):
    """More elements than one launch takes (2^30): a stretch's bytes and values are those of the stretch
    alone, on both sides of the border and at the ragged end."""
    import torch

    n = (1 << 30) + 256 * 5 + 77
    gen = torch.Generator(device=gpu)
    gen.manual_seed(3)
    level = torch.exp2(torch.randint(-20, 4, (1 << 20,), generator=gen, device=gpu).float())
    m = repeated(torch.randn(1 << 20, generator=gen, device=gpu) * level, n)
    v = repeated((torch.randn(1 << 20, generator=gen, device=gpu) * level) ** 2, n)
    m[1 << 30] = 1e3  # the second launch's first block and the last one are like no other
    v[-1] = 1e6
    rows = optim.moment_scales(n)
    m8, v8 = (torch.full((n + 1,), 77, dtype=torch.uint8, device=gpu) for _ in "mv")
    ms, vs = (torch.full((rows + 1,), 7.0, device=gpu) for _ in "mv")
    optim.moments8_encode_(m8[:n], ms[:rows], v8[:n], vs[:rows], m, v)
    mo, vo = (torch.full((n + 1,), 7.0, dtype=torch.bfloat16, device=gpu) for _ in "mv")
    optim.moments8_decode_(mo[:n], vo[:n], m8[:n], ms[:rows], v8[:n], vs[:rows])
    for x in (m8, v8, ms, vs, mo, vo):
        assert x[-1].item() in (77, 7.0)
    for at, end in ((0, 4096), ((1 << 30) - 2048, (1 << 30) + 1024), ((1 << 30) - 256, 1 << 30), (1 << 30, n), (n // 256 * 256, n)):
        k, first, last = end - at, at // 256, -(-end // 256)
        a8, b8 = (torch.zeros(k, dtype=torch.uint8, device=gpu) for _ in "mv")
        sa, sb = (torch.zeros(last - first, device=gpu) for _ in "mv")
        optim.moments8_encode_(a8, sa, b8, sb, m[at:end], v[at:end])
        ao, bo = (torch.zeros(k, dtype=torch.bfloat16, device=gpu) for _ in "mv")
        optim.moments8_decode_(ao, bo, a8, sa, b8, sb)
        for got, want in ((m8[at:end], a8), (v8[at:end], b8), (ms[first:last], sa), (vs[first:last], sb), (mo[at:end], ao), (vo[at:end], bo)):
            assert torch.equal(got, want), (at, end)
    assert ms[1 << 22].item() > 500 and vs[rows - 1].item() > 500


def test_step_beyond_32_bits(gpu):
    """fp32 moments of more than 2^32 elements, at an odd offset."""
    import torch

    n = (1 << 32) + 4096 * 3 + 77
    bf = torch.bfloat16
    pattern = (torch.randn(1 << 20, device=gpu) * 0.01).to(bf)
    g = repeated(pattern, n + 3)[3:]
    p = torch.zeros(n + 4, dtype=bf, device=gpu)
    m, v = (torch.zeros(n + 2, device=gpu) for _ in "mv")
    plan = optim.AdamW([p[3:n + 3]], [g], [m[1:n + 1]], [v[1:n + 1]], weight_decay=0.0)
    ctrl = optim.Control(gpu, lr=0.5)
    plan.grad_norm_(ctrl)
    total = float((f64(pattern) ** 2).sum()) * 4096 + float((f64(g[(1 << 32) - 3:]) ** 2).sum())
    assert abs(ctrl.norm.item() - np.sqrt(total)) <= np.sqrt(total) * (R.U32 + 2.0 ** -30)
    plan.step_(ctrl=ctrl)
    for at in (0, (1 << 30) - 100, (1 << 31) - 512, (1 << 32) - 512, n - 3000):
        end = min(n, at + 5120)
        x = f64(g[at:end])
        zero = np.zeros(x.size)
        (want, wm, wv), (ep, em, ev) = R.step64(zero, x, zero, zero, lr=0.5, t=1)
        assert (np.abs(f64(m[at + 1:end + 1]) - wm) <= em).all() and (np.abs(f64(v[at + 1:end + 1]) - wv) <= ev).all(), at
        assert (np.abs(f64(p[at + 3:end + 3]) - want) <= ep + 2.0 ** -8 * (np.abs(want) + ep)).all(), at
    assert (p[:3] == 0).all() and p[n + 3] == 0 and all(x[0] == 0 and x[n + 1] == 0 for x in (m, v))


def test_a_copied_control_has_its_own_memory(gpu):
    """The calls go to the copy's addresses, not to the first one's."""
    import copy
    import pickle

    import torch

    grads = [torch.randn(n, device=gpu) for n in (200_000, 5)]
    plan, first = optim.AdamW(None, grads), optim.Control(gpu, lr=0.25, step=7)
    plan.grad_norm_(first)
    before = first.buffer.clone()
    for make in (copy.copy, copy.deepcopy, lambda c: pickle.loads(pickle.dumps(c))):
        c = make(first)
        assert torch.equal(c.buffer, before) and c.ptr == c.buffer.data_ptr() != first.ptr
        plan.grad_norm_(c)
        assert (c.step.item(), c.lr.item(), c.norm.item()) == (9, 0.25, first.norm.item())
        assert torch.equal(first.buffer, before)
