"""GPU tests of how a program calls the optimizer step: streams, captures, threads, alignments and
sizes beyond one launch's or 32 bits (hydra_amd/optim.py); the operators' values are tested in
test_gpu_optim.py."""
import pytest

import optim_ref as R
from hydra_amd import optim
from test_gpu_optim import Setup, f64

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
