"""How hydra_amd.optim makes its calls, without a GPU: plans whose library is a stand-in."""
import ctypes

import pytest

from hydra_amd import optim

torch = pytest.importorskip("torch")


class Library:
    """Takes every call and keeps its arguments."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0

        return call


class Plan(optim.AdamW):
    def __del__(self):  # its handle is none
        pass


def plan_of(library, workspace=16384):
    plan = Plan.__new__(Plan)
    plan._h, plan._L, plan._index, plan.device = ctypes.c_void_p(1), library, 0, torch.device("cuda", 0)
    plan._bucket, plan._bucket_at, plan._workspace, plan._keep = None, None, workspace, []
    return plan


def control(monkeypatch):
    """A Control whose memory is the host's."""
    zeros = torch.zeros

    class Memory:
        def __init__(self, n):
            self.t = zeros(n, dtype=torch.uint8)
            self.is_cuda = True

        def __getitem__(self, at):
            m = Memory(0)
            m.t = self.t[at]
            return m

        def __getattr__(self, name):
            return getattr(self.t, name)

        def get_device(self):
            return 0

    monkeypatch.setattr(optim.torch, "zeros", lambda n, dtype, device: Memory(n))
    c = optim.Control("cuda:0", lr=0.5, step=3)
    monkeypatch.setattr(optim.torch, "zeros", zeros)
    return c


@pytest.mark.parametrize("stream", [None, 1234])
def test_norm_takes_its_partial_sums_from_the_control(monkeypatch, stream):
    """A call allocates nothing: memory from torch's allocator belongs to the current stream, and work
    still queued there may use it while the call runs on another one.  The partial sums lie in the
    Control, which is ordered between streams by its owner."""
    ctrl, library = control(monkeypatch), Library()

    def empty(*a, **k):
        raise AssertionError("grad_norm_ allocates")

    monkeypatch.setattr(optim.torch, "empty", empty)
    monkeypatch.setattr(optim, "_current_stream", lambda index: 77)
    plan = plan_of(library)
    plan.grad_norm_(ctrl, max_norm=1.0, stream=stream)
    (name, (_, bucket, scale, max_norm, at, ws, size, s)), = library.calls
    assert (name, bucket, scale, max_norm, s) == ("hydra_adamw_grad_norm", None, 1.0, 1.0, stream or 77)
    assert at == ctrl.ptr and ctrl.buffer.numel() == 64
    memory = ctrl.buffer.untyped_storage()
    assert size == 16384 and at + 64 <= ws and ws + size <= memory.data_ptr() + memory.nbytes() and ws % 8 == 0


def left():
    return [h.value for h in optim._left]


def test_a_dropped_plan_waits(monkeypatch):
    """Dropping a plan calls nothing: releasing it waits for the device, which would end a capture that
    any thread makes.  The next plan that is made or closed releases it, once."""
    library = Library()
    monkeypatch.setattr(optim._lib, "lib", lambda: library)
    monkeypatch.setattr(optim.torch.cuda, "is_current_stream_capturing", lambda: False)
    assert left() == []
    plan = optim.AdamW.__new__(optim.AdamW)
    plan._h, plan._keep = ctypes.c_void_p(11), []
    del plan
    assert library.calls == [] and left() == [11]
    with pytest.raises(optim.HydraError, match="no tensors"):
        optim.AdamW([], [], [], [])
    assert [(name, h.value) for name, (h,) in library.calls] == [("hydra_adamw_destroy", 11)] and left() == []
    plans = [optim.AdamW.__new__(optim.AdamW) for _ in range(2)]
    for i, plan in enumerate(plans):
        plan._h, plan._keep = ctypes.c_void_p(20 + i), []
    del library.calls[:], plan
    last = plans.pop()
    del plans[0]
    last.close()
    last.close()
    del last
    assert sorted(h.value for _, (h,) in library.calls) == [20, 21] and left() == []


def test_plans_left_during_a_capture_stay(monkeypatch):
    library = Library()
    monkeypatch.setattr(optim._lib, "lib", lambda: library)
    monkeypatch.setattr(optim.torch.cuda, "is_current_stream_capturing", lambda: True)
    optim._left.append(ctypes.c_void_p(5))
    with pytest.raises(optim.HydraError, match="no tensors"):
        optim.AdamW([], [], [], [])
    assert library.calls == [] and left() == [5]
    optim._left.clear()


def test_two_threads_release_at_once(monkeypatch):
    """The other thread takes the last one between the look and the taking."""
    library = Library()
    monkeypatch.setattr(optim._lib, "lib", lambda: library)

    def capturing():
        optim._left.clear()
        return False

    monkeypatch.setattr(optim.torch.cuda, "is_current_stream_capturing", capturing)
    optim._left.append(ctypes.c_void_p(5))
    with pytest.raises(optim.HydraError, match="no tensors"):
        optim.AdamW([], [], [], [])
    assert library.calls == []


@pytest.mark.parametrize("seed", [-1, 1 << 64, (1 << 64) + 5])
def test_seeds_beyond_64_bits_are_refused(monkeypatch, seed):
    """2^64 would wrap to 0, which rounds to nearest."""
    library, ctrl = Library(), control(monkeypatch)
    monkeypatch.setattr(optim, "_current_stream", lambda index: 77)
    plan = plan_of(library)
    for kw in (dict(lr=1e-3, step=1), dict(ctrl=ctrl)):
        with pytest.raises(optim.HydraError, match="seed"):
            plan.step_(seed=seed, **kw)
    assert library.calls == []
    plan.step_(lr=1e-3, step=1, seed=(1 << 64) - 1)
    plan.step_(ctrl=ctrl, seed=0)
    assert [name for name, _ in library.calls] == ["hydra_adamw_step", "hydra_adamw_step_ctrl"]


def test_plans_are_not_copied():
    """A copy would hold the first one's handle, and release it again."""
    import copy
    import pickle

    for make in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(optim.HydraError, match="copied"):
            make(plan_of(Library()))
