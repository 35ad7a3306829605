"""The optimizer step on a reduced gradient bucket (include/hydra_optim.h).

What a training program does with a bucket once it is allreduced, on the device and on torch's
current stream: the norm of all gradients with the clip factor and the finite check, the AdamW step
over many tensors in one launch, and the conversion of 8-bit moments.  The reference has no
counterpart; the formulas and the 8-bit format stand in include/hydra_optim.h.

    plan = AdamW(params, grads, m, v, weight_decay=0.1)         # fp32 moments
    ctrl = Control(device, lr=3e-4)
    peer.allreduce_(bucket)                                     # grads are views of the bucket
    plan.grad_norm_(ctrl, max_norm=1.0, grad_scale=1.0 / world) # norm, clip factor, finite check
    plan.step_(ctrl=ctrl)                                       # skipped where a gradient overflowed

8-bit moments: uint8 tensors of the params' lengths and moment_scales(n) fp32 scales each,
zeroed to start with, and a seed that stays the same for the whole training:

    plan = AdamW(params, grads, m8, v8, m_scale=ms, v_scale=vs)
    plan.step_(lr=3e-4, step=1, seed=1234)
"""
from __future__ import annotations

import collections
import ctypes

import numpy as np
import torch

from . import _lib
from ._lib import HydraError, check

MOMENT_BLOCK = 256  # elements that share one scale of an 8-bit moment
_SEEDS = (1 << 64) - 1
_WORKSPACE = 16384  # HYDRA_ADAMW_WORKSPACE_MAX (include/hydra_optim.h)
_CODES = {torch.float32: _lib.FLOAT32, torch.bfloat16: _lib.BFLOAT16, torch.float16: _lib.FLOAT16}
# the current stream's handle by device index (torch.cuda.current_stream builds a Stream object
# around it: 2 us, as long as a small step's kernel runs)
_current_stream = torch._C._cuda_getCurrentRawStream
_left = collections.deque()  # handles of dropped plans: released when the next plan is made or closed


def moment_scales(n: int) -> int:
    """Scales of an 8-bit moment of n elements."""
    return -(-n // MOMENT_BLOCK)


def _code(dtype) -> int:
    try:
        return _CODES[dtype]
    except KeyError:
        raise HydraError(_lib.ERR_INVALID, f"unsupported dtype {dtype}") from None


def _list(x) -> list:
    return [x] if isinstance(x, torch.Tensor) else list(x)


def _refuse(msg: str):
    raise HydraError(_lib.ERR_INVALID, msg)


def _release_left() -> None:
    while True:
        try:
            h = _left.popleft()  # (another thread may have taken the last one)
        except IndexError:
            return
        _lib.lib().hydra_adamw_destroy(h)


class Control:
    """hydra_adamw_ctrl_t: 64 bytes on the device that carry a step's scalars from grad_norm_ to
    step_ without a host round trip.  Its fields are 0-d device tensors: lr and step are set by the
    program (ctrl.lr.fill_(x)), the others are written by grad_norm_.  Behind them lies grad_norm_'s
    workspace: calls on one Control go to one stream or are ordered by events, whatever their plans,
    and a graph that holds such calls needs its Control."""

    def __init__(self, device, lr: float = 0.0, step: int = 0):
        memory = torch.zeros(64 + _WORKSPACE, dtype=torch.uint8, device=device)
        if not memory.is_cuda:
            _refuse("Control: a GPU device is required")
        self.buffer = memory[:64]
        self.index, self.ptr = self.buffer.get_device(), self.buffer.data_ptr()
        self.workspace = self.ptr + 64
        f, i = self.buffer.view(torch.float32), self.buffer.view(torch.int32)
        self.step, self.skipped = self.buffer.view(torch.int64)[:2]
        self.lr, self.mult, self.norm = f[4], f[5], f[6]
        self.skip = i[7]
        self.lr.fill_(lr)
        self.step.fill_(step)

    def __reduce__(self):  # a copy, also by way of a file, has memory of its own
        return _control_of, (self.buffer,)


def _control_of(buffer) -> Control:
    c = Control(buffer.device)
    c.buffer.copy_(buffer)
    return c


class AdamW:
    """A plan (hydra_adamw_t): the tensors that are stepped together, laid out once.

    params, grads, m, v: lists of contiguous tensors on one GPU, alike in length; params and grads
    in fp32, bf16 or fp16, m and v in fp32, or uint8 with m_scale and v_scale (fp32,
    moment_scales(n) each).  master: fp32 weights beside 16-bit params, which a step then only
    writes.  weight_decay and lr_scale: a number, or one for each tensor.  params None: a plan for
    grad_norm_ alone.  bucket: a 1-d tensor whose views the grads are; each call may then name
    another bucket of that layout (two buckets in turn, one being reduced while the other is
    stepped).  The plan keeps the tensors alive; a graph that holds its calls does not.  Calls write
    the tensors past autograd: nothing that a backward pass still needs may be among them.

    Plans are made and closed while no thread captures a stream.  One that is dropped without close()
    waits with its device tables (88 bytes a tensor and 4 for 1024 elements) until the next one is made or
    closed, so plans may be dropped at any time.  close() waits for the device's work, dropping does not:
    what a plan alone kept alive and used on another stream than its own follows torch's rule for such
    tensors (record_stream, or close() first)."""

    def __init__(self, params, grads, m=None, v=None, *, master=None, m_scale=None, v_scale=None,
                 betas=(0.9, 0.999), eps: float = 1e-8, weight_decay=0.01, lr_scale=1.0,
                 bucket=None):
        self._h = ctypes.c_void_p()
        if _left and not torch.cuda.is_current_stream_capturing():
            _release_left()
        grads = _list(grads)
        if not grads:
            _refuse("AdamW: no tensors")
        k, norm_only = len(grads), params is None
        lists = {"params": params, "m": m, "v": v, "master": master, "m_scale": m_scale,
                 "v_scale": v_scale}
        if norm_only and any(x is not None for x in lists.values()):
            _refuse("AdamW: a plan without params holds gradients alone")
        if not norm_only and (m is None or v is None):
            _refuse("AdamW: m and v are required")
        lists = {name: _list(x) for name, x in lists.items() if x is not None}
        index = grads[0].get_device()
        for name, ts in [("grads", grads), *lists.items()]:
            if len(ts) != k:
                _refuse(f"AdamW: {len(ts)} {name} for {k} grads")
            dtype = ts[0].dtype
            for t in ts:
                if t.get_device() != index or index < 0:
                    _refuse(f"AdamW: {name} must be on one GPU, that of the grads")
                if not t.is_contiguous():
                    _refuse(f"AdamW: {name} must be contiguous")
                if t.dtype != dtype:
                    _refuse(f"AdamW: {name} must share one dtype")
        eight = not norm_only and lists["m"][0].dtype == torch.uint8
        if not norm_only:
            for name in ("m", "v"):
                if lists[name][0].dtype != (torch.uint8 if eight else torch.float32):
                    _refuse("AdamW: m and v must both be float32 or both uint8")
            if eight != ("m_scale" in lists) or eight != ("v_scale" in lists):
                _refuse("AdamW: m_scale and v_scale belong to uint8 moments, and to them only")
            for name in ("master", "m_scale", "v_scale"):
                if name in lists and lists[name][0].dtype != torch.float32:
                    _refuse(f"AdamW: {name} must be float32")
        sizes = [g.numel() for g in grads]
        rows = [moment_scales(n) for n in sizes] if eight else None
        for name, ts in lists.items():
            have, want = [t.numel() for t in ts], rows if name.endswith("_scale") else sizes
            if have != want:
                i = next(i for i in range(k) if have[i] != want[i])
                _refuse(f"AdamW: {name} of {have[i]} elements where {want[i]} are needed")
        wd = list(weight_decay) if hasattr(weight_decay, "__iter__") else [weight_decay] * k
        ls = list(lr_scale) if hasattr(lr_scale, "__iter__") else [lr_scale] * k
        if len(wd) != k or len(ls) != k:
            _refuse("AdamW: weight_decay and lr_scale: a number, or one for each tensor")

        base = 0
        self._bucket_bytes = None
        if bucket is not None:
            self._check_bucket_tensor(bucket, grads[0])
            base = bucket.data_ptr()
            self._bucket_bytes = bucket.numel() * bucket.element_size()
            for g in grads:
                end = g.data_ptr() + g.numel() * g.element_size()
                if g.numel() and not (base <= g.data_ptr() and end <= base + self._bucket_bytes):
                    _refuse("AdamW: a grad is not a view of the bucket")
        self.device, self._index = grads[0].device, index
        self._grad_dtype, self._bucket = grads[0].dtype, bucket
        # what the launches touch; with buckets of the caller's choice, not the first one's views
        self._keep = [*lists.values(), grads if bucket is None else ()]
        table = np.zeros(k, _lib.ADAMW_TENSOR)
        columns = {"params": "param"}
        for name, ts in lists.items():
            table[columns.get(name, name)] = [t.data_ptr() for t in ts]
        table["grad"] = [g.data_ptr() - base if n else 0 for g, n in zip(grads, sizes)]
        table["n"], table["lr_scale"], table["weight_decay"] = sizes, ls, wd
        flags = (_lib.ADAMW_MASTER if master is not None else 0) | \
                (_lib.ADAMW_BUCKET if bucket is not None else 0) | \
                (_lib.ADAMW_NORM_ONLY if norm_only else 0)
        cfg = _lib.AdamWConfig(0 if norm_only else _code(lists["params"][0].dtype),
                               _code(self._grad_dtype),
                               _lib.UINT8 if eight else _lib.FLOAT32, flags, betas[0], betas[1], eps)
        self._bucket_at = base if bucket is not None else None
        L = self._L = _lib.lib()
        check(L.hydra_adamw_create(self._index, ctypes.byref(cfg), table.ctypes.data, k,
                                   ctypes.byref(self._h)))
        size = ctypes.c_size_t()
        check(L.hydra_adamw_workspace(self._h, ctypes.byref(size)))
        self._workspace = size.value  # 0: the norm is one launch

    @staticmethod
    def _check_bucket_tensor(b, like):
        if not b.is_cuda or b.device != like.device or b.dtype != like.dtype or b.dim() != 1 or \
                not b.is_contiguous():
            _refuse("AdamW: the bucket must be a contiguous 1-d tensor like the grads")

    def _bucket_ptr(self, bucket):
        if self._bucket is None:
            _refuse("AdamW: the plan was made without a bucket")
        if bucket is None:
            return self._bucket_at
        self._check_bucket_tensor(bucket, self._bucket)
        if bucket.numel() * bucket.element_size() < self._bucket_bytes:
            _refuse("AdamW: the bucket is shorter than the plan's")
        return bucket.data_ptr()

    def __reduce__(self):
        _refuse("AdamW: a plan cannot be copied: make another over the tensors of the copy")

    def _closed(self):
        _refuse("AdamW: the plan is closed")

    def grad_norm_(self, ctrl: Control, max_norm: float = 0.0, grad_scale: float = 1.0, bucket=None,
                   stream: int | None = None) -> None:
        """hydra_adamw_grad_norm: norm, clip factor and finite check of all gradients into ctrl, and
        the next step's number.  max_norm 0: no clipping.  stream: a raw handle; the tensors' ordering and
        lifetime on another stream than torch's current one are the caller's."""
        h = self._h or self._closed()
        b = self._bucket_ptr(bucket) if self._bucket is not bucket else self._bucket_at
        if ctrl.index != self._index:
            _refuse("grad_norm_: ctrl is on another device")
        s = _current_stream(self._index) if stream is None else stream
        # the workspace is the Control's: memory allocated here would belong to the current stream, whose
        # queued work may still use it when another stream writes it
        check(self._L.hydra_adamw_grad_norm(h, b, grad_scale, max_norm, ctrl.ptr, ctrl.workspace,
                                            _WORKSPACE, s))

    def step_(self, lr: float | None = None, step: int | None = None, grad_scale: float = 1.0,
              ctrl: Control | None = None, seed: int = 0, bucket=None,
              stream: int | None = None) -> None:
        """One AdamW step in place: with lr and step (1, 2, ...) from the arguments, or with ctrl
        from the last grad_norm_ on it.  seed: that of the 8-bit moments' rounding (0: to nearest)."""
        h = self._h or self._closed()
        b = self._bucket_ptr(bucket) if self._bucket is not bucket else self._bucket_at
        s = _current_stream(self._index) if stream is None else stream
        if not 0 <= seed <= _SEEDS:
            _refuse("step_: a seed has 64 bits")
        if ctrl is not None:
            if lr is not None or step is not None or grad_scale != 1.0:
                _refuse("step_: lr, step and grad_scale come from ctrl")
            if ctrl.index != self._index:
                _refuse("step_: ctrl is on another device")
            rc = self._L.hydra_adamw_step_ctrl(h, b, ctrl.ptr, seed, s)
        else:
            if lr is None or step is None:
                _refuse("step_: lr and step, or ctrl")
            rc = self._L.hydra_adamw_step(h, b, lr, step, grad_scale, seed, s)
        if rc:
            check(rc)

    def close(self) -> None:
        """Waits for the device's work, then releases the plan."""
        if self._h:
            _left.append(self._h)
            self._h = ctypes.c_void_p()
            self._keep = []
        _release_left()

    def __del__(self):
        # releasing waits for the device, which would end a capture of any thread's: that is left to
        # the next plan made or closed (while the interpreter is finalizing, the deque may be gone)
        if _left is not None and self._h:
            _left.append(self._h)


def _moments(m, v, m8, m_scale, v8, v_scale):
    """Checks a conversion's tensors; (device index, dtype code, n, m's pointers, v's)."""
    some = m if m is not None else v
    if some is None:
        _refuse("moments8: neither moment given")
    n, dtype, index = some.numel(), some.dtype, some.get_device()
    if index < 0:
        _refuse("moments8: contiguous tensors on one GPU are required")
    rows = -(-n // MOMENT_BLOCK)

    def pointers(x, codes, scale, name):
        if x is None:
            if codes is not None or scale is not None:
                _refuse(f"moments8: codes or scales of {name} without its values")
            return None, None, None
        if codes is None or scale is None:
            _refuse(f"moments8: {name} needs its codes and its scales")
        if not (x.get_device() == codes.get_device() == scale.get_device() == index
                and x.is_contiguous() and codes.is_contiguous() and scale.is_contiguous()):
            _refuse("moments8: contiguous tensors on one GPU are required")
        if codes.dtype is not torch.uint8 or scale.dtype is not torch.float32 or x.dtype is not dtype:
            _refuse("moments8: uint8 codes, float32 scales and values of one dtype are required")
        if x.numel() != n or codes.numel() != n or scale.numel() != rows:
            _refuse(f"moments8: {name}: lengths do not fit {n} elements")
        return x.data_ptr(), codes.data_ptr(), scale.data_ptr()

    return index, _code(dtype), n, pointers(m, m8, m_scale, "m"), pointers(v, v8, v_scale, "v")


def _on(index: int, call, *args) -> None:
    """A C call that works on the current device, made on device `index`."""
    if torch.cuda.current_device() == index:
        check(call(*args))
    else:
        with torch.cuda.device(index):
            check(call(*args))


def moments8_encode_(m8, m_scale, v8, v_scale, m, v, stream: int | None = None) -> None:
    """One tensor's moments (fp32 or bf16) into 8 bits, to nearest; either moment may be None."""
    index, code, n, pm, pv = _moments(m, v, m8, m_scale, v8, v_scale)
    s = _current_stream(index) if stream is None else stream
    _on(index, _lib.lib().hydra_moments8_encode, pm[1], pm[2], pv[1], pv[2], pm[0], pv[0], code, n, s)


def moments8_decode_(m, v, m8, m_scale, v8, v_scale, stream: int | None = None) -> None:
    """The values that 8-bit moments stand for, into fp32 or bf16; either moment may be None."""
    index, code, n, pm, pv = _moments(m, v, m8, m_scale, v8, v_scale)
    s = _current_stream(index) if stream is None else stream
    _on(index, _lib.lib().hydra_moments8_decode, pm[0], pv[0], code, pm[1], pm[2], pv[1], pv[2], n, s)
