"""AdamW over many tensors at once, with states in 32 or in 8 bits (over the C ABI).

`MultiAdamW` is the optimizer of the AZ trainer (candle-nn's AdamW,
src/az/train_gpu_candle.rs:113-122, :159) for parameters that do not live in
one flat buffer: one launch per 384 tensors, any mix of fp32, bf16 and fp16
parameters and gradients.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import numpy as np
import torch

from ._lib import AdamwTensor, check, lib

BLOCK = 256     # elements per scale of an 8-bit state
NO_DECAY = 1    # cnnue_adamw_tensor flag
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _span(t: torch.Tensor):
    return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()


class MultiAdamW:
    """AdamW on a list of tensors, in place.

    params: contiguous CUDA tensors (float32, bfloat16 or float16) on one
        device; grads: their gradients (any of the three dtypes, contiguous,
        same sizes), whose buffers every step reads (`bind` changes them).
    state_bits=32: moments m and v in float32, the arithmetic of the flat
        optimizer (cnnue_adamw) bit for bit.  state_bits=8: m and sqrt(v) as
        float8_e4m3fn with one float32 scale per block of 256 elements (2.03
        instead of 8 bytes per parameter); the update uses the new moments
        before they are rounded.
    copies (optional): per parameter a bfloat16 or float16 tensor (or None) that
        receives the rounded new parameter.
    no_decay (optional): per parameter a truth value, True = no weight decay.
    state (optional): {"m": [...], "v": [...]} and, for 8 bits, "m_scale" and
        "v_scale" lists, to step on; made as zeros otherwise.  step: steps
        already taken.
    device_state=True keeps the hyper-parameters and the step counter in device
        memory and advances the counter there, so that a captured CUDA graph
        replays step after step.

    The buffers are held by the object and read and written at every step; a
    parameter or gradient whose storage is replaced has to be bound anew."""

    def __init__(self, params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], lr: float = 1e-3,
                 beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8, weight_decay: float = 1e-4,
                 state_bits: int = 32, state: Optional[dict] = None,
                 copies: Optional[Sequence[Optional[torch.Tensor]]] = None,
                 no_decay: Optional[Sequence[bool]] = None, step: int = 0, device_state: bool = False):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        self.params = [p.detach() for p in params]
        if not self.params:
            raise ValueError("no parameters")
        self.device = self.params[0].device
        if self.device.type != "cuda":
            raise ValueError("parameters must be CUDA tensors")
        n = len(self.params)
        self.state_bits = state_bits
        self.lr, self.beta1, self.beta2, self.eps, self.weight_decay = lr, beta1, beta2, eps, weight_decay
        self._step = step
        for i, p in enumerate(self.params):
            self._check(p, f"params[{i}]", _TYPES, None)
        state = state or {}
        names = ("m", "v") if state_bits == 32 else ("m", "v", "m_scale", "v_scale")
        if state and set(state) != set(names):
            raise ValueError(f"state must hold {names}, has {tuple(state)}")
        self.state = {}
        for k in names:
            scale = k.endswith("_scale")
            dtype = torch.float8_e4m3fn if state_bits == 8 and not scale else torch.float32
            size = [(p.numel() + BLOCK - 1) // BLOCK if scale else p.numel() for p in self.params]
            if state:
                if len(state[k]) != n:
                    raise ValueError(f"state {k} has {len(state[k])} tensors for {n} parameters")
                for i, t in enumerate(state[k]):
                    self._check(t, f"state {k}[{i}]", (dtype,), size[i])
                self.state[k] = list(state[k])
            else:  # one buffer, every tensor on a 256-byte boundary
                each = torch.empty(0, dtype=dtype).element_size()
                places = np.concatenate([[0], np.cumsum([(s * each + 255) // 256 * 256 for s in size])])
                flat = torch.zeros(int(places[-1]), dtype=torch.uint8, device=self.device)
                self.state[k] = [flat[a:a + s * each].view(dtype) for a, s in zip(places.tolist(), size)]
        copies = [None] * n if copies is None else list(copies)
        if len(copies) != n or (no_decay is not None and len(no_decay) != n):
            raise ValueError("copies and no_decay have one entry per parameter")
        for i, c in enumerate(copies):
            if c is not None:
                self._check(c, f"copies[{i}]", (torch.bfloat16, torch.float16), self.params[i].numel())
        self.copies = copies
        self._table = (AdamwTensor * n)()
        for i, (e, p) in enumerate(zip(self._table, self.params)):
            e.param, e.n, e.param_type = p.data_ptr(), p.numel(), _TYPES[p.dtype]
            e.m, e.v = self.state["m"][i].data_ptr(), self.state["v"][i].data_ptr()
            if state_bits == 8:
                e.m_scale, e.v_scale = self.state["m_scale"][i].data_ptr(), self.state["v_scale"][i].data_ptr()
            if copies[i] is not None:
                e.copy, e.copy_type = copies[i].data_ptr(), _TYPES[copies[i].dtype]
            e.flags = NO_DECAY if no_decay is not None and no_decay[i] else 0
        self._dstate = None
        if device_state:
            host = np.zeros(12, np.float64)
            host[:5] = [lr, beta1, beta2, eps, weight_decay]
            host.view(np.int64)[5] = step
            self._dstate = torch.from_numpy(host.view(np.uint8).copy()).to(self.device)
        self.bind(grads)

    def _check(self, t: torch.Tensor, name: str, dtypes, size: Optional[int]) -> None:
        if t.device != self.device:
            raise ValueError(f"{name} must be on {self.device}, is on {t.device}")
        if t.dtype not in dtypes:
            raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if size is not None and t.numel() != size:
            raise ValueError(f"{name} must hold {size} elements, has {t.numel()}")

    def bind(self, grads: Sequence[torch.Tensor]) -> None:
        """The gradient buffers that the following steps read."""
        grads = list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"{len(grads)} gradients for {len(self.params)} parameters")
        for i, (g, p) in enumerate(zip(grads, self.params)):
            self._check(g, f"grads[{i}]", _TYPES, p.numel())
        # a buffer that is written may not share memory with any other
        spans = [(*_span(t), True, k) for k, ts in (("params", self.params), *self.state.items(), ("copies", self.copies))
                 for t in ts if t is not None and t.numel()]
        spans += [(*_span(g), False, "grads") for g in grads if g.numel()]
        spans.sort(key=lambda s: (s[0], s[1]))
        end, end_written, kind, last = 0, 0, "", ""
        for lo, hi, written, k in spans:
            if lo < end_written or (written and lo < end):
                raise ValueError(f"{k} overlaps {last if lo < end_written else kind}")
            if hi > end:
                end, kind = hi, k
            if written and hi > end_written:
                end_written, last = hi, k
        self.grads = grads
        for e, g in zip(self._table, grads):
            e.grad, e.grad_type = g.data_ptr(), _TYPES[g.dtype]

    @property
    def step_count(self) -> int:
        """Steps taken (with device_state: read from the device, skipped steps
        not counted; otherwise the calls of step())."""
        if self._dstate is not None:
            return int(self._dstate[40:48].view(torch.int64).item())
        return self._step

    def set_learning_rate(self, lr: float) -> None:
        self.lr = lr
        if self._dstate is not None:
            self._dstate[:8].copy_(torch.from_numpy(np.array([lr], np.float64).view(np.uint8)))

    def step(self, grad_scale: float = 1.0, skip: Optional[torch.Tensor] = None) -> None:
        """One step on the device's current stream, without a synchronisation.
        Gradients are multiplied by grad_scale first; with `skip` (float32
        device flags) any nonzero flag leaves everything unchanged."""
        if skip is not None and (skip.device != self.device or skip.dtype != torch.float32 or not skip.is_contiguous()):
            raise ValueError(f"skip must be a contiguous float32 tensor on {self.device}")
        if torch.cuda.current_device() != self.device.index:
            with torch.cuda.device(self.device):
                return self._run(grad_scale, skip)
        return self._run(grad_scale, skip)

    def _run(self, grad_scale: float, skip: Optional[torch.Tensor]) -> None:
        stream = torch.cuda.current_stream(self.device).cuda_stream
        flags = (None, 0) if skip is None else (skip.data_ptr(), skip.numel())
        if self._dstate is not None:
            check(lib().cnnue_adamw_multi_device(C.addressof(self._table), len(self._table), self.state_bits,
                                                 self._dstate.data_ptr(), grad_scale, *flags, stream),
                  "cnnue_adamw_multi_device")
            return
        check(lib().cnnue_adamw_multi(C.addressof(self._table), len(self._table), self.state_bits, self.lr, self.beta1,
                                      self.beta2, self.eps, self.weight_decay, self._step + 1, grad_scale, *flags,
                                      stream), "cnnue_adamw_multi")
        self._step += 1
