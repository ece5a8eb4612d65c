"""AdamW over many tensors at once, with states in 32 or in 8 bits (over the C ABI).

`MultiAdamW` is the optimizer of the AZ trainer (candle-nn's AdamW,
src/az/train_gpu_candle.rs:113-122, :159) for parameters that do not live in
one flat buffer: one launch per 384 tensors, any mix of fp32, bf16 and fp16
parameters and gradients.
"""
from __future__ import annotations

from typing import Optional, Sequence

import numpy as np
import torch

from ._lib import check, lib
from .quantized import _device_stream

BLOCK = 256     # elements per scale of an 8-bit state
NO_DECAY = 1    # cnnue_adamw_tensor flag
STOCHASTIC = 256  # added to state_bits
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


# cnnue_adamw_tensor
_TENSOR = np.dtype([(k, np.uint64) for k in ("param", "grad", "m", "v", "m_scale", "v_scale", "copy")] + [("n", np.int64)]
                   + [(k, np.int16) for k in ("param_type", "grad_type", "copy_type", "flags")])


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
    stochastic (state_bits=8): rounds sqrt(v) up with the probability that the
        remainder says, by a hash of the step, the tensor's place in the list
        and the element (the same step gives the same state, on any rank).
        Without it sqrt(v) is rounded to nearest, and with beta2 = 0.999 hardly
        follows the gradients once it has settled: a step moves it by 0.05 %,
        half a step of the format is 3 to 6 %.  After 6,000 steps of normal
        gradients it holds 0.64 to 1.62 of the true root (1 % to 99 %), and 7.6
        times the root in the median where half of a block's gradients fell
        tenfold after step 1,000; stochastic: 0.65 to 1.9, medians 0.98 to 1.02.
        For training of more than some hundred steps, switch it on.
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
                 no_decay: Optional[Sequence[bool]] = None, step: int = 0, device_state: bool = False,
                 stochastic: bool = False):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if stochastic and state_bits != 8:
            raise ValueError("stochastic rounding is for state_bits=8")
        self.params = list(params)
        if not self.params:
            raise ValueError("no parameters")
        self.device = self.params[0].device
        if self.device.type != "cuda":
            raise ValueError("parameters must be CUDA tensors")
        n = len(self.params)
        self.state_bits = state_bits
        self._bits = state_bits | (STOCHASTIC if stochastic else 0)
        self.lr, self.beta1, self.beta2, self.eps, self.weight_decay = lr, beta1, beta2, eps, weight_decay
        self._step = step
        self._table = np.zeros(n, _TENSOR)
        self._address = self._table.ctypes.data
        self._sizes = [p.numel() for p in self.params]
        self._table["n"] = self._sizes
        self._table["param_type"] = self._buffers("params", self.params, _TYPES, self._sizes, "param")
        self._hold_state(state or {})
        copies = [None] * n if copies is None else list(copies)
        if len(copies) != n or (no_decay is not None and len(no_decay) != n):
            raise ValueError("copies and no_decay have one entry per parameter")
        self.copies = copies
        with_copy = [i for i, c in enumerate(copies) if c is not None]
        if with_copy:
            some = [copies[i] for i in with_copy]
            types = self._buffers("copies", some, (torch.bfloat16, torch.float16), [self._sizes[i] for i in with_copy])
            self._table["copy"][with_copy] = [c.data_ptr() for c in some]
            self._table["copy_type"][with_copy] = types
        if no_decay is not None:
            self._table["flags"] = [NO_DECAY if d else 0 for d in no_decay]
        self._check_written()
        self._changed = self.params + [c for c in copies if c is not None]
        self._dstate = None
        if device_state:
            host = np.zeros(12, np.float64)
            host[:5] = [lr, beta1, beta2, eps, weight_decay]
            host.view(np.int64)[5] = step
            self._dstate = torch.from_numpy(host.view(np.uint8).copy()).to(self.device)
        self.bind(grads)

    def _buffers(self, name: str, tensors, dtypes, sizes, column: Optional[str] = None) -> list:
        """Checks the buffers, writes their addresses to a column of the
        table; returns their type codes (None for state types)."""
        dev = self.device.index
        for i, (t, size) in enumerate(zip(tensors, sizes)):
            if t.dtype not in dtypes:
                raise TypeError(f"{name}[{i}] must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
            if t.get_device() != dev:
                raise ValueError(f"{name}[{i}] must be on {self.device}, is on {t.device}")
            if not t.is_contiguous():
                raise ValueError(f"{name}[{i}] must be contiguous")
            if t.numel() != size:
                raise ValueError(f"{name}[{i}] must hold {size} elements, has {t.numel()}")
        if column is not None:
            self._table[column] = [t.data_ptr() for t in tensors]
        return [_TYPES.get(t.dtype) for t in tensors]

    def _hold_state(self, state: dict) -> None:
        eight = self.state_bits == 8
        names = ("m", "v", "m_scale", "v_scale") if eight else ("m", "v")
        if state and set(state) != set(names):
            raise ValueError(f"state must hold {names}, has {tuple(state)}")
        self.state = {}
        for k in names:
            scale = k.endswith("_scale")
            dtype = torch.float8_e4m3fn if eight and not scale else torch.float32
            sizes = [-(-s // BLOCK) for s in self._sizes] if scale else self._sizes
            if state:
                if len(state[k]) != len(sizes):
                    raise ValueError(f"state {k} has {len(state[k])} tensors for {len(sizes)} parameters")
                self.state[k] = list(state[k])
            else:  # one buffer, every tensor on a 256-byte boundary
                each = 1 if dtype is torch.float8_e4m3fn else 4
                places = np.concatenate([[0], np.cumsum([(s * each + 255) // 256 * 256 for s in sizes])]).tolist()
                flat = torch.zeros(places[-1], dtype=torch.uint8, device=self.device)
                self.state[k] = [flat[a:a + s * each].view(dtype) for a, s in zip(places, sizes)]
            self._buffers(f"state {k}", self.state[k], (dtype,), sizes, k)

    def _check_written(self) -> None:
        """No buffer that is written shares memory with another one."""
        t, n = self._table, self._table["n"]
        blocks = -(-n // BLOCK)
        each = 1 if self.state_bits == 8 else 4
        spans = [(t["param"], n * np.where(t["param_type"] == 0, 4, 2), "params"), (t["m"], n * each, "state m"),
                 (t["v"], n * each, "state v"), (t["copy"], np.where(t["copy"] != 0, n * 2, 0), "copies")]
        if self.state_bits == 8:
            spans += [(t["m_scale"], blocks * 4, "state m_scale"), (t["v_scale"], blocks * 4, "state v_scale")]
        lo = np.concatenate([s[0] for s in spans]).astype(np.int64)
        size = np.concatenate([s[1] for s in spans])
        kind = np.repeat([s[2] for s in spans], len(n))
        order = np.argsort(lo, kind="stable")
        order = order[size[order] > 0]
        lo, hi, kind = lo[order], (lo + size)[order], kind[order]
        clash = np.nonzero(lo[1:] < np.maximum.accumulate(hi)[:-1])[0]
        if len(clash):
            raise ValueError(f"{kind[clash[0] + 1]} overlaps {kind[clash[0]]}")
        self._written = lo, hi, kind

    def bind(self, grads: Sequence[torch.Tensor]) -> None:
        """The gradient buffers that the following steps read."""
        grads = list(grads)
        if len(grads) != len(self.params):
            raise ValueError(f"{len(grads)} gradients for {len(self.params)} parameters")
        types = np.array(self._buffers("grads", grads, _TYPES, self._sizes))
        g_lo = np.array([g.data_ptr() for g in grads], np.int64)
        g_hi = g_lo + self._table["n"] * np.where(types == 0, 4, 2)
        lo, hi, kind = self._written
        if len(lo):
            before = np.searchsorted(lo, g_hi, "left") - 1  # the last written buffer that starts before the gradient ends
            clash = np.nonzero((before >= 0) & (hi[before] > g_lo) & (g_hi > g_lo))[0]
            if len(clash):
                raise ValueError(f"grads[{clash[0]}] overlaps {kind[before[clash[0]]]}")
        self.grads = grads
        self._table["grad"], self._table["grad_type"] = g_lo, types

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
        stream = _device_stream(self.device.index)
        flags = (None, 0) if skip is None else (skip.data_ptr(), skip.numel())
        if self._dstate is not None:
            check(lib().cnnue_adamw_multi_device(self._address, len(self.params), self._bits,
                                                 self._dstate.data_ptr(), grad_scale, *flags, stream),
                  "cnnue_adamw_multi_device")
            torch.autograd.graph.increment_version(self._changed)
            return
        check(lib().cnnue_adamw_multi(self._address, len(self.params), self._bits, self.lr, self.beta1,
                                      self.beta2, self.eps, self.weight_decay, self._step + 1, grad_scale, *flags,
                                      stream), "cnnue_adamw_multi")
        self._step += 1
        # told to autograd, as in-place operations are: a graph that saved a parameter refuses its backward pass
        torch.autograd.graph.increment_version(self._changed)
