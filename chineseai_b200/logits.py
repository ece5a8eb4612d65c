"""Logits a model answers with and learns from (over the C ABI).

`process_logits` applies penalties for repeated tokens, biases and packed
masks to rows of logits; `policy_loss` (with autograd) and `policy_loss_grad`
(loss and gradient in one pass) are the softmax cross entropy over the same
masks.  A token is anything a policy ranks: one of the 2086 dense moves
(`az.dense_moves`; `mcts.legal_mask` packs the legal ones), one of the 8100
from-to pairs, or an entry of a vocabulary.  The masked policy loss takes the
role of the policy part of compute_batch_loss
(src/az/train_gpu_candle.rs:221-305) for whole rows of logits.

All tensors are CUDA tensors on one device; calls run on that device's current
stream, allocate only their results and can be captured in a CUDA graph when
`status` is given.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import numpy as np
import torch

from ._lib import LogitRules, LossTargets, check, lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def pack_mask(allowed) -> "torch.Tensor | np.ndarray":
    """Truth values [..., V] as packed words int32 [..., ceil(V / 32)]: bit j of
    word w is token 32 w + j.  Takes and returns a tensor or a numpy array."""
    if isinstance(allowed, np.ndarray):
        return pack_mask(torch.from_numpy(np.ascontiguousarray(allowed))).numpy()
    a = allowed.bool()
    words = (a.shape[-1] + 31) // 32
    pad = torch.zeros(a.shape[:-1] + (words * 32,), dtype=torch.bool, device=a.device)
    pad[..., :a.shape[-1]] = a
    bit = torch.ones((), dtype=torch.int64, device=a.device) << torch.arange(32, device=a.device)
    w = (pad.view(a.shape[:-1] + (words, 32)) * bit).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _rows(x: torch.Tensor, name: str) -> torch.Tensor:
    if x.dim() != 2:
        raise ValueError(f"{name} must be [rows, vocab], got {tuple(x.shape)}")
    if not x.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if x.dtype not in _TYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {x.dtype}")
    return x if x.shape[1] <= 1 or x.stride(1) == 1 else x.contiguous()


def _per_row(x: Optional[torch.Tensor], like: torch.Tensor, dtype: torch.dtype, name: str, keep: list):
    """Pointer of a per-row vector, or None."""
    if x is None:
        return None
    if x.device != like.device:
        raise ValueError(f"{name} must be on {like.device}, is on {x.device}")
    if x.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {x.dtype}")
    if x.shape != like.shape[:1]:
        raise ValueError(f"{name} must be [{like.shape[0]}], got {tuple(x.shape)}")
    if not x.is_contiguous():
        x = x.contiguous()
        keep.append(x)
    return x.data_ptr()


def _lists(x: torch.Tensor, like: torch.Tensor, dtypes, name: str, keep: list) -> Tuple[int, int, int]:
    """(pointer, row stride, length) of lists [rows, n], or [n] for all rows."""
    if x.device != like.device:
        raise ValueError(f"{name} must be on {like.device}, is on {x.device}")
    if x.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {x.dtype}")
    if x.dim() not in (1, 2) or (x.dim() == 2 and x.shape[0] != like.shape[0]):
        raise ValueError(f"{name} must be [{like.shape[0]}, n] or [n], got {tuple(x.shape)}")
    n = x.shape[-1]
    if n > 1 and x.stride(-1) != 1:
        x = x.contiguous()
        keep.append(x)
    # an empty list has no storage and is never read: any address says that it is there
    return x.data_ptr() or like.data_ptr(), (x.stride(0) if x.dim() == 2 else 0), n


def _set_mask(s, mask, mask_index, like: torch.Tensor, keep: list) -> None:
    """Fills the mask fields of a LogitRules or LossTargets."""
    if mask is None:
        if mask_index is not None:
            raise ValueError("mask_index without a mask")
        return
    if mask.device != like.device:
        raise ValueError(f"mask must be on {like.device}, is on {mask.device}")
    if mask.dtype != torch.int32:
        raise TypeError(f"mask must hold packed int32 words (pack_mask), got {mask.dtype}")
    words = (like.shape[1] + 31) // 32
    if mask.dim() not in (1, 2) or mask.shape[-1] != words:
        raise ValueError(f"mask must be [masks, {words}] or [{words}], got {tuple(mask.shape)}")
    if words > 1 and mask.stride(-1) != 1:
        mask = mask.contiguous()
        keep.append(mask)
    n = 1 if mask.dim() == 1 else mask.shape[0]
    if mask_index is None and n != 1 and n != like.shape[0]:
        raise ValueError(f"mask has {n} rows for {like.shape[0]} rows of logits and no mask_index")
    s.mask, s.mask_stride, s.mask_rows = mask.data_ptr(), (0 if mask.dim() == 1 else mask.stride(0)), n
    s.mask_index = _per_row(mask_index, like, torch.int32, "mask_index", keep)


class _Call:
    """The status word, the stream and the device of one call: with `status`
    None the word is read here (a host synchronisation) and raised."""

    def __init__(self, like: torch.Tensor, status: Optional[torch.Tensor]):
        self.device = like.device
        self.own = status is None
        if self.own:
            status = torch.zeros(1, dtype=torch.int32, device=like.device)
        elif status.device != like.device or status.dtype != torch.int32 or status.numel() < 1:
            raise ValueError(f"status must be an int32 tensor on {like.device}")
        self.status = status

    def __call__(self, name: str, *args) -> None:
        if torch.cuda.current_device() != self.device.index:
            with torch.cuda.device(self.device):
                return self._run(name, *args)
        return self._run(name, *args)

    def _run(self, name: str, *args) -> None:
        stream = torch.cuda.current_stream(self.device).cuda_stream
        check(getattr(lib(), name)(*args, self.status.data_ptr(), stream), name)
        if self.own:
            st = C.c_int(0)
            check(lib().cnnue_read_status(self.status.data_ptr(), stream, C.byref(st)), "cnnue_read_status")
            check(st.value, f"{name} (kernel status)")


def process_logits(logits: torch.Tensor, *, history: Optional[torch.Tensor] = None,
                   lengths: Optional[torch.Tensor] = None, prompt_lengths: Optional[torch.Tensor] = None,
                   repetition: Optional[torch.Tensor] = None, frequency: Optional[torch.Tensor] = None,
                   presence: Optional[torch.Tensor] = None, bias_tokens: Optional[torch.Tensor] = None,
                   bias_values: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                   mask_index: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                   out_dtype: Optional[torch.dtype] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Penalties, biases and masks on logits [R, V] (float32, bfloat16 or
    float16), in this order, in fp32, rounded once:

    history int32 or int64 [R, L] (or [L]): tokens so far, negative = padding;
        the first lengths[r] (int32; default all) count, of which the first
        prompt_lengths[r] (int32; default none) are the prompt.  A token that
        occurs anywhere: x / repetition[r] when x > 0, else x * repetition[r].
        One that occurs c > 0 times after the prompt: x - frequency[r] * c,
        then - presence[r].  (repetition, frequency, presence: float32 [R].)
    bias_tokens int32 [R, K] (or [K]; negative = no entry) with bias_values
        float32 of the same shape: x + value; a repeated token takes its
        values in list order.
    mask int32 [G, ceil(V / 32)] packed words (`pack_mask`,
        `mcts.legal_mask`): tokens not allowed become -inf, whatever their
        logit.  Row r uses mask_index[r] (int32; negative = no mask), or row
        r, or the only row.

    Returns `out` (the logits' dtype or float32; `out=logits` works in place)
    or a new tensor of `out_dtype` (default: the logits').  A token >= V raises
    CnnueError (bad index; the token is skipped), a length outside [0, L] too
    (bad offsets; clamped); with `status` (int32 device tensor) the bits are
    collected there instead and nothing synchronises.  Not differentiable."""
    if torch.is_grad_enabled() and logits.requires_grad:
        raise ValueError("process_logits is not differentiable: detach the logits or use policy_loss")
    z = _rows(logits, "logits")
    if out is None:
        dtype = z.dtype if out_dtype is None else out_dtype
        if dtype != z.dtype and dtype != torch.float32:
            raise TypeError(f"out_dtype must be {z.dtype} or float32, got {dtype}")
        out = torch.empty(z.shape, dtype=dtype, device=z.device)
    else:
        if out.shape != z.shape or out.device != z.device:
            raise ValueError(f"out must be {tuple(z.shape)} on {z.device}, is {tuple(out.shape)} on {out.device}")
        if (out.dtype != z.dtype and out.dtype != torch.float32) or (out_dtype is not None and out.dtype != out_dtype):
            raise TypeError(f"out must be {z.dtype} or float32 (and out_dtype, if given), got {out.dtype}")
        if out.shape[1] > 1 and out.stride(1) != 1:
            raise ValueError("out: the vocabulary must be contiguous")
        if torch.is_grad_enabled() and out.requires_grad:
            raise ValueError("out requires a gradient")
    keep: list = [z]
    r = LogitRules()
    if history is not None:
        r.history, r.history_stride, r.history_len = _lists(history, z, (torch.int32, torch.int64), "history", keep)
        r.history_bytes = history.element_size()
        r.lengths = _per_row(lengths, z, torch.int32, "lengths", keep)
        r.prompt_lengths = _per_row(prompt_lengths, z, torch.int32, "prompt_lengths", keep)
        r.repetition = _per_row(repetition, z, torch.float32, "repetition", keep)
        r.frequency = _per_row(frequency, z, torch.float32, "frequency", keep)
        r.presence = _per_row(presence, z, torch.float32, "presence", keep)
    elif any(x is not None for x in (lengths, prompt_lengths, repetition, frequency, presence)):
        raise ValueError("penalties need a history")
    if (bias_tokens is None) != (bias_values is None):
        raise ValueError("bias_tokens and bias_values come together")
    if bias_tokens is not None:
        if bias_tokens.shape != bias_values.shape:
            raise ValueError(f"bias_tokens {tuple(bias_tokens.shape)} and bias_values {tuple(bias_values.shape)} differ")
        r.bias_tokens, r.bias_tokens_stride, r.bias_count = _lists(bias_tokens, z, (torch.int32,), "bias_tokens", keep)
        r.bias_values, r.bias_values_stride, _ = _lists(bias_values, z, (torch.float32,), "bias_values", keep)
    _set_mask(r, mask, mask_index, z, keep)
    _Call(z, status)("cnnue_logits_process", z.data_ptr(), z.stride(0), _TYPES[z.dtype], out.data_ptr(), out.stride(0),
                     _TYPES[out.dtype], z.shape[0], z.shape[1], C.addressof(r))
    return out


def _targets(z: torch.Tensor, targets, target_index, target_prob, mask, mask_index, weights, keep: list) -> LossTargets:
    t = LossTargets()
    if (targets is None) == (target_index is None):
        raise ValueError("give either dense targets or target_index")
    if targets is not None:
        if target_prob is not None:
            raise ValueError("target_prob goes with target_index")
        if targets.shape != z.shape or targets.device != z.device:
            raise ValueError(f"targets must be {tuple(z.shape)} on {z.device}, are {tuple(targets.shape)} on {targets.device}")
        d = _rows(targets, "targets")
        keep.append(d)
        t.dense, t.dense_stride, t.dense_type = d.data_ptr(), d.stride(0), _TYPES[d.dtype]
    else:
        if target_index.dim() == 1:  # labels: one token per row
            target_index = target_index[:, None]
            if target_prob is not None and target_prob.dim() == 1:
                target_prob = target_prob[:, None]
        if target_index.dim() != 2:
            raise ValueError(f"target_index must be [rows] or [rows, n], got {tuple(target_index.shape)}")
        t.index, t.index_stride, t.count = _lists(target_index, z, (torch.int32, torch.int64), "target_index", keep)
        t.index_bytes = target_index.element_size()
        if target_prob is not None:
            if target_prob.shape != target_index.shape:
                raise ValueError(f"target_prob must be {tuple(target_index.shape)}, got {tuple(target_prob.shape)}")
            t.prob, t.prob_stride, _ = _lists(target_prob, z, (torch.float32,), "target_prob", keep)
    _set_mask(t, mask, mask_index, z, keep)
    t.weights = _per_row(weights, z, torch.float32, "weights", keep)
    return t


def _refuse_gradients(**named) -> None:
    for name, x in named.items():
        if x is not None and x.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name}: the loss is differentiable in the logits only")


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, target_index, target_prob, mask, mask_index, weights, status):
        z = _rows(logits, "logits")
        keep: list = []
        t = _targets(z, targets, target_index, target_prob, mask, mask_index, weights, keep)
        loss = torch.empty(z.shape[0], dtype=torch.float32, device=z.device)
        stats = torch.empty((z.shape[0], 3), dtype=torch.float32, device=z.device)
        _Call(z, status)("cnnue_policy_loss_fwd", z.data_ptr(), z.stride(0), _TYPES[z.dtype], z.shape[0], z.shape[1],
                         C.addressof(t), loss.data_ptr(), stats.data_ptr())
        ctx.save_for_backward(logits, targets, target_index, target_prob, mask, mask_index, weights, stats)
        ctx.status = status
        return loss

    @staticmethod
    def backward(ctx, upstream):
        logits, targets, target_index, target_prob, mask, mask_index, weights, stats = ctx.saved_tensors
        z = _rows(logits, "logits")
        keep: list = []
        t = _targets(z, targets, target_index, target_prob, mask, mask_index, weights, keep)
        up = upstream.float().contiguous()
        grad = torch.empty(z.shape, dtype=z.dtype, device=z.device)
        _Call(z, ctx.status)("cnnue_policy_loss_bwd", z.data_ptr(), z.stride(0), _TYPES[z.dtype], z.shape[0],
                             z.shape[1], C.addressof(t), stats.data_ptr(), up.data_ptr(), grad.data_ptr(),
                             grad.stride(0))
        return grad, None, None, None, None, None, None, None


def policy_loss(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, *,
                target_index: Optional[torch.Tensor] = None, target_prob: Optional[torch.Tensor] = None,
                mask: Optional[torch.Tensor] = None, mask_index: Optional[torch.Tensor] = None,
                weights: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Masked softmax cross entropy per row: logits [R, V] -> float32 [R],
    differentiable in the logits (the gradient has their dtype).

    Over the allowed tokens of a row: loss = weight * sum t (log sum exp z -
    z).  The targets t are dense `targets` [R, V] (float32, bfloat16 or
    float16), or lists: target_index int32 or int64 [R, K] (or labels [R];
    negative = no entry) with target_prob float32 of the same shape (default:
    1 each; repeated tokens add up).  They need not sum to 1.  `mask` and
    `mask_index` as in process_logits; targets on tokens that are not allowed
    are dropped.  weights float32 [R], default 1: divide by the row count for a
    mean.  A row with nothing allowed, or of weight 0, has loss 0 and gradient
    0; a NaN at an allowed token makes its row NaN.  A listed token >= V raises
    CnnueError, or sets a bit of `status` (int32 device tensor) when given."""
    _refuse_gradients(targets=targets, target_prob=target_prob, weights=weights)
    return _PolicyLoss.apply(logits, targets, target_index, target_prob, mask, mask_index, weights, status)


def policy_loss_grad(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, *,
                     target_index: Optional[torch.Tensor] = None, target_prob: Optional[torch.Tensor] = None,
                     mask: Optional[torch.Tensor] = None, mask_index: Optional[torch.Tensor] = None,
                     weights: Optional[torch.Tensor] = None, grad: Optional[torch.Tensor] = None,
                     status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss float32 [R], gradient of its sum over the rows [R, V] in the
    logits' dtype), in one pass over the logits: policy_loss and its backward
    for training loops that know the row weights beforehand.  Arguments as in
    policy_loss; `grad`: where to write the gradient (not the logits)."""
    _refuse_gradients(targets=targets, target_prob=target_prob, weights=weights)
    z = _rows(logits.detach(), "logits")
    keep: list = []
    t = _targets(z, targets, target_index, target_prob, mask, mask_index, weights, keep)
    if grad is None:
        grad = torch.empty(z.shape, dtype=z.dtype, device=z.device)
    else:
        if grad.shape != z.shape or grad.device != z.device or grad.dtype != z.dtype:
            raise ValueError(f"grad must be {z.dtype} {tuple(z.shape)} on {z.device}")
        if grad.shape[1] > 1 and grad.stride(1) != 1:
            raise ValueError("grad: the vocabulary must be contiguous")
    loss = torch.empty(z.shape[0], dtype=torch.float32, device=z.device)
    _Call(z, status)("cnnue_policy_loss_grad", z.data_ptr(), z.stride(0), _TYPES[z.dtype], z.shape[0], z.shape[1],
                     C.addressof(t), loss.data_ptr(), grad.data_ptr(), grad.stride(0))
    return loss, grad
