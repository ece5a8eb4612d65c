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
stream, allocate only their results (and contiguous copies of inputs whose last
dimension is strided) and can be captured in a CUDA graph when `status` is
given.  While policy_loss's backward pass is captured, no eager graph of the
same leaf may live: torch ends the capture with an error then, as for its own
operations.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Tuple

import numpy as np
import torch

from ._lib import check, lib
from .quantized import _device_stream

# What a kernel wrote into a caller's tensor, told to autograd: a graph that saved it refuses its backward pass.
_written = torch.autograd.graph.increment_version

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


# The C structs as bytes (native layout): much quicker to fill than field by
# field, and these calls run once per generated token.
_RULES = struct.Struct("@PqqiPPPPPPqPqqPqqP")    # cnnue_logit_rules
_TARGETS = struct.Struct("@PqiPqiPqqPqqPP")       # cnnue_loss_targets
_NO_MASK = (0, 0, 0, 0)
_INTS = {torch.int32: 4, torch.int64: 8}


def _rows(x: torch.Tensor, name: str) -> torch.Tensor:
    if x.dim() != 2:
        raise ValueError(f"{name} must be [rows, vocab], got {tuple(x.shape)}")
    if not x.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if x.dtype not in _TYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {x.dtype}")
    return x if x.stride(1) == 1 or x.size(1) <= 1 else x.contiguous()


def _per_row(x: Optional[torch.Tensor], n: int, dev: int, dtype: torch.dtype, name: str, keep: list) -> int:
    """Address of a per-row vector, 0 for None."""
    if x is None:
        return 0
    if x.dtype is dtype and x.get_device() == dev and x.dim() == 1 and x.numel() == n:
        if not x.is_contiguous():
            x = x.contiguous()
            keep.append(x)
        return x.data_ptr()
    if x.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {x.dtype}")
    if x.get_device() != dev:
        raise ValueError(f"{name} must be on cuda:{dev}, is on {x.device}")
    raise ValueError(f"{name} must be [{n}], got {tuple(x.shape)}")


def _lists(x: torch.Tensor, n: int, dev: int, dtypes, name: str, keep: list) -> Tuple[int, int, int]:
    """(address, row stride, length) of lists [rows, n], or [n] for all rows."""
    if x.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {x.dtype}")
    if x.get_device() != dev:
        raise ValueError(f"{name} must be on cuda:{dev}, is on {x.device}")
    shape = x.shape
    dim = len(shape)
    if dim not in (1, 2) or (dim == 2 and shape[0] != n):
        raise ValueError(f"{name} must be [{n}, n] or [n], got {tuple(shape)}")
    length = shape[-1]
    strides = x.stride()
    if length > 1 and strides[-1] != 1:
        x = x.contiguous()
        keep.append(x)
        strides = x.stride()
    # an empty list has no storage and is never read: any address says that it is there
    return x.data_ptr() or 1 << 12, (strides[0] if dim == 2 else 0), length


def _mask(mask: Optional[torch.Tensor], mask_index, n: int, vocab: int, dev: int, keep: list):
    """The mask fields of a struct: address, stride, rows, index."""
    if mask is None:
        if mask_index is not None:
            raise ValueError("mask_index without a mask")
        return _NO_MASK
    if mask.dtype is not torch.int32:
        raise TypeError(f"mask must hold packed int32 words (pack_mask), got {mask.dtype}")
    if mask.get_device() != dev:
        raise ValueError(f"mask must be on cuda:{dev}, is on {mask.device}")
    words, shape = (vocab + 31) // 32, mask.shape
    dim = len(shape)
    if dim not in (1, 2) or shape[-1] != words:
        raise ValueError(f"mask must be [masks, {words}] or [{words}], got {tuple(shape)}")
    strides = mask.stride()
    if words > 1 and strides[-1] != 1:
        mask = mask.contiguous()
        keep.append(mask)
        strides = mask.stride()
    m = 1 if dim == 1 else shape[0]
    if mask_index is None and m != 1 and m != n:
        raise ValueError(f"mask has {m} rows for {n} rows of logits and no mask_index")
    index = 0 if mask_index is None else _per_row(mask_index, n, dev, torch.int32, "mask_index", keep)
    return mask.data_ptr() or 1 << 12, (0 if dim == 1 else strides[0]), m, index


def _call(name: str, dev: int, status: Optional[torch.Tensor], *args) -> None:
    """One entry point on the device's current stream.  With `status` None the
    kernels' status word is read here (a host synchronisation) and raised."""
    if torch.cuda.current_device() != dev:
        with torch.cuda.device(dev):
            return _call(name, dev, status, *args)
    own = status is None
    if own:
        status = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", dev))
    elif status.dtype is not torch.int32 or status.get_device() != dev or status.numel() < 1:
        raise ValueError(f"status must be an int32 tensor on cuda:{dev}")
    stream = _device_stream(dev)
    st = getattr(lib(), name)(*args, status.data_ptr(), stream)
    if st:
        check(st, name)
    if own:
        word = C.c_int(0)
        check(lib().cnnue_read_status(status.data_ptr(), stream, C.byref(word)), "cnnue_read_status")
        check(word.value, f"{name} (kernel status)")


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
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("process_logits is not differentiable: detach the logits or use policy_loss")
    z = _rows(logits, "logits")
    n, vocab = z.shape
    dev = z.get_device()
    code = _TYPES[z.dtype]
    given = out
    if out is None:
        if out_dtype is None or out_dtype is z.dtype:
            out, out_code = torch.empty_like(z), code
        elif out_dtype is torch.float32:
            out, out_code = torch.empty_like(z, dtype=torch.float32), 0
        else:
            raise TypeError(f"out_dtype must be {z.dtype} or float32, got {out_dtype}")
    else:
        if out.shape != z.shape or out.get_device() != dev:
            raise ValueError(f"out must be {tuple(z.shape)} on {z.device}, is {tuple(out.shape)} on {out.device}")
        if (out.dtype != z.dtype and out.dtype != torch.float32) or (out_dtype is not None and out.dtype != out_dtype):
            raise TypeError(f"out must be {z.dtype} or float32 (and out_dtype, if given), got {out.dtype}")
        if vocab > 1 and out.stride(1) != 1:
            raise ValueError("out: the vocabulary must be contiguous")
        if torch.is_grad_enabled() and out.requires_grad:
            raise ValueError("out requires a gradient")
        out_code = _TYPES[out.dtype]
    keep: list = []
    if history is not None:
        f32 = torch.float32
        h, h_stride, h_len = _lists(history, n, dev, _INTS, "history", keep)
        part = (h, h_stride, h_len, _INTS[history.dtype], _per_row(lengths, n, dev, torch.int32, "lengths", keep),
                _per_row(prompt_lengths, n, dev, torch.int32, "prompt_lengths", keep),
                _per_row(repetition, n, dev, f32, "repetition", keep), _per_row(frequency, n, dev, f32, "frequency", keep),
                _per_row(presence, n, dev, f32, "presence", keep))
    else:
        for x in (lengths, prompt_lengths, repetition, frequency, presence):
            if x is not None:
                raise ValueError("penalties need a history")
        part = (0, 0, 0, 0, 0, 0, 0, 0, 0)
    if bias_tokens is not None and bias_values is not None:
        if bias_tokens.shape != bias_values.shape:
            raise ValueError(f"bias_tokens {tuple(bias_tokens.shape)} and bias_values {tuple(bias_values.shape)} differ")
        t, t_stride, count = _lists(bias_tokens, n, dev, (torch.int32,), "bias_tokens", keep)
        v, v_stride, _ = _lists(bias_values, n, dev, (torch.float32,), "bias_values", keep)
        bias = (t, t_stride, v, v_stride, count)
    elif bias_tokens is None and bias_values is None:
        bias = (0, 0, 0, 0, 0)
    else:
        raise ValueError("bias_tokens and bias_values come together")
    rules = _RULES.pack(*part, *bias, *_mask(mask, mask_index, n, vocab, dev, keep))
    _call("cnnue_logits_process", dev, status, z.data_ptr(), z.stride(0), code, out.data_ptr(), out.stride(0), out_code, n,
          vocab, rules)
    if given is not None:
        _written(given)
    return out


def _targets(z: torch.Tensor, targets, target_index, target_prob, mask, mask_index, weights, keep: list) -> bytes:
    n, vocab = z.shape
    dev = z.get_device()
    if targets is not None:
        if target_index is not None:
            raise ValueError("give either dense targets or target_index")
        if target_prob is not None:
            raise ValueError("target_prob goes with target_index")
        if targets.shape != z.shape or targets.get_device() != dev:
            raise ValueError(f"targets must be {tuple(z.shape)} on {z.device}, are {tuple(targets.shape)} on {targets.device}")
        d = _rows(targets, "targets")
        if d is not targets:
            keep.append(d)
        part = (d.data_ptr(), d.stride(0), _TYPES[d.dtype], 0, 0, 0, 0, 0, 0)
    else:
        if target_index is None:
            raise ValueError("give either dense targets or target_index")
        if target_index.dim() == 1:  # labels: one token per row
            target_index = target_index[:, None]
            if target_prob is not None and target_prob.dim() == 1:
                target_prob = target_prob[:, None]
        if target_index.dim() != 2:
            raise ValueError(f"target_index must be [rows] or [rows, n], got {tuple(target_index.shape)}")
        i, i_stride, count = _lists(target_index, n, dev, _INTS, "target_index", keep)
        p = p_stride = 0
        if target_prob is not None:
            if target_prob.shape != target_index.shape:
                raise ValueError(f"target_prob must be {tuple(target_index.shape)}, got {tuple(target_prob.shape)}")
            p, p_stride, _ = _lists(target_prob, n, dev, (torch.float32,), "target_prob", keep)
        part = (0, 0, 0, i, i_stride, _INTS[target_index.dtype], p, p_stride, count)
    return _TARGETS.pack(*part, *_mask(mask, mask_index, n, vocab, dev, keep),
                         _per_row(weights, n, dev, torch.float32, "weights", keep))


def _refuse_gradients(*tensors) -> None:
    for x in tensors:
        if x is not None and x.requires_grad and torch.is_grad_enabled():
            raise ValueError("targets, target_prob and weights: the loss is differentiable in the logits only")


def _places(tensors) -> list:
    """Where tensors of known shapes and types lie: all that a struct holds of them."""
    return [None if x is None else (x.data_ptr(), x.stride()) for x in tensors]


def _as_read(x: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """x with its last dimension contiguous, as the kernels read it."""
    return x if x is None or x.dim() == 0 or x.stride(-1) == 1 or x.size(-1) <= 1 else x.contiguous()


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, target_index, target_prob, mask, mask_index, weights, status):
        z = _rows(logits, "logits")
        inputs = [_as_read(x) for x in (targets, target_index, target_prob, mask, mask_index, weights)]
        t = _targets(z, *inputs, [])
        n, vocab = z.shape
        dev = z.get_device()
        loss = z.new_empty(n, dtype=torch.float32)
        stats = z.new_empty(3 * n, dtype=torch.float32)
        _call("cnnue_policy_loss_fwd", dev, status, z.data_ptr(), z.stride(0), _TYPES[z.dtype], n, vocab, t,
              loss.data_ptr(), stats.data_ptr())
        # copies that were made are saved in the place of what they are copies of, and freed with the graph
        saved = (z, *inputs, stats)
        ctx.save_for_backward(*saved)
        ctx.status = status
        # the struct, for a backward pass over the same storage (saved-tensor hooks may bring another, or another layout)
        ctx.packed = _places(saved), t
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, upstream):
        saved = ctx.saved_tensors
        z, stats = saved[0], saved[7]
        places, t = ctx.packed
        keep: list = []
        if _places(saved) != places:
            z = _rows(z, "logits")
            t = _targets(z, *saved[1:7], keep)
        n, vocab = z.shape
        up = upstream if upstream.dtype is torch.float32 and upstream.is_contiguous() else upstream.float().contiguous()
        grad = torch.empty_like(z)
        _call("cnnue_policy_loss_bwd", z.get_device(), ctx.status, z.data_ptr(), z.stride(0), _TYPES[z.dtype], n, vocab, t,
              stats.data_ptr(), up.data_ptr(), grad.data_ptr(), grad.stride(0))
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
    _refuse_gradients(targets, target_prob, weights)
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
    _refuse_gradients(targets, target_prob, weights)
    z = _rows(logits, "logits")
    keep: list = []
    t = _targets(z, targets, target_index, target_prob, mask, mask_index, weights, keep)
    n, vocab = z.shape
    dev = z.get_device()
    given = grad
    if grad is None:
        grad = torch.empty_like(z)
    else:
        if grad.shape != z.shape or grad.get_device() != dev or grad.dtype != z.dtype:
            raise ValueError(f"grad must be {z.dtype} {tuple(z.shape)} on {z.device}")
        if vocab > 1 and grad.stride(1) != 1:
            raise ValueError("grad: the vocabulary must be contiguous")
        if torch.is_grad_enabled() and grad.requires_grad:
            raise ValueError("grad requires a gradient")
    loss = z.new_empty(n, dtype=torch.float32)
    _call("cnnue_policy_loss_grad", dev, status, z.data_ptr(), z.stride(0), _TYPES[z.dtype], n, vocab, t, loss.data_ptr(),
          grad.data_ptr(), grad.stride(0))
    if given is not None:
        _written(given)
    return loss, grad
