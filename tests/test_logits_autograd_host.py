"""CPU tests of what policy_loss hands to the kernels of its backward pass: the
entry points are replaced by a recorder, the tensors lie on the CPU."""
import pytest
import torch

from chineseai_b200 import logits as lg

TARGET_FIELDS = ("dense", "dense_stride", "dense_type", "index", "index_stride", "index_bytes", "prob", "prob_stride", "count",
                 "mask", "mask_stride", "mask_rows", "mask_index", "weights")


@pytest.fixture
def calls(monkeypatch):
    """[(entry point, arguments)] of the calls, with CPU tensors let through."""
    made = []
    monkeypatch.setattr(lg, "_rows", lambda x, name: x if x.stride(1) == 1 or x.size(1) <= 1 else x.contiguous())
    monkeypatch.setattr(lg, "_call", lambda name, dev, status, *args: made.append((name, args)))
    return made


def fields(call):
    return dict(zip(TARGET_FIELDS, lg._TARGETS.unpack(call[1][5])))


def padded(shape, dtype, pad=3):
    return torch.zeros(shape[0], shape[1] + pad, dtype=dtype)[:, :shape[1]]


def packed_in_place(x):
    """A contiguous tensor of x's shape in x's own storage: the same address, other strides."""
    return x.as_strided(x.shape, (x.shape[1], 1)) if x.dim() == 2 else x


@pytest.mark.parametrize("kind", ["dense", "lists"])
def test_backward_takes_the_strides_that_saved_tensor_hooks_bring(calls, kind):
    R, V, K = 4, 70, 5
    z = padded((R, V), torch.float32).requires_grad_(True)
    kw = dict(mask=padded((R, 3), torch.int32))
    if kind == "dense":
        kw["targets"] = padded((R, V), torch.float32)
    else:
        kw.update(target_index=padded((R, K), torch.int32), target_prob=padded((R, K), torch.float32))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, packed_in_place):
        loss = lg.policy_loss(z, **kw)
    loss.sum().backward()
    (_, fwd), (name, bwd) = calls
    assert name == "cnnue_policy_loss_bwd"
    before, after = fields(calls[0]), fields(calls[1])
    assert fwd[1] == V + 3 and bwd[1] == V
    assert (before["mask_stride"], after["mask_stride"]) == (6, 3)
    if kind == "dense":
        assert (before["dense_stride"], after["dense_stride"]) == (V + 3, V)
    else:
        assert (before["index_stride"], after["index_stride"]) == (K + 3, K)
        assert (before["prob_stride"], after["prob_stride"]) == (K + 3, K)
    assert all(before[k] == after[k] for k in ("dense", "index", "prob", "mask"))
