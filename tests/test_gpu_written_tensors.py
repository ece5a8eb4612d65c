"""Tensors that the logit operators and MultiAdamW write in place: a graph that
saved one of them refuses its backward pass, as after torch's own in-place
operations."""
import pytest
import torch

from chineseai_b200 import logits as lg
from chineseai_b200.optim import MultiAdamW

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
MODIFIED = "modified by an inplace operation"


def test_process_logits_in_place():
    z = torch.randn(4, 100, device=DEV, requires_grad=True)
    mask = lg.pack_mask(torch.rand(4, 100, device=DEV) < 0.5)
    label = torch.zeros(4, dtype=torch.int64, device=DEV)
    for loss in (lg.policy_loss(z, target_index=label), torch.logsumexp(z, 1), lg.policy_loss(z, target_index=label)):
        lg.process_logits(z.detach(), mask=mask, out=z.detach())
        with pytest.raises(RuntimeError, match=MODIFIED):
            loss.sum().backward()
    a = z * 1.0
    p = torch.softmax(a, 1)
    lg.process_logits(p.detach(), mask=mask)  # another tensor gets the result: nothing changes
    p.sum().backward()


def test_policy_loss_grad_into_a_saved_tensor():
    z = torch.randn(4, 100, device=DEV)
    x = torch.randn(4, 100, device=DEV, requires_grad=True)
    buf = torch.empty_like(z)
    y = x * buf
    lg.policy_loss_grad(z, target_index=torch.zeros(4, dtype=torch.int64, device=DEV), grad=buf)
    with pytest.raises(RuntimeError, match=MODIFIED):
        y.sum().backward()


@pytest.mark.parametrize("device_state", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_between_forward_and_backward(bits, device_state):
    w = torch.nn.Parameter(torch.randn(8, 16, device=DEV))
    copy = w.detach().to(torch.bfloat16)
    g = torch.randn(8, 16, device=DEV)
    opt = MultiAdamW([w], [g], state_bits=bits, copies=[copy], device_state=device_state)
    x = torch.randn(4, 16, device=DEV, requires_grad=True)
    for y in (x @ w.t(), x.to(torch.bfloat16) @ copy.t()):
        opt.step()
        with pytest.raises(RuntimeError, match=MODIFIED):
            y.sum().backward()
    w.grad = None
    (x @ w.t()).sum().backward()  # a graph of the new values is fine
    opt.bind([w.grad])
    opt.step()
