"""CPU tests of what the many-tensor AdamW refuses about the form of its states."""
import ctypes as C

import pytest
import torch

from chineseai_b200 import _lib
from chineseai_b200.optim import MultiAdamW

INVALID, A = 1, 1 << 20  # an address that no call below gets to use


@pytest.mark.parametrize("bits", [0, 256, 32 | 256, 8 | 512, 8 | 1, -8])
def test_forms_of_the_states(bits):
    t = (_lib.AdamwTensor * 1)(_lib.AdamwTensor(param=A, grad=A, m=A, v=A, m_scale=A, v_scale=A, n=4))
    L = _lib.lib()
    assert L.cnnue_adamw_multi(C.addressof(t), 1, bits, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, None, 0, None) == INVALID
    assert L.cnnue_adamw_multi_device(C.addressof(t), 1, bits, A, 1.0, None, 0, None) == INVALID


@pytest.mark.parametrize("missing", ["m_scale", "v_scale"])
def test_stochastic_states_need_their_scales(missing):
    t = (_lib.AdamwTensor * 1)(_lib.AdamwTensor(param=A, grad=A, m=A, v=A, m_scale=A, v_scale=A, n=4))
    setattr(t[0], missing, None)
    L = _lib.lib()
    assert L.cnnue_adamw_multi(C.addressof(t), 1, 8 | 256, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, None, 0, None) == INVALID


def test_stochastic_is_for_8_bits():
    x = torch.zeros(4)
    with pytest.raises(ValueError, match="stochastic"):
        MultiAdamW([x], [x], stochastic=True)
