"""What the device-state AdamW entry points write to cnnue_adamw_state, and to
the 8-bit states over many steps."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from chineseai_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
LR, B1, B2, EPS, WD = 3e-3, 0.9, 0.999, 1e-8, 0.01


def device_state(step, mark):
    """cnnue_adamw_state: five doubles, the step, 9 scalars, 3 floats of padding (filled with `mark`)."""
    host = np.zeros(12, np.float64)
    host[:5] = [LR, B1, B2, EPS, WD]
    host.view(np.int64)[5] = step
    host.view(np.float32)[21:24] = mark
    return torch.from_numpy(host.view(np.uint8).copy()).to(DEV)


def pads(state):
    return state.cpu().numpy().view(np.float32)[21:24]


@pytest.mark.parametrize("step", [0, 1, 99, 12345])
def test_the_root_factor_is_formed_by_8_bit_steps_only(step):
    """The other device steps, the AZ trainer's among them, do not form it."""
    p, g, m, v = (torch.zeros(512, device=DEV) for _ in range(4))
    scales = torch.zeros(2, 2, device=DEV)
    t = (_lib.AdamwTensor * 1)(_lib.AdamwTensor(param=p.data_ptr(), grad=g.data_ptr(), m=m.data_ptr(), v=v.data_ptr(),
                                                m_scale=scales[0].data_ptr(), v_scale=scales[1].data_ptr(), n=512))
    L, mark = _lib.lib(), 7.5
    flat = (p.data_ptr(), m.data_ptr(), v.data_ptr(), g.data_ptr(), 512)
    stream = torch.cuda.current_stream().cuda_stream
    for call in (lambda s: L.cnnue_adamw_device(*flat, s, stream),
                 lambda s: L.cnnue_adamw_device_scaled(*flat, s, 0.5, None, 0, stream),
                 lambda s: L.cnnue_adamw_multi_device(C.addressof(t), 1, 32, s, 1.0, None, 0, stream)):
        state = device_state(step, mark)
        assert call(state.data_ptr()) == 0
        assert pads(state)[0] == 0 and (pads(state)[1:] == mark).all()
    state = device_state(step, mark)
    assert L.cnnue_adamw_multi_device(C.addressof(t), 1, 8, state.data_ptr(), 1.0, None, 0, stream) == 0
    want = math.sqrt(1.0 / (1.0 - B2 ** (step + 1)))
    # fp64 rounding (the power's, grown by the difference from 1) is far below fp32's half step
    assert abs(pads(state)[1] - want) <= want * 2.0 ** -23 and pads(state)[2] == mark
