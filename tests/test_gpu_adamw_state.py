"""What the device-state AdamW entry points write to cnnue_adamw_state, and to
the 8-bit states over many steps."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from tests.test_gpu_multi_adamw import B1, B2, EPS, EPS32, LR, SIZES, WD, check_codes, expect, f64, held, placed, tensors
from chineseai_b200 import _lib
from chineseai_b200.optim import MultiAdamW

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


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


# ---- 8-bit states, the second moment rounded stochastically ----------------------------
def steps_around(want, scale):
    """The e4m3 values times `scale` around each value (64 bits): (below, above)."""
    grid = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()  # 0 .. 448
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(scale > 0, want / scale, 0.0)
    at = np.clip(np.searchsorted(grid, q, "right") - 1, 0, len(grid) - 2)
    return grid[at] * scale, grid[at + 1] * scale


def pair_of(ps, gs, state, offset=0, **kw):
    """Two optimizers from the same parameters, gradients and state: nearest and stochastic."""
    out = []
    for stochastic in (False, True):
        p, _ = placed(ps, offset)
        g, _ = placed(gs, offset)
        st = None if state is None else {k: [t.clone() for t in v] for k, v in state.items()}
        out.append(MultiAdamW(p, g, lr=LR, weight_decay=WD, state_bits=8, state=st, stochastic=stochastic, **kw))
    return out


def all_bytes(opt):
    return torch.cat([t.contiguous().reshape(-1).view(torch.uint8) for v in [opt.params, *opt.state.values()] for t in v])


def some_state(ps, gs, steps=3):
    """A state that has seen gradients of different sizes."""
    p, _ = placed(ps, 0)
    g, _ = placed(gs, 0)
    opt = MultiAdamW(p, g, lr=LR, weight_decay=WD, state_bits=8)
    for i in range(steps):
        for t in g:
            t.mul_(-0.7)
        opt.step()
    return opt.state


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("ptype,gtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                         (torch.bfloat16, torch.float16), (torch.float16, torch.float32)])
def test_stochastic_rounding_takes_one_of_the_two_codes(ptype, gtype, offset):
    """Parameters, first moments and scales are the other form's bits; each code of the root is a neighbour of its value."""
    ps, gs = tensors(SIZES, ptype, 30), tensors(SIZES, gtype, 31, 0.1)
    state = some_state(ps, gs)
    a, b = pair_of(ps, gs, state, offset, step=3)
    a.step()
    b.step()
    up = total = 0
    for i, n in enumerate(SIZES):
        assert torch.equal(a.params[i], b.params[i])
        for k in ("m", "m_scale", "v_scale"):
            assert torch.equal(a.state[k][i].view(torch.uint8), b.state[k][i].view(torch.uint8)), k
        m, u = (held(state[k][i], state[k + "_scale"][i]) for k in "mv")
        _, _, u1, _, _, e = expect(f64(ps[i]), f64(gs[i]), m, u, None, 4, True, True)
        each = np.repeat(f64(b.state["v_scale"][i]), 256)[:n]
        # the kernel's u' is off by e, its scale and its product with 448 / max by four roundings
        slack = e + 4 * EPS32 * u1
        low, high = steps_around(u1 - slack, each)[0], steps_around(u1 + slack, each)[1]
        got = held(b.state["v"][i], b.state["v_scale"][i])
        assert ((got >= low * (1 - 2 * EPS32)) & (got <= high * (1 + 2 * EPS32))).all(), n
        assert (got[(u1 > 2.0 ** -62) & (each > 0)] > 0).all()
        up, total = up + int((got > u1).sum()), total + n
    assert 0.3 * total < up < 0.7 * total


def test_stochastic_rounding_is_unbiased_and_independent():
    """Over elements and over steps: the codes' mean is the value, and one step's rounding says nothing of another's."""
    n, steps = 1 << 18, 16
    ps, gs = tensors([n], torch.float32, 32), tensors([n], torch.float32, 33, 0.1)
    state = some_state(ps, gs)
    m, u = (held(state[k][0], state[k + "_scale"][0]) for k in "mv")
    u1 = expect(f64(ps[0]), f64(gs[0]), m, u, None, 4, True, True)[2]
    rest = []
    for step in range(100, 100 + steps):
        _, b = pair_of(ps, gs, state, step=step)
        b.step()
        each = np.repeat(f64(b.state["v_scale"][0]), 256)
        low, high = steps_around(u1, each)
        p = (u1 - low) / (high - low)
        live = (p > 0.001) & (p < 0.999)  # values next to a code may fall on its other side in fp32
        got = held(b.state["v"][0], b.state["v_scale"][0])
        rest.append(np.where(live, (got > (low + high) / 2) - p, 0.0))
        var = (p * (1 - p))[live].sum()
        # 6 standard deviations; the probability is good to 2^-17 (the random bits) and to u's 2^-20 and a few roundings,
        # 16 times that of a code's step
        assert abs(rest[-1].sum()) < 6 * math.sqrt(var) + live.sum() * 2.0 ** -15
        assert abs((rest[-1] ** 2).sum() - var) < 6 * math.sqrt(n) * 0.25 + n * 2.0 ** -15  # each square varies by 1/4 at most
    for i in range(steps):
        for j in range(i):
            assert abs((rest[i] * rest[j]).sum()) < 6 * math.sqrt(n) * 0.25 + n * 2.0 ** -15
    for lag in (1, 2, 3, 128, 256):
        assert abs((rest[0][lag:] * rest[0][:-lag]).sum()) < 6 * math.sqrt(n) * 0.25 + n * 2.0 ** -15


@pytest.mark.parametrize("kind", ["still", "fall", "grow"])
def test_stochastic_root_moments_follow_the_gradients(kind):
    """3,000 steps of normal gradients; in half of every block they change tenfold, or threefold, after step 500.

    The spread, by arithmetic: v falls by 1 - beta2 per step at most, sqrt(v) by f = 0.0005 of itself.  A code's step is
    d = 1/16 to 1/8 of its value, so a code moves with probability f / d, and one step adds f d to the variance of log u,
    at most 0.0000625; while v falls, nothing takes an error back.  After 2,500 steps: 0.156 at most, a standard deviation
    of 0.395, so 1 % and 99 % lie at exp(-+ 2.33 0.395) = 0.40 and 2.5 times the median; the mean of u is kept, so the
    median is exp(-0.156 / 2) = 0.92 at least; sampling adds less than a twentieth: 0.36 to 2.8.  (Where v does not fall,
    errors are taken back and the spread is a fifth.)  Rounded to nearest, a CPU model has medians of 4.1 in `fall` and of
    3.0 in the other half of `grow`."""
    n = 1 << 14
    p, g = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    opt = MultiAdamW([p], [g], lr=LR, weight_decay=WD, state_bits=8, stochastic=True)
    half = torch.arange(n, device=DEV) % 2 == 0
    factor = torch.where(half, {"still": 1.0, "fall": 0.1, "grow": 3.0}[kind], 1.0)
    v = torch.zeros(n, device=DEV, dtype=torch.float64)
    rng = torch.Generator(device=DEV).manual_seed(34)
    for t in range(3000):
        g.normal_(generator=rng)
        if t >= 500:
            g.mul_(factor)
        opt.step()
        v.mul_(B2).addcmul_(g.double(), g.double(), value=1 - B2)
    u = opt.state["v"][0].double() * opt.state["v_scale"][0].double().repeat_interleave(256)
    ratio = u / v.sqrt()
    for part in (ratio[half], ratio[~half]):
        low, mid, high = torch.quantile(part, torch.tensor([0.01, 0.5, 0.99], device=DEV, dtype=torch.float64)).tolist()
        assert 0.36 < low and 0.9 < mid < 1.1 and high < 2.8, (low, mid, high)


def test_stochastic_steps_do_not_depend_on_launch_alignment_or_run():
    """The same bits at other alignments, from run to run, from a resumed state, and from a replayed graph."""
    sizes = SIZES + [(i * 37) % 300 + 1 for i in range(800)]  # three launches
    ps, gs = tensors(sizes, torch.float32, 35), tensors(sizes, torch.bfloat16, 36)
    want = []
    for offset, device_state in ((0, False), (1, False), (4, True)):
        p, _ = placed(ps, offset)
        g, _ = placed(gs, offset)
        opt = MultiAdamW(p, g, lr=LR, weight_decay=WD, state_bits=8, stochastic=True, device_state=device_state)
        got = []
        if device_state:
            opt.step()
            got.append(all_bytes(opt))
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step()
            for _ in range(2):
                graph.replay()
                got.append(all_bytes(opt))
        else:
            for _ in range(3):
                opt.step()
                got.append(all_bytes(opt))
        if want:
            assert all(torch.equal(x, y) for x, y in zip(got, want))
        want = got
    state = {k: [t.clone() for t in v] for k, v in opt.state.items()}
    again = MultiAdamW([t.clone() for t in opt.params], opt.grads, lr=LR, weight_decay=WD, state_bits=8, stochastic=True,
                       state=state, step=3)
    again.step()
    graph.replay()
    assert torch.equal(all_bytes(again), all_bytes(opt))


def test_tensors_and_steps_round_by_themselves():
    """Equal tensors of one list get other random bits, and so do later steps."""
    n = 4096
    ps, gs = tensors([n], torch.float32, 37) * 2, tensors([n], torch.float32, 38) * 2
    codes = []
    for step in (5, 6):
        p, _ = placed(ps, 0)
        g, _ = placed(gs, 0)
        opt = MultiAdamW(p, g, lr=LR, weight_decay=WD, state_bits=8, stochastic=True, step=step)
        opt.step()
        assert torch.equal(p[0], p[1])
        codes += [t.view(torch.uint8) for t in opt.state["v"]]
    for i in range(4):
        for j in range(i):
            assert 0.1 * n < int((codes[i] != codes[j]).sum()) < 0.6 * n


def test_stochastic_blocks_with_a_nan_zeros_and_tiny_values():
    n = 1279
    g = torch.ones(n, device=DEV)
    g[256:512] = 0
    g[600] = float("nan")
    g[700] = float("inf")
    g[768:1024] = 1e-38
    g[1278] = float("nan")
    p = torch.zeros(n, device=DEV)
    opt = MultiAdamW([p], [g], state_bits=8, lr=LR, stochastic=True)
    opt.step()
    u, s = opt.state["v"][0].float().cpu(), opt.state["v_scale"][0].cpu()
    assert torch.isfinite(u[:512]).all() and (u[:256] == 448).all() and not u[256:512].any() and s[1] == 0
    assert not torch.isfinite(s[2]) and u[512:768].isnan().all() and torch.isfinite(u[768:1024]).all()
    assert not torch.isfinite(s[4]) and u[1024:].isnan().all()
    assert torch.isfinite(p[:600]).all() and torch.isfinite(p[768:1024]).all()


def test_stochastic_rounding_is_refused_for_32_bits():
    p, g = torch.zeros(8, device=DEV), torch.zeros(8, device=DEV)
    with pytest.raises(ValueError, match="stochastic"):
        MultiAdamW([p], [g], stochastic=True)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("native", [True, False])
def test_az_trainer_with_8_bit_states_steps_by_the_formula(native, graph):
    """Each step's parameters and states against the formula in 64 bits, from the state and the gradients of that step."""
    from chineseai_b200 import az, az_train
    w = az.AzWeights.random(32, 7)
    batch = az_train.pack_batch(az_train.random_samples(48, 5), caps=(96, 160, 256), fixed=True)
    tr = az_train.AzTrainer(w, lr=LR, graph=graph, native=native, state_bits=8, weight_decay=WD)
    opt, moved = tr.optimizer, set()
    for step in range(1, 6):
        before = [(f64(p), held(*(opt.state[k][i] for k in ("m", "m_scale"))), held(*(opt.state[k][i] for k in ("v", "v_scale"))))
                  for i, p in enumerate(opt.params)]
        tr.step(batch)
        assert opt.step_count == step
        for i, (p, m, u) in enumerate(before):
            g = f64(opt.grads[i])
            p1, m1, u1, e_p, e_m, e_u = expect(p, g, m, u, None, step, True, True)
            clear = (u1 > 2.0 ** -55) | (u1 == 0)  # below, a root outside fp32's normal range says nothing of the step
            assert (np.abs(f64(opt.params[i]) - p1) <= e_p)[clear].all(), (step, i)
            check_codes(opt.state["m"][i], opt.state["m_scale"][i], m1, e_m, False)
            each = np.repeat(f64(opt.state["v_scale"][i]), 256)[:len(u1)]
            slack = e_u + 4 * EPS32 * u1
            low, high = steps_around(u1 - slack, each)[0], steps_around(u1 + slack, each)[1]
            got = held(opt.state["v"][i], opt.state["v_scale"][i])
            assert ((got >= low * (1 - 2 * EPS32)) & (got <= high * (1 + 2 * EPS32)))[each > 0].all(), (step, i)
            if (g != 0).any():
                moved.add(i)
    assert len(moved) > len(before) // 2  # the output layers start at zero, and with them the first step's other gradients
    tr.close()
