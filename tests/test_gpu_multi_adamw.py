"""MultiAdamW against the oracle's AdamW (fp32 throughout: bit for bit) and the
formula in 64 bits (every type, both forms of the states)."""
import numpy as np
import pytest
import torch

import oracle
from chineseai_b200 import optim
from chineseai_b200.optim import MultiAdamW

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
F = np.float32
EPS32 = 2.0 ** -24
SIZES = [1, 2, 3, 4, 5, 31, 127, 128, 129, 255, 256, 257, 1000, 1024, 4095, 4096, 4097, 20011]
LR, B1, B2, EPS, WD = 3e-3, 0.9, 0.999, 1e-8, 0.01


def tensors(sizes, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale).to(dtype) for n in sizes]


def placed(ts, offset):
    """Device copies, each `offset` elements into a buffer of its own, with the buffers."""
    out, bufs = [], []
    for t in ts:
        b = torch.full((t.numel() + 2 * offset + 8,), 3.0, device=DEV).to(t.dtype)
        v = b[offset:offset + t.numel()]
        v.copy_(t)
        out.append(v)
        bufs.append(b)
    return out, bufs


def f64(x):
    return (x.float() if isinstance(x, torch.Tensor) else x).cpu().double().numpy()


def held(codes, scale):
    """The values that 8-bit codes and their blocks' scales stand for, in 64 bits."""
    return f64(codes) * np.repeat(f64(scale), optim.BLOCK)[:codes.numel()]


def check_codes(codes, scale, want, rel, root):
    """`codes` and `scale` hold `want` (64 bits; the kernel's fp32 value is off by at most `rel` of its parts):
    the scale is max / 448 and each value within half a step of e4m3 (2^-4 of it, 2^-10 of the scale below the normal
    codes), widened by `rel` and three fp32 roundings; a root moment above zero stays above zero."""
    n = len(want)
    pad = np.zeros(-(-n // 256) * 256)
    pad[:n] = np.abs(want)
    err = np.zeros_like(pad)
    err[:n] = rel
    top, slack = pad.reshape(-1, 256).max(1), err.reshape(-1, 256).max(1)
    s = f64(scale)
    live = top / 448 > 2.0 ** -125
    assert (np.abs(s - top / 448)[live] <= (slack / 448 + 2 * EPS32 * top / 448)[live]).all()
    assert (s[top / 448 < 2.0 ** -127] == 0).all()
    each = np.repeat(s, 256)[:n]
    got = held(codes, scale)
    tol = np.maximum(np.abs(want) * 2.0 ** -4, each * 2.0 ** -10) * (1 + 2.0 ** -18) + 2 * rel + 2.0 ** -117
    if root:
        tol = np.where((want > 0) & (want < each * 2.0 ** -9), np.maximum(tol, each * 2.0 ** -9), tol)
        assert (got[(want > 2.0 ** -62) & (each > 0)] > 0).all()
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)
    assert (got[want == 0] == 0).all()


def expect(p, g, m, u, v, step, decay, eight):
    """(p', m', u' or v', bound of p', bound of m', bound of u' or v') of the formula in 64 bits.  m' and v' carry up to 5
    roundings of their parts (the constants' among them), the root and the quotient 2^-22 each in the 8-bit form, the
    step 10 roundings more, p' three."""
    v = u * u if eight else v
    m1 = B1 * m + (1 - B1) * g
    v1 = B2 * v + (1 - B2) * g * g
    e_m = 5 * EPS32 * (np.abs(B1 * m) + np.abs((1 - B1) * g)) + 2.0 ** -148
    den = np.sqrt(v1 / (1 - B2 ** step)) + EPS
    move = LR * m1 / (1 - B1 ** step) / den
    p1 = p * (1 - LR * WD if decay else 1.0) - move
    hard = 2.0 ** -21 if eight else 0.0
    e_p = 4 * EPS32 * np.abs(p) + LR / (1 - B1 ** step) * e_m / den + (16 * EPS32 + hard) * np.abs(move) + 2.0 ** -148
    if eight:  # v1 off by 2^-126 where it is flushed or leaves the normal range: its root by 2^-63
        u1 = np.sqrt(v1)
        return p1, m1, u1, e_p + LR * np.abs(m1) / (1 - B1 ** step) / den ** 2 * 2.0 ** -62, e_m, u1 * (8 * EPS32 + 2.0 ** -22) + 2.0 ** -62
    return p1, m1, v1, e_p, e_m, 8 * EPS32 * v1 + 2.0 ** -148


@pytest.mark.parametrize("offset", [0, 1, 4])
def test_32_bit_states_equal_the_flat_optimizer(offset):
    ps, gs = tensors(SIZES, torch.float32, 1), tensors(SIZES, torch.float32, 2, 0.1)
    p, bufs = placed(ps, offset)
    g, _ = placed(gs, offset)
    opt = MultiAdamW(p, g, lr=LR, weight_decay=WD)
    ref = [(a.numpy().copy(), np.zeros(a.numel(), F), np.zeros(a.numel(), F)) for a in ps]
    for step in (1, 2, 3):
        opt.step()
        for (rp, rm, rv), gg in zip(ref, gs):
            oracle.adamw(rp, rm, rv, gg.numpy(), LR, B1, B2, EPS, WD, step)
    for i, (rp, rm, rv) in enumerate(ref):
        assert np.array_equal(p[i].cpu().numpy(), rp), SIZES[i]
        assert np.array_equal(opt.state["m"][i].cpu().numpy(), rm) and np.array_equal(opt.state["v"][i].cpu().numpy(), rv)
        b = bufs[i].cpu()
        assert (b[:offset] == 3).all() and (b[offset + SIZES[i]:] == 3).all(), "wrote outside the tensor"
    assert opt.step_count == 3


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1, 4])
@pytest.mark.parametrize("ptype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gtype", [torch.float32, torch.bfloat16, torch.float16])
def test_types_against_64_bits(ptype, gtype, offset, bits):
    """Three steps, each against the formula from the state before it; 16-bit parameters and copies round once."""
    ps, gs = tensors(SIZES, ptype, 3), tensors(SIZES, gtype, 4, 0.1)
    p, pb = placed(ps, offset)
    g, _ = placed(gs, offset)
    c, cb = placed([torch.zeros(n, dtype=torch.bfloat16) for n in SIZES], offset)
    opt = MultiAdamW(p, g, lr=LR, weight_decay=WD, state_bits=bits, copies=c, no_decay=[i % 2 == 1 for i in range(len(SIZES))])
    st = opt.state
    for step in (1, 2, 3):
        before = []
        for i in range(len(SIZES)):
            if bits == 8:
                m, u = (held(st[k][i], st[k + "_scale"][i]) for k in "mv")
                before.append((f64(p[i]), f64(g[i]), m, u, None))
            else:
                before.append((f64(p[i]), f64(g[i]), f64(st["m"][i]), None, f64(st["v"][i])))
        opt.step()
        for i, n in enumerate(SIZES):
            p1, m1, s1, e_p, e_m, e_s = expect(*before[i], step, i % 2 == 0, bits == 8)
            half = torch.finfo(ptype).eps / 2 if ptype != torch.float32 else 0.0
            tiny = torch.finfo(ptype).smallest_normal * torch.finfo(ptype).eps / 2
            assert (np.abs(f64(p[i]) - p1) <= e_p + half * (np.abs(p1) + e_p) + tiny).all(), (n, step)
            assert (np.abs(f64(c[i]) - p1) <= e_p + 2.0 ** -8 * (np.abs(p1) + e_p) + 2.0 ** -134).all(), (n, step)
            if ptype != torch.float16:
                assert torch.equal(c[i], p[i].to(torch.bfloat16)), "the copy is the rounded parameter"
            if bits == 8:
                check_codes(st["m"][i], st["m_scale"][i], m1, e_m, False)
                check_codes(st["v"][i], st["v_scale"][i], s1, e_s, True)
            else:
                assert (np.abs(f64(st["m"][i]) - m1) <= e_m).all() and (np.abs(f64(st["v"][i]) - s1) <= e_s).all()
    for bufs in (pb, cb):
        for b, n in zip(bufs, SIZES):
            assert (b[:offset] == 3).all() and (b[offset + n:] == 3).all(), "wrote outside the tensor"


def test_8_bit_results_do_not_depend_on_the_alignment():
    ps, gs = tensors(SIZES, torch.float32, 20), tensors(SIZES, torch.bfloat16, 21)
    got = []
    for offset in (0, 1):
        p, _ = placed(ps, offset)
        g, _ = placed(gs, offset)
        opt = MultiAdamW(p, g, state_bits=8)
        opt.step()
        opt.step()
        got.append(torch.cat([t.reshape(-1).float() for t in p + [x for v in opt.state.values() for x in v]]))
    assert torch.equal(*got)


def test_8_bit_states_hold_a_wide_range_of_moments():
    n = 100_000
    g = (torch.randn(n, generator=torch.Generator().manual_seed(5)) ** 5).float()
    g[::7] = 0
    p, gd = torch.zeros(n, device=DEV), g.to(DEV)
    opt = MultiAdamW([p], [gd], lr=LR, weight_decay=WD, state_bits=8)
    opt.step()
    z = np.zeros(n)
    p1, m1, u1, e_p, e_m, e_u = expect(z, f64(g), z, z, None, 1, True, True)
    check_codes(opt.state["m"][0], opt.state["m_scale"][0], m1, e_m, False)
    check_codes(opt.state["v"][0], opt.state["v_scale"][0], u1, e_u, True)
    # where the root moment is below fp32's reach (2^-63) the bound of the step says nothing
    assert (np.abs(f64(p) - p1) <= e_p)[(u1 > 2.0 ** -55) | (u1 == 0)].all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [1, 15, 16, 17, 383, 384, 385, 1000])
def test_many_tensors(count, bits):
    """More tensors than one launch carries, empty ones among them."""
    sizes = [(i * 37) % 300 for i in range(count)]
    sizes[0] = 5000
    ps, gs = tensors(sizes, torch.float32, 6), tensors(sizes, torch.float32, 7)
    p, g = [t.to(DEV) for t in ps], [t.to(DEV) for t in gs]
    opt = MultiAdamW(p, g, lr=LR, weight_decay=WD, state_bits=bits)
    opt.step()
    for i, n in enumerate(sizes):
        if n == 0:
            continue
        if bits == 8:
            z = np.zeros(n)
            p1, m1, u1, e_p, e_m, e_u = expect(f64(ps[i]), f64(gs[i]), z, z, None, 1, True, True)
            assert (np.abs(f64(p[i]) - p1) <= e_p).all(), i
            check_codes(opt.state["m"][i], opt.state["m_scale"][i], m1, e_m, False)
            check_codes(opt.state["v"][i], opt.state["v_scale"][i], u1, e_u, True)
        else:
            want, m, v = ps[i].numpy().copy(), np.zeros(n, F), np.zeros(n, F)
            oracle.adamw(want, m, v, gs[i].numpy(), LR, B1, B2, EPS, WD, 1)
            assert np.array_equal(p[i].cpu().numpy(), want), i


@pytest.mark.parametrize("bits", [32, 8])
def test_skip_scale_learning_rate_and_state(bits):
    p = torch.randn(1000, device=DEV)
    g = torch.randn(1000, device=DEV)
    a, b = p.clone(), p.clone()
    half = (g * 2.0)
    x, y = MultiAdamW([a], [g], state_bits=bits), MultiAdamW([b], [half], state_bits=bits)
    flags = torch.zeros(3, device=DEV)
    for _ in range(3):
        x.step(skip=flags)
        y.step(grad_scale=0.5)
    assert torch.equal(a, b)
    before = a.clone(), [t.clone().view(torch.uint8) for v in x.state.values() for t in v]
    flags[2] = 1
    x.step(skip=flags)
    assert torch.equal(a, before[0])
    assert all(torch.equal(t.view(torch.uint8), u) for t, u in zip([t for v in x.state.values() for t in v], before[1]))
    # another object steps on from the state
    c = b.clone()
    z = MultiAdamW([c], [half], state_bits=bits, state={k: [t.clone() for t in v] for k, v in y.state.items()}, step=3, lr=0.5)
    z.set_learning_rate(1e-3)
    z.step(grad_scale=0.5)
    y.step(grad_scale=0.5)
    assert torch.equal(b, c) and z.step_count == 4


@pytest.mark.parametrize("bits", [32, 8])
def test_device_state_in_a_captured_graph(bits):
    sizes = [3, 700, 5000]
    ps, gs = tensors(sizes, torch.float32, 8), tensors(sizes, torch.bfloat16, 9)
    p, g = [t.to(DEV) for t in ps], [t.to(DEV) for t in gs]
    q = [t.to(DEV) for t in ps]
    host = MultiAdamW(q, g, lr=LR, weight_decay=WD, state_bits=bits)
    opt = MultiAdamW(p, g, lr=LR, weight_decay=WD, state_bits=bits, device_state=True)
    skip = torch.zeros(1, device=DEV)
    opt.step(skip=skip)
    host.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(skip=skip)
    for i in range(3):
        for t in g:
            t.mul_(-0.5)
        graph.replay()
        host.step()
    assert all(torch.equal(a, b) for a, b in zip(p, q)) and opt.step_count == 4
    skip.fill_(1)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(p, q)) and opt.step_count == 4
    skip.zero_()
    opt.set_learning_rate(0.25)
    host.set_learning_rate(0.25)
    graph.replay()
    host.step()
    assert all(torch.equal(a, b) for a, b in zip(p, q)) and opt.step_count == 5


def test_a_block_with_a_nan_becomes_one_and_the_others_do_not():
    n = 1024
    g = torch.ones(n, device=DEV)
    g[300] = float("nan")
    g[600] = float("inf")
    p = torch.zeros(n, device=DEV)
    opt = MultiAdamW([p], [g], state_bits=8, lr=LR)
    opt.step()
    m, ms = opt.state["m"][0].float().cpu(), opt.state["m_scale"][0].cpu()
    assert not torch.isfinite(ms[1]) and not torch.isfinite(ms[2]) and torch.isfinite(ms[[0, 3]]).all()
    assert m[256:512].isnan().all() and torch.isfinite(m[:256]).all() and torch.isfinite(m[768:]).all()
    assert torch.isfinite(p[[0, 299, 301, 599, 601, 1023]]).all() and p[300].isnan()


def test_gradients_whose_square_overflows():
    """v' saturates: the step stays finite, and the rest of the block's root moments with it."""
    g = torch.full((512,), 1e-3, device=DEV)
    g[5] = 1e25
    p = torch.ones(512, device=DEV)
    opt = MultiAdamW([p], [g], state_bits=8, lr=LR, weight_decay=0.0)
    opt.step()
    opt.step()
    u = opt.state["v"][0].float() * opt.state["v_scale"][0].repeat_interleave(256)
    assert torch.isfinite(p).all() and torch.isfinite(u).all() and u[5] > 1e19


def test_a_tensor_of_more_than_two_to_the_31_elements():
    n, tail = 2 ** 31 + 777, 2000
    small_p = torch.randn(tail, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    small_g = torch.randn(tail, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    off = (n - tail) % 256  # the same blocks of 256 at the end of both
    p, g = torch.zeros(n, dtype=torch.bfloat16, device=DEV), torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    q, h = torch.zeros(off + tail, dtype=torch.bfloat16, device=DEV), torch.zeros(off + tail, dtype=torch.bfloat16, device=DEV)
    for t, v in ((p, small_p), (g, small_g), (q, small_p), (h, small_g)):
        t[-tail:] = v.to(DEV)
    for bits in (8, 32):
        a, b = MultiAdamW([p], [g], state_bits=bits), MultiAdamW([q], [h], state_bits=bits)
        a.step()
        b.step()
        assert torch.equal(p[-tail:], q[-tail:]) and not p[:4096].any()
        assert torch.equal(a.state["m"][0][-tail:].float(), b.state["m"][0][-tail:].float())
        del a


def test_tiny_and_zero_blocks():
    g = torch.zeros(768, device=DEV)
    g[256:512] = 1e-38
    g[512] = 1e-30
    p = torch.ones(768, device=DEV)
    opt = MultiAdamW([p], [g], state_bits=8, lr=LR, weight_decay=0.0)
    opt.step()
    assert (opt.state["m_scale"][0][:2] == 0).all() and not opt.state["m"][0].float()[:512].any()
    assert (p[:256] == 1).all() and torch.isfinite(p).all()


def test_refusals():
    p, g = torch.zeros(8, device=DEV), torch.zeros(8, device=DEV)
    for args, kw in [(([p, p], [g, g]), {}), (([p], [p]), {}), (([p[:6], p[4:]], [g[:6], g[4:]]), {}),
                     (([p], [g]), dict(copies=[p.view(torch.bfloat16)[:8]])),
                     (([p], [g, g]), {}), (([p], [g[:4]]), {}), (([p[::2]], [g[:4]]), {}), (([p], [g.cpu()]), {}),
                     (([p], [g]), dict(state={"m": [p]})), (([p], [g]), dict(state={"m": [torch.zeros_like(p)], "v": [g]})),
                     (([p], [g]), dict(copies=[None, None]))]:
        with pytest.raises(ValueError):
            MultiAdamW(*args, **kw)
    for args, kw in [(([p.double()], [g]), {}), (([p], [g.int()]), {}), (([p], [g]), dict(copies=[torch.zeros_like(p)])),
                     (([p], [g]), dict(state_bits=8, state={k: [torch.zeros(8, device=DEV)] for k in
                                                            ("m", "v", "m_scale", "v_scale")}))]:
        with pytest.raises(TypeError):
            MultiAdamW(*args, **kw)
    opt = MultiAdamW([p], [g])
    with pytest.raises(ValueError):
        opt.step(skip=torch.zeros(1))
    shared = MultiAdamW([p, torch.zeros(8, device=DEV)], [g, g])  # one gradient buffer read twice is fine
    shared.step()


def test_results_do_not_change_from_run_to_run():
    got = []
    for _ in range(2):
        ps, gs = tensors([70_000, 333], torch.bfloat16, 10), tensors([70_000, 333], torch.bfloat16, 11)
        p, g = [t.to(DEV) for t in ps], [t.to(DEV) for t in gs]
        opt = MultiAdamW(p, g, state_bits=8)
        for _ in range(4):
            opt.step()
        got.append(torch.cat([t.float() for t in p] + [t.float() for t in opt.state["v"]]))
    assert torch.equal(*got)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("native", [True, False])
def test_az_trainer_with_8_bit_states(native, graph):
    """The first step from zero moments is the 32-bit trainer's (the update comes before the rounding, and root and
    quotient are good to 2^-21 of the step); later steps stay near it, replayed or not; a bad batch changes nothing."""
    from chineseai_b200 import az, az_train
    from chineseai_b200._lib import CnnueError
    w = az.AzWeights.random(32, 7)
    batch = az_train.pack_batch(az_train.random_samples(48, 5), caps=(96, 160, 256), fixed=True)
    a = az_train.AzTrainer(w, lr=LR, graph=graph, native=native)
    b = az_train.AzTrainer(w, lr=LR, graph=graph, native=native, state_bits=8)
    start = a.flat.clone()
    sa, sb = a.step(batch), b.step(batch)
    assert sa.loss == sb.loss or not native
    move = (a.flat - start).abs()
    # gradients of the autograd path may differ by their summation; the native step's are the same bits
    if native:
        assert ((a.flat - b.flat).abs() <= 4 * EPS32 * start.abs() + (2.0 ** -20 + 16 * EPS32) * move + 2.0 ** -140).all()
    for _ in range(3):
        sa, sb = a.step(batch), b.step(batch)
    assert b.optimizer.step_count == 4 and torch.isfinite(b.flat).all()
    # with nearly constant gradients each of the 3 later steps moves a parameter by about lr, on either side by moments
    # that are good to 2^-4 each (m over its root)
    assert (a.flat - b.flat).abs().max() < 3 * LR * (1 + (1 + 2.0 ** -4) / (1 - 2.0 ** -4)) * 1.01
    before = b.flat.clone()
    bad = az_train.pack_batch(az_train.random_samples(48, 5), caps=(96, 160, 256), fixed=True)
    bad.feature_items[3, 0] = 1700
    with pytest.raises(CnnueError):
        b.step(bad)
    assert torch.equal(b.flat, before) and b.optimizer.step_count == 4
    if native:
        with pytest.raises(ValueError, match="state_bits"):
            b.native_loss(b.to_device(batch), adamw=True)
    b.set_learning_rate(0.0)
    b.step(batch)
    assert torch.equal(b.flat, before * 1.0) and b.optimizer.step_count == 5
    a.close()
    b.close()
