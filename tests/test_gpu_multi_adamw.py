"""MultiAdamW against the oracle's AdamW (32-bit states: bit for bit), a plain
fp32 restatement in numpy (8-bit states: bit for bit, codes and scales too) and
the formula in 64 bits."""
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


def to16(x, dtype):
    return torch.from_numpy(x).to(dtype).float().numpy()


def scalars(step):
    d = dict(b1=F(B1), o1=F(1 - B1), b2=F(B2), o2=F(1 - B2), c1=F(1 / (1 - B1 ** step)), c2=F(1 / (1 - B2 ** step)),
             decay=F(1 - LR * WD), lr=F(LR), eps=F(EPS))
    d["root"] = F(np.sqrt(1 / (1 - B2 ** step)))
    return d


def decode(codes, scale):
    c = codes.float().numpy()
    return c * np.repeat(scale, optim.BLOCK)[:len(c)]


def encode(x, floor):
    n = len(x)
    pad = np.zeros(-(-n // 256) * 256, F)
    pad[:n] = x
    b = pad.reshape(-1, 256)
    top = np.abs(b).max(1)
    scale = top * F(1 / 448)
    live = scale >= F(2.0 ** -126)
    factor = np.where(live, F(448) / np.where(top > 0, top, F(1)), F(0)).astype(F)
    q = np.clip(b * factor[:, None], F(-448), F(448))
    if floor:
        q = np.where((b > 0) & live[:, None], np.maximum(q, F(2.0 ** -9)), q)
    codes = torch.from_numpy(q.astype(F).reshape(-1)[:n]).to(torch.float8_e4m3fn)
    return codes, np.where(live, scale, F(0)).astype(F)


def step8(p, g, m, u, k):
    """One 8-bit step on fp32 numpy values: every operation rounds to fp32."""
    v = u * u
    m = m * k["b1"] + g * k["o1"]
    u = np.sqrt(v * k["b2"] + (g * g) * k["o2"])
    p = p * k["decay"] - ((m * k["c1"]) / (u * k["root"] + k["eps"])) * k["lr"]
    return p, m, u


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
def test_types_against_fp32_and_64_bits(ptype, gtype, offset, bits):
    ps, gs = tensors(SIZES, ptype, 3), tensors(SIZES, gtype, 4, 0.1)
    cs = [torch.zeros(n, dtype=torch.bfloat16) for n in SIZES]
    p, _ = placed(ps, offset)
    g, _ = placed(gs, offset)
    c, _ = placed(cs, offset)
    opt = MultiAdamW(p, g, lr=LR, weight_decay=WD, state_bits=bits, copies=c, no_decay=[i % 2 == 1 for i in range(len(SIZES))])
    now = [t.float().numpy() for t in ps]
    if bits == 8:
        st = [(torch.zeros(n, dtype=torch.float8_e4m3fn), np.zeros(-(-n // 256), F)) for n in SIZES]
        st = [[a, (a[0].clone(), a[1].copy())] for a in st]
    else:
        st = [[np.zeros(n, F), np.zeros(n, F)] for n in SIZES]
    for step in (1, 2, 3):
        opt.step()
        k = scalars(step)
        for i, n in enumerate(SIZES):
            ki = dict(k, decay=F(1)) if i % 2 else k
            gg = gs[i].float().numpy()
            if bits == 8:
                m0, u0 = decode(*st[i][0]), decode(*st[i][1])
                new, m, u = step8(now[i], gg, m0, u0, ki)
                v0, v = u0.astype(np.float64) ** 2, None
                st[i] = [encode(m, False), encode(u, True)]
            else:
                m0, v0 = st[i]
                m = m0 * k["b1"] + gg * k["o1"]
                v = v0 * k["b2"] + (gg * gg) * k["o2"]
                new = now[i] * ki["decay"] - ((m * k["c1"]) / (np.sqrt(v * k["c2"]) + k["eps"])) * k["lr"]
                st[i] = [m, v]
            # the formula in 64 bits: m' and v' carry 4 roundings (the constants' among them), the step 9 more
            d = lambda x: np.asarray(x, np.float64)  # noqa: E731
            m64 = B1 * d(m0) + (1 - B1) * d(gg)
            v64 = B2 * d(v0) + (1 - B2) * d(gg) ** 2
            den = np.sqrt(v64 / (1 - B2 ** step)) + EPS
            move = LR * m64 / (1 - B1 ** step) / den
            p64 = d(now[i]) * (1.0 if i % 2 else 1 - LR * WD) - move
            e_m = 4 * EPS32 * (np.abs(B1 * d(m0)) + np.abs((1 - B1) * d(gg))) + 2.0 ** -149
            bound = 4 * EPS32 * np.abs(d(now[i])) + LR / (1 - B1 ** step) * e_m / den + 14 * EPS32 * np.abs(move) + 2.0 ** -149
            assert (np.abs(new - p64) <= bound).all()
            now[i] = to16(new, ptype) if ptype != torch.float32 else new
            rounded = torch.from_numpy(new).to(torch.bfloat16)
            assert torch.equal(c[i].cpu(), rounded), (n, step)
    for i, n in enumerate(SIZES):
        assert np.array_equal(p[i].float().cpu().numpy(), now[i]), n
        if bits == 8:
            for name, (codes, scale) in zip("mv", st[i]):
                assert torch.equal(opt.state[name][i].cpu().view(torch.uint8), codes.view(torch.uint8)), (n, name)
                assert np.array_equal(opt.state[name + "_scale"][i].cpu().numpy(), scale), (n, name)
        else:
            assert np.array_equal(opt.state["m"][i].cpu().numpy(), st[i][0])
            assert np.array_equal(opt.state["v"][i].cpu().numpy(), st[i][1])


def test_8_bit_states_hold_the_moments_to_half_a_code():
    """|stored - m'| <= half a step of e4m3 (2^-4 of the value, 2^-10 of the scale below the normal codes); a root
    moment above zero stays above zero."""
    n = 100_000
    g = (torch.randn(n, generator=torch.Generator().manual_seed(5)) ** 5).float()
    g[::7] = 0
    p, gd = torch.zeros(n, device=DEV), g.to(DEV)
    opt = MultiAdamW([p], [gd], state_bits=8)
    opt.step()
    s = {k: v[0].cpu() for k, v in opt.state.items()}
    for name, want in (("m", g.double() * (1 - B1)), ("v", g.double().abs() * np.sqrt(1 - B2))):
        scale = s[name + "_scale"].double().repeat_interleave(256)[:n]
        got = s[name].double() * scale
        tol = torch.maximum(want.abs() * 2.0 ** -4, scale * 2.0 ** -10) * (1 + 2.0 ** -20)
        if name == "v":
            # The squares are fp32: below its normal range the two products are off by up to 2^-150 each, so v' by at
            # most 2^-148 with the sum's own rounding, and |sqrt a - sqrt b| <= sqrt |a - b| <= 2^-74; v' above
            # 2^-126 (u' above 2^-63) stays above zero.
            tol = torch.where((want > 0) & (want < scale * 2.0 ** -9), scale * 2.0 ** -9, tol) + 2.0 ** -74
            assert (got[want > 2.0 ** -62] > 0).all()
        assert ((got - want).abs() <= tol).all()
        assert (got[want == 0] == 0).all()


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
    k = scalars(1)
    for i, n in enumerate(sizes):
        if n == 0:
            continue
        z = np.zeros(n, F)
        if bits == 8:
            want, _, _ = step8(ps[i].numpy(), gs[i].numpy(), z, z, k)
        else:
            want, m, v = ps[i].numpy().copy(), z.copy(), z.copy()
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
