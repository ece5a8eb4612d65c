"""process_logits, policy_loss and policy_loss_grad against plain 64-bit forms
(tests/_logitsref.py), at the sizes, types, strides and masks where rows,
slices and vectors end."""
import math
import threading

import numpy as np
import pytest
import torch

from tests import _logitsref as ref
from chineseai_b200 import logits as lg
from chineseai_b200._lib import CnnueError

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [(1, 1), (3, 2), (5, 7), (2, 8), (4, 31), (3, 33), (7, 2086), (2, 8100), (3, 8192), (2, 8193), (2, 50001)]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def dev(x):
    return None if x is None else x.to(DEV)


def rows(r, v, dtype, g, pad=0, offset=0):
    """[r, v] logits inside a larger buffer: row stride v + pad, `offset` elements in."""
    buf = torch.randn(offset + r * (v + pad) + 16, generator=g) * 3
    return buf.to(dtype)[offset:offset + r * (v + pad)].view(r, v + pad)[:, :v]


def to_dev_strided(x, pad, offset):
    """x on the device with the same padding and offset."""
    r, v = x.shape
    buf = torch.full((offset + r * (v + pad) + 16,), 77.0, dtype=x.dtype, device=DEV)
    y = buf[offset:offset + r * (v + pad)].view(r, v + pad)[:, :v]
    y.copy_(x)
    return y, buf


def history_of(r, v, n, g, dtype=torch.int32):
    h = (torch.rand(r, n, generator=g) ** 3 * v).long().clamp(0, v - 1)
    h[torch.rand(r, n, generator=g) < 0.05] = -1
    return h.to(dtype)


def mask_of(r, v, share, g):
    return lg.pack_mask(torch.rand(r, v, generator=g) < share)


# ---- process_logits -------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_process_sizes(size, dtype):
    R, V = size
    g = gen(V * 7 + R)
    x = rows(R, V, dtype, g)
    kw = dict(history=history_of(R, V, 37, g), lengths=torch.randint(0, 38, (R,), generator=g).int(),
              prompt_lengths=torch.randint(0, 30, (R,), generator=g).int(), repetition=1 + torch.rand(R, generator=g),
              frequency=torch.rand(R, generator=g), presence=torch.rand(R, generator=g) - 0.5,
              bias_tokens=torch.randint(-1, V, (R, 9), generator=g).int(), bias_values=torch.randn(R, 9, generator=g),
              mask=mask_of(R, V, 0.6, g))
    out = lg.process_logits(dev(x), **{k: dev(t) for k, t in kw.items()})
    assert out.dtype == dtype
    want, bound = ref.process(x, **kw)
    ref.close(out, want, bound, dtype)


@pytest.mark.parametrize("part", ["none", "history", "bias", "mask", "history+mask", "bias+mask", "history+bias"])
@pytest.mark.parametrize("dtype", TYPES)
def test_process_parts(part, dtype):
    R, V = 5, 2086
    g = gen(len(part))
    x = rows(R, V, dtype, g)
    kw = {}
    if "history" in part:
        kw.update(history=history_of(R, V, 300, g, torch.int64), repetition=0.5 + torch.rand(R, generator=g))
    if "bias" in part:
        kw.update(bias_tokens=torch.randperm(V, generator=g)[:40].int(), bias_values=torch.randn(40, generator=g))
    if "mask" in part:
        kw.update(mask=mask_of(1, V, 0.02, g)[0])
    out = lg.process_logits(dev(x), out_dtype=torch.float32, **{k: dev(t) for k, t in kw.items()})
    want, bound = ref.process(x, **kw)
    ref.close(out, want, bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,offset", [(0, 1), (3, 0), (5, 3), (8, 8)])
def test_process_strides_in_place_and_neighbours(pad, offset, dtype):
    R, V = 6, 1003
    g = gen(pad * 10 + offset)
    x = rows(R, V, dtype, g)
    kw = dict(history=history_of(R, V, 50, g), frequency=torch.rand(R, generator=g), mask=mask_of(3, V, 0.5, g),
              mask_index=torch.tensor([2, -1, 0, 1, -5, 2], dtype=torch.int32))
    want, bound = ref.process(x, **kw)
    d = {k: dev(t) for k, t in kw.items()}
    y, buf = to_dev_strided(x, pad, offset)
    before = buf.clone()
    ref.close(lg.process_logits(y, **d), want, bound, dtype)
    assert torch.equal(buf, before), "the logits were written"
    o, obuf = to_dev_strided(torch.zeros(R, V, dtype=dtype), pad + 1, 2)
    marks = obuf.clone()
    lg.process_logits(y, out=o, **d)
    ref.close(o, want, bound, dtype)
    o.copy_(marks[2:2 + R * (V + pad + 1)].view(R, -1)[:, :V])
    assert torch.equal(obuf, marks), "wrote outside the rows"
    assert lg.process_logits(y, out=y, **d) is y
    ref.close(y, want, bound, dtype)
    y.copy_(x)
    assert torch.equal(buf, before), "in place: wrote outside the rows"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [100, 2086, 16_384, 16_385, 40_001])
def test_process_in_place_with_penalties_biases_and_masks_rounds_once(vocab, dtype):
    """The same bits as out of place: biased tokens among the penalised ones, repeated, masked."""
    g = gen(vocab)
    R = 4
    x = rows(R, vocab, dtype, g)
    h = history_of(R, vocab, 200, g)
    kw = dict(history=h, repetition=1 + torch.rand(R, generator=g), frequency=torch.rand(R, generator=g),
              bias_tokens=torch.cat([h[:, :20], h[:, 5:10], torch.randint(0, vocab, (R, 10), generator=g).int()], 1),
              bias_values=torch.randn(R, 35, generator=g), mask=mask_of(R, vocab, 0.8, g))
    d = {k: dev(t) for k, t in kw.items()}
    out = lg.process_logits(dev(x), **d)
    want, bound = ref.process(x, **kw)
    ref.close(out, want, bound, dtype)
    y = dev(x).clone()
    lg.process_logits(y, out=y, **d)
    assert torch.equal(y, out)


def test_process_broadcast_row_and_transposed_logits():
    g = gen(5)
    x = rows(1, 500, torch.float32, g)
    m = mask_of(4, 500, 0.5, g)
    want, bound = ref.process(x.expand(4, -1), mask=m)
    ref.close(lg.process_logits(dev(x).expand(4, -1), mask=dev(m)), want, bound)
    want, bound = ref.process(x.expand(4, -1), mask=m[:1].expand(4, -1))
    ref.close(lg.process_logits(dev(x).expand(4, -1), mask=dev(m)[:1].expand(4, -1)), want, bound)
    t = torch.randn(500, 4, generator=g)
    want, bound = ref.process(t.t(), mask=m)
    ref.close(lg.process_logits(dev(t).t(), mask=dev(m)), want, bound)


@pytest.mark.parametrize("dtype", TYPES)
def test_process_extremes(dtype):
    """Infinities, NaN, the type's lowest value, in allowed and masked places; a row that allows nothing."""
    V = 70
    lowest = torch.finfo(dtype).min
    x = torch.zeros(4, V, dtype=dtype)
    x[:, :6] = torch.tensor([math.inf, -math.inf, math.nan, lowest, -0.0, 1.0]).to(dtype)
    a = torch.ones(4, V, dtype=torch.bool)
    a[1] = False
    a[2, :4] = False
    a[3] = False
    a[3, 69] = True
    h = torch.tensor([0, 1, 2, 3, 4, 5], dtype=torch.int32)
    kw = dict(history=h, repetition=torch.full((4,), 2.0), mask=lg.pack_mask(a))
    out = lg.process_logits(dev(x), **{k: dev(t) for k, t in kw.items()}).cpu()
    assert (out[1] == -math.inf).all()
    assert (out[2, :4] == -math.inf).all() and (out[2, 6:] == 0).all()
    assert (out[3, :69] == -math.inf).all() and out[3, 69] == 0
    assert out[0, 0] == math.inf and out[0, 1] == -math.inf and math.isnan(out[0, 2]) and out[0, 5] == 0.5
    assert out[0, 3] == -math.inf or dtype == torch.float32 and out[0, 3] == torch.tensor(lowest) * 2


def test_process_repeated_bias_tokens_in_list_order():
    """1e8 + 1 - 1e8: the order of fp32 additions shows."""
    x = torch.zeros(1, 40)
    tok = torch.tensor([[3, 3, 5, 3, -1, 5, 39]], dtype=torch.int32)
    val = torch.tensor([[1e8, 1.0, 2.0, -1e8, 9.0, 0.5, 7.0]])
    out = lg.process_logits(dev(x), bias_tokens=dev(tok), bias_values=dev(val)).cpu()
    want = torch.zeros(1, 40)
    want[0, 3] = (torch.tensor(1e8) + 1.0) - 1e8
    want[0, 5], want[0, 39] = 2.5, 7.0
    assert torch.equal(out, want)


def test_process_one_token_many_times():
    V, L = 4096, 100_000
    x = torch.full((2, V), 1.0)
    h = torch.full((2, L), 17, dtype=torch.int64)
    kw = dict(history=dev(h), lengths=dev(torch.tensor([L, 1], dtype=torch.int32)),
              prompt_lengths=dev(torch.tensor([5, 1], dtype=torch.int32)), frequency=dev(torch.full((2,), 0.5)),
              presence=dev(torch.full((2,), 0.25)), repetition=dev(torch.full((2,), 2.0)))
    out = lg.process_logits(dev(x), **kw).cpu()
    assert out[0, 17] == 0.5 - 0.5 * (L - 5) - 0.25 and out[1, 17] == 0.5
    out[:, 17] = 1.0
    assert (out == 1.0).all()


def test_process_bad_data_is_reported_and_skipped():
    x = torch.ones(3, 50)
    h = torch.tensor([[1, 50, 2], [3, 2**31 - 1, 4], [5, 6, 7]], dtype=torch.int32)
    f = torch.ones(3)
    with pytest.raises(CnnueError, match="index"):
        lg.process_logits(dev(x), history=dev(h), frequency=dev(f))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    wide = h.long()
    wide[1, 1] = 2**40
    out = lg.process_logits(dev(x), history=dev(wide), frequency=dev(f), status=status).cpu()
    want = torch.ones(3, 50)
    for r, ts in enumerate(([1, 2], [3, 4], [5, 6, 7])):
        want[r, ts] = 0.0
    assert torch.equal(out, want) and int(status) == 1
    status.zero_()
    out = lg.process_logits(dev(x), history=dev(h[2:3].expand(3, 3).contiguous()), frequency=dev(f), status=status,
                            lengths=dev(torch.tensor([-1, 4, 1], dtype=torch.int32))).cpu()
    assert int(status) == 2
    assert (out[0] == 1).all() and (out[1, 5:8] == 0).all() and out[2, 5] == 0 and (out[2, 6:8] == 1).all()
    status.zero_()
    out = lg.process_logits(dev(x), bias_tokens=dev(torch.tensor([50, 4], dtype=torch.int32)),
                            bias_values=dev(torch.tensor([3.0, 1.0])), status=status).cpu()
    assert int(status) == 1 and out[0, 4] == 2 and out.sum() == 153
    status.zero_()
    m = lg.pack_mask(torch.ones(2, 50, dtype=torch.bool))
    out = lg.process_logits(dev(x), mask=dev(m), mask_index=dev(torch.tensor([0, 2, 1], dtype=torch.int32)),
                            status=status).cpu()
    assert int(status) == 1 and (out[1] == -math.inf).all() and (out[[0, 2]] == 1).all()


@pytest.mark.parametrize("count", [1, 500, 1500, 4000])
def test_process_long_bias_lists(count):
    """More entries than threads; more than a hash table holds; every token of the vocabulary named."""
    R, V = 2, 20_000
    g = gen(count)
    x = rows(R, V, torch.float32, g)
    tok = torch.stack([torch.randperm(V, generator=g)[:count] for _ in range(R)]).int()
    tok[0, count // 2:] = tok[0, 0]  # one token again and again
    kw = dict(bias_tokens=tok, bias_values=torch.randn(R, count, generator=g), history=tok.flip(1)[:, :1000],
              frequency=torch.ones(R), mask=mask_of(1, V, 0.7, g)[0])
    want, bound = ref.process(x, **kw)
    ref.close(lg.process_logits(dev(x), **{k: dev(t) for k, t in kw.items()}), want, bound)


def test_process_hash_neighbours_and_the_last_token():
    """Tokens that meet in a hash table, and the ends of a large vocabulary."""
    V, n = 1 << 20, 1000
    x = torch.ones(1, V)
    h = (torch.arange(n) * 1021 % V).int()
    h[-3:] = torch.tensor([V - 1, 0, V - 1])
    kw = dict(history=h, frequency=torch.ones(1))
    want, bound = ref.process(x, **kw)
    ref.close(lg.process_logits(dev(x), history=dev(h), frequency=dev(torch.ones(1))), want, bound)


def test_process_empty():
    assert lg.process_logits(torch.empty(0, 5, device=DEV)).shape == (0, 5)
    x = torch.ones(2, 9, device=DEV)
    none = torch.empty(2, 0, dtype=torch.int32, device=DEV)
    out = lg.process_logits(x, history=none, frequency=torch.ones(2, device=DEV), bias_tokens=none,
                            bias_values=torch.empty(2, 0, device=DEV))
    assert torch.equal(out, x)


@pytest.mark.parametrize("L", [1, 2047, 2048, 2049, 5000, 20_000, 32_767, 32_768, 60_000])
@pytest.mark.parametrize("dtype", TYPES)
def test_process_long_history_and_large_vocabulary(dtype, L):
    R, V = 3, 100_003
    g = gen(9)
    x = rows(R, V, dtype, g)
    kw = dict(history=history_of(R, V, L, g), frequency=torch.rand(R, generator=g), repetition=1 + torch.rand(R, generator=g),
              prompt_lengths=torch.tensor([0, L // 2, L], dtype=torch.int32),
              bias_tokens=torch.randint(0, V, (R, 300), generator=g).int(), bias_values=torch.randn(R, 300, generator=g),
              mask=mask_of(R, V, 0.9, g))
    want, bound = ref.process(x, **kw)
    ref.close(lg.process_logits(dev(x), **{k: dev(t) for k, t in kw.items()}), want, bound, dtype)


@pytest.mark.parametrize("V,L", [(2086, 64), (40_000, 64), (40_000, 4000)])
def test_process_captured_and_replayed_on_new_data(V, L):
    """One launch, and two that overlap (short and long histories); two graphs of the same buffers in turn."""
    g = gen(3)
    R = 4
    x, h, n = dev(rows(R, V, torch.float32, g)), dev(history_of(R, V, L, g)), dev(torch.full((R,), 10, dtype=torch.int32))
    f, m = dev(torch.rand(R, generator=g)), dev(mask_of(R, V, 0.5, g))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.empty_like(x)
    kw = dict(history=h, lengths=n, frequency=f, mask=m)
    lg.process_logits(x, out=out, status=status, **kw)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for graph in graphs:
        with torch.cuda.graph(graph):
            lg.process_logits(x, out=out, status=status, **kw)
    for k in (20, L):
        for graph in graphs:
            n.fill_(k)
            x.mul_(0.5)
            graph.replay()
            want, bound = ref.process(x.cpu(), **{k: t.cpu() for k, t in kw.items()})
            ref.close(out, want, bound)
    assert int(status) == 0


def test_process_calls_in_a_row_and_on_two_streams():
    """Calls that follow each other without a wait, the output of one the input of the next, and two streams at once."""
    g = gen(21)
    R, V = 8, 30_000
    x = rows(R, V, torch.bfloat16, g)
    h = history_of(R, V, 300, g)
    kw = dict(history=h, frequency=torch.rand(R, generator=g), mask=mask_of(R, V, 0.5, g))
    d = {k: dev(t) for k, t in kw.items()}
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    first = lg.process_logits(dev(x), **d).cpu()
    second = lg.process_logits(first.to(DEV), **d).cpu()
    third = lg.process_logits(second.to(DEV), **d).cpu()
    a = dev(x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                y = lg.process_logits(a, status=status, **d)
                y = lg.process_logits(y, status=status, **d)
                lg.process_logits(y, out=y, status=status, **d)
                got.append(y)
    torch.cuda.synchronize()
    assert all(torch.equal(y.cpu(), third) for y in got) and int(status) == 0


def test_process_on_another_stream():
    g = gen(4)
    x = rows(64, 8100, torch.float32, g)
    m = mask_of(64, 8100, 0.3, g)
    want, bound = ref.process(x, mask=m)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        out = lg.process_logits(x.to(DEV), mask=m.to(DEV), status=torch.zeros(1, dtype=torch.int32, device=DEV))
    s.synchronize()
    ref.close(out, want, bound)


# ---- policy_loss ------------------------------------------------------------------
def loss_inputs(R, V, dtype, kind, g, pad=0, share=0.5):
    x = rows(R, V, dtype, g, pad)
    kw = {}
    if kind == "dense":
        kw["targets"] = torch.rand(R, V, generator=g) ** 2
    elif kind == "dense16":
        kw["targets"] = (torch.rand(R, V, generator=g) ** 2).to(torch.bfloat16 if dtype != torch.float16 else dtype)
    elif kind == "labels":
        kw["target_index"] = torch.randint(-1 if R > 1 else 0, V, (R,), generator=g)
    else:
        kw["target_index"] = torch.randint(-1, V, (R, 17), generator=g).int()
        kw["target_prob"] = torch.rand(R, 17, generator=g)
    if share < 1:
        kw["mask"] = mask_of(R, V, share, g)
    kw["weights"] = torch.rand(R, generator=g) + 0.25
    return x, kw


def check_all(x, kw, dtype, up=None):
    """The fused form and autograd against the 64-bit form."""
    R = x.shape[0]
    d = {k: dev(t) for k, t in kw.items()}
    want, grad, b_loss, b_grad = ref.loss(x, **kw)
    loss, got = lg.policy_loss_grad(dev(x), d.pop("targets", None), **d)
    ref.close(loss, want, b_loss)
    ref.close(got, grad, b_grad, dtype)
    up = torch.linspace(-1, 2, R) if up is None else up
    _, grad, _, b_grad = ref.loss(x, **kw, upstream=up)
    leaf = dev(x).requires_grad_(True)
    d = {k: dev(t) for k, t in kw.items()}
    loss = lg.policy_loss(leaf, d.pop("targets", None), **d)
    ref.close(loss, want, b_loss)
    (got,) = torch.autograd.grad(loss, leaf, dev(up))
    ref.close(got, grad, b_grad, dtype)


@pytest.mark.parametrize("kind", ["dense", "dense16", "labels", "lists"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_loss_sizes(size, dtype, kind):
    g = gen(size[1] + size[0] * 3)
    x, kw = loss_inputs(*size, dtype, kind, g)
    check_all(x, kw, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_loss_large_vocabulary(dtype):
    g = gen(11)
    x, kw = loss_inputs(2, 140_001, dtype, "lists", g, share=1.0)
    check_all(x, kw, dtype)
    x, kw = loss_inputs(1, 300_007, dtype, "dense", g, share=0.9)
    check_all(x, kw, dtype)


@pytest.mark.parametrize("kind", ["dense", "labels"])
@pytest.mark.parametrize("size", [(2, 190_003), (20, 190_003), (2, 260_000), (20, 260_000), (1, 400_001), (1, 1_000_003)])
def test_loss_of_rows_kept_or_read_twice(size, kind):
    """fp32 rows at both sides of each limit of what a cluster keeps, few and many of them."""
    g = gen(size[1])
    x, kw = loss_inputs(*size, torch.float32, kind, g)
    d = {k: dev(t) for k, t in kw.items()}
    targets = d.pop("targets", None)
    loss, got = lg.policy_loss_grad(dev(x), targets, **d)
    one = slice(size[0] - 1, size[0])
    want, grad, bl, bg = ref.loss(x[one], **{k: t[one] for k, t in kw.items()})
    ref.close(loss[one], want, bl)
    ref.close(got[one], grad, bg)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,offset", [(0, 1), (3, 0), (5, 3)])
def test_loss_strides_and_neighbours(pad, offset, dtype):
    R, V = 5, 2087
    g = gen(pad + offset)
    x, kw = loss_inputs(R, V, dtype, "dense", g)
    want, grad, b_loss, b_grad = ref.loss(x, **kw)
    d = {k: dev(t) for k, t in kw.items()}
    y, _ = to_dev_strided(x, pad, offset)
    t, _ = to_dev_strided(kw["targets"], 1, 3)
    d.pop("targets")
    o, obuf = to_dev_strided(torch.zeros(R, V, dtype=dtype), pad, 2)
    marks = obuf.clone()
    loss, got = lg.policy_loss_grad(y, t, grad=o, **d)
    assert got is o
    ref.close(loss, want, b_loss)
    ref.close(o, grad, b_grad, dtype)
    o.copy_(marks[2:2 + R * (V + pad)].view(R, -1)[:, :V])
    assert torch.equal(obuf, marks), "wrote outside the gradient"


@pytest.mark.parametrize("dtype", TYPES)
def test_loss_of_a_common_offset_keeps_its_digits(dtype):
    g = gen(2)
    x = (torch.randn(3, 2086, generator=g) + 1000).to(dtype)
    check_all(x, {"target_index": torch.tensor([5, 0, 2085]), "mask": mask_of(3, 2086, 0.9, g) | -1}, dtype)


@pytest.mark.parametrize("offset", [3e4, 65530.0, 1e6, -65530.0, -1e7, 1e10, -1e12, 1e20, -1e30, 2e37])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loss_of_large_logits(offset, dtype):
    """Logits around any size, with steps of their type's own spacing and rows that reach across sizes."""
    g = gen(23)
    step = abs(offset) * torch.finfo(dtype).eps
    x = (offset + torch.randint(-3, 4, (4, 900), generator=g).double() * step).to(dtype)
    x[1, ::3] = 0.0  # far below or above the others
    x[2, 5:] = torch.finfo(dtype).min
    x[3] = torch.linspace(-1, 1, 900) * 70000 if abs(offset) < 1e8 else x[3]
    check_all(x, {"target_index": torch.tensor([[5, 7], [0, 1], [3, 899], [898, 4]]), "target_prob": torch.rand(4, 2, generator=g)},
              dtype)


@pytest.mark.parametrize("kind", ["dense", "labels", "lists"])
@pytest.mark.parametrize("dtype", TYPES)
def test_loss_rows_where_little_or_nothing_is_left(kind, dtype):
    """Nothing allowed; only -inf allowed; NaN and infinities in masked places; weight 0 over NaN; the lowest value;
    one token; no target; targets all masked."""
    R, V = 10, 1000
    g = gen(6)
    x, kw = loss_inputs(R, V, dtype, kind, g, share=2.0)
    lowest = torch.finfo(dtype).min
    a = torch.rand(R, V, generator=g) < 0.5
    a[:, 7] = True
    a[0] = False
    x[1] = -math.inf
    x[2][~a[2]] = math.nan
    x[3][~a[3]] = math.inf
    x[4] = math.nan
    kw["weights"][4] = 0.0
    x[5] = lowest
    a[6] = False
    a[6, 7] = True
    if kind == "dense":
        kw["targets"][7] = 0.0
        kw["targets"][8] = torch.where(a[8], 0.0, kw["targets"][8])
        kw["targets"][2][~a[2]] = math.nan
    else:
        kw["target_index"][7] = -1
        kw["target_index"][8] = int((~a[8]).nonzero()[0])
    kw["mask"] = lg.pack_mask(a)
    if kind == "dense":  # the plain form multiplies: give it zeros where the operator must not look
        clean = dict(kw, targets=torch.where(a, kw["targets"], 0.0))
    else:
        clean = kw
    want, grad, b_loss, b_grad = ref.loss(torch.where(a, x, torch.zeros((), dtype=dtype)), **clean)
    d = {k: dev(t) for k, t in kw.items()}
    loss, got = lg.policy_loss_grad(dev(x), d.pop("targets", None), **d)
    ref.close(loss, want, b_loss)
    ref.close(got, grad, b_grad, dtype)
    for r in (0, 1, 4, 7, 8):
        assert float(loss[r]) == 0 and not got[r].any()
    leaf = dev(x).requires_grad_(True)
    d = {k: dev(t) for k, t in kw.items()}
    loss = lg.policy_loss(leaf, d.pop("targets", None), **d)
    ref.close(loss, want, b_loss)
    loss.sum().backward()
    ref.close(leaf.grad, grad, b_grad, dtype)


def test_loss_nan_and_infinite_logits_at_allowed_tokens():
    x = torch.zeros(4, 64)
    x[0, 3] = math.nan
    x[1, 3] = math.inf
    x[2, 3] = -math.inf  # no target there
    x[3, 5] = -math.inf  # a target there
    label = torch.tensor([5, 5, 5, 5])
    loss, grad = lg.policy_loss_grad(dev(x), target_index=dev(label))
    loss, grad = loss.cpu(), grad.cpu()
    assert math.isnan(loss[0]) and grad[0].isnan().all()
    assert math.isnan(loss[1]) or loss[1] == math.inf
    assert abs(float(loss[2]) - math.log(63)) < 1e-6 and grad[2, 3] == 0
    assert loss[3] == math.inf and grad[3, 5] == -1 and abs(float(grad[3, 0]) - 1 / 63) < 1e-7


def test_loss_masses_other_than_one_and_repeated_tokens():
    g = gen(8)
    x = torch.randn(3, 100, generator=g)
    kw = dict(target_index=torch.tensor([[4, 4, 4, 9], [0, 99, 0, 99], [-1, 3, -1, 3]]),
              target_prob=torch.tensor([[0.5, 2.0, -1.0, 0.1], [3.0, 0.0, 1.0, 0.25], [5.0, 0.5, 5.0, 0.5]]))
    check_all(x, kw, torch.float32)


def test_loss_gradient_against_differences():
    g = gen(10)
    x = torch.randn(2, 40, generator=g)
    kw = dict(target_index=torch.randint(0, 40, (2, 5), generator=g), target_prob=torch.rand(2, 5, generator=g),
              mask=mask_of(2, 40, 0.7, g), weights=torch.tensor([0.7, 1.3]))
    _, grad = lg.policy_loss_grad(dev(x), **{k: dev(t) for k, t in kw.items()})
    h = 1e-5
    for j in range(40):
        up, down = x.double().clone(), x.double().clone()
        up[:, j] += h
        down[:, j] -= h
        d = (ref.loss(up, **kw)[0] - ref.loss(down, **kw)[0]) / (2 * h)
        # third derivative of the loss is at most 1 (times weight and mass): h^2; the kernel's own bound above it
        ref.close(grad[:, j], d, torch.full((2,), 8 * h * h + 1e-10 / h + 1e-6).double())


def test_loss_broadcast_logits_sum_their_gradients():
    g = gen(12)
    x = torch.randn(1, 333, generator=g)
    label = torch.randint(0, 333, (6,), generator=g)
    leaf = dev(x).requires_grad_(True)
    lg.policy_loss(leaf.expand(6, -1), target_index=dev(label)).sum().backward()
    _, grad, _, b = ref.loss(x.expand(6, -1), target_index=label)
    ref.close(leaf.grad, grad.sum(0, keepdim=True), b.sum(0, keepdim=True) + 6 * ref.EPS32 * grad.abs().sum(0, keepdim=True))


def test_loss_bad_tokens_are_reported_and_skipped():
    x = torch.zeros(2, 50)
    t = torch.tensor([[3, 50], [2**40, 4]])
    with pytest.raises(CnnueError, match="index"):
        lg.policy_loss(dev(x), target_index=dev(t))
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    loss, grad = lg.policy_loss_grad(dev(x), target_index=dev(t), status=status)
    assert int(status) == 1
    want, g, bl, bg = ref.loss(x, target_index=torch.tensor([[3, -1], [-1, 4]]))
    ref.close(loss, want, bl)
    ref.close(grad, g, bg)


def test_loss_gradient_may_not_replace_its_inputs():
    x, t = torch.randn(2, 64, device=DEV), torch.rand(2, 64, device=DEV)
    for grad in (x, t):
        with pytest.raises(CnnueError, match="overlaps"):
            lg.policy_loss_grad(x, t, grad=grad)


def test_loss_survives_offloaded_and_released_tensors():
    """Saved-tensor hooks bring other storage to the backward pass; a second pass over a kept graph gives the same."""
    g = gen(22)
    x, kw = loss_inputs(3, 700, torch.float32, "lists", g)
    d = {k: dev(t) for k, t in kw.items()}
    leaf = dev(x).requires_grad_(True)
    plain = torch.autograd.grad(lg.policy_loss(leaf, **d).sum(), leaf)[0]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(DEV)):
        loss = lg.policy_loss(leaf, **d)
    assert torch.equal(torch.autograd.grad(loss.sum(), leaf)[0], plain)
    loss = lg.policy_loss(leaf.t().contiguous().t(), **d)  # a copy is made of it
    first = torch.autograd.grad(loss.sum(), leaf, retain_graph=True)[0]
    assert torch.equal(first, plain) and torch.equal(torch.autograd.grad(loss.sum(), leaf)[0], plain)


def test_loss_empty():
    loss, grad = lg.policy_loss_grad(torch.empty(0, 5, device=DEV), target_index=torch.empty(0, dtype=torch.int64, device=DEV))
    assert loss.shape == (0,) and grad.shape == (0, 5)
    x = torch.randn(2, 9, device=DEV)
    loss, grad = lg.policy_loss_grad(x, target_index=torch.empty(2, 0, dtype=torch.int32, device=DEV))
    assert not loss.any() and not grad.any()


def test_loss_step_captured_and_replayed():
    g = gen(13)
    x, kw = loss_inputs(8, 2086, torch.bfloat16, "lists", g)
    d = {k: dev(t) for k, t in kw.items()}
    y = dev(x).clone()
    grad = torch.empty_like(y)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    lg.policy_loss_grad(y, grad=grad, status=status, **d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, _ = lg.policy_loss_grad(y, grad=grad, status=status, **d)
    y.mul_(0.5)
    graph.replay()
    want, gr, bl, bg = ref.loss(y.cpu(), **kw)
    ref.close(loss, want, bl)
    ref.close(grad, gr, bg, torch.bfloat16)


@pytest.mark.parametrize("dtype", TYPES)
def test_results_do_not_change_from_run_to_run(dtype):
    g = gen(14)
    x, kw = loss_inputs(33, 30_011, dtype, "lists", g)
    d = {k: dev(t) for k, t in kw.items()}
    first = lg.policy_loss_grad(dev(x), **d)
    for _ in range(3):
        again = lg.policy_loss_grad(dev(x), **d)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_more_than_32_bits_apart(dtype):
    """Elements and bytes past 2^32, of the logits, the results and the targets."""
    g = gen(31)
    R, V, far = 4, 20_001, (1 << 30) + 3
    x = rows(R, V, dtype, g)
    kw = dict(history=history_of(R, V, 100, g), frequency=torch.rand(R, generator=g), mask=mask_of(R, V, 0.5, g))
    size = (R - 1) * far + V
    a, b = (torch.empty(size, dtype=dtype, device=DEV).as_strided((R, V), (far, 1)) for _ in range(2))
    a.copy_(x)
    want, bound = ref.process(x, **kw)
    ref.close(lg.process_logits(a, out=b, **{k: dev(t) for k, t in kw.items()}), want, bound, dtype)
    t = torch.rand(R, V, generator=g)
    want, grad, bl, bg = ref.loss(x, t, mask=kw["mask"])
    loss, got = lg.policy_loss_grad(a, dev(t), mask=dev(kw["mask"]), grad=b)
    ref.close(loss, want, bl)
    ref.close(got, grad, bg, dtype)


# ---- together, as they are used -----------------------------------------------------
def test_legal_moves_choose_learn_and_update():
    """The ResNet's logits under the rules of the game: legal-move priors; then
    a policy head learns visit counts under the same masks, with 8-bit AdamW."""
    from chineseai_b200 import az, mcts, resnet
    from chineseai_b200.optim import MultiAdamW
    n = 6
    boards = az.random_boards(n, 3)
    sides = np.arange(n, dtype=np.uint8) % 2
    mask = torch.from_numpy(mcts.legal_mask(boards, sides)).to(DEV)
    model = resnet.ResNetModel(resnet.ResNetWeights.synthetic(5))
    planes = torch.from_numpy(resnet.synthetic_planes(n, 6).view(np.int16)).to(DEV)
    probs, logits, _ = model.forward(planes, with_logits=True)
    a = ref.unpack(mask.cpu(), 2086)
    want, bound = ref.process(logits.cpu(), mask=mask.cpu())
    ref.close(lg.process_logits(logits, mask=mask), want, bound)
    answer, _ = model.move_logits(planes, mask=mask)
    ref.close(answer, want, bound)
    model.close()

    g = gen(1)
    feats = torch.randn(n, 32, generator=g)
    head = [torch.randn(2086, 32, generator=g) * 0.1, torch.zeros(2086)]
    visits = torch.rand(n, 2086, generator=g) * a
    visits = visits / visits.sum(1, keepdim=True).clamp(min=1e-9)
    w = torch.full((n,), 1.0 / n)
    p = [dev(t).clone() for t in head]
    grads = [torch.empty_like(t) for t in p]
    opt = MultiAdamW(p, grads, lr=1e-2, state_bits=8)
    z = torch.addmm(p[1], dev(feats), p[0].t())
    loss, gz = lg.policy_loss_grad(z, dev(visits), mask=mask, weights=dev(w))
    torch.mm(gz.t(), dev(feats), out=grads[0])
    torch.sum(gz, 0, out=grads[1])
    opt.step()
    # the same step in 64 bits
    hp = [t.double().requires_grad_(True) for t in head]
    zz = torch.addmm(hp[1], feats.double(), hp[0].t()).masked_fill(~a, -math.inf)
    lse = torch.logsumexp(zz, 1, keepdim=True)
    total = (-(visits.double() * torch.where(a, zz - lse, 0.0)).sum(1) * w.double())
    total.sum().backward()
    # logits differ by the fp32 matmul's rounding (33 terms of size < 5) and so does the loss
    assert (loss.cpu().double() - total.detach()).abs().max() < 40 * 5 * 33 * ref.EPS32
    for q, h, gr in zip(p, hp, grads):
        # gradients: the fp32 sum over the boards and the logits' error
        assert (gr.cpu().double() - h.grad).abs().max() < 1e-4 * h.grad.abs().max()
        # a first AdamW step moves every parameter by lr * g / (|g| + eps), less the decay
        g64 = gr.cpu().double()
        step = h.detach() * (1 - 1e-2 * 1e-4) - 1e-2 * g64 / (g64.abs() + 1e-8)
        # below 2^-60 the squares leave fp32's normal range and the root loses digits
        big = (g64.abs() > 2.0 ** -55) | (g64 == 0)
        assert ((q.cpu().double() - step).abs()[big] <= 16 * ref.EPS32 * (step.abs() + 1e-2)[big]).all()


def test_calls_of_other_sizes_in_other_threads():
    """Calls in several threads that need different amounts of shared memory give what they give alone."""
    def jobs(seed):
        g = gen(seed)
        made = []
        for vocab in (8_192, 60_001, 126_000, 190_000):
            x = dev(torch.randn(3, vocab, generator=g))
            label = dev(torch.randint(0, vocab, (3,), generator=g))
            history = dev(torch.randint(0, vocab, (3, 3000), generator=g, dtype=torch.int32))
            rule = dict(history=history, frequency=dev(torch.full((3,), 0.25)))
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            made.append((lambda x=x, label=label, status=status: lg.policy_loss_grad(x, target_index=label, status=status)[1]))
            made.append((lambda x=x, rule=rule, status=status: lg.process_logits(x, **rule, status=status)))
        return made

    work = [jobs(seed) for seed in range(4)]
    alone = [[f() for f in fs] for fs in work]
    torch.cuda.synchronize()
    faults = []

    def run(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(50):
                    j = (i * (2 * k + 1) + k) % len(work[k])
                    if not torch.equal(work[k][j](), alone[k][j]):
                        faults.append((k, j))
        except Exception as e:  # noqa: BLE001
            faults.append((k, repr(e)))

    threads = [threading.Thread(target=run, args=(k,)) for k in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not faults and not any(t.is_alive() for t in threads)
