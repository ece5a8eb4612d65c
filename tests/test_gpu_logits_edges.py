"""The masked policy loss and process_logits where single targets, NaNs and
arguments are unusual: signed targets, NaNs that few threads see, rows without
target mass, histories without penalties; against the plain 64-bit forms."""
import math

import pytest
import torch

from tests import _logitsref as ref
from tests.test_gpu_logits import DEV, TYPES, check_all, dev, gen
from chineseai_b200 import logits as lg
from chineseai_b200._lib import CnnueError

pytestmark = pytest.mark.gpu


# ---- targets of both signs --------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [100, 2086, 131_072])
@pytest.mark.parametrize("kind", ["lists", "dense"])
def test_loss_of_targets_that_cancel(kind, vocab, dtype):
    """+p and -p in one vector, one warp, two warps, two CTAs of a cluster; alone, and beside other targets."""
    g = gen(vocab)
    pairs = [(4, 5), (0, vocab - 1), (8, vocab // 2), (vocab // 3, vocab // 3 + 9), (5, 9), (1, 96)]
    x = (torch.randn(2 * len(pairs), vocab, generator=g) * 3).to(dtype)
    K = 300  # entries of a list: the second of a pair is another warp's
    index = torch.full((len(x), K), -1, dtype=torch.int64)
    prob = torch.zeros(len(x), K)
    for r, (a, b) in enumerate(pairs * 2):
        at = (0, 1) if r % 2 else (3, 290)
        index[r, at[0]], index[r, at[1]] = a, b
        prob[r, at[0]], prob[r, at[1]] = 0.75, -0.75
        if r >= len(pairs):
            index[r, 100], prob[r, 100] = vocab // 2 + 1, 0.5
    if kind == "lists":
        return check_all(x, dict(target_index=index, target_prob=prob), dtype)
    targets = torch.zeros(len(x), vocab).scatter_add_(1, index.clamp(min=0), torch.where(index >= 0, prob, 0.0))
    check_all(x, dict(targets=targets), dtype)


def test_loss_of_a_pair_at_any_two_tokens():
    """A preference pair is the difference of two logits, wherever its tokens lie."""
    g = gen(3)
    V = 2086
    x = torch.randn(64, V, generator=g)
    pair = torch.stack([torch.randperm(V, generator=g)[:2] for _ in range(64)])
    pair[0] = torch.tensor([5, 9])
    prob = torch.tensor([1.0, -1.0]).expand(64, 2)
    check_all(x, dict(target_index=pair, target_prob=prob), torch.float32)
    loss, _ = lg.policy_loss_grad(dev(x), target_index=dev(pair), target_prob=dev(prob))
    z = x.double().gather(1, pair)
    d = z[:, 1] - z[:, 0]
    # every value on the way is below 10; a target's difference is rounded once, in each of two joins it is moved to
    # the joint maximum (two roundings) and added up (at most four that round)
    assert ((loss.cpu().double() - d).abs() <= 2 * 13 * ref.EPS32 * 10).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["lists", "dense"])
def test_loss_of_targets_on_minus_infinity(kind, dtype):
    """t (M - z) there is an infinity of the target's sign, whichever thread meets it, before or after a finite logit;
    infinities of both signs are NaN."""
    g = gen(17)
    V, R, K = 2086, 12, 300
    x = torch.randn(R, V, generator=g).to(dtype)
    x[:, 4:2000] = x[:, 2008:] = -math.inf  # most threads see nothing else
    index = torch.full((R, K), -1, dtype=torch.int64)
    prob = torch.zeros(R, K)
    for r in range(R):
        sign = -1.0 if r % 2 else 1.0
        token = (100, 700, 1499)[r % 3]
        entry, finite = ((26, 282), (282, 26), (40, 41))[r // 2 % 3]  # a thread's first or second entry, another thread's
        index[r, entry], prob[r, entry] = token, sign * 0.5
        index[r, finite], prob[r, finite] = (2000, 3)[r % 2], 1.0
    index[10, 100], prob[10, 100] = 101, -prob[10, index[10] >= 100].max()
    index[11, 0:2], prob[11, 0:2] = torch.tensor([600, 601]), torch.tensor([0.5, -0.25])
    if kind == "lists":
        kw = dict(target_index=index, target_prob=prob)
    else:
        kw = dict(targets=torch.zeros(R, V).scatter_add_(1, index.clamp(min=0), torch.where(index >= 0, prob, 0.0)))
    want = ref.loss(x, **kw)[0]
    assert torch.isinf(want[:10]).all() and (want[:10] < 0).any() and want[10:].isnan().all()
    check_all(x, kw, dtype)


# ---- NaNs at allowed tokens ---------------------------------------------------------
def check_nan_rows(x, a, kw, dtype):
    """Every row of x is NaN: its loss, and its gradient at the allowed tokens; 0 at the others."""
    d = {k: dev(t) for k, t in kw.items()}
    targets = d.pop("targets", None)
    loss, got = lg.policy_loss_grad(dev(x), targets, **d)
    leaf = dev(x).requires_grad_(True)
    again = lg.policy_loss(leaf, targets, **d)
    again.sum().backward()
    for rows, grad in ((loss, got), (again, leaf.grad)):
        assert rows.isnan().all(), rows
        assert torch.equal(grad.isnan().cpu(), a) and not grad.cpu()[~a].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["dense", "labels", "lists"])
@pytest.mark.parametrize("rows,vocab", [(1, 64), (3, 2086), (1, 8100), (2, 50_001), (3, 131_072), (1, 900_001)])
@pytest.mark.parametrize("hidden", ["mask", "-inf"])
def test_loss_keeps_a_nan_that_nothing_finite_follows(hidden, rows, vocab, kind, dtype):
    """One allowed token, a NaN, among masked ones or logits of -inf: at the row's start, where the thread that meets it
    has all its other vectors to go, in the middle and at the end; one CTA and clusters, rows kept and read twice."""
    g = gen(vocab)
    for at in (5, vocab // 2, vocab - 1):
        x = torch.randn(rows, vocab, generator=g).to(dtype)
        a = torch.ones(rows, vocab, dtype=torch.bool)
        kw = {}
        if hidden == "mask":
            a[:] = False
            a[:, at] = True
            kw["mask"] = lg.pack_mask(a)
        else:
            x[:] = -math.inf
        x[:, at] = math.nan
        if kind == "dense":
            kw["targets"] = torch.rand(rows, vocab, generator=g)
        elif kind == "labels":
            kw["target_index"] = torch.full((rows,), at)
        else:
            kw["target_index"] = torch.tensor([[-1, at, at, 0]]).expand(rows, 4).contiguous()
            kw["target_prob"] = torch.tensor([[1.0, 0.5, 0.25, 0.125]]).expand(rows, 4).contiguous()
        check_nan_rows(x, a, kw, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [100, 2086, 131_072, 900_001])
@pytest.mark.parametrize("kind", ["dense", "lists", "labels"])
def test_loss_of_a_nan_row_without_target_mass(kind, vocab, dtype):
    """No target at all, targets on masked tokens only, masses that cancel: the NaN is there all the same."""
    g = gen(vocab + 1)
    R = 6
    x = torch.randn(R, vocab, generator=g).to(dtype)
    x[:3, vocab // 3] = math.nan  # among finite logits
    x[3:] = -math.inf  # alone
    x[3:, 7] = math.nan
    a = torch.rand(R, vocab, generator=g) < 0.7
    a[:, :20] = a[:, vocab // 3] = True
    a[:, 20] = False
    index = torch.tensor([[-1, -1, -1], [20, 20, -1], [4, 9, -1]]).repeat(2, 1)  # nothing, masked, +0.5 and -0.5
    prob = torch.tensor([0.5, -0.5, 1.0]).expand(R, 3)
    if kind == "lists":
        kw = dict(target_index=index, target_prob=prob)
    elif kind == "labels":
        kw = dict(target_index=torch.tensor([-1, 20, -1, 20, -1, 9]))  # the last has its mass on another token
    else:
        kw = dict(targets=torch.zeros(R, vocab).scatter_add_(1, index.clamp(min=0), torch.where(index >= 0, prob, 0.0)))
    check_nan_rows(x, a, dict(kw, mask=lg.pack_mask(a)), dtype)
    idle = dict(kw, mask=lg.pack_mask(a), weights=torch.zeros(R))  # rows of weight 0 are not read
    d = {k: dev(t) for k, t in idle.items()}
    loss, got = lg.policy_loss_grad(dev(x), d.pop("targets", None), **d)
    assert not loss.any() and not got.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", [(200, 100), (33, 2086), (5, 131_072), (2, 500_009)])
def test_loss_both_forms_give_the_same_bits(rows, vocab, dtype):
    g = gen(vocab + 2)
    x = dev((torch.randn(rows, vocab, generator=g) * 3).to(dtype)).requires_grad_(True)
    kw = dict(target_index=dev(torch.randint(0, vocab, (rows, 5), generator=g)), target_prob=dev(torch.rand(rows, 5, generator=g)),
              weights=dev(torch.rand(rows, generator=g)))
    loss, grad = lg.policy_loss_grad(x.detach(), **kw)
    again = lg.policy_loss(x, **kw)
    again.sum().backward()
    assert torch.equal(loss, again) and torch.equal(grad, x.grad)


# ---- saved tensors ------------------------------------------------------------------
def test_loss_of_tensors_that_hooks_pack_together():
    """Hooks that bring the saved tensors back without their padding, at the same addresses."""
    g = gen(19)
    R, V, K, pad = 16, 700, 9, 5
    x = torch.randn(R, V, generator=g)

    def padded(t):
        buf = torch.zeros(R, t.shape[1] + pad, dtype=t.dtype, device=DEV)
        buf[:, :t.shape[1]] = dev(t)
        return buf[:, :t.shape[1]]

    def close_up(t):
        if t.dim() != 2:
            return t
        kept = t.clone()
        u = t.as_strided(t.shape, (t.shape[1], 1))
        u.copy_(kept)
        return u

    for kw in (dict(targets=torch.rand(R, V, generator=g)),
               dict(target_index=torch.randint(0, V, (R, K), generator=g), target_prob=torch.rand(R, K, generator=g))):
        kw["mask"] = lg.pack_mask(torch.rand(R, V, generator=g) < 0.5)
        want, grad, bl, bg = ref.loss(x, **kw)
        leaf = dev(x).requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), close_up):
            loss = lg.policy_loss(leaf, **{k: padded(t) for k, t in kw.items()})
        ref.close(loss, want, bl)
        ref.close(torch.autograd.grad(loss.sum(), leaf)[0], grad, bg)


def test_loss_keeps_no_copy_after_the_backward_pass():
    """Copies of strided logits, targets and masks are freed with the graph, though the loss lives on."""
    g = gen(20)
    R, V = 16, 200_000
    x, t = (torch.randn(V, R, generator=g).to(DEV).t() for _ in range(2))
    m = lg.pack_mask(torch.rand(R, V, generator=g) < 0.5).t().contiguous().to(DEV).t()
    x.requires_grad_(True)
    before = torch.cuda.memory_allocated()
    loss = lg.policy_loss(x, t, mask=m)
    grad, = torch.autograd.grad(loss.sum(), x)
    want = lg.policy_loss_grad(x.detach(), t, mask=m)
    assert torch.equal(loss, want[0]) and torch.equal(grad, want[1])
    del grad, want
    assert torch.cuda.memory_allocated() - before < R * V  # a quarter of one copy's bytes
    first = lg.policy_loss(x, t, mask=m)
    a, = torch.autograd.grad(first.sum(), x, retain_graph=True)
    b, = torch.autograd.grad(first.sum(), x)
    assert torch.equal(a, b)


# ---- a history without penalties ------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab,length", [(50, 30), (2086, 200), (40_000, 100), (40_000, 5000), (40_000, 40_000)])
def test_process_checks_a_history_without_penalties(vocab, length, dtype):
    """Bad tokens and lengths are reported as with penalties, and nothing but the mask changes the rows."""
    g = gen(vocab + length)
    R = 3
    x = (torch.randn(R, vocab, generator=g) * 3).to(dtype)
    x[0, :3] = torch.tensor([math.inf, -math.inf, -0.0]).to(dtype)
    h = torch.randint(-1, vocab, (R, length), generator=g)
    h[:, :3] = torch.arange(3)
    m = lg.pack_mask(torch.rand(R, vocab, generator=g) < 0.8)
    want, bound = ref.process(x, mask=m)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)

    def run(history, lengths, **kw):
        status.zero_()
        out = lg.process_logits(dev(x), history=dev(history), lengths=dev(lengths), status=status, **kw)
        return out, int(status)

    out, word = run(h, None, mask=dev(m))
    ref.close(out, want, bound, dtype)
    assert word == 0
    bits = {torch.float32: torch.int32}.get(dtype, torch.int16)
    out, word = run(h, None)
    assert torch.equal(out.cpu().view(bits), x.view(bits)) and word == 0
    bad = h.clone()
    bad[1, length - 1] = vocab
    out, word = run(bad, None)
    assert torch.equal(out.cpu().view(bits), x.view(bits)) and word == 1
    out, word = run(bad, torch.tensor([length, length - 1, length], dtype=torch.int32))  # the bad token does not count
    assert torch.equal(out.cpu().view(bits), x.view(bits)) and word == 0
    out, word = run(h, torch.tensor([0, length + 1, -1], dtype=torch.int32))
    assert torch.equal(out.cpu().view(bits), x.view(bits)) and word == 2
    out, word = run(h[:, :0], torch.tensor([0, 1, 0], dtype=torch.int32))
    assert torch.equal(out.cpu().view(bits), x.view(bits)) and word == 2
    y = dev(x).clone()
    status.zero_()
    lg.process_logits(y, history=dev(bad), out=y, status=status)  # in place, without a mask
    assert torch.equal(y.cpu().view(bits), x.view(bits)) and int(status) == 1


# ---- rows between each other -----------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gap", [0, 3])
@pytest.mark.parametrize("first", ["in", "out"])
def test_column_ranges_of_one_matrix(first, gap, dtype):
    """Logits and results in one matrix, side by side, as the operators' inputs and outputs; one column nearer is refused."""
    g = gen(41)
    R, V = 9, 333
    x = (torch.randn(R, V, generator=g) * 3).to(dtype)
    m = lg.pack_mask(torch.rand(R, V, generator=g) < 0.5)
    label = torch.randint(0, V, (R,), generator=g)
    buf = torch.full((R, 2 * V + gap + 2), 7.0, dtype=dtype, device=DEV)
    a, b = buf[:, 1:1 + V], buf[:, 1 + V + gap:1 + 2 * V + gap]
    z, out = (a, b) if first == "in" else (b, a)
    z.copy_(x)
    before = buf.clone()
    want, bound = ref.process(x, mask=m)
    lg.process_logits(z, mask=dev(m), out=out)
    ref.close(out, want, bound, dtype)
    loss, grad, bl, bg = ref.loss(x, target_index=label, mask=m)
    got, _ = lg.policy_loss_grad(z, target_index=dev(label), mask=dev(m), grad=out)
    ref.close(got, loss, bl)
    ref.close(out, grad, bg, dtype)
    out.copy_(before[:, 1 + V + gap:1 + 2 * V + gap] if first == "in" else before[:, 1:1 + V])
    assert torch.equal(buf, before), "wrote outside the columns"
    near = buf[:, V:2 * V] if first == "in" else buf[:, 2 + gap:2 + gap + V]
    with pytest.raises(CnnueError, match="overlaps"):
        lg.process_logits(z, out=near)
    with pytest.raises(CnnueError, match="overlaps"):
        lg.policy_loss_grad(z, target_index=dev(label), grad=near)
    t = torch.empty(R, V + 1, dtype=dtype, device=DEV)  # rows at another distance over the same memory
    with pytest.raises(CnnueError, match="overlaps"):
        lg.process_logits(t[:, :V], out=t.view(-1)[:R * V].view(R, V))


# ---- captured calls at the sizes that take more shared memory ---------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [2086, 131_072, 250_001])
def test_loss_forward_and_backward_captured(vocab, dtype):
    """policy_loss with its gradient and policy_loss_grad in one graph, replayed on new logits."""
    g = gen(vocab + 5)
    R = 3
    x = torch.randn(2, R, vocab, generator=g).to(dtype)
    label = torch.randint(0, vocab, (R,), generator=g)
    m = lg.pack_mask(torch.rand(R, vocab, generator=g) < 0.9)
    kw = dict(target_index=dev(label), mask=dev(m), status=torch.zeros(1, dtype=torch.int32, device=DEV))
    leaf = dev(x[0]).clone().requires_grad_(True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = lg.policy_loss(leaf, **kw)
        grad, = torch.autograd.grad(loss.sum(), leaf)
        fused = lg.policy_loss_grad(leaf.detach(), **kw)
    with torch.no_grad():
        leaf.copy_(x[1])
    graph.replay()
    want, gr, bl, bg = ref.loss(x[1], target_index=label, mask=m)
    for a, b in ((loss, grad), fused):
        ref.close(a, want, bl)
        ref.close(b, gr, bg, dtype)
    assert int(kw["status"]) == 0


@pytest.mark.parametrize("vocab,length", [(16_384, 40_000), (131_072, 5000), (131_072, 40_000)])
def test_process_captured_with_many_counters(vocab, length):
    g = gen(length)
    x = torch.randn(2, vocab, generator=g)
    h = torch.randint(0, vocab, (2, length), generator=g).int()
    f, a, hist = torch.rand(2, generator=g), dev(x).clone(), dev(h)
    status, fd = torch.zeros(1, dtype=torch.int32, device=DEV), dev(f)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lg.process_logits(a, history=hist, frequency=fd, status=status)
    hist.copy_(dev(h.flip(0)))
    graph.replay()
    want, bound = ref.process(x, history=h.flip(0), frequency=f)
    ref.close(out, want, bound)
    assert int(status) == 0


# ---- the largest and the most rows -------------------------------------------------------
def test_the_largest_vocabulary():
    """2^30 tokens: sums of that many equal terms are exact, so losses and gradients are known."""
    V = 1 << 30
    x = torch.zeros(1, V, dtype=torch.bfloat16, device=DEV)
    label = torch.tensor([V - 1], device=DEV)
    loss, grad = lg.policy_loss_grad(x, target_index=label)
    assert abs(float(loss) - 30 * math.log(2)) < 21 * 2.0 ** -21
    assert float(grad[0, V - 1]) == -1.0 and float(grad[0, 0]) == 2.0 ** -30 and float(grad[0, V // 2]) == 2.0 ** -30
    assert int((grad == 2.0 ** -30).sum()) == V - 1
    del grad
    x.requires_grad_(True)
    again = lg.policy_loss(x, target_index=label)
    assert torch.equal(again, loss)
    grad, = torch.autograd.grad(again.sum(), x)
    assert float(grad[0, V - 1]) == -1.0 and int((grad == 2.0 ** -30).sum()) == V - 1
    del grad, again
    x = x.detach()
    for length in (3, 3000):  # hash table; counters of 2^15 CTAs
        h = torch.full((length,), V - 1, dtype=torch.int32, device=DEV)
        h[0], h[1] = 0, V // 2
        mask = torch.full((1, V // 32), -1, dtype=torch.int32, device=DEV)
        mask[0, V // 64] = 0
        out = lg.process_logits(x, history=h, frequency=torch.full((1,), 0.5, device=DEV), mask=mask)
        far = torch.tensor(-0.5 * (length - 2)).to(torch.bfloat16)  # rounded once
        assert float(out[0, V - 1]) == float(far) and float(out[0, 0]) == -0.5
        assert int((out == 0).sum()) == V - 32 - 2 and int((out == -math.inf).sum()) == 32
        del out


@pytest.mark.parametrize("vocab", [1, 2, 7])
def test_many_short_rows(vocab):
    R = 1_000_003
    x = torch.arange(R * vocab, device=DEV).view(R, vocab).remainder(5).float()
    label = torch.arange(R, device=DEV).remainder(vocab)
    loss, grad = lg.policy_loss_grad(x, target_index=label)
    z = x.double()
    want = torch.logsumexp(z, 1) - z.gather(1, label[:, None])[:, 0]
    assert ((loss.double() - want).abs() <= 2.0 ** -19).all()  # logits of 0 .. 4: a few roundings of sums below 8
    p = torch.softmax(z, 1).scatter_add(1, label[:, None], torch.full((R, 1), -1.0, device=DEV, dtype=torch.float64))
    assert ((grad.double() - p).abs() <= 2.0 ** -19).all()
    h = label[:, None].int()
    out = lg.process_logits(x, history=h, frequency=torch.ones(R, device=DEV))
    assert torch.equal(out, x.scatter_add(1, label[:, None], torch.full((R, 1), -1.0, device=DEV)))
