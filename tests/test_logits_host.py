"""CPU tests of the logit operators' host side: packed masks, legal-move masks,
and what the entry points refuse before anything reaches a GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

from chineseai_b200 import _lib, az, logits, mcts
from chineseai_b200.optim import MultiAdamW

INVALID = 1


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 64, 2086])
def test_pack_mask(vocab):
    rng = np.random.default_rng(vocab)
    a = rng.random((3, vocab)) < 0.5
    w = logits.pack_mask(a)
    assert w.dtype == np.int32 and w.shape == (3, (vocab + 31) // 32)
    u = w.view(np.uint32)
    for r in range(3):
        for t in range(vocab):
            assert bool(u[r, t // 32] >> np.uint32(t % 32) & np.uint32(1)) == a[r, t]
    assert torch.equal(logits.pack_mask(torch.from_numpy(a)), torch.from_numpy(w))


@pytest.mark.parametrize("threads", [1, 0, 3])
def test_legal_mask_is_the_legal_moves(threads):
    n = 200
    boards = az.random_boards(n, 11)
    sides = (np.arange(n) % 2).astype(np.uint8)
    m = mcts.legal_mask(boards, sides, threads).view(np.uint32)
    assert m.shape == (n, 66)
    _, s2d = az.dense_moves()
    for i in range(n):
        got = {t for t in range(66 * 32) if m[i, t // 32] >> np.uint32(t % 32) & np.uint32(1)}
        want = set()
        for f, t in mcts.legal_moves(boards[i], int(sides[i])):
            f, t = (int(f), int(t)) if sides[i] == 0 else (89 - int(f), 89 - int(t))
            if s2d[f * 90 + t] < 2086:
                want.add(int(s2d[f * 90 + t]))
        assert got == want
    b0, s0 = az.board_from_fen("rnbakabnr/9/1c5c1/p1p1p1p1p/9/9/P1P1P1P1P/1C5C1/9/RNBAKABNR w - - 0 1")
    words = mcts.legal_mask(b0, np.array([s0])).view(np.uint32)
    assert sum(bin(int(w)).count("1") for w in words.reshape(-1)) == 44


def test_legal_mask_refuses():
    b = np.zeros((2, 90), np.int8)
    with pytest.raises(ValueError):
        mcts.legal_mask(b, np.zeros(3, np.uint8))
    with pytest.raises(_lib.CnnueError):
        mcts.legal_mask(b, np.array([0, 2], np.uint8))
    b[1, 5] = 9
    with pytest.raises(_lib.CnnueError):
        mcts.legal_mask(b, np.zeros(2, np.uint8))
    assert mcts.legal_mask(np.zeros((0, 90)), np.zeros(0)).shape == (0, 66)


def rules(**kw):
    r = _lib.LogitRules()
    for k, v in kw.items():
        setattr(r, k, v)
    return C.addressof(r), r


@pytest.mark.parametrize("packed,declared", [(logits._RULES, _lib.LogitRules), (logits._TARGETS, _lib.LossTargets)])
def test_packed_structs_have_the_declared_layout(packed, declared):
    values = list(range(1, len(declared._fields_) + 1))
    data = packed.pack(*values)
    assert len(data) == C.sizeof(declared)
    back = declared.from_buffer_copy(data)
    assert [getattr(back, name) for name, _ in declared._fields_] == values


def test_optimizer_table_has_the_declared_layout():
    from chineseai_b200.optim import _TENSOR
    assert _TENSOR.itemsize == C.sizeof(_lib.AdamwTensor)
    for name, kind in _lib.AdamwTensor._fields_:
        assert _TENSOR.fields[name][1] == getattr(_lib.AdamwTensor, name).offset
        assert _TENSOR.fields[name][0].itemsize == C.sizeof(kind)


A, B, S = 1 << 20, 1 << 24, 1 << 28  # addresses that no call below gets to use


def process(r=None, logits=A, ls=100, lt=0, out=B, os=100, ot=0, rows=4, vocab=100, status=S):
    addr, keep = rules(**(r or {}))
    return _lib.lib().cnnue_logits_process(logits, ls, lt, out, os, ot, rows, vocab, addr, status, None)


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(vocab=-1), dict(vocab=(1 << 30) + 1), dict(status=None), dict(logits=None), dict(out=None),
    dict(lt=3), dict(ot=-1), dict(lt=1, ot=2), dict(lt=0, ot=1), dict(logits=A + 2), dict(out=B + 1), dict(ls=-1),
    dict(os=99), dict(os=0), dict(out=A + 4), dict(out=A, os=101), dict(lt=1, out=A), dict(out=A + 4 * 399),
    dict(r=dict(repetition=A)), dict(r=dict(lengths=A)), dict(r=dict(history=A, history_bytes=2)),
    dict(r=dict(history=A, history_bytes=4, history_len=-1)), dict(r=dict(history=A, history_bytes=4, history_len=1 << 31)),
    dict(r=dict(history=A, history_bytes=8, history_stride=-1)), dict(r=dict(bias_tokens=A)), dict(r=dict(bias_values=A)),
    dict(r=dict(bias_tokens=A, bias_values=A, bias_count=-1)), dict(r=dict(mask_index=A)),
    dict(r=dict(mask=A, mask_rows=3, mask_stride=4)), dict(r=dict(mask=A, mask_rows=4, mask_stride=-1)),
    dict(r=dict(mask=A, mask_rows=-1, mask_stride=4, mask_index=A)),
])
def test_process_refuses(bad):
    assert process(**bad) == INVALID
    assert _lib.last_error()


def test_nothing_to_do_is_ok():
    assert process(rows=0, logits=None, out=None) == 0
    assert process(vocab=0, logits=None, out=None) == 0
    t = _lib.LossTargets(index=A, index_bytes=4, count=1)
    assert _lib.lib().cnnue_policy_loss_grad(None, 0, 0, 0, 5, C.addressof(t), None, None, 0, S, None) == 0
    assert _lib.lib().cnnue_adamw_multi(None, 0, 32, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 1.0, None, 0, None) == 0


def targets(**kw):
    t = _lib.LossTargets(index=A, index_bytes=4, count=1, index_stride=1)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


@pytest.mark.parametrize("bad", [
    dict(rows=-1), dict(vocab=0), dict(vocab=1 << 31), dict(status=None), dict(logits=None), dict(grad=None),
    dict(loss=None), dict(lt=4), dict(logits=A + 1), dict(grad=A), dict(grad=A + 4), dict(gs=99), dict(ls=-5),
    dict(t=dict(index=None)), dict(t=dict(dense=A)), dict(t=dict(index_bytes=2)), dict(t=dict(count=-1)),
    dict(t=dict(index_stride=-1)), dict(t=dict(index=None, dense=A, dense_type=7)),
    dict(t=dict(index=None, dense=A + 2)), dict(t=dict(index=None, dense=B, dense_stride=100)), dict(t=dict(index=None, dense=A, prob=A)),
    dict(t=dict(mask=A, mask_rows=2, mask_stride=4)), dict(t=dict(mask_index=A)),
])
def test_loss_refuses(bad):
    kw = dict(logits=A, ls=100, lt=0, rows=4, vocab=100, loss=A, grad=B, gs=100, status=S, t={})
    kw.update(bad)
    t = targets(**kw["t"])
    L = _lib.lib()
    head = (kw["logits"], kw["ls"], kw["lt"], kw["rows"], kw["vocab"], C.addressof(t))
    assert L.cnnue_policy_loss_grad(*head, kw["loss"], kw["grad"], kw["gs"], kw["status"], None) == INVALID
    if kw["loss"] is not None and not {"grad", "gs"} & set(bad) and kw["t"].get("dense") != B:
        assert L.cnnue_policy_loss_fwd(*head, A, A, kw["status"], None) == INVALID
    if kw["loss"] is not None:
        assert L.cnnue_policy_loss_bwd(*head, A, None, kw["grad"], kw["gs"], kw["status"], None) == INVALID
    assert L.cnnue_policy_loss_grad(A, 100, 0, 4, 100, None, A, B, 100, S, None) == INVALID


@pytest.mark.parametrize("bad", [
    dict(n=-1), dict(param=None), dict(grad=None), dict(m=None), dict(v=None), dict(param=A + 2), dict(grad=A + 1),
    dict(param_type=3), dict(grad_type=-1), dict(m=A + 2), dict(copy=A, copy_type=0), dict(copy=A + 1, copy_type=1),
    dict(bits=8, m_scale=None), dict(bits=8, v_scale=A + 2), dict(bits=16), dict(step=0), dict(n_skip=-1),
    dict(n_skip=1), dict(count=-1),
])
def test_multi_adamw_refuses(bad):
    t = (_lib.AdamwTensor * 1)(_lib.AdamwTensor(param=A, grad=A, m=A, v=A, m_scale=A, v_scale=A, n=4))
    kw = dict(bits=32, step=1, n_skip=0, count=1)
    for k, v in bad.items():
        if k in kw:
            kw[k] = v
        else:
            setattr(t[0], k, v)
    L = _lib.lib()
    assert L.cnnue_adamw_multi(C.addressof(t), kw["count"], kw["bits"], 1e-3, 0.9, 0.999, 1e-8, 0.0, kw["step"], 1.0, None,
                               kw["n_skip"], None) == INVALID
    assert L.cnnue_adamw_multi_device(C.addressof(t), kw["count"], kw["bits"], None if "step" in bad else A, 1.0, None,
                                      kw["n_skip"], None) == INVALID


def test_python_refusals_without_a_gpu():
    x = torch.zeros(2, 10)
    with pytest.raises(ValueError, match="CUDA"):
        logits.process_logits(x)
    with pytest.raises(ValueError, match="CUDA"):
        logits.policy_loss(x, target_index=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        MultiAdamW([x], [x])
    with pytest.raises(ValueError, match="no parameters"):
        MultiAdamW([], [])
    with pytest.raises(ValueError, match="state_bits"):
        MultiAdamW([x], [x], state_bits=16)
    with pytest.raises(ValueError, match="not differentiable"):
        logits.process_logits(x.requires_grad_(True))
