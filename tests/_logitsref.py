"""Plain 64-bit (CPU, torch double) forms of the logit operators, with bounds
of what fp32 arithmetic may add."""
import math

import torch

EPS32 = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the smallest subnormal."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def unpack(mask, vocab):
    bits = (mask[..., None].long() >> torch.arange(32)) & 1
    return bits.reshape(mask.shape[:-1] + (-1,))[..., :vocab].bool()


def allowed(rows, vocab, mask=None, mask_index=None):
    a = torch.ones(rows, vocab, dtype=torch.bool)
    if mask is None:
        return a
    m = unpack(mask if mask.dim() == 2 else mask[None], vocab)
    for r in range(rows):
        i = int(mask_index[r]) if mask_index is not None else (0 if len(m) == 1 else r)
        if i >= len(m):
            a[r] = False
        elif i >= 0:
            a[r] = m[i]
    return a


def process(logits, history=None, lengths=None, prompt_lengths=None, repetition=None, frequency=None, presence=None,
            bias_tokens=None, bias_values=None, mask=None, mask_index=None):
    """(result in 64 bits, bound of the fp32 error per element)."""
    x = logits.double().clone()
    R, V = x.shape
    size = x.abs()  # largest magnitude on the way
    ops = torch.zeros(R, V, dtype=torch.double)
    for r in range(R):
        if history is not None:
            h = (history if history.dim() == 2 else history[None].expand(R, -1))[r]
            n = h.numel() if lengths is None else min(max(int(lengths[r]), 0), h.numel())
            seen, count = {}, {}
            for i, t in enumerate(h[:n].tolist()):
                if 0 <= t < V:
                    seen[t] = True
                    if i >= (0 if prompt_lengths is None else int(prompt_lengths[r])):
                        count[t] = count.get(t, 0) + 1
            rep = 1.0 if repetition is None else float(repetition[r])
            fr = 0.0 if frequency is None else float(frequency[r])
            pr = 0.0 if presence is None else float(presence[r])
            for t in seen:
                v = float(x[r, t])
                v = v / rep if v > 0 else v * rep
                c = count.get(t, 0)
                if c:
                    v = v - fr * c - pr
                size[r, t] = max(float(size[r, t]) * max(rep, 1 / rep), 0) + abs(fr) * c + abs(pr)
                ops[r, t] += 4
                x[r, t] = v
        if bias_tokens is not None:
            bt = (bias_tokens if bias_tokens.dim() == 2 else bias_tokens[None].expand(R, -1))[r].tolist()
            bv = (bias_values if bias_values.dim() == 2 else bias_values[None].expand(R, -1))[r].tolist()
            for t, b in zip(bt, bv):
                if 0 <= t < V:
                    x[r, t] += b
                    size[r, t] += abs(b)
                    ops[r, t] += 1
    x[~allowed(R, V, mask, mask_index)] = -math.inf
    return x, ops * EPS32 * size * 1.01


def loss(logits, targets=None, target_index=None, target_prob=None, mask=None, mask_index=None, weights=None,
         upstream=None):
    """(loss, gradient, bound of the loss's fp32 error, bound of the gradient's), in 64 bits.

    Bounds: exp(z - M) through exp2: the difference and its product with
    log2(e) are rounded (2 half steps of a magnitude up to the spread, times
    ln 2 / ln 2), the constant (one more), the instruction is good to 2^-21; a
    sum of n terms in any order adds n half steps (n = V here)."""
    z = logits.double()
    R, V = z.shape
    a = allowed(R, V, mask, mask_index)
    t = torch.zeros(R, V, dtype=torch.double)
    terms = torch.ones(R, V, dtype=torch.double)
    if targets is not None:
        t = targets.double().clone()
    else:
        ti = target_index if target_index.dim() == 2 else target_index[:, None]
        tp = None if target_prob is None else (target_prob if target_prob.dim() == 2 else target_prob[:, None])
        for r in range(R):
            for k in range(ti.shape[1]):
                j = int(ti[r, k])
                if 0 <= j < V:
                    t[r, j] += 1.0 if tp is None else float(tp[r, k])
                    terms[r, j] += 1
    t[~a] = 0
    w = torch.ones(R, dtype=torch.double) if weights is None else weights.double()
    up = torch.ones(R, dtype=torch.double) if upstream is None else upstream.double()
    out = torch.zeros(R, dtype=torch.double)
    grad = torch.zeros(R, V, dtype=torch.double)
    b_loss, b_grad = torch.zeros(R, dtype=torch.double), torch.zeros(R, V, dtype=torch.double)
    for r in range(R):
        zr = z[r][a[r]]
        if w[r] == 0 or zr.numel() == 0 or (zr == -math.inf).all():
            continue
        tr = t[r][a[r]]
        m = zr.max() if not zr.isnan().any() else torch.tensor(math.nan, dtype=torch.double)
        e = torch.exp(zr - m)
        s, mass = e.sum(), tr.sum()
        # M - z is formed in fp32: from FLT_MAX and half a step on it is infinite (2e37 + 3.4028e38 > 3.4029e38)
        apart = torch.where(m - zr >= 2.0 ** 128 - 2.0 ** 103, torch.full_like(zr, math.inf), m - zr)
        d = torch.where(tr != 0, tr * apart, torch.zeros_like(zr))
        log_s = torch.log(s) if mass != 0 else torch.zeros(())
        out[r] = w[r] * (mass * log_s + d.sum())
        p = mass * e / s if mass != 0 else torch.zeros_like(e)
        g = w[r] * up[r] * (p - tr)
        grad[r][a[r]] = g
        spread = (m - zr).clamp(max=104.0)  # beyond, exp is below fp32
        rel_exp = 2.0 ** -21 + 3 * EPS32 * spread * 1.4427
        rel_s = float(((rel_exp * e).sum() / s)) + V * EPS32
        n = V + terms[r].max()
        mag = tr.abs().sum()
        b_loss[r] = abs(w[r]) * (abs(mass) * rel_s + 4 * EPS32 * mag * log_s.abs() + n * EPS32 * mag * (1 + log_s.abs())
                                 + (n + 4) * EPS32 * d.abs().sum() + mag * 2.0 ** -21)
        gb = abs(w[r] * up[r]) * (p.abs() * (rel_exp + rel_s + (n + 8) * EPS32) + (terms[r][a[r]] + 4) * EPS32 * tr.abs()
                                  + 2.0 ** -126)
        b_grad[r][a[r]] = gb
    return out, grad, b_loss, b_grad


def close(got, ref, bound, dtype=torch.float32):
    """got (any dtype) equals ref up to bound and one rounding to dtype; the
    same infinities and NaNs."""
    g, ref = got.detach().cpu().double(), ref.double()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(g), torch.isnan(ref)), "NaNs differ"
    inf = torch.isinf(ref)
    assert torch.equal(g[inf], ref[inf]), "infinities differ"
    assert torch.isfinite(g[fine]).all(), "not finite where the reference is"
    tol = bound.double() + half_step(dtype) * (ref.abs() + bound.double()) + tiny(dtype)
    bad = ((g - ref).abs() > tol) & fine
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, worst {float(((g - ref).abs() / tol)[bad].max()):.3g} "
                           f"times the bound, first at {bad.nonzero()[0].tolist()}")
