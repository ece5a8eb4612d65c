"""Cases of the policy-logit and optimizer operators: what is measured, their plain forms, and their definition in 64 bits.

Three operators of chineseai_b200 over four kinds of case:
  process  logits.process_logits: penalties for repeated tokens, sparse biases and packed masks on rows of logits
  loss     logits.policy_loss_grad: the masked softmax cross entropy and its gradient in one call
  ploss    logits.policy_loss: the same loss through autograd (forward, then backward)
  adamw    optim.MultiAdamW: an AdamW step over many tensors, states in 32 or in 8 bits
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
BETA1, BETA2, EPS, WEIGHT_DECAY, LR = 0.9, 0.999, 1e-8, 1e-4, 1e-3  # the AZ trainer's
BLOCK = 256       # elements of one 8-bit state block
E4M3_MAX = 448.0  # largest e4m3 value
E4M3_MIN = 2.0 ** -9  # smallest e4m3 value above zero
NORMAL = 2.0 ** -126  # smallest normal fp32


def listed():
    return [
        # one board at the root of a game: pick among the legal moves of the 2086-move space, played moves penalised
        {"name": "process_one_board", "op": "process", "rows": 1, "vocab": 2086, "hist": 48, "bias": 0, "type": "f32",
         "grammars": 1},
        # a leaf batch of the search: every board has its own legal moves and its game's moves so far
        {"name": "process_leaf_batch", "op": "process", "rows": 1024, "vocab": 2086, "hist": 200, "bias": 0, "type": "f32",
         "grammars": 1024},
        # a decoding batch over a large vocabulary: long histories, a bias list, a few grammars shared by the rows
        {"name": "process_decode", "op": "process", "rows": 64, "vocab": 131072, "hist": 8192, "bias": 64, "type": "bf16",
         "grammars": 4},
        # many rows of an odd vocabulary, half precision
        {"name": "process_odd_vocab", "op": "process", "rows": 2048, "vocab": 50001, "hist": 512, "bias": 16, "type": "f16",
         "grammars": 16},
        # a few boards over the 90 x 90 from-to space, visit counts of the searched moves as lists
        {"name": "loss_few_boards", "op": "loss", "rows": 8, "vocab": 8100, "targets": 40, "type": "f32", "grammars": 8},
        # the AZ training batch over the move space: dense visit distributions, legal-move masks
        {"name": "loss_az_batch", "op": "loss", "rows": 1024, "vocab": 2086, "targets": -1, "type": "f32", "grammars": 1024},
        # next-token training rows over a large vocabulary, hard labels
        {"name": "loss_large_vocab", "op": "loss", "rows": 4096, "vocab": 131072, "targets": 1, "type": "bf16", "grammars": 0},
        # distillation lists over an odd vocabulary through autograd
        {"name": "ploss_distil", "op": "ploss", "rows": 500, "vocab": 32003, "targets": 64, "type": "bf16", "grammars": 2},
        # the AZ trainer's 17 leaves at hidden 128, fp32 throughout
        {"name": "adamw32_az_leaves", "op": "adamw", "set": "az", "count": 17, "shapes": 0, "top": 0, "bits": 32, "param": "f32",
         "grad": "f32", "copy": False, "align": 64},
        # a few hundred matrices and vectors, fp32 masters, bf16 gradients and bf16 copies for the next forward
        {"name": "adamw32_mixed", "op": "adamw", "set": "spread", "count": 300, "shapes": 7, "top": 4194304, "bits": 32,
         "param": "f32", "grad": "bf16", "copy": True, "align": 64},
        # the policy/value ResNet's tensors, 8-bit states
        {"name": "adamw8_resnet", "op": "adamw", "set": "resnet", "count": 52, "shapes": 0, "top": 0, "bits": 8, "param": "f32",
         "grad": "f32", "copy": False, "align": 256},
        # large matrices, 8-bit states, bf16 gradients
        {"name": "adamw8_large", "op": "adamw", "set": "large", "count": 16, "shapes": 0, "top": 16777216, "bits": 8,
         "param": "f32", "grad": "bf16", "copy": False, "align": 256},
    ]


def _log(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["process", "loss", "ploss", "adamw", "adamw"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "adamw":
        bits = rng.choice([8, 32])
        param = rng.choice(["f32", "f32", "bf16"])
        return {"op": op, "set": "spread", "count": _log(rng, 1, 600), "shapes": rng.randrange(1 << 20),
                "top": _log(rng, 64, 1 << 21), "bits": bits, "param": param, "grad": rng.choice(["f32", "bf16", "f16"]),
                "copy": param == "f32" and rng.random() < 0.4, "align": 256 if bits == 8 else rng.choice([1, 64])}
    vocab = rng.choice([2086, 8100, _log(rng, 2, 262144), _log(rng, 200, 200000) | 1])
    rows = max(1, _log(rng, 1, max(2, min(8192, (1 << 28) // vocab))))
    grammars = rng.choice([0, 1, rows, _log(rng, 1, 64)])
    if op == "process":
        long = _log(rng, 512, 32768 if rows <= 512 else 2048)
        return {"op": op, "rows": rows, "vocab": vocab, "hist": rng.choice([0, _log(rng, 1, 512), long]),
                "bias": rng.choice([0, min(vocab, _log(rng, 1, 300))]), "type": kind, "grammars": grammars}
    dense = rows * vocab <= 1 << 27 and rng.random() < 0.3
    listed_targets = min(vocab, rng.choice([1, _log(rng, 2, 128)]))
    return {"op": op, "rows": rows, "vocab": vocab, "targets": -1 if dense else listed_targets, "type": kind,
            "grammars": grammars}


# ---- inputs -------------------------------------------------------------------------------------------------------
def _sizes(case):
    """Element counts of the case's tensors."""
    if case["set"] == "az":  # the 17 leaves of the AZ training step at hidden 128
        h = 128
        return [1545 * h, 7 * h, h, 96 * h, 96, 3 * 96, 57702 * 64, 3 * 128, 16 * 128, 2086, 32, 16 * h, 2086 * 16, 32 * h,
                2086 * 32, 2596273, 934976]
    if case["set"] == "resnet":  # stem, 10 blocks of two convolutions, heads: weights and biases
        return [128 * 15 * 9, 128] + [128 * 128 * 9, 128] * 20 + [256, 2, 2086 * 180, 2086, 128, 1, 256 * 90, 256, 256, 1]
    if case["set"] == "large":
        return [case["top"]] * case["count"]
    r = random.Random(case["shapes"])  # matrices and vectors of all sizes, odd ones among them
    return [_log(r, 1, case["top"]) for _ in range(case["count"])]


def _places(sizes, align):
    """Start of every tensor in the flat buffer, and the buffer's length."""
    at, starts = 0, []
    for n in sizes:
        starts.append(at)
        at += -(-n // align) * align
    return starts, at


def _mask_words(rows, vocab, dense, gen):
    """Packed masks [rows][ceil(vocab / 32)]: a row allows about its share `dense` of the vocabulary."""
    words = -(-vocab // 32)
    bits = torch.rand(rows, words * 32, generator=gen, device=DEV) < dense[:, None]
    weights = torch.ones(32, dtype=torch.int64, device=DEV) << torch.arange(32, device=DEV)
    packed = (bits.view(rows, words, 32).long() * weights).sum(2)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)


def _shares(case, gen):
    """The share of the vocabulary that each grammar allows: legal moves are few; other grammars allow little or nearly all."""
    g = case["grammars"]
    if case["vocab"] in (2086, 8100):
        return torch.full((g,), 40.0 / case["vocab"], device=DEV)
    return torch.where(torch.arange(g, device=DEV) % 2 == 0, 0.98, 0.02)


def _prepare_rows(case, gen):
    R, V, G = case["rows"], case["vocab"], case["grammars"]
    s = {"case": case, "status": torch.zeros(1, dtype=torch.int32, device=DEV), "mask": None, "mask_index": None}
    s["logits"] = (2.5 * torch.randn(R, V, generator=gen, device=DEV)).to(TYPES[case["type"]])
    if G:
        s["mask"] = _mask_words(G, V, _shares(case, gen), gen)
        if 1 < G != R:  # shared by the rows; one row in 8 has no grammar
            s["mask_index"] = torch.where(torch.arange(R, device=DEV) % 8 == 7, -1,
                                          torch.randint(0, G, (R,), generator=gen, device=DEV)).to(torch.int32)
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    if case["op"] == "adamw":
        return _prepare_adamw(case, gen)
    s = _prepare_rows(case, gen)
    R, V = case["rows"], case["vocab"]
    if case["op"] == "process":
        L, K = case["hist"], case["bias"]
        s.update(dict.fromkeys(("history", "lengths", "prompt", "rep", "freq", "pres", "bias_tokens", "bias_values")))
        if L:  # tokens repeat, as text and play do: most come from a small part of the vocabulary
            u = torch.rand(R, L, generator=gen, device=DEV, dtype=torch.float64)
            s["history"] = (u * u * u * V).to(torch.int32).clamp_(0, V - 1)
            s["lengths"] = torch.randint(L // 2, L + 1, (R,), generator=gen, device=DEV).to(torch.int32)
            s["prompt"] = (s["lengths"] * torch.rand(R, generator=gen, device=DEV)).to(torch.int32)
            s["rep"] = 1.0 + 0.3 * torch.rand(R, generator=gen, device=DEV)
            s["freq"] = 0.2 * torch.rand(R, generator=gen, device=DEV)
            s["pres"] = 0.5 * torch.rand(R, generator=gen, device=DEV)
        if K:  # distinct tokens, a value each
            first = torch.randint(0, V, (R, 1), generator=gen, device=DEV)
            s["bias_tokens"] = ((first + torch.arange(K, device=DEV) * max(1, V // K)) % V).to(torch.int32)
            s["bias_values"] = 3.0 * torch.randn(R, K, generator=gen, device=DEV)
        return s
    K = case["targets"]
    # the mean over the rows; half-precision gradients carry a loss scale instead, or they would fall under fp16's range
    s["weights"] = (0.1 + torch.rand(R, generator=gen, device=DEV)) * (256.0 if case["type"] == "f16" else 1.0 / R)
    s["targets"] = s["index"] = s["prob"] = None
    if K < 0:  # visit shares over the whole space
        t = torch.rand(R, V, generator=gen, device=DEV) ** 4
        s["targets"] = t / t.sum(1, keepdim=True)
    else:
        first = torch.randint(0, V, (R, 1), generator=gen, device=DEV)
        s["index"] = ((first + torch.arange(K, device=DEV) * max(1, V // K)) % V).to(torch.int32)
        if K > 1:
            p = torch.rand(R, K, generator=gen, device=DEV) ** 2
            s["prob"] = p / p.sum(1, keepdim=True)
    if case["op"] == "ploss":
        s["logits"].requires_grad_(True)
        s["upstream"] = torch.rand(R, generator=gen, device=DEV) + 0.5
    return s


def _prepare_adamw(case, gen):
    sizes = _sizes(case)
    starts, total = _places(sizes, case["align"])
    real = torch.ones(total, device=DEV)
    ends = [a + n for a, n in zip(starts, sizes)]
    for a, b in zip(ends, starts[1:] + [total]):  # what fills up to the next tensor's start stays zero
        real[a:b] = 0
    randn = lambda: torch.randn(total, generator=gen, device=DEV) * real  # noqa: E731
    g = 0.01 * randn()
    s = {"case": case, "step": 100, "param": (0.05 * randn()).to(TYPES[case["param"]]), "grad": g.to(TYPES[case["grad"]])}
    s["copy"] = torch.zeros(total, dtype=torch.bfloat16, device=DEV) if case["copy"] else None
    m, u = 0.003 * randn(), 0.01 * (0.2 + torch.rand(total, generator=gen, device=DEV)) * real
    if case["bits"] == 8:
        s["m"], s["m_scale"] = _encode(m.view(-1, BLOCK), False)
        s["v"], s["v_scale"] = _encode(u.view(-1, BLOCK), True)
    else:
        s["m"], s["v"] = m, u * u
    if own:
        from chineseai_b200.optim import MultiAdamW

        def cut(flat, each=1):
            return None if flat is None else [flat[a // each:-(-(a + n) // each)] for a, n in zip(starts, sizes)]

        state = {"m": cut(s["m"]), "v": cut(s["v"])}
        if case["bits"] == 8:
            state.update(m_scale=cut(s["m_scale"], BLOCK), v_scale=cut(s["v_scale"], BLOCK))
        s["plan"] = MultiAdamW(cut(s["param"]), cut(s["grad"]), lr=LR, beta1=BETA1, beta2=BETA2, eps=EPS,
                               weight_decay=WEIGHT_DECAY, state_bits=case["bits"], state=state, copies=cut(s["copy"]),
                               step=s["step"])
    return s


# ---- plain forms --------------------------------------------------------------------------------------------------
def _allowed(s):
    """bool [rows or 1][vocab] of the packed masks, or None."""
    if s["mask"] is None:
        return None
    bits = (s["mask"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
    a = bits.view(len(s["mask"]), -1)[:, :s["case"]["vocab"]].bool()
    if s["mask_index"] is not None:
        a = a[s["mask_index"].clamp(min=0).long()] | (s["mask_index"] < 0)[:, None]
    return a


def _process(s):
    x = s["logits"].float()
    R, V = x.shape
    if s["history"] is not None:
        at = torch.arange(s["history"].shape[1], device=DEV)
        live = at < s["lengths"][:, None]
        tok = torch.where(live, s["history"].long(), V)
        out = (live & (at >= s["prompt"][:, None])).float()
        count = torch.zeros(R, V + 1, device=DEV).scatter_add_(1, tok, out)[:, :V]
        seen = torch.zeros(R, V + 1, dtype=torch.bool, device=DEV).scatter_(1, tok, True)[:, :V]
        rep = s["rep"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        x = x - s["freq"][:, None] * count
        x = x - s["pres"][:, None] * (count > 0)
    if s["bias_tokens"] is not None:
        x = x.scatter_add(1, s["bias_tokens"].long(), s["bias_values"])
    a = _allowed(s)
    if a is not None:
        x = torch.where(a, x, -math.inf)
    return x.to(s["logits"].dtype)


def _loss(s, upstream=None):
    z = s["logits"].detach().float()
    R, V = z.shape
    a = _allowed(s)
    if s["targets"] is not None:
        t = s["targets"]
    else:
        p = s["prob"] if s["prob"] is not None else torch.ones_like(s["index"], dtype=torch.float32)
        t = torch.zeros(R, V, device=DEV).scatter_add_(1, s["index"].long(), p)
    if a is not None:
        z = torch.where(a, z, -math.inf)
        t = torch.where(a, t, 0.0)
    top = z.amax(1, keepdim=True)
    some = top > -math.inf
    z = torch.where(some, z - top, -math.inf)
    e = torch.exp(z)
    total = torch.where(some, e.sum(1, keepdim=True), 1.0)
    mass = t.sum(1, keepdim=True)
    each = torch.where(t != 0, t * (torch.log(total) - z), 0.0)
    loss = s["weights"] * torch.where(some, each, 0.0).sum(1)
    w = s["weights"] if upstream is None else s["weights"] * upstream
    grad = w[:, None] * (mass * (e / total) - torch.where(some, t, 0.0))
    return loss, grad.to(s["logits"].dtype)


def _encode(x, floor):
    """The blocks' e4m3 values and scales of x [blocks][256]; values above zero do not fall under `floor`."""
    top = x.abs().amax(1, keepdim=True)
    scale = top * (1.0 / E4M3_MAX)
    live = scale >= NORMAL
    q = x * torch.where(live, torch.full_like(top, E4M3_MAX) / top, 0.0)
    q = q.clamp(-E4M3_MAX, E4M3_MAX)
    if floor:
        q = torch.where((x > 0) & live, q.clamp(min=E4M3_MIN), q)
    return q.to(torch.float8_e4m3fn).view(-1), torch.where(live, scale, 0.0).view(-1)


def _adamw(s):
    c = s["case"]
    s["step"] += 1
    corr1, corr2 = 1.0 / (1.0 - BETA1 ** s["step"]), 1.0 / (1.0 - BETA2 ** s["step"])
    p, g = s["param"].float(), s["grad"].float()
    if c["bits"] == 8:
        m = (s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        u = (s["v"].float().view(-1, BLOCK) * s["v_scale"][:, None]).view(-1)
        v = u * u
    else:
        m, v = s["m"], s["v"]
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * g) * (1.0 - BETA2)
    if c["bits"] == 8:
        u = torch.sqrt(v)
        den = u * math.sqrt(corr2) + EPS
    else:
        den = torch.sqrt(v * corr2) + EPS
    p = p * (1.0 - LR * WEIGHT_DECAY) - ((m * corr1) / den) * LR
    s["param"].copy_(p)
    if s["copy"] is not None:
        s["copy"].copy_(p)
    if c["bits"] == 8:
        for name, x, floor in (("m", m, False), ("v", u, True)):
            q, scale = _encode(x.view(-1, BLOCK), floor)
            s[name].copy_(q)
            s[name + "_scale"].copy_(scale)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return _adamw_out(s)


def _adamw_out(s):
    return {k: s[k] for k in ("param", "m", "v", "m_scale", "v_scale", "copy") if s.get(k) is not None}


def run(s):
    op = s["case"]["op"]
    if own:
        if op == "adamw":
            s["plan"].step()
            return _adamw_out(s)
        from chineseai_b200 import logits
        if op == "process":
            return logits.process_logits(
                s["logits"], history=s["history"], lengths=s["lengths"], prompt_lengths=s["prompt"], repetition=s["rep"],
                frequency=s["freq"], presence=s["pres"], bias_tokens=s["bias_tokens"], bias_values=s["bias_values"],
                mask=s["mask"], mask_index=s["mask_index"], status=s["status"])
        named = dict(target_index=s["index"], target_prob=s["prob"], mask=s["mask"], mask_index=s["mask_index"],
                     weights=s["weights"], status=s["status"])
        if op == "loss":
            return logits.policy_loss_grad(s["logits"], s["targets"], **named)
        loss = logits.policy_loss(s["logits"], s["targets"], **named)
        return loss.detach(), torch.autograd.grad(loss, s["logits"], s["upstream"])[0]
    if op == "adamw":
        return _adamw(s)
    return _process(s) if op == "process" else _loss(s, s.get("upstream"))


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        each = 2 * BYTES[case["param"]] + BYTES[case["grad"]] + (2 if case["copy"] else 0)
        each += 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": n * each, "flops": 16 * n}
    R, V, G, b = case["rows"], case["vocab"], case["grammars"], BYTES[case["type"]]
    share = 1.0  # of the logits that are read: what no mask excludes
    if G:
        share = 40.0 / V if V in (2086, 8100) else (0.98 * ((G + 1) // 2) + 0.02 * (G // 2)) / G
        share = share * 7 / 8 + 1 / 8 if 1 < G != R else share
    moved = R * V * b * (share + 1) + 4 * min(G, R) * (-(-V // 32))
    if case["op"] == "process":
        return {"bytes": moved + 4 * R * case["hist"] * 3 / 4 + 8 * R * case["bias"], "flops": 8 * R * V}
    K = case["targets"]
    moved += R * V * 4 * share if K < 0 else R * K * (8 if K > 1 else 4)
    if case["op"] == "ploss":  # the backward pass reads the logits again
        moved += R * V * b * share
    return {"bytes": moved + 8 * R, "flops": 10 * R * V}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------
def _unpacked(s, V):
    """The masks' truth values, word by word from the low bit up."""
    if s["mask"] is None:
        return None
    words = s["mask"].long() & 0xFFFFFFFF
    at = torch.arange(V, device=DEV)
    a = torch.remainder(torch.div(words[:, at // 32], 2 ** (at % 32), rounding_mode="floor"), 2) == 1
    if s["mask_index"] is None:
        return a.expand(s["case"]["rows"], V)
    free = torch.ones(1, V, dtype=torch.bool, device=DEV)
    return torch.cat([free, a])[s["mask_index"].long() + 1]


def _exact_process(s, lo, hi, a):
    z = s["logits"][lo:hi].double()
    R, V = z.shape
    count, seen, extra = torch.zeros_like(z), torch.zeros_like(z), torch.zeros_like(z)
    if s["history"] is not None:
        at = torch.arange(s["history"].shape[1], device=DEV)[None]
        rows, at = torch.nonzero(at < s["lengths"][lo:hi, None], as_tuple=True)
        flat = rows * V + s["history"][lo:hi][rows, at].long()
        said = (at >= s["prompt"][lo:hi][rows].long()).double()
        seen = torch.bincount(flat, minlength=R * V).view(R, V)
        count = torch.bincount(flat, weights=said, minlength=R * V).view(R, V)
        rep, freq, pres = (s[k][lo:hi].double()[:, None] for k in ("rep", "freq", "pres"))
        z = torch.where(seen > 0, z * torch.where(z > 0, 1 / rep, rep), z) - freq * count - pres * (count > 0).double()
    if s["bias_tokens"] is not None:
        where = (torch.arange(R, device=DEV)[:, None] * V + s["bias_tokens"][lo:hi].long()).view(-1)
        extra = torch.bincount(where, weights=s["bias_values"][lo:hi].double().reshape(-1), minlength=R * V).view(R, V)
        z = z + extra
    if a is not None:
        z = z.masked_fill(~a[lo:hi], -math.inf)
    return z


def _exact_loss(s, lo, hi, a):
    z = s["logits"].detach()[lo:hi].double()
    R, V = z.shape
    if s["targets"] is not None:
        t = s["targets"][lo:hi].double()
    else:
        p = (torch.ones_like(s["index"]) if s["prob"] is None else s["prob"])[lo:hi].double()
        where = (torch.arange(R, device=DEV)[:, None] * V + s["index"][lo:hi].long()).view(-1)
        t = torch.bincount(where, weights=p.reshape(-1), minlength=R * V).view(R, V)
    if a is not None:
        t = t * a[lo:hi]
        z = z.masked_fill(~a[lo:hi], -math.inf)
    some = torch.isfinite(z).any(1, keepdim=True)
    lse = torch.logsumexp(z, 1, keepdim=True)
    logp = torch.where(some & torch.isfinite(z), z - lse, 0.0)
    prob = torch.where(some & torch.isfinite(z), logp.exp(), 0.0)
    w = s["weights"][lo:hi].double()
    loss = -w * (t * logp).sum(1)
    if "upstream" in s:
        w = w * s["upstream"][lo:hi].double()
    return loss, w[:, None] * (t.sum(1, keepdim=True) * prob - torch.where(some, t, 0.0))


def _exact_blocks(x, lowest):
    x = x.view(-1, BLOCK)
    scale = x.abs().amax(1) / E4M3_MAX
    scale = torch.where(scale < NORMAL, 0.0, scale)
    q = torch.where(scale[:, None] > 0, x / scale[:, None], 0.0)
    q = torch.where((x > 0) & (q > 0), q.clamp(min=lowest), q)
    return q.float().clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).double().view(-1), scale


def _exact_adamw(s):
    c, t = s["case"], s["step"] + 1
    p, g = s["param"].double(), s["grad"].double()
    if c["bits"] == 8:
        each = lambda k: s[k].double() * s[k + "_scale"].double().repeat_interleave(BLOCK)  # noqa: E731
        m, v = each("m"), each("v") ** 2
    else:
        m, v = s["m"].double(), s["v"].double()
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    p = p - LR * WEIGHT_DECAY * p - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
    out = {"param": p}
    if c["bits"] == 8:
        out["m"], out["m_scale"] = _exact_blocks(m, 0.0)
        out["v"], out["v_scale"] = _exact_blocks(torch.sqrt(v), E4M3_MIN)
    else:
        out["m"], out["v"] = m, v
    if s["copy"] is not None:
        out["copy"] = p
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    if case["rows"] * case["vocab"] > 1 << 30:
        return None
    a = _unpacked(s, case["vocab"])
    step = max(1, (1 << 26) // case["vocab"])
    f = _exact_process if case["op"] == "process" else _exact_loss
    parts = [f(s, lo, min(case["rows"], lo + step), a) for lo in range(0, case["rows"], step)]
    if case["op"] == "process":
        return torch.cat(parts)
    return torch.cat([x for x, _ in parts]), torch.cat([x for _, x in parts])
