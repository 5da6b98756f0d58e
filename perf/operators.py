"""The operators of a training step of a categorical model, as a user calls them, and their plain forms.

Four operators, in the order of a step:

* ``logprob``     log-probabilities of labels (and the entropy) from logits, and their gradient
* ``preference``  a preference loss over pairs of sequences (paired log ratios) with its gradient
* ``policy``      a clipped policy loss with a KL term and an entropy bonus, with its gradient
* ``adamw``       an AdamW step over many tensors at once, states in 32 or in 8 bits, clipped by the global gradient norm

``own`` False: elementary torch operations; True: the calls of ``dorpatch_amd``.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 128                     # elements that share a scale where AdamW's states have 8 bits; also the padding of a tensor's part
BETA1, BETA2, EPS, LR, DECAY = 0.9, 0.999, 1e-8, 1e-3, 0.05
CLIP_LOW, CLIP_HIGH, KL, ENTROPY = 0.2, 0.28, 0.04, 0.01
PREF_BETA, SMOOTHING = 0.1, 0.1
FIRST_STEP = 100                # the states that prepare() makes have this many steps behind them

#: the stages of the repository's ResNetV2-50 backbone: (blocks, channels in, in the middle, out)
STAGES = ((3, 64, 64, 256), (4, 256, 128, 512), (6, 512, 256, 1024), (3, 1024, 512, 2048))


def listed():
    return [
        # the classes of one masked image: the smallest call, latency alone
        {"name": "logprob 1x1000 fp32", "op": "logprob", "rows": 1, "vocab": 1000, "dtype": "fp32", "grad": False},
        # a step's 64 images x 32 masks over the 1000 classes, with the gradient: rows of a likelihood loss
        {"name": "logprob 2048x1000 fp32 grad", "op": "logprob", "rows": 2048, "vocab": 1000, "dtype": "fp32", "grad": True},
        # log-probabilities of a reference model over a large vocabulary, forward alone
        {"name": "logprob 4096x131072 bf16", "op": "logprob", "rows": 4096, "vocab": 131072, "dtype": "bf16", "grad": False},
        # pairs of cell selections of a patch: 1024 cells of 7 x 7 pixels, 20 to 60 picked
        {"name": "preference 64 pairs, 1024 fp32", "op": "preference", "pairs": 64, "length": 40, "vocab": 1024, "dtype": "fp32"},
        # ordinary pairs of answers of a few hundred tokens, an odd vocabulary: rows that start off 16 bytes
        {"name": "preference 8 pairs, 50001 fp16", "op": "preference", "pairs": 8, "length": 200, "vocab": 50001, "dtype": "fp16"},
        # the largest: long answers, large vocabulary
        {"name": "preference 4 pairs, 131072 bf16", "op": "preference", "pairs": 4, "length": 480, "vocab": 131072, "dtype": "bf16"},
        # a policy over the 2520 double masks, one draw of 128, a tenth of the masks not allowed
        {"name": "policy 128x2520 fp32", "op": "policy", "rows": 128, "vocab": 2520, "dtype": "fp32"},
        # an ordinary batch of tokens
        {"name": "policy 2048x32768 bf16", "op": "policy", "rows": 2048, "vocab": 32768, "dtype": "bf16"},
        # the largest
        {"name": "policy 4096x131072 bf16", "op": "policy", "rows": 4096, "vocab": 131072, "dtype": "bf16"},
        # patterns and masks of 64 images of 224 x 224: 128 tensors that are optimised side by side
        {"name": "adamw 64 patches fp32", "op": "adamw", "set": "patches", "size": 64, "dtype": "fp32", "bits": 32, "clip": False},
        # the 153 tensors of the backbone, as its fine-tuning takes them: clipped by the global norm, no decay on vectors
        {"name": "adamw backbone fp32 clip", "op": "adamw", "set": "backbone", "size": 1, "classes": 1000, "dtype": "fp32", "bits": 32, "clip": True},
        # a large model's matrices in bf16, states in 8 bits, clipped
        {"name": "adamw 2^28 bf16 8-bit clip", "op": "adamw", "set": "matrices", "size": 2 ** 28, "dtype": "bf16", "bits": 8, "clip": True},
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["logprob", "preference", "policy", "adamw"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "adamw":
        which = rng.choice(["patches", "backbone", "matrices"])
        size = {"patches": _log_uniform(rng, 1, 256), "backbone": rng.randint(1, 4), "matrices": _log_uniform(rng, 1000, 2 ** 28)}[which]
        case = {"op": op, "set": which, "size": size, "dtype": rng.choice(["fp32", "bf16"]), "bits": rng.choice([8, 32]), "clip": rng.random() < 0.5}
        return {**case, "classes": _log_uniform(rng, 2, 20000)} if which == "backbone" else case
    vocab = _log_uniform(rng, 500, 131072)
    most = 2 ** (28 if dtype == "fp32" else 29) // vocab
    if op == "preference":
        pairs = _log_uniform(rng, 1, 64)
        return {"op": op, "pairs": pairs, "length": _log_uniform(rng, 2, max(2, min(600, most // (2 * pairs)))), "vocab": vocab, "dtype": dtype}
    rows = _log_uniform(rng, 1, min(16384, most))
    case = {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype}
    if op == "logprob":
        case["grad"] = rng.random() < 0.5
    return case


# ---------------------------------------------------------------- sizes that a case stands for
def _lengths(case):
    """The 2 * pairs lengths of a preference case: ragged, by the case alone."""
    return [max(1, int(case["length"] * (0.4 + 1.2 * ((0.618 * (i + 1)) % 1.0)))) for i in range(2 * case["pairs"])]


def _shapes(case):
    """(shapes with decay, shapes without) of an adamw case."""
    n = case["size"]
    if case["set"] == "patches":
        return [(3, 224, 224), (1, 224, 224)] * n, []
    if case["set"] == "matrices":
        cols = max(1, min(8192, math.isqrt(n // 8)))
        return [(max(1, n // (8 * cols)), cols)] * 8, [(cols,)] * 8
    matrices, vectors = [], []
    for _ in range(n):
        matrices.append((64, 3, 7, 7))
        for blocks, first, mid, out in STAGES:
            for b in range(blocks):
                c = first if b == 0 else out
                matrices += [(out, c, 1, 1)] * (b == 0) + [(mid, c, 1, 1), (mid, mid, 3, 3), (out, mid, 1, 1)]
                vectors += [(c,), (c,), (mid,), (mid,), (mid,), (mid,)]
        matrices.append((case["classes"], 2048, 1, 1))
        vectors += [(2048,), (2048,), (case["classes"],)]
    return matrices, vectors


def _padded(shapes):
    return sum(-(-math.prod(s) // BLOCK) * BLOCK for s in shapes)


def _rows(case):
    return sum(_lengths(case)) if case["op"] == "preference" else case["rows"]


def work(case):
    """Each input read once, each output written once; an element of logits costs an exponential, its sum and, with a gradient, three
    operations more; an element of AdamW about fourteen."""
    if case["op"] == "adamw":
        n = sum(math.prod(s) for part in _shapes(case) for s in part)
        e = 4 if case["dtype"] == "fp32" else 2
        states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": n * (3 * e + states), "flops": 14 * n}
    rows, e = _rows(case), 4 if case["dtype"] == "fp32" else 2
    n = rows * case["vocab"]
    grad = case["op"] != "logprob" or case["grad"]
    small = {"logprob": 8 + 4 + 4 + (4 if grad else 0), "preference": 8, "policy": 8 + 4 * 4 + 3 * 4}[case["op"]]
    return {"bytes": n * e * (2 if grad else 1) + rows * small, "flops": n * (7 if grad else 4)}


# ---------------------------------------------------------------- what a program has in hand
def _logits(gen, rows, vocab, dtype, labels, ban):
    """Logits as a model gives them: spread over about +-10, the label's raised; `ban`: that share of the others is -inf (not allowed)."""
    x = torch.empty(rows, vocab, device="cuda", dtype=dtype)
    step = max(1, 2 ** 26 // vocab)
    for r in range(0, rows, step):
        part = torch.randn(min(step, rows - r), vocab, device="cuda", generator=gen) * 2.5
        if ban:
            part.masked_fill_(torch.rand(part.shape, device="cuda", generator=gen) < ban, -math.inf)
        lift = torch.rand(part.shape[0], 1, device="cuda", generator=gen) * 10
        part.scatter_(1, labels[r:r + step, None], lift)
        x[r:r + step] = part
    return x


def _label_logp(x, labels):
    """log-probabilities of the labels, 64 bits, a band of rows at a time."""
    out = torch.empty(x.shape[0], device=x.device, dtype=torch.float64)
    step = max(1, 2 ** 26 // x.shape[1])
    for r in range(0, x.shape[0], step):
        part = x[r:r + step].double()
        out[r:r + step] = part.gather(1, labels[r:r + step, None])[:, 0] - part.logsumexp(1)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "adamw":
        return _prepare_adamw(case, gen, dtype)
    rows, vocab = _rows(case), case["vocab"]
    labels = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
    x = _logits(gen, rows, vocab, dtype, labels, 0.1 if case["op"] == "policy" and vocab < 8192 else 0.0)
    state = {"case": case, "logits": x}
    if case["op"] == "logprob":
        state["g"] = torch.randn(rows, device="cuda", generator=gen)
    elif case["op"] == "preference":
        bounds = [0]
        for n in _lengths(case):
            bounds.append(bounds[-1] + n)
        state["cu_seqlens"] = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    else:
        logp = _label_logp(x, labels)
        # the ratio to the policy that drew the label; no draw lies on an edge of the clip range, where its gradient jumps
        shift = torch.randn(rows, device="cuda", generator=gen, dtype=torch.float64) * 0.2
        for edge in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
            shift = torch.where((shift - edge).abs() < 1e-3, torch.full_like(shift, edge + 2e-3), shift)
        state["old_logp"] = (logp - shift).float()
        state["ref_logp"] = (logp + torch.randn(rows, device="cuda", generator=gen) * 0.1).float()
        state["advantage"] = torch.randn(rows, device="cuda", generator=gen)
        state["weight"] = torch.rand(rows, device="cuda", generator=gen) * 0.5 + 0.5
    if rows > 1:                # prompts and padding: rows that count for nothing
        labels = torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.1, torch.full_like(labels, -100), labels)
    state["labels"] = labels
    if case["op"] == "preference":      # what the reference model said: near what the model says
        logp = torch.where(labels < 0, 0.0, _label_logp(x, labels.clamp(min=0)))
        sums = torch.stack([t.sum() for t in logp.split(_lengths(case))])
        state["ref_logp"] = (sums + torch.randn(len(sums), device="cuda", generator=gen) * 2).float()
    state["upstream"] = 1.0 if case["dtype"] == "fp16" else 1.0 / (case["pairs"] if case["op"] == "preference" else rows)   # fp16: a scaled loss
    return state


def _prepare_adamw(case, gen, dtype):
    """Parameters and gradients as views of two flat buffers (every tensor's part padded to a multiple of BLOCK), the ones with decay
    first; the states' buffers have the same places."""
    parts = _shapes(case)
    ends = [_padded(parts[0]), _padded(parts[0]) + _padded(parts[1])]
    flat = torch.zeros(ends[1], device="cuda", dtype=dtype)
    grads = torch.zeros(ends[1], device="cuda", dtype=dtype)
    m, v = torch.zeros(ends[1], device="cuda"), torch.zeros(ends[1], device="cuda")
    params, grad_views, at = [], [], 0
    for shape in parts[0] + parts[1]:
        n = math.prod(shape)
        scale = 10.0 ** (2 * torch.rand((), device="cuda", generator=gen) - 4)          # gradients of 1e-4 to 1e-2
        flat[at:at + n] = (torch.randn(n, device="cuda", generator=gen) * 0.05).to(dtype)
        grads[at:at + n] = (torch.randn(n, device="cuda", generator=gen) * scale).to(dtype)
        m[at:at + n] = torch.randn(n, device="cuda", generator=gen) * (scale * 0.25)
        v[at:at + n] = torch.randn(n, device="cuda", generator=gen).square() * (scale * scale * 0.1)
        params.append(flat[at:at + n].view(shape))
        grad_views.append(grads[at:at + n].view(shape))
        at += -(-n // BLOCK) * BLOCK
    state = {"case": case, "flat": flat, "grads": grads, "ends": ends, "steps": FIRST_STEP, "max_norm": 1.0 if case["clip"] else None}
    if case["bits"] == 8:
        r = torch.zeros(m.numel(), dtype=torch.int64, device="cuda")
        state["m"], state["m_scale"] = _to_8_bits(m, r, False)
        state["v"], state["v_scale"] = _to_8_bits(v, r, True)
    else:
        state["m"], state["v"] = m, v
    if own:                     # the handle that a program keeps
        from dorpatch_amd.optim import AdamW
        decay = [DECAY] * len(parts[0]) + [0.0] * len(parts[1])
        opt = AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=decay, state_bits=case["bits"], max_norm=state["max_norm"], seed=7)
        opt.load_state(state["m"], state["v"], FIRST_STEP, *([state["m_scale"], state["v_scale"]] if case["bits"] == 8 else []))
        state["opt"], state["grad_views"] = opt, grad_views
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    return {"logprob": _run_logprob, "preference": _run_preference, "policy": _run_policy, "adamw": _run_adamw}[state["case"]["op"]](state)


def _run_logprob(s):
    grad = s["case"]["grad"]
    if own:
        from dorpatch_amd import ops
        logp, entropy, stats = ops.label_logprob(s["logits"], s["labels"], want_entropy=True)
        if not grad:
            return {"logp": logp, "entropy": entropy}
        return {"logp": logp, "entropy": entropy, "dlogits": ops.label_logprob_bwd(s["logits"], s["labels"], stats, s["g"])}
    e, p, logp, entropy, dead = _softmax(s["logits"], s["labels"])
    out = {"logp": logp.float(), "entropy": entropy.float()}
    if grad:
        out["dlogits"] = _gradient(s["logits"], s["labels"], p, torch.where(dead, 0.0, s["g"]))
    return out


def _run_preference(s):
    if own:
        from dorpatch_amd import ops
        loss, dlogits, seq_logp = ops.preference_loss(s["logits"], s["labels"], s["cu_seqlens"], s["ref_logp"], PREF_BETA, s["upstream"],
                                                      label_smoothing=SMOOTHING)
        return {"loss": loss, "dlogits": dlogits, "seq_logp": seq_logp}
    e, p, logp, entropy, dead = _softmax(s["logits"], s["labels"])
    cu = s["cu_seqlens"].long()
    total = torch.cat([logp.new_zeros(1), logp.cumsum(0)])
    seq = total[cu[1:]] - total[cu[:-1]]
    ratio = seq - s["ref_logp"].double()
    h = PREF_BETA * (ratio[0::2] - ratio[1::2])
    loss = (1 - SMOOTHING) * (1 + (-h).exp()).log() + SMOOTHING * (1 + h.exp()).log()
    slope = s["upstream"] * PREF_BETA * (SMOOTHING / (1 + (-h).exp()) - (1 - SMOOTHING) / (1 + h.exp()))
    g = torch.stack([slope, -slope], 1).reshape(-1).repeat_interleave(cu[1:] - cu[:-1], output_size=logp.numel())
    return {"loss": loss.float(), "dlogits": _gradient(s["logits"], s["labels"], p, torch.where(dead, 0.0, g)), "seq_logp": seq.float()}


def _run_policy(s):
    if own:
        from dorpatch_amd import ops
        loss, dlogits, logp, entropy = ops.policy_loss(s["logits"], s["labels"], s["old_logp"], s["advantage"], CLIP_LOW, CLIP_HIGH, s["upstream"],
                                                       ref_logp=s["ref_logp"], kl_coef=KL, entropy_coef=ENTROPY, weight=s["weight"])
        return {"loss": loss, "dlogits": dlogits, "logp": logp, "entropy": entropy}
    e, p, logp, entropy, dead = _softmax(s["logits"], s["labels"])
    ratio = (logp - s["old_logp"].double()).exp()
    adv = s["advantage"].double()
    plain, clipped = -adv * ratio, -adv * ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
    far = s["ref_logp"].double() - logp
    loss = torch.maximum(plain, clipped) + KL * (far.exp() - far - 1) - ENTROPY * entropy
    slope = torch.where(plain >= clipped, plain, 0.0) + KL * (1 - far.exp())
    w = torch.where(dead, 0.0, s["upstream"] * s["weight"].double())
    # the entropy bonus: - ENTROPY * dH/dx = ENTROPY * p (log p + H)
    bonus = (w * ENTROPY).float()[:, None] * p * (e + entropy.float()[:, None])
    return {"loss": torch.where(dead, 0.0, loss).float(), "dlogits": _gradient(s["logits"], s["labels"], p, w * slope, bonus),
            "logp": logp.float(), "entropy": entropy.float()}


def _softmax(logits, labels):
    """(log p, finite where p is 0; p; label's log p in 64 bits; entropy in 64 bits; rows without a label), the last two zero there."""
    dead = labels < 0
    x = logits.float()
    x = x - x.amax(1, keepdim=True)
    e = x.exp()
    total = e.sum(1, keepdim=True)
    log_total = total.double().log()
    logp = x.gather(1, labels.clamp(min=0)[:, None]).double() - log_total
    x = x.clamp(min=-1e30)
    entropy = log_total - ((e * x).sum(1, keepdim=True) / total).double()
    return x - log_total.float(), e / total, torch.where(dead, 0.0, logp[:, 0]), torch.where(dead, 0.0, entropy[:, 0]), dead


def _gradient(logits, labels, p, g, more=None):
    """g (1[j = label] - p) + more, rounded to the logits' type."""
    d = p * (-g).float()[:, None]
    if more is not None:
        d += more
    return d.scatter_add_(1, labels.clamp(min=0)[:, None], g.float()[:, None]).to(logits.dtype)


# ---------------------------------------------------------------- AdamW
def _hash(n, seed, step, device):
    """32 random bits for each of n elements, from (seed, step, element)."""
    low = 0xFFFFFFFF
    i = torch.arange(n, device=device)
    key = _mix((seed * 0x9E3779B1 + step) & low)
    h = (i & low) ^ ((i >> 32) * 0x85EBCA77 & low) ^ key
    return _mix(h)


def _mix(h):
    low = 0xFFFFFFFF
    h = (h ^ (h >> 16)) * 0x9E3779B1 & low
    h = (h ^ (h >> 15)) * 0x85EBCA77 & low
    return h ^ (h >> 16)


def _to_8_bits(x, r, second):
    """x -> (e4m3 codes, a scale for each BLOCK): the scale is the power of two that puts the block's largest magnitude into [128, 256);
    rounding is up with the probability of the part cut off (r: 16 random bits).  A second moment over zero never becomes zero."""
    a = x.abs().view(-1, BLOCK)
    field = ((a.amax(1).view(torch.int32) >> 23) - 7).clamp(min=1)
    scale = (field << 23).view(torch.float32)
    y = (a * ((254 - field) << 23).view(torch.float32)[:, None]).view(-1)
    normal = ((y.view(torch.int32) + (r << 4).int()) & -0x100000).view(torch.float32)
    small = (y * 512 + r.float() * 2.0 ** -16).floor()
    if second:
        small = torch.where((small == 0) & (x > 0), 1.0, small)
    q = torch.where(y >= 2.0 ** -6, normal, small / 512)
    return torch.copysign(q, x).to(torch.float8_e4m3fn), scale


def _from_8_bits(codes, scale):
    return (codes.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _run_adamw(s):
    case = s["case"]
    if own:
        opt = s["opt"]
        norm = opt.step(s["grad_views"])
        m, v, scales = opt.exp_avg, opt.exp_avg_sq, (opt.exp_avg_scale, opt.exp_avg_sq_scale)
    else:
        norm = _plain_adamw(s)
        m, v, scales = s["m"], s["v"], (s.get("m_scale"), s.get("v_scale"))
    out = {"params": s["flat"], "m": m, "v": v}
    if case["bits"] == 8:
        out["m_scale"], out["v_scale"] = scales
    if case["clip"]:
        out["norm"] = norm
    return out


def _plain_adamw(s):
    """One step on the flat buffers, in place; every operation rounded by itself."""
    s["steps"] += 1
    t, eight = s["steps"], s["case"]["bits"] == 8
    g, norm = s["grads"].float(), None
    if s["max_norm"] is not None:
        norm = s["grads"].double().square().sum().sqrt()
        g = g * torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0).float()
        norm = norm.float()
    m = _from_8_bits(s["m"], s["m_scale"]) if eight else s["m"]
    v = _from_8_bits(s["v"], s["v_scale"]) if eight else s["v"]
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    change = (m / (v.sqrt() * (1 / math.sqrt(1 - BETA2 ** t)) + EPS)) * (LR / (1 - BETA1 ** t))
    a = s["ends"][0]
    p = s["flat"].float()
    p[:a] *= 1 - LR * DECAY
    s["flat"].copy_(p - change)
    if eight:
        h = _hash(m.numel(), 7, t, m.device)
        m, m_scale = _to_8_bits(m, h & 0xFFFF, False)
        v, v_scale = _to_8_bits(v, h >> 16, True)
        s["m_scale"].copy_(m_scale)
        s["v_scale"].copy_(v_scale)
    s["m"].copy_(m)
    s["v"].copy_(v)
    return norm


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    x, y = s["logits"], s["labels"]
    rows, vocab = x.shape
    live = y >= 0
    up = s["upstream"]
    # a band of rows at a time: log-probabilities first, then the gradient's bands from each row's coefficients
    logp = torch.zeros(rows, dtype=torch.float64, device=x.device)
    entropy = torch.zeros_like(logp)
    band = max(1, 2 ** 25 // vocab)
    for r in range(0, rows, band):
        lp = torch.log_softmax(x[r:r + band].double(), 1)
        logp[r:r + band] = lp.gather(1, y[r:r + band].clamp(min=0)[:, None])[:, 0]
        entropy[r:r + band] = -(lp.exp() * lp.clamp(min=-1e300)).sum(1)
    logp, entropy = logp * live, entropy * live
    extra = None
    if case["op"] == "logprob":
        out, slope = {"logp": logp, "entropy": entropy}, s["g"].double()
        if not case["grad"]:
            return out
    elif case["op"] == "preference":
        seqs = logp.split(_lengths(case))
        total = torch.stack([t.sum() for t in seqs])
        margin = total - s["ref_logp"].double()
        h = PREF_BETA * (margin[0::2] - margin[1::2])
        log_sigmoid = torch.nn.functional.logsigmoid
        out = {"loss": -(1 - SMOOTHING) * log_sigmoid(h) - SMOOTHING * log_sigmoid(-h), "seq_logp": total}
        d = PREF_BETA * up * (torch.sigmoid(h) - (1 - SMOOTHING))
        slope = torch.cat([d[i // 2].expand(len(t)) * (1 if i % 2 == 0 else -1) for i, t in enumerate(seqs)])
    else:
        ratio = torch.exp(logp - s["old_logp"].double())
        a = s["advantage"].double()
        held = torch.where(a >= 0, torch.clamp(ratio, max=1 + CLIP_HIGH), torch.clamp(ratio, min=1 - CLIP_LOW))
        back = torch.exp(s["ref_logp"].double() - logp)
        out = {"loss": live * (-a * held + KL * (back - torch.log(back) - 1) - ENTROPY * entropy), "logp": logp, "entropy": entropy}
        w = up * s["weight"].double()
        slope = w * (torch.where(held == ratio, -a * ratio, 0.0) + KL * (1 - back))
        extra = w * ENTROPY
    slope = slope * live
    d = torch.empty(rows, vocab, dtype=torch.float64 if rows * vocab <= 2 ** 28 else torch.float32, device=x.device)
    for r in range(0, rows, band):
        lp = torch.log_softmax(x[r:r + band].double(), 1)
        p = lp.exp()
        part = -slope[r:r + band, None] * p
        if extra is not None:
            part += (extra * live)[r:r + band, None] * torch.special.xlogy(p, p) + (extra * live * entropy)[r:r + band, None] * p
        part[torch.arange(len(part), device=x.device), y[r:r + band].clamp(min=0)] += slope[r:r + band]
        d[r:r + band] = part
    out["dlogits"] = d
    return out


def _exact_adamw(s):
    case, t = s["case"], FIRST_STEP + 1
    g = s["grads"].double()
    out = {}
    if case["clip"]:
        out["norm"] = g.norm()
        g = g * min(1.0, s["max_norm"] / (float(out["norm"]) + 1e-6))
    m, v = s["m"].double(), s["v"].double()
    if case["bits"] == 8:
        m, v = m * s["m_scale"].double().repeat_interleave(BLOCK), v * s["v_scale"].double().repeat_interleave(BLOCK)
    m.mul_(BETA1).add_(g, alpha=1 - BETA1)
    v.mul_(BETA2).addcmul_(g, g, value=1 - BETA2)
    p = s["flat"].double()
    p[:s["ends"][0]] *= 1 - LR * DECAY
    out["params"] = p - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    if case["bits"] == 32:
        return {**out, "m": m, "v": v}
    h = _hash(m.numel(), 7, t, m.device)
    for name, x, r in (("m", m, h & 0xFFFF), ("v", v, h >> 16)):
        top = x.abs().view(-1, BLOCK).amax(1)
        scale = torch.ldexp(torch.ones_like(top), (torch.frexp(top)[1] - 8).clamp(min=-126))
        y = x.abs() / scale.repeat_interleave(BLOCK)
        step = torch.ldexp(torch.ones_like(y), (torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
        q = torch.floor(y / step + r.double() / 65536) * step
        if name == "v":
            q = torch.where((q == 0) & (x > 0), 2.0 ** -9, q)
        out[name], out[name + "_scale"] = torch.copysign(q, x), scale
    return out
