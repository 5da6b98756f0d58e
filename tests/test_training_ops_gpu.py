"""ops.label_logprob / preference_loss / policy_loss and optim.AdamW against plain implementations in 64 bits.

test_training_ops_emu.py runs the same tests on CPU tensors through the host emulation of the kernels.

Tolerances (u = 2^-24, the rounding of fp32).  A term 2^z of the sum s, z = (x - m) log2 e, is off by |z| u from its argument's
rounding and 2 u from v_exp_f32; weighted with its probability |z| averages to less than log2 V + 2 <= 20.  A lane adds up to 64
terms in order and a tree joins the lanes: 64 u + 20 u + 2 u < 6e-6 relative for s, so as much absolute for log s.  p is off by
that and by its own |z| u."""
import math

import pytest
import torch

from dorpatch_amd import _lib, ops, optim

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
LOG_S = 6e-6
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
NAN, INF = float("nan"), float("inf")


def rand(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


def make_logits(shape, dtype, seed=0, scale=3.0):
    return rand(*shape, seed=seed, scale=scale).to(DTYPES[dtype])


def make_labels(shape, V, seed=0, ignored=0.25):
    g = torch.Generator().manual_seed(seed + 1)
    y = torch.randint(0, V, shape, generator=g)
    if y.numel() > 1:
        y = torch.where(torch.rand(shape, generator=g) < ignored, torch.full_like(y, -100), y)
    return y


def softmax64(x, y):
    """(p, logp, entropy) in 64 bits on the CPU; rows that count for nothing are 0."""
    x = x.detach().cpu().double()
    y = y.cpu()
    dead = (y < 0) | (x == -INF).all(-1)
    x = torch.where(dead[..., None], torch.zeros_like(x), x)
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    logp = lp.gather(-1, y.clamp(0, x.shape[-1] - 1)[..., None])[..., 0]
    entropy = -torch.xlogy(p, p).sum(-1)
    return p, torch.where(dead, 0.0, logp), torch.where(dead, 0.0, entropy), dead


def onehot(y, V):
    return torch.nn.functional.one_hot(y.cpu().clamp(0, V - 1), V).double()


def check_logp(got, want, where=""):
    err = (got.cpu().double() - want).abs()
    assert (err <= LOG_S + 2 * U * want.abs()).all(), (where, err.max())


def check_grad(got, want, g, p, y, dtype, g_err=0.0, entropy=0.0):
    """got: the gradient; want: the same in 64 bits; g (rows): what multiplies (onehot - p), itself off by g_err; entropy (rows): what
    multiplies p (log p + H).  p is off by LOG_S and (|z| <= 60) 62 u: 1e-5 of itself; the products and the sum at the label round 4
    times; |log p + H| <= 40 and off by 2 (LOG_S + 60 u) in all; at last the rounding to the type, or half its smallest step."""
    t = DTYPES[dtype]
    hot = onehot(y, want.shape[-1])
    g, g_err, entropy = (torch.as_tensor(v, dtype=torch.float64).expand(want.shape[:-1])[..., None] for v in (g, g_err, entropy))
    bound = g.abs() * (2e-5 * p + 4 * U * hot) + g_err * (p + hot) + entropy.abs() * p * (40 * 2e-5 + 2e-5)
    bound = bound + torch.finfo(t).eps / 2 * (want.abs() + bound) + torch.finfo(t).tiny * torch.finfo(t).eps
    err = (got.cpu().double() - want).abs()
    assert (err <= bound).all(), (float((err - bound).max()), float(err.max()))


# ---------------------------------------------------------------- log-probabilities of labels
SHAPES = [((1,), 1), ((1,), 2), ((7,), 10), ((5,), 63), ((3,), 1000), ((9,), 1024), ((4,), 2520), ((6,), 2049), ((2,), 4099), ((3,), 8193), ((1,), 20011),
          ((2, 3), 130), ((2, 3), 5001), ((), 77)]


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("shape,V", SHAPES)
def test_label_logprob_and_its_gradient(shape, V, dtype):
    x = make_logits(shape + (V,), dtype, seed=V)
    y = make_labels(shape, V, seed=V)
    p, logp, entropy, dead = softmax64(x, y)
    xd, yd = x.to(DEV), y.to(DEV)
    got, ent, stats = ops.label_logprob(xd, yd, want_entropy=True)
    assert got.shape == y.shape and ent.shape == y.shape and stats.shape == (y.numel(), 2)
    check_logp(got, logp), check_logp(ent, entropy)
    plain, none, again = ops.label_logprob(xd, yd)
    assert none is None and torch.equal(plain, got) and torch.equal(stats, again)
    g = rand(*shape, seed=3) if shape else torch.tensor(0.7)
    d = ops.label_logprob_bwd(xd, yd, stats, g.to(DEV))
    live = (~dead).double() * g.double()
    check_grad(d, live[..., None] * (onehot(y, V) - p), live, p, y, dtype)
    assert (d.cpu()[dead] == 0).all() and (got.cpu()[dead] == 0).all() and (ent.cpu()[dead] == 0).all()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("V", [37, 1001, 4100])
def test_logits_as_they_lie(V, dtype):
    """The shifted slice of a (B, T, V) tensor, columns cut off in front, transposed batches, a broadcast row: no copy is made."""
    base = make_logits((3, 5, V), dtype, seed=9).to(DEV)
    for view in (base[:, :-1], base[:, 1:, 3:], base.transpose(0, 1), base[1, ::2], base[:1, 0].expand(4, V), base[..., :V - 1]):
        y = make_labels(tuple(view.shape[:-1]), view.shape[-1], seed=4).to(DEV)
        a, ent, stats = ops.label_logprob(view, y, want_entropy=True)
        p, logp, entropy, dead = softmax64(view, y)
        check_logp(a, logp), check_logp(ent, entropy)
        g = rand(*y.shape, seed=5)
        d = ops.label_logprob_bwd(view, y, stats, g.to(DEV))
        live = (~dead).double() * g.double()
        check_grad(d, live[..., None] * (onehot(y, view.shape[-1]) - p), live, p, y, dtype)
        assert d.is_contiguous() and d.shape == view.shape
    into = torch.full((3, 5, V + 9), 7.0, dtype=base.dtype, device=DEV)
    y = make_labels((3, 5), V, seed=4).to(DEV)
    stats = ops.label_logprob(base, y)[2]
    g = rand(3, 5, seed=5).to(DEV)
    want = ops.label_logprob_bwd(base, y, stats, g)
    assert torch.equal(ops.label_logprob_bwd(base, y, stats, g, out=into[..., 1:V + 1]), want)
    assert (into[..., :1] == 7).all() and (into[..., V + 1:] == 7).all()         # the padding stays
    work = base.clone()
    assert torch.equal(ops.label_logprob_bwd(work, y, stats, g, out=work), want) and torch.equal(work, want)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("V", [9, 1000, 9001])
def test_banned_entries_and_strange_rows(V, dtype):
    t = DTYPES[dtype]
    x = make_logits((9, V), dtype, seed=2)
    y = torch.randint(0, V, (9,), generator=torch.Generator().manual_seed(1))
    x[0, torch.arange(V) != int(y[0])] = -INF       # one entry is left: p = 1
    x[1] = -INF                                     # nothing is left
    x[2] = torch.finfo(t).min                       # the type's lowest value everywhere: uniform
    x[3, ::2] = torch.finfo(t).min
    x[3, y[3]] = 0.5
    x[4] = NAN                                      # a row that does not count may hold anything
    x[5] = INF
    y[4] = y[5] = -1
    x[6, y[6]] = -INF                               # the label itself is banned
    y[7] = V                                        # no category at all
    x[8, 0] = NAN                                   # a NaN that counts
    xd, yd = x.to(DEV), y.to(DEV)
    logp, ent, stats = ops.label_logprob(xd, yd, want_entropy=True)
    d = ops.label_logprob_bwd(xd, yd, stats, torch.ones(9).to(DEV)).cpu().double()
    p, want, entropy, dead = softmax64(x, y)
    logp, ent = logp.cpu(), ent.cpu()
    # the one term of s is within 2 u of a power of two's: log s as near to 0, and 1 - e (1 / s) is off by 3 roundings
    assert -LOG_S <= logp[0] <= 0 and 0 <= ent[0] <= LOG_S and (d[0].abs() <= 4 * U).all()
    assert logp[1] == 0 and ent[1] == 0 and (d[1] == 0).all()
    check_logp(logp[2:4], want[2:4]), check_logp(ent[2:4], entropy[2:4])
    assert (logp[4:6] == 0).all() and (ent[4:6] == 0).all() and (d[4:6] == 0).all()
    assert logp[6] == -INF and torch.isfinite(ent[6])
    check_grad(d[6:7], (onehot(y, V) - p)[6:7], torch.ones(1), p[6:7], y[6:7], dtype)
    assert torch.isnan(logp[7]) and torch.isnan(d[7]).all()
    assert torch.isnan(logp[8]) and torch.isnan(d[8]).all()


@pytest.mark.parametrize("R,V", [(3, 7), (3, 2000), (70, 5000), (2, 40000)])
def test_rows_of_nan_alone_count(R, V):
    """Short rows, one workgroup a row, rows cut into slices; the fused and the two-pass policy loss."""
    for dtype in sorted(DTYPES):
        x = make_logits((R, V), dtype)
        x[1] = NAN
        y = torch.ones(R, dtype=torch.int64)
        xd, yd, one = x.to(DEV), y.to(DEV), torch.ones(R).to(DEV)
        logp, ent, stats = ops.label_logprob(xd, yd, want_entropy=True)
        d = ops.label_logprob_bwd(xd, yd, stats, one)
        loss, dp, lp, h = ops.policy_loss(xd, yd, one, one, 0.2, 0.2, 1.0, entropy_coef=0.1)
        for t in (logp, ent, d, loss, dp, lp, h):
            t = t.cpu()
            assert torch.isnan(t[1]).all() and torch.isfinite(t[0]).all() and torch.isfinite(t[R - 1 if R > 2 else 0]).all()
        cu = torch.tensor([0, 2, R], dtype=torch.int32).to(DEV)
        loss, d, seq = ops.preference_loss(xd, yd, cu, None, 0.1, 1.0)
        assert torch.isnan(loss).all() and torch.isnan(seq[0]) and torch.isnan(d).all()


def test_an_entry_far_above_long_sums():
    """Lanes that hold sums over 2^28 meet an entry of 2^101: nothing is left of them, and no 0 * infinity."""
    x = torch.full((1, 16384), 16.0)
    x[0, :1024] = 0.0
    x[0, 5000] = 2.0 ** 101
    y, one = torch.tensor([5000]).to(DEV), torch.ones(1).to(DEV)
    for logp, ent in (ops.label_logprob(x.to(DEV), y, want_entropy=True)[:2],
                      ops.policy_loss(x.to(DEV), y, one, one, 0.2, 0.2, 1.0, entropy_coef=0.1)[2:]):
        assert logp[0] == 0 and ent[0] == 0


# ---------------------------------------------------------------- preference loss
def preference64(x, y, cu, ref, beta, smoothing, average, upstream):
    """(loss, dlogits, seq_logp, g) by autograd in 64 bits."""
    _, _, _, dead = softmax64(x, y)
    x = torch.where(dead[:, None], torch.zeros((), dtype=torch.float64), x.cpu().double()).requires_grad_(True)
    lp = torch.log_softmax(x, -1).gather(1, y.cpu().clamp(min=0)[:, None])[:, 0] * (~dead)
    sums = []
    for a, b in zip(cu[:-1], cu[1:]):
        n = int((~dead[a:b]).sum())
        sums.append(lp[a:b].sum() / (max(n, 1) if average else 1))
    sums = torch.stack(sums)
    m = sums - (0 if ref is None else ref.double())
    h = beta * (m[0::2] - m[1::2])
    loss = -(1 - smoothing) * torch.nn.functional.logsigmoid(h) - smoothing * torch.nn.functional.logsigmoid(-h)
    glp, = torch.autograd.grad((upstream * loss).sum(), lp, retain_graph=True)
    d, = torch.autograd.grad((upstream * loss).sum(), x)
    return loss.detach(), d, sums.detach(), glp * (~dead), dead


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("V,smoothing,average,with_ref", [(11, 0.0, False, True), (1024, 0.1, False, True), (1001, 0.5, True, False), (4500, 0.0, True, True)])
def test_preference_loss(V, smoothing, average, with_ref, dtype):
    cu = [2, 5, 5, 12, 13, 13, 13, 20, 24]          # rows in front, an empty sequence, a pair of nothing, rows behind
    R, P = 27, 4
    x = make_logits((R, V), dtype, seed=V + 1)
    y = make_labels((R,), V, seed=V)
    y[13:20] = torch.where(torch.arange(7) < 6, y[13:20], torch.full((7,), -1))
    x[3] = -INF                                     # allows nothing: not counted, in a mean either
    x[y < 0] = NAN
    ref = rand(2 * P, seed=8, scale=5.0) if with_ref else None
    up, beta = 0.37, 0.3
    loss, d, seq = ops.preference_loss(x.to(DEV), y.to(DEV), torch.tensor(cu, dtype=torch.int32).to(DEV), None if ref is None else ref.to(DEV), beta, up,
                                       label_smoothing=smoothing, average=average)
    wl, wd, ws, g, dead = preference64(x, y, cu, ref, beta, smoothing, average, up)
    n = 7                                           # labels of the longest sequence
    assert ((seq.cpu().double() - ws).abs() <= n * LOG_S + 2 * U * ws.abs()).all()
    dh = beta * 2 * n * LOG_S
    assert ((loss.cpu().double() - wl).abs() <= dh + 2 * U * wl.abs()).all()
    p = softmax64(x, y)[0]
    # the slope's derivative by h is at most 1/4
    check_grad(d, wd, g, p, y, dtype, g_err=(up * beta * dh / 4 + 2 * U * g.abs()) * (g != 0))
    assert (d.cpu()[:2] == 0).all() and (d.cpu()[24:] == 0).all() and (d.cpu()[dead] == 0).all()
    only, none, seq2 = ops.preference_loss(x.to(DEV), y.to(DEV), torch.tensor(cu, dtype=torch.int32).to(DEV), None if ref is None else ref.to(DEV), beta, up,
                                           label_smoothing=smoothing, average=average, want_grad=False)
    assert none is None and torch.equal(only, loss) and torch.equal(seq, seq2)
    work = x.to(DEV).clone()
    ops.preference_loss(work, y.to(DEV), torch.tensor(cu, dtype=torch.int32).to(DEV), None if ref is None else ref.to(DEV), beta, up,
                        label_smoothing=smoothing, average=average, out=work)
    assert torch.equal(work, d)


def test_preference_loss_far_apart():
    """h of +-300 and +-1e4: the loss is -h or 0, the slope 1 or 0, nothing overflows."""
    x = make_logits((4, 50), "fp32")
    y = torch.zeros(4, dtype=torch.int64)
    cu = torch.arange(5, dtype=torch.int32)
    for far in (300.0, -300.0, 1e4, -1e4):
        ref = torch.tensor([-far, 0.0, far, 0.0])
        loss, d, seq = ops.preference_loss(x.to(DEV), y.to(DEV), cu.to(DEV), ref.to(DEV), 1.0, 1.0)
        wl, wd, ws, g, _ = preference64(x, y, cu.tolist(), ref, 1.0, 0.0, False, 1.0)
        assert torch.isfinite(loss).all() and torch.isfinite(d).all()
        assert ((loss.cpu().double() - wl).abs() <= 2 * LOG_S + 2 * U * wl.abs()).all()
        check_grad(d, wd, g, softmax64(x, y)[0], y, "fp32", g_err=2 * LOG_S + 2 * U)


def test_preference_loss_with_a_banned_label():
    """An impossible sequence: h is infinite, the loss 0 and without gradient, or infinite with the whole slope."""
    x = make_logits((2, 60), "fp32")
    x[1, 5] = -INF
    y = torch.tensor([3, 5])
    for first, second, want, slope in ((0, 1, 0.0, 0.0), (1, 0, INF, 0.5)):
        xs, ys = x[[first, second]], y[[first, second]]
        loss, d, seq = ops.preference_loss(xs.to(DEV), ys.to(DEV), torch.tensor([0, 1, 2], dtype=torch.int32).to(DEV), None, 0.5, 1.0)
        assert loss[0] == want and seq[second] == -INF and torch.isfinite(seq[first])
        p = softmax64(xs, ys)[0]
        g = torch.tensor([slope, -slope])
        check_grad(d, g[:, None] * (p - onehot(ys, 60)), -g, p, ys, "fp32")
    loss, _, _ = ops.preference_loss(x.to(DEV), y.to(DEV), torch.tensor([0, 1, 2], dtype=torch.int32).to(DEV), None, 0.5, 1.0, label_smoothing=0.1)
    assert loss[0] == INF                           # with a weight of its own the other term counts


def test_preference_loss_of_nothing():
    e = torch.zeros(0, 8).to(DEV)
    y0 = torch.zeros(0, dtype=torch.int64).to(DEV)
    loss, d, seq = ops.preference_loss(e, y0, torch.zeros(5, dtype=torch.int32).to(DEV), torch.tensor([1.0, 0.0, 0.0, 2.0]).to(DEV), 0.5, 1.0, label_smoothing=0.25)
    h = 0.5 * torch.tensor([-1.0, 2.0]).double()
    want = -0.75 * torch.nn.functional.logsigmoid(h) - 0.25 * torch.nn.functional.logsigmoid(-h)
    assert torch.allclose(loss.cpu().double(), want, rtol=0, atol=8 * U) and (seq == 0).all() and d.shape == (0, 8)
    loss, d, seq = ops.preference_loss(make_logits((3, 8), "fp32").to(DEV), torch.zeros(3, dtype=torch.int64).to(DEV), torch.zeros(1, dtype=torch.int32).to(DEV), None, 0.5, 1.0)
    assert loss.shape == (0,) and seq.shape == (0,) and (d == 0).all()


def test_preference_loss_stays_inside_its_rows_whatever_the_bounds_say():
    """Bounds that descend or point past the rows are not what the call is for, but no access leaves the tensors."""
    x, y = make_logits((6, 40), "fp32").to(DEV), torch.ones(6, dtype=torch.int64).to(DEV)
    for cu in ([0, 900, 7], [-5, 3, 2000000000], [6, 3, 0], [2147483647, -2147483648, 1]):
        loss, d, seq = ops.preference_loss(x, y, torch.tensor(cu, dtype=torch.int32).to(DEV), None, 0.1, 1.0)
        assert loss.shape == (1,) and d.shape == x.shape and torch.isfinite(loss).all() and torch.isfinite(d).all()


# ---------------------------------------------------------------- clipped policy loss
def policy64(x, y, old, adv, lo, hi, up, ref, kl, ent, weight):
    """(loss, dlogits, logp, entropy, what multiplies (onehot - p)) from the formulas in 64 bits."""
    p, logp, entropy, dead = softmax64(x, y)
    live = (~dead).double()
    ratio = torch.exp(logp - old.double())
    adv = adv.double()
    plain, held = -adv * ratio, -adv * ratio.clamp(1 - lo, 1 + hi)
    loss, slope = torch.maximum(plain, held), torch.where(plain >= held, plain, 0.0)
    if ref is not None:
        k = ref.double() - logp
        loss = loss + kl * (torch.expm1(k) - k)
        slope = slope - kl * torch.expm1(k)
    loss = loss - ent * entropy
    w = up * (1.0 if weight is None else weight.double())
    g = torch.where(dead, 0.0, w * slope)
    d = g[..., None] * (onehot(y, p.shape[-1]) - p) + (live * w * ent)[..., None] * (torch.xlogy(p, p) + p * entropy[..., None])
    return torch.where(dead, 0.0, loss), d, logp, entropy, g, dead


def away_from_edges(shift, lo, hi):
    for edge in (math.log(1 - lo) if lo < 1 else -80.0, math.log(1 + hi)):
        shift = torch.where((shift - edge).abs() < 1e-3, torch.full_like(shift, edge + 2e-3), shift)
    return shift


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("shape,V,kl,ent,weighted", [((1,), 2, 0.0, 0.0, False), ((33,), 10, 0.1, 0.0, True), ((20,), 2520, 0.04, 0.01, True),
                                                     ((2, 6), 4099, 0.0, 0.02, False), ((5,), 9001, 0.04, 0.0, False), ((3,), 33001, 0.1, 0.05, True)])
def test_policy_loss(shape, V, kl, ent, weighted, dtype):
    lo, hi, up = 0.2, 0.28, 0.9
    x = make_logits(shape + (V,), dtype, seed=V)
    y = make_labels(shape, V, seed=V)
    if V > 100:
        ban = torch.rand(x.shape, generator=torch.Generator().manual_seed(6)) < 0.1
        ban.scatter_(-1, y.clamp(min=0)[..., None], False)
        x[ban] = -INF
    _, logp, _, dead = softmax64(x, y)
    old = (logp - away_from_edges(rand(*shape, seed=1, scale=0.4).double(), lo, hi)).float()
    adv = rand(*shape, seed=2)
    ref = (logp + rand(*shape, seed=3, scale=0.3)).float() if kl else None
    weight = rand(*shape, seed=4).abs() if weighted else None
    for t in (old, adv, ref, weight):
        if t is not None:
            t[dead] = NAN                           # rows that do not count may hold anything
    x[dead] = NAN
    dev = [None if t is None else t.to(DEV) for t in (old, adv, ref, weight)]
    loss, d, lp, h = ops.policy_loss(x.to(DEV), y.to(DEV), dev[0], dev[1], lo, hi, up, ref_logp=dev[2], kl_coef=kl, entropy_coef=ent, weight=dev[3],
                                     want_entropy=True)
    wl, wd, wlp, wh, g, _ = policy64(x, y, old.nan_to_num(), adv.nan_to_num(), lo, hi, up, None if ref is None else ref.nan_to_num(), kl, ent,
                                     None if weight is None else weight.nan_to_num())
    check_logp(lp, wlp), check_logp(h, wh)
    # logp is off by LOG_S: the ratios by that much of themselves (and 4 roundings), the entropy by 2 LOG_S
    slope = adv.nan_to_num().abs() * torch.exp(wlp - old.nan_to_num().double())
    if kl:
        slope = slope + kl * (1 + torch.exp(ref.nan_to_num().double() - wlp))
    off = slope * (LOG_S + 4 * U) * (~dead)
    assert ((loss.cpu().double() - wl).abs() <= off + ent * 2 * LOG_S + 4 * U * (wl.abs() + ent * wh)).all()
    w = up * (1.0 if weight is None else weight.nan_to_num().double()) * (~dead)
    check_grad(d, wd, g, softmax64(x, y)[0], y, dtype, g_err=w * off + 4 * U * g.abs(), entropy=w * ent)
    assert (d.cpu()[dead] == 0).all() and (loss.cpu()[dead] == 0).all()
    only, none, lp2, h2 = ops.policy_loss(x.to(DEV), y.to(DEV), dev[0], dev[1], lo, hi, up, ref_logp=dev[2], kl_coef=kl, entropy_coef=ent, weight=dev[3],
                                          want_grad=False)
    assert none is None and torch.equal(only, loss) and torch.equal(lp, lp2) and ((h2 is None) == (ent == 0.0))
    work = x.to(DEV).clone()
    ops.policy_loss(work, y.to(DEV), dev[0], dev[1], lo, hi, up, ref_logp=dev[2], kl_coef=kl, entropy_coef=ent, weight=dev[3], out=work)
    assert torch.equal(work, d)


@pytest.mark.parametrize("rows,V,dtype", [(2, v, "fp32") for v in (1024, 1025, 2048, 2049, 4096, 4097, 8192, 8193, 16384, 16385, 32768, 32769)]
                         + [(3, v, "bf16") for v in (2047, 4095, 8191, 16383, 32767, 65535)] + [(66, 33003, "fp32")])
def test_policy_loss_where_the_row_length_changes_the_kernel(rows, V, dtype):
    test_policy_loss((rows,), V, 0.04, 0.01, True, dtype)


def test_policy_loss_on_its_own_draws_and_its_clip():
    """ratio = 1 (the first step after the draw): the gradient of the plain branch; far outside the range: none on the clipped
    side, the plain one on the other."""
    x = make_logits((6, 30), "fp32", seed=5)
    y = torch.arange(6)
    lp = ops.label_logprob(x.to(DEV), y.to(DEV))[0]
    adv = torch.tensor([1.0, -1.0, 2.0, -2.0, 1.0, -1.0])
    old = lp.cpu() - torch.tensor([0.0, 0.0, 1.0, -1.0, -1.0, 1.0])        # ratio 1, 1, e, 1/e, 1/e, e
    loss, d, _, _ = ops.policy_loss(x.to(DEV), y.to(DEV), old.to(DEV), adv.to(DEV), 0.2, 0.3, 1.0)
    want = torch.tensor([-1.0, 1.0, -2 * 1.3, 2 * 0.8, -math.exp(-1), math.e]).double()
    assert ((loss.cpu().double() - want).abs() <= want.abs() * (4 * LOG_S)).all()
    assert (d.cpu()[2:4] == 0).all()
    p = softmax64(x, y)[0]
    slope = torch.tensor([-1.0, 1.0, 0.0, 0.0, -math.exp(-1), math.e]).double()
    check_grad(d, slope[:, None] * (onehot(y, 30) - p), slope, p, y, "fp32", g_err=slope.abs() * 2 * LOG_S)


def test_policy_loss_keeps_what_is_not_finite():
    x = make_logits((5, 40), "fp32", seed=5)
    y = torch.arange(5)
    old, adv = torch.full((5,), -3.0), torch.ones(5)
    old[0], adv[1], x[2, 7] = NAN, NAN, NAN
    x[3, 3] = -INF                                  # drawn, and now banned: ratio 0
    loss, d, lp, h = ops.policy_loss(x.to(DEV), y.to(DEV), old.to(DEV), adv.to(DEV), 0.2, 0.2, 1.0, entropy_coef=0.1)
    assert torch.isnan(loss.cpu()[:3]).all() and torch.isfinite(loss.cpu()[3:]).all()
    assert torch.isnan(d.cpu()[:3]).all() and torch.isfinite(d.cpu()[3:]).all()
    assert lp.cpu()[3] == -INF and torch.isfinite(h.cpu()[3:]).all()


def test_gradients_against_differences():
    """The losses' gradients against central differences of the losses themselves in 64 bits, so that loss and gradient belong together."""
    V, eps = 6, 1e-6
    x, y = make_logits((4, V), "fp32", seed=11).double(), torch.tensor([1, 2, 0, 5])
    old, adv, ref = rand(4, seed=1).double() - 2, rand(4, seed=2).double(), rand(4, seed=3).double() - 2

    def policy(z):
        return policy64(z, y, old, adv, 0.2, 0.3, 1.0, ref, 0.2, 0.1, None)[0].sum()

    def preference(z):
        return preference64(z, y, [0, 1, 2, 3, 4], ref, 0.7, 0.1, False, 1.0)[0].sum()

    got_policy = ops.policy_loss(x.float().to(DEV), y.to(DEV), old.float().to(DEV), adv.float().to(DEV), 0.2, 0.3, 1.0, ref_logp=ref.float().to(DEV), kl_coef=0.2,
                                 entropy_coef=0.1)[1].cpu().double()
    got_preference = ops.preference_loss(x.float().to(DEV), y.to(DEV), torch.arange(5, dtype=torch.int32).to(DEV), ref.float().to(DEV), 0.7, 1.0,
                                         label_smoothing=0.1)[1].cpu().double()
    for f, got in ((policy, got_policy), (preference, got_preference)):
        for r in range(4):
            for j in range(V):
                step = torch.zeros_like(x)
                step[r, j] = eps
                slope = float(f(x + step) - f(x - step)) / (2 * eps)
                # differences: 1e-16 / eps = 1e-10 and eps^2; the kernel: 2e-5 of gradients of order 1
                assert abs(slope - float(got[r, j])) <= 1e-4, (r, j)


# ---------------------------------------------------------------- refusals
def refused(kind, call, *a, **k):
    with pytest.raises(kind):
        call(*a, **k)


def test_losses_refuse_what_they_do_not_take():
    x, y = make_logits((4, 9), "fp32").to(DEV), torch.zeros(4, dtype=torch.int64).to(DEV)
    r = torch.zeros(4).to(DEV)
    refused(TypeError, ops.label_logprob, x.double(), y)
    refused(TypeError, ops.label_logprob, x, y.int())
    refused(ValueError, ops.label_logprob, x, y[:3])
    refused(ValueError, ops.label_logprob, x.t(), torch.zeros(9, dtype=torch.int64).to(DEV))
    refused(ValueError, ops.label_logprob, x[:, :0], y)
    refused(ValueError, ops.label_logprob, x[None, None], y[None, None])
    refused(ValueError, ops.label_logprob, x, torch.zeros(8, dtype=torch.int64).to(DEV)[::2])
    stats = ops.label_logprob(x, y)[2]
    refused(ValueError, ops.label_logprob_bwd, x, y, stats[:3], r)
    refused(TypeError, ops.label_logprob_bwd, x, y, stats, r.double())
    refused(ValueError, ops.label_logprob_bwd, x, y, stats, r, out=x[:3])
    refused(ValueError, ops.label_logprob_bwd, x[:, 1:], y, stats, r, out=x[:, :-1])        # overlaps, and is not the same
    refused(ValueError, ops.label_logprob_bwd, x, y, stats, r, out=torch.zeros(1, 9).to(DEV).expand(4, 9))
    refused(ValueError, ops.label_logprob_bwd, x[None], y[None], stats, r[None], out=torch.zeros(40).to(DEV).as_strided((1, 4, 9), (0, 8, 1)))
    cu = torch.tensor([0, 2, 4], dtype=torch.int32).to(DEV)
    refused(ValueError, ops.preference_loss, x, y, cu[:2], None, 0.1, 1.0)
    refused(TypeError, ops.preference_loss, x, y, cu.long(), None, 0.1, 1.0)
    refused(ValueError, ops.preference_loss, x, y, cu, r, 0.1, 1.0)
    refused(ValueError, ops.preference_loss, x, y, cu, None, 0.1, 1.0, label_smoothing=1.5)
    refused(ValueError, ops.preference_loss, x[None], y[None], cu, None, 0.1, 1.0)
    refused(ValueError, ops.policy_loss, x, y, r[:3], r, 0.2, 0.2, 1.0)
    refused(TypeError, ops.policy_loss, x, y, None, r, 0.2, 0.2, 1.0)
    refused(ValueError, ops.policy_loss, x, y, r, r, -0.1, 0.2, 1.0)
    refused(ValueError, ops.policy_loss, x, y, r, r, 0.2, 0.2, 1.0, kl_coef=0.1)
    e = torch.zeros(0, 9).to(DEV)
    y0, r0 = torch.zeros(0, dtype=torch.int64).to(DEV), torch.zeros(0).to(DEV)
    assert ops.label_logprob(e, y0)[0].shape == (0,)
    assert ops.policy_loss(e, y0, r0, r0, 0.2, 0.2, 1.0)[1].shape == (0, 9)


# ---------------------------------------------------------------- AdamW
def adamw64(p, g, m, v, t, lr, betas, eps, decay, clip=1.0):
    g = g.double() * clip
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    p = p * (1 - lr * decay) - lr / (1 - betas[0] ** t) * m / ((v / (1 - betas[1] ** t)).sqrt() + eps)
    return p, m, v


SIZES = [1, 3, 127, 128, 129, 0, 1000, 4096, 4097, 9001]


@pytest.mark.parametrize("pt,gt", [("fp32", "fp32"), ("bf16", "bf16"), ("fp32", "bf16"), ("fp16", "fp16"), ("bf16", "fp32")])
@pytest.mark.parametrize("max_norm", [None, 1.0])
def test_adamw_steps_in_32_bits(pt, gt, max_norm):
    betas, eps, steps = (0.9, 0.99), 1e-8, 4
    params = [rand(n, seed=n).to(DTYPES[pt]) for n in SIZES]
    lrs = [1e-2 / (k + 1) for k in range(len(SIZES))]
    decays = [0.1 * (k % 2) for k in range(len(SIZES))]
    on = [p.clone().to(DEV) for p in params]
    opt = optim.AdamW(on, lr=lrs, betas=betas, eps=eps, weight_decay=decays, max_norm=max_norm)
    p64 = [p.double() for p in params]
    m64, v64 = [torch.zeros(n).double() for n in SIZES], [torch.zeros(n).double() for n in SIZES]
    half = torch.finfo(DTYPES[pt]).eps / 2
    for t in range(1, steps + 1):
        grads = [rand(n, seed=100 * t + n, scale=0.3 / t).to(DTYPES[gt]) for n in SIZES]
        norm = opt.step([g.to(DEV) for g in grads])
        all_g = torch.cat([g.double() for g in grads])
        clip = 1.0
        if max_norm is not None:
            assert abs(float(norm) / float(all_g.norm()) - 1) <= 2 * U
            clip = min(1.0, max_norm / (float(all_g.norm()) + 1e-6))
        else:
            assert norm is None
        for k in range(len(SIZES)):
            # the kernel goes on from its own rounded parameters
            p64[k], m64[k], v64[k] = adamw64(on_before[k] if t > 1 else params[k].double(), grads[k], m64[k], v64[k], t, lrs[k], betas, eps, decays[k], clip)
        on_before = [p.cpu().double() for p in on]
        for k, n in enumerate(SIZES):
            got = on_before[k]
            # an update is at most about lr / sqrt(1 - beta2) and off by 20 roundings; the parameter by its own rounding
            bound = half * p64[k].abs() * (1 + 1e-3) + 4 * U * p64[k].abs() + 20 * U * 10 * lrs[k] + torch.finfo(DTYPES[pt]).tiny
            assert ((got - p64[k]).abs() <= bound).all(), (n, t)
            m, v = opt.moments(k)
            assert ((m.cpu().double() - m64[k]).abs() <= 6 * U * t * 0.3).all() and ((v.cpu().double() - v64[k]).abs() <= 8 * U * t * (v64[k] + 1e-30)).all()
    assert opt.steps == steps


def test_adamw_many_tensors_some_without_gradients_and_off_alignment():
    """More tensors than a launch takes, parts of one buffer that start anywhere, gradients that are missing."""
    sizes = [(7 * k) % 300 + 1 for k in range(160)]
    flat = rand(sum(sizes) + 1, seed=1).to(DEV)
    gflat = rand(sum(sizes) + 3, seed=2).to(DEV)
    params, grads, at = [], [], 1
    for k, n in enumerate(sizes):
        params.append(flat[at:at + n])
        grads.append(None if k % 11 == 5 else gflat[at + 2:at + 2 + n])
        at += n
    before = [p.cpu().clone() for p in params]
    first = flat[0].item()
    opt = optim.AdamW(params, lr=1e-2, weight_decay=0.1, box=(-1.0, 0.5))
    opt.step(grads)
    for k, n in enumerate(sizes):
        if grads[k] is None:
            assert torch.equal(params[k].cpu(), before[k]) and (opt.moments(k)[0] == 0).all()
            continue
        want, m, v = adamw64(before[k].double(), grads[k].cpu(), torch.zeros(n).double(), torch.zeros(n).double(), 1, 1e-2, (0.9, 0.999), 1e-8, 0.1)
        assert ((params[k].cpu().double() - want.clamp(-1.0, 0.5)).abs() <= 4 * U * (want.abs() + 0.1)).all()
        assert ((opt.moments(k)[0].cpu().double() - m).abs() <= 2 * U * m.abs()).all()
    assert flat[0].item() == first
    for a, b in zip(opt.offsets, opt.offsets[1:] + [opt.exp_avg.numel()]):
        k = opt.offsets.index(a)
        assert (opt.exp_avg[a + sizes[k]:b] == 0).all() and (opt.exp_avg_sq[a + sizes[k]:b] == 0).all()         # padding


def mix32(h):
    low = 0xFFFFFFFF
    h = (h ^ (h >> 16)) * 0x9E3779B1 & low
    h = (h ^ (h >> 15)) * 0x85EBCA77 & low
    return h ^ (h >> 16)


def encode8(x, bits16, second):
    """The 8-bit form of moments x (a multiple of 128 of them, fp32) from 16 random bits each: (values, scales), by its definition in 64 bits."""
    a = x.double().abs().view(-1, 128)
    top = a.amax(1)
    scale = torch.ldexp(torch.ones_like(top), (torch.frexp(top)[1] - 8).clamp(min=-126))
    scale = torch.where(top == 0, 2.0 ** -126, scale)
    y = (a / scale[:, None]).view(-1)
    step = torch.ldexp(torch.ones_like(y), (torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
    step = torch.where(y == 0, 2.0 ** -9, step)
    q = torch.floor(y / step + bits16.double() / 65536) * step
    if second:
        q = torch.where((q == 0) & (x > 0), 2.0 ** -9, q)
    return torch.copysign(q, x.double()).float(), scale.float()


@pytest.mark.parametrize("pt,max_norm", [("fp32", None), ("bf16", 1.0)])
def test_adamw_steps_in_8_bits(pt, max_norm):
    """The codes, bit for bit: the moments are products and sums of fp32 in a fixed order, the scale a power of two."""
    sizes, seed, b1, b2 = [5, 128, 300, 4500], 77, 0.9, 0.999
    params = [rand(n, seed=n).to(DTYPES[pt]).to(DEV) for n in sizes]
    opt = optim.AdamW(params, lr=1e-2, betas=(b1, b2), weight_decay=0.0, state_bits=8, max_norm=max_norm, seed=seed)
    total = opt.exp_avg.numel()
    m = v = torch.zeros(total)
    e = torch.arange(total)
    live = torch.zeros(total, dtype=torch.bool)
    for at, n in zip(opt.offsets, sizes):
        live[at:at + n] = True
    for t in range(1, 5):
        # magnitudes over many powers of two in one block, zeroes among them
        grads = [(rand(n, seed=t * 1000 + n) * torch.exp2(-torch.arange(n) % 23).float() * (torch.arange(n) % 7 > 0)).to(DTYPES[pt]) for n in sizes]
        old = [p.cpu().float().clone() for p in params]
        norm = opt.step([g.to(DEV) for g in grads])
        g = torch.zeros(total)
        for at, n, gr in zip(opt.offsets, sizes, grads):
            g[at:at + n] = gr.float()
        if max_norm is not None:
            total_norm = g.double().square().sum().sqrt()
            assert abs(float(norm) / float(total_norm) - 1) <= 2 * U
            g = g * torch.clamp(max_norm / (total_norm + 1e-6), max=1.0).float()
        m = m * b1 + g * (1 - b1)
        v = v * b2 + (g * g) * (1 - b2)
        m_before, v_before = m, v
        h = mix32(((e & 0xFFFFFFFF) ^ mix32((seed * 0x9E3779B1 + t) & 0xFFFFFFFF)))
        (m8, ms), (v8, vs) = encode8(m, h & 0xFFFF, False), encode8(v, h >> 16, True)
        assert torch.equal(opt.exp_avg_scale.cpu(), ms) and torch.equal(opt.exp_avg_sq_scale.cpu(), vs)
        assert torch.equal(opt.exp_avg.cpu().float(), m8) and torch.equal(opt.exp_avg_sq.cpu().float(), v8)
        m, v = (m8.view(-1, 128) * ms[:, None]).view(-1), (v8.view(-1, 128) * vs[:, None]).view(-1)
        assert (v[live & (v_before > 0)] > 0).all() and (m[~live] == 0).all()
        for k, (at, n) in enumerate(zip(opt.offsets, sizes)):
            mk, vk = m_before[at:at + n].double(), v_before[at:at + n].double()
            want = old[k].double() - 1e-2 / (1 - b1 ** t) * mk / ((vk / (1 - b2 ** t)).sqrt() + 1e-8)
            change = (want - old[k]).abs()
            half = torch.finfo(DTYPES[pt]).eps / 2
            assert ((params[k].cpu().double() - want).abs() <= half * want.abs() * 1.001 + 20 * U * change + 4 * U * want.abs() + torch.finfo(DTYPES[pt]).tiny).all()


def test_eight_bit_rounding_keeps_the_expectation():
    """beta2 = 0.999 moves a second moment by a thousandth a step, an eightieth of a code's distance: the mean over many elements
    follows all the same.  40 000 elements: the mean's standard deviation is under 0.06 of a code's width / sqrt(40000)."""
    n = 40064
    p = torch.zeros(n).to(DEV)
    opt = optim.AdamW([p], lr=0.0, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8, seed=3)
    g = torch.ones(n)
    g[::128] = 4.0                                  # holds the blocks' scales
    want = 0.0
    for t in range(12):
        opt.step([(g * (1.0 + t)).to(DEV)])
        want = want * 0.999 + 0.001 * (1.0 + t) ** 2
    v = opt.moments(0)[1].cpu().double().view(-1, 128)[:, 1:]
    # every step rounds by less than an eighth of the value, 12 of them, over sqrt(39751) elements: 4 standard deviations
    assert abs(float(v.mean()) / want - 1) <= 4 * 0.125 / 2 * math.sqrt(12.0 / v.numel())
    assert float(v.std()) > 0


def test_adamw_does_not_take_a_step_whose_norm_is_not_finite():
    for bad in (NAN, INF):
        for bits in (32, 8):
            p = rand(300, seed=1).to(DEV)
            opt = optim.AdamW([p], state_bits=bits, max_norm=1.0)
            opt.step([rand(300, seed=2).to(DEV)])
            kept = [t.clone() for t in (p, opt.exp_avg.view(torch.uint8), opt.exp_avg_sq.view(torch.uint8))]
            g = rand(300, seed=3)
            g[7] = bad
            norm = opt.step([g.to(DEV)])
            assert not torch.isfinite(norm).any() and opt.steps == 1
            for a, b in zip(kept, (p, opt.exp_avg.view(torch.uint8), opt.exp_avg_sq.view(torch.uint8))):
                assert torch.equal(a, b)
            opt.step([rand(300, seed=4).to(DEV)])
            assert opt.steps == 2


def test_adamw_stores_what_is_not_finite_as_nan_in_8_bits():
    p = torch.zeros(256).to(DEV)
    opt = optim.AdamW([p], state_bits=8)
    g = torch.ones(256)
    g[3], g[200] = INF, NAN
    opt.step([g.to(DEV)])
    m, v = (t.cpu() for t in opt.moments(0))
    for t in (m, v):
        assert torch.isnan(t[[3, 200]]).all() and torch.isfinite(t).sum() == 254 and (t[torch.isfinite(t)] > 0).all()


def test_adamw_goes_on_from_a_saved_state():
    for bits in (32, 8):
        a, b = rand(500, seed=1).to(DEV), rand(500, seed=1).to(DEV)
        one, two = optim.AdamW([a], state_bits=bits, seed=5), optim.AdamW([b], state_bits=bits, seed=5)
        one.step([rand(500, seed=2).to(DEV)])
        two.load_state_dict(one.state_dict())
        b.copy_(a)
        one.step([rand(500, seed=3).to(DEV)]), two.step([rand(500, seed=3).to(DEV)])
        assert torch.equal(a, b) and one.steps == two.steps == 2
        assert torch.equal(one.exp_avg.view(torch.uint8), two.exp_avg.view(torch.uint8))


def test_adamw_of_parameters_with_grad():
    """Module parameters: .grad is taken, requires_grad is no obstacle, autograd notices the change."""
    lin = torch.nn.Linear(5, 3).to(DEV)
    opt = optim.AdamW(lin.parameters(), lr=1e-2, weight_decay=0.0)
    x = rand(4, 5).to(DEV)
    lin(x).sum().backward()
    out = lin(x).square().sum()                     # saves the weight for its backward of x
    xs = x.clone().requires_grad_(True)
    held = lin(xs).square().sum()
    before = [p.detach().clone() for p in lin.parameters()]
    assert opt.step() is None
    for p, b in zip(lin.parameters(), before):
        # step 1 moves every element by lr against its gradient's sign (here the sums of inputs are far over eps)
        assert ((p - b).abs() - 1e-2).abs().max() <= 1e-2 * 1e-4 or (p.grad == 0).any()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        held.backward()
    assert torch.isfinite(out)


def test_adamw_refuses_what_it_does_not_take():
    p = torch.zeros(10).to(DEV)
    refused(ValueError, optim.AdamW, [])
    refused(ValueError, optim.AdamW, [p, p])
    refused(ValueError, optim.AdamW, [p[:6], p[5:]])
    refused(TypeError, optim.AdamW, [p.double()])
    refused(ValueError, optim.AdamW, [torch.zeros(4, 5).to(DEV).t()])
    refused(ValueError, optim.AdamW, [p], state_bits=16)
    refused(ValueError, optim.AdamW, [p], betas=(1.0, 0.9))
    refused(ValueError, optim.AdamW, [p], max_norm=0.0)
    refused(ValueError, optim.AdamW, [p], box=(1.0, 0.0))
    refused(ValueError, optim.AdamW, [p], lr=[1e-3, 1e-3])
    refused(ValueError, optim.AdamW, [p], weight_decay=-0.1)
    opt = optim.AdamW([p])
    refused(ValueError, opt.step, [])
    refused(ValueError, opt.step, [torch.zeros(9).to(DEV)])
    refused(TypeError, opt.step, [torch.zeros(10).double().to(DEV)])
    refused(ValueError, opt.step, [torch.zeros(20).to(DEV)[::2]])
    refused(ValueError, opt.load_state, torch.zeros(5).to(DEV), torch.zeros(5).to(DEV), 1)
    refused(ValueError, opt.load_state, opt.exp_avg, opt.exp_avg_sq, -1)
    refused(ValueError, optim.AdamW, [p], lr=INF)
    refused(ValueError, opt.step, [p.clone()], lr=NAN)
    assert opt.steps == 0 and (p == 0).all()


def test_adamw_of_nothing():
    e = torch.zeros(0, 3).to(DEV)
    for bits, max_norm in ((32, None), (8, 1.0)):
        opt = optim.AdamW([e], state_bits=bits, max_norm=max_norm)
        norm = opt.step([e.clone()])
        assert opt.steps == 1 and (norm is None or norm == 0)
        norm = opt.step([None])
        assert opt.steps == 2 and (norm is None or norm == 0) and opt.moments(0)[0].shape == (0, 3)


def test_adamw_refuses_parameters_that_have_changed():
    """`.data` given another type, size or stride since: the states no longer fit, and nothing is written."""
    for change in (lambda t: t.half(), lambda t: t[:5].clone(), lambda t: torch.zeros(20).to(DEV)[::2], lambda t: torch.zeros(1).to(DEV).expand(10)):
        p = torch.nn.Parameter(torch.zeros(10).to(DEV))
        opt = optim.AdamW([p])
        p.data = change(p.data)
        refused(ValueError, opt.step, [torch.ones(10).to(DEV)])
        assert (p == 0).all() and opt.steps == 0
    p = torch.nn.Parameter(torch.zeros(10).to(DEV))
    opt = optim.AdamW([p], weight_decay=0.0)
    p.data = torch.ones(10).to(DEV)                 # other data of the same kind: taken where it lies
    opt.step([torch.ones(10).to(DEV)])
    assert ((p - (1 - 1e-3)).abs() <= 1e-7).all()


def test_c_entries_refuse_what_the_kernels_do_not_take():
    """The C ABI's own checks: status 1 (invalid value), nothing launched."""
    import ctypes
    lib = _lib.load()
    x, y, o = torch.zeros(4, 8).to(DEV), torch.zeros(4, dtype=torch.int64).to(DEV), torch.zeros(64).to(DEV)
    P = ctypes.c_void_p

    def rows(**k):
        d = dict(data=x.data_ptr(), dtype=0, rows=4, vocab=8, inner=4, outer_stride=0, row_stride=8)
        d.update(k)
        return ctypes.byref(_lib.DpLogits(**d))
    for bad in (dict(data=0), dict(data=x.data_ptr() + 2), dict(dtype=3), dict(rows=0), dict(rows=2 ** 23 + 1), dict(vocab=0), dict(inner=0), dict(row_stride=-8)):
        assert lib.dp_label_logprob(rows(**bad), P(y.data_ptr()), P(o.data_ptr()), None, None, None, ops._stream()) == 1, bad
    assert lib.dp_label_logprob(rows(), None, P(o.data_ptr()), None, None, None, ops._stream()) == 1
    assert lib.dp_logits_workspace(7, 4, 8, 0) == 0 and lib.dp_logits_workspace(_lib.DP_PREFERENCE, 4, 8, 0) >= 4 * 28
    table = (_lib.DpAdamwTensor * 2)()
    for k in range(2):
        table[k].param, table[k].grad, table[k].n, table[k].at = o.data_ptr() + 64 * k, x.data_ptr(), 16, 128 * k
    cfg = _lib.DpAdamwCfg(0.9, 0.999, 1e-8, 0.0, 0.0, 0.0, 0, 32, 1, 0)
    m = torch.zeros(256).to(DEV)

    def step():
        return lib.dp_adamw_step(ctypes.byref(cfg), table, 2, P(m.data_ptr()), None, P(m.data_ptr()), None, None, None, None, ops._stream())
    table[1].param = o.data_ptr() + 4               # overlapping parameters
    assert step() == 1
    table[1].param, table[1].at = o.data_ptr() + 64, 64
    assert step() == 1
    table[1].at = 0                                 # the same part of the states
    assert step() == 1
    table[1].at, table[1].n = 128, -1
    assert step() == 1
    table[1].n, table[1].grad_dtype = 16, 5
    assert step() == 1
    table[1].grad_dtype, cfg.state_bits = 0, 8      # no scales
    assert step() == 1
    cfg.state_bits, cfg.max_norm = 32, 1.0          # no counter
    assert step() == 1


# ---------------------------------------------------------------- together
def adamw_reference(state, p, g, t, lr, decay, clip):
    m, v = state
    p, state[0], state[1] = adamw64(p, g, m, v, t, lr, (0.9, 0.999), 1e-8, decay, clip)
    return p


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_of_a_policy_and_a_preference_together(bits):
    """A linear model over 60 categories: three steps of the policy loss, then three of the preference loss against the model
    before, each with the gradient through the product and a clipped AdamW step: the parameters as in 64 bits throughout.

    32 bits: a step's gradient is off by about 3e-5 of itself (check_grad's 2e-5 and the product's roundings); Adam's first steps
    scale every element to about lr, an element of the gradient much under the others moves by lr times its own relative error,
    so that few elements may be off more than 1e-3 lr and none more than 2 lr a step.  8 bits: the first step is the same; what is kept after
    it is a code off by at most an eighth (m) and an eighth (v, so a sixteenth in its root): a step differs by less than a third."""
    V, d, R, lr = 60, 16, 24, 1e-2
    w = rand(V, d, seed=1, scale=0.3)
    bias = rand(V, seed=2, scale=0.1)
    x = rand(R, d, seed=3)
    y = make_labels((R,), V, seed=4)
    adv = rand(R, seed=5)
    cu = [0, 5, 9, 16, R]
    params = [w.clone().to(DEV), bias.clone().to(DEV)]
    opt = optim.AdamW(params, lr=lr, weight_decay=[0.1, 0.0], state_bits=bits, max_norm=0.5, seed=9)
    p64 = [w.double(), bias.double()]
    states = [[torch.zeros_like(p), torch.zeros_like(p)] for p in p64]
    xd, yd = x.to(DEV), y.to(DEV)
    old = ref = None
    for t in range(1, 7):
        logits = (xd @ params[0].t() + params[1]).contiguous()
        l64 = x.double() @ p64[0].t() + p64[1]
        if t <= 3:
            if old is None:
                old, old64 = ops.label_logprob(logits, yd)[0], softmax64(l64, y)[1]
            loss, dl, _, _ = ops.policy_loss(logits, yd, old, adv.to(DEV), 0.2, 0.2, 1.0 / R, entropy_coef=0.01, out=logits)
            dl64 = policy64(l64, y, old64, adv, 0.2, 0.2, 1.0 / R, None, 0.0, 0.01, None)[1]
        else:
            if ref is None:
                lp, lp64 = ops.label_logprob(logits, yd)[0], softmax64(l64, y)[1]
                ref = torch.stack([lp[a:b].sum() for a, b in zip(cu[:-1], cu[1:])])
                ref64 = torch.stack([lp64[a:b].sum() for a, b in zip(cu[:-1], cu[1:])])
            loss, dl, _ = ops.preference_loss(logits, yd, torch.tensor(cu, dtype=torch.int32).to(DEV), ref, 0.5, 0.5)
            dl64 = preference64(l64, y, cu, ref64, 0.5, 0.0, False, 0.5)[1]
        norm = opt.step([(dl.t() @ xd).contiguous(), dl.sum(0)])
        g64 = [dl64.t() @ x.double(), dl64.sum(0)]
        n64 = math.sqrt(sum(float(g.square().sum()) for g in g64))
        clip = min(1.0, 0.5 / (n64 + 1e-6))
        for k, decay in enumerate((0.1, 0.0)):
            p64[k] = adamw_reference(states[k], p64[k], g64[k], t, lr, decay, clip)
        if bits == 32:
            assert abs(float(norm) / n64 - 1) <= 1e-3
        for p, q in zip(params, p64):
            err = (p.cpu().double() - q).abs()
            if bits == 32:
                assert err.max() <= 2 * lr * t and (err > 1e-3 * lr * t).float().mean() <= 0.02, (t, err.max())
            else:
                assert err.mean() <= lr / 3 * t and err.max() <= 2 * lr * t, (t, err.mean(), err.max())
        if bits == 8 and t == 1:
            for p, q in zip(params, p64):
                assert ((p.cpu().double() - q).abs() <= 1e-3 * lr).float().mean() >= 0.98
    assert opt.steps == 6 and torch.isfinite(loss).all()
