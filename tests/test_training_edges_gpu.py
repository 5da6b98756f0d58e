"""Calls of ops.label_logprob / preference_loss / policy_loss, optim.AdamW and generate(update="adamw") at the edges of what they take.

test_training_edges_emu.py runs the same tests on CPU tensors through the host emulation of the kernels, test_training_edges_asan.py under
AddressSanitizer.  Tolerances: those of test_training_ops_gpu.py."""
import numpy as np
import pytest
import torch

from dorpatch_amd import ops, optim
from dorpatch_amd.attack import DorPatch
from dorpatch_amd.utils import NormModel, get_normalize
from oracle import toy_models
from test_training_ops_gpu import DTYPES, INF, LOG_S, U, check_grad, check_logp, onehot, policy64, preference64, rand, softmax64

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ---------------------------------------------------------------- logits of every magnitude
MAGNITUDES = [2.0 ** 20, 2.0 ** 22 - 1, 2.0 ** 22, 2.0 ** 24 + 2, 1e9, 2.0 ** 30, 3e9, 1e10, 1e18, 1e20, 1e30, 2.0 ** 100, 2.0 ** 101, 1e38]


def large_rows(V, dtype, few):
    """(logits, labels): for each magnitude of either sign a row of it alone; of it and its neighbour below; ordinary logits beside a
    negative fill in the first half, in every other column, everywhere but at three entries; ordinary logits under one that large."""
    t = DTYPES[dtype]
    base = rand(V, seed=V, scale=3.0)
    rows, labels = [], []
    for k, big in enumerate(MAGNITUDES[::3] if few else MAGNITUDES):
        y = (37 * k + 1) % V
        big = torch.tensor(big).to(t).item()
        for a in (big, -big):
            alone = torch.full((V,), a)
            # the next value of the type away from zero or towards it, whichever is below
            below = torch.tensor(a).to(t).view(torch.int32 if dtype == "fp32" else torch.int16)
            below = (below + (1 if a < 0 else -1)).view(t).float()
            pair = alone.clone()
            pair[1::4] = below
            pair[y] = a
            rows += [alone, pair]
        first, every, most, under = base.clone(), base.clone(), torch.full((V,), -big), base.clone()
        first[:V // 2] = -big
        every[::2] = -big
        most[[0, V // 3, V - 1]] = base[:3]
        under[V // 2] = big
        for r in (first, every, most):
            r[y] = 0.25
        under[y] = 0.25 if y != V // 2 else big
        rows += [first, every, most, under]
        labels += [y] * 8
    x = torch.stack(rows).to(t)
    assert torch.isfinite(x).all()
    return x, torch.tensor(labels)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("V,few,repeat", [(300, False, 1), (2520, False, 1), (9001, True, 1), (40003, True, 1), (33003, True, 2)])
def test_logits_of_every_magnitude(V, few, repeat, dtype):
    """Statistics a wave, a workgroup and slices a row; the policy loss in registers, walked twice (33003: 80 rows), and in slices."""
    x, y = large_rows(V, dtype, few)
    x, y = x.repeat(repeat, 1), y.repeat(repeat)
    R = len(y)
    xd, yd = x.to(DEV), y.to(DEV)
    p, want, entropy, _ = softmax64(x, y)
    logp, ent, stats = ops.label_logprob(xd, yd, want_entropy=True)
    check_logp(logp, want), check_logp(ent, entropy)
    g = rand(R, seed=3)
    check_grad(ops.label_logprob_bwd(xd, yd, stats, g.to(DEV)), g.double()[:, None] * (onehot(y, V) - p), g, p, y, dtype)
    old = (want.clamp(min=-30) - 0.05).float()           # in the clip range, or (the label far under the others) a ratio of 0
    adv, ref = rand(R, seed=4), (want.clamp(min=-30) + 0.1).float()
    weight = torch.where(want < -30, 0.0, 1.0)           # a label that far down has no part in the loss; exp(ref - logp) would be infinite
    ref = torch.where(want < -30, -INF, ref)
    loss, d, lp, h = ops.policy_loss(xd, yd, old.to(DEV), adv.to(DEV), 0.2, 0.28, 0.9, ref_logp=ref.to(DEV), kl_coef=0.04, entropy_coef=0.01, weight=weight.to(DEV))
    wl, wd, wlp, wh, slope, _ = policy64(x, y, old, adv, 0.2, 0.28, 0.9, ref, 0.04, 0.01, weight)
    check_logp(lp, wlp), check_logp(h, wh)
    live = want >= -30
    # as in test_policy_loss: the ratios are off by LOG_S of themselves and four roundings
    off = (adv.abs().double() * torch.exp(wlp - old.double()) + 0.04 * (1 + torch.exp(ref.double() - wlp))) * (LOG_S + 4 * U)
    assert ((loss.cpu().double() - wl).abs() <= off + 0.01 * 2 * LOG_S + 4 * U * (wl.abs() + 0.01 * wh))[live].all()
    check_grad(d.cpu()[live], wd[live], slope[live], p[live], y[live], dtype, g_err=(0.9 * off + 4 * U * slope.abs())[live], entropy=(0.9 * weight * 0.01)[live])
    assert torch.isfinite(d).all() and (d.cpu()[~live] == 0).all()
    keep = live.nonzero()[:, 0]
    keep = keep[:len(keep) // 2 * 2]
    xs, ys = x[keep], y[keep]
    cu = torch.arange(len(keep) + 1, dtype=torch.int32)
    loss, d, seq = ops.preference_loss(xs.to(DEV), ys.to(DEV), cu.to(DEV), None, 0.3, 0.5)
    wl, wd, ws, slope, _ = preference64(xs, ys, cu.tolist(), None, 0.3, 0.0, False, 0.5)
    check_logp(seq, ws)
    assert ((loss.cpu().double() - wl).abs() <= 0.6 * LOG_S + 2 * U * wl.abs()).all()
    check_grad(d, wd, slope, p[keep], ys, dtype, g_err=0.5 * 0.3 * 0.6 * LOG_S / 4 + 2 * U * slope.abs())


# ---------------------------------------------------------------- gradients written into the caller's tensors
def loss_calls(y, r, cu):
    """The losses' calls that write into `out`, by name."""
    return {"label_logprob_bwd": lambda x, out: ops.label_logprob_bwd(x, y, ops.label_logprob(x, y)[2], r, out=out),
            "preference_loss": lambda x, out: ops.preference_loss(x, y, cu, None, 0.3, 1.0, out=out)[1],
            "policy_loss": lambda x, out: ops.policy_loss(x, y, r, r, 0.2, 0.2, 1.0, out=out)[1]}


@pytest.mark.parametrize("name", sorted(loss_calls(None, None, None)))
def test_autograd_notices_a_gradient_written_over_the_logits(name):
    """What an operation before the logits has kept of them is gone: its backward has to say so, not to use the gradient in its place."""
    y, r, cu = torch.tensor([1, 2, 3, 4]).to(DEV), torch.full((4,), -2.0).to(DEV), torch.tensor([0, 2, 4], dtype=torch.int32).to(DEV)
    call = loss_calls(y, r, cu)[name]
    w = rand(6, 9, seed=1).to(DEV).requires_grad_(True)
    h = rand(4, 6, seed=2).to(DEV)
    x = torch.tanh(h @ w)                           # (its backward takes its result)
    before = x._version
    want = call(x.detach(), None)
    assert x._version == before                     # a gradient of its own: nothing of the caller's was written
    d = call(x.detach(), x.detach())
    assert torch.equal(d, want) and torch.equal(x.detach(), want) and x._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        x.backward(d.clone())
    other = torch.zeros(4, 12).to(DEV)
    z = (other * w[0, 0]).sum()                     # keeps `other` for the backward of w
    call(want.clone(), other[:, 1:10])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
    with torch.inference_mode():
        x = rand(4, 9, seed=3).to(DEV)
        assert torch.equal(call(x, x), x)


@pytest.mark.parametrize("cu", [[0, 2147483647, 5], [2147483647, 5, 6], [2147483600, 2147483647, 3], [0, 2147483584, -1], [-2147483648, 2147483647, 2147483647]])
def test_sequences_that_start_behind_every_row(cu):
    """Bounds that are no row at all name no rows: what is inside the tensors counts, and a start near 2^31 does not wrap round."""
    x, y = rand(6, 40, seed=1).to(DEV), torch.ones(6, dtype=torch.int64).to(DEV)
    bounds = torch.tensor(cu, dtype=torch.int32).to(DEV)
    want = softmax64(x, y)[1].sum()
    for grad in (False, True):
        loss, d, seq = ops.preference_loss(x, y, bounds, None, 0.1, 1.0, want_grad=grad)
        assert torch.isfinite(loss).all() and (d is None or torch.isfinite(d).all())
        if cu[0] <= 0 and cu[2] >= 6:               # the first sequence holds all rows
            assert abs(float(seq[0]) - float(want)) <= 6 * LOG_S + 2 * U * abs(float(want)) and seq[1] == 0


# ---------------------------------------------------------------- the attack's AdamW
def attack(stages=None, n_it=2, B=1, hook=None, **extra):
    """A short run on one directory's path: (mask, pattern) on the CPU; `stages`: the stage of every step."""
    H = 56
    model = NormModel(toy_models.make_toy(gain=2.0), get_normalize("imagenet", "resnetv2")).to(DEV)
    g = torch.Generator().manual_seed(5)
    x = torch.rand(B, 3, H, H, generator=g).to(DEV)

    def seen(d):
        if stages is not None:
            stages.append(int(d["stage"]))
        if hook is not None:
            hook(d)
    extra.setdefault("init_mask", torch.rand(B, 1, H, H, generator=g))
    out = DorPatch(verbose=False).generate(model, x, 0.12, 10, "res/cfg/sub", 0, y=torch.arange(1, B + 1).to(DEV), targeted=True, lr=0.01, sampling_size=4,
                                           max_iterations=n_it, init_pattern=torch.rand(B, 3, H, H, generator=g),
                                           rngs=[np.random.RandomState(b) for b in range(B)], step_hook=seen, **extra)
    return [t.cpu() for t in out]


@pytest.mark.parametrize("first,second", [(dict(), dict(update="adamw")), (dict(update="adamw"), dict()),
                                          (dict(update="adamw", adamw=dict(state_bits=8, seed=3)), dict(update="adamw", adamw=dict(state_bits=8, seed=4)))])
def test_attack_stage_0_of_another_update_is_not_taken_for_ones_own(tmp_path, monkeypatch, first, second):
    """Two runs in one directory: each has its own first stage, and gives what it gives alone; a run again takes its own up."""
    for name in ("alone", "both"):
        (tmp_path / name).mkdir()
    monkeypatch.chdir(tmp_path / "alone")
    alone = attack(**second)
    monkeypatch.chdir(tmp_path / "both")
    attack(**first)
    stages = []
    got = attack(stages, **second)
    assert stages == [0, 0, 1, 1] and all(torch.equal(a, b) for a, b in zip(got, alone))
    for options in (first, second):
        stages = []
        attack(stages, **options)
        assert stages == [1, 1]


def test_attack_adamw_takes_a_gradient_that_is_not_finite_for_none(tmp_path, monkeypatch):
    """One step's gradient holds infinities and a NaN: there it counts as 0 in pattern and mask, and both go on as by the formula."""
    monkeypatch.chdir(tmp_path)
    seen, bad = [], [(0, 20, 30, INF), (1, 33, 9, -INF), (2, 41, 40, float("nan"))]

    def plant(d):
        seen.append({k: (d[k].detach().cpu().clone() if torch.is_tensor(d[k]) else np.array(d[k])) for k in ("stage", "grad_pattern", "grad_mask", "mask", "pattern", "lr")})
        if d["i"] == 1:
            for c, h, w, value in bad:
                d["g_adv"][0, c, h, w] = value
                seen[-1]["grad_pattern"][0, c, h, w] = seen[-1]["grad_mask"][0, 0, h, w] = 0.0
    attack(n_it=4, hook=plant, update="adamw", adamw=dict(betas=(0.8, 0.95)))
    for name, learned_in in (("pattern", (0, 1)), ("mask", (0,))):
        for stage in learned_in:
            steps = [d for d in seen if d["stage"] == stage]
            m = v = torch.zeros_like(steps[0][name]).double()
            for t, (d, after) in enumerate(zip(steps, steps[1:]), 1):
                g = d["grad_" + name].double().nan_to_num(nan=0.0)
                m, v = 0.8 * m + 0.2 * g, 0.95 * v + 0.05 * g * g
                lr = torch.from_numpy(d["lr"]).double().view(-1, 1, 1, 1)
                change = lr * (m / (1 - 0.8 ** t)) / ((v / (1 - 0.95 ** t)).sqrt() + 1e-8)
                want = (d[name].double() - change).clamp(0, 1)
                # as in test_pattern_and_mask_follow_adamw
                assert ((after[name].double() - want).abs() <= 2 * U * (want.abs() + d[name].abs()) + (3 * t + 8) * U * (change.abs() + lr)).all(), (name, stage, t)
    assert len(seen) == 8 and all(torch.isfinite(d[k]).all() for d in seen for k in ("pattern", "mask"))


# ---------------------------------------------------------------- sizes beyond the kernels' own numbers
def test_losses_refuse_sizes_that_do_not_fit_their_32_bits():
    """A row of 2^32 + 8 categories is none of 8, nor 2^32 + 1 pairs one: the sizes are looked at before they become C integers.  (The
    tensors are broadcast or lie on the meta device: no memory is behind them.)"""
    def refused(match, call, *a, **k):
        with pytest.raises(ValueError, match=match):
            call(*a, **k)
    y = torch.tensor(3).to(DEV)
    for V in (2 ** 30 + 1, 2 ** 31, 2 ** 32 + 8):
        refused("categories", ops._rows, torch.empty(V, dtype=torch.bfloat16, device="meta"))
    for rows in (2 ** 23 + 1, 2 ** 31, 2 ** 32 + 5):
        refused("rows", ops._rows, torch.zeros(1, 1).to(DEV).expand(rows, 1))
        refused("rows", ops._rows, torch.zeros(1, 1, 1).to(DEV).expand(2, rows, 1))
    x = torch.zeros(4, 8).to(DEV)
    for pairs in (2 ** 24, 2 ** 31, 2 ** 32 + 1):
        refused("pairs", ops._pairs, torch.empty(2 * pairs + 1, dtype=torch.int32, device="meta"))
    assert ops._rows(x)[1] == 4 and ops._pairs(torch.zeros(5, dtype=torch.int32)) == 2


def test_c_entry_refuses_more_pairs_than_a_launch_takes():
    """2^24 workgroups of 256 are 2^32 threads, one more than a launch has."""
    import ctypes
    from dorpatch_amd import _lib
    lib, P = _lib.load(), ctypes.c_void_p
    x, y, o = torch.zeros(4, 8).to(DEV), torch.zeros(4, dtype=torch.int64).to(DEV), torch.zeros(64).to(DEV)
    d = _lib.DpLogits(data=x.data_ptr(), dtype=0, rows=4, vocab=8, inner=4, outer_stride=0, row_stride=8)
    for pairs in (2 ** 24, 2 ** 30, 2 ** 31 - 1, 0, -1):        # (nothing is read of what the pointers name)
        assert lib.dp_preference_loss(ctypes.byref(d), P(y.data_ptr()), P(y.data_ptr()), pairs, None, 0.1, 1.0, 0.0, 0, P(o.data_ptr()), P(o.data_ptr()), None,
                                      P(o.data_ptr()), ops._stream()) == 1, pairs


# ---------------------------------------------------------------- AdamW
def test_adamw_refuses_gradients_that_lie_on_parameters():
    """A step writes its parameters while others of its workgroups still read gradients: a gradient on another parameter, or askew on
    its own, would be read before or after, as it happens.  A parameter that is its own gradient is read where it is written."""
    def parameters():
        return [torch.full((5000,), 1.0).to(DEV), torch.full((5000,), 2.0).to(DEV), torch.full((300,), 3.0).to(DEV)]
    one = torch.ones(5000).to(DEV)
    for max_norm in (None, 1.0):
        a, b, c = parameters()
        opt = optim.AdamW([a, b, c], weight_decay=0.0, max_norm=max_norm)
        for grads in ([b, a, c], [one, a, None], [one, one, b[4000:4300]], [one, one, a[:300]]):
            with pytest.raises(RuntimeError, match="dp_adamw_step"):
                opt.step(grads)
        flat = torch.ones(5001).to(DEV)
        askew = optim.AdamW([flat[1:]], max_norm=max_norm)
        with pytest.raises(RuntimeError, match="dp_adamw_step"):
            askew.step([flat[:-1]])
        assert opt.steps == askew.steps == 0 and (flat == 1).all()
        assert all(torch.equal(p, q) for p, q in zip((a, b, c), parameters()))
        opt.step([a, None, b[:300]])                # its own; a parameter that this step does not write
        assert (b == 2).all() and opt.steps == 1
        for p, before in ((a, 1.0), (c, 3.0)):      # step 1 moves an element by lr against its gradient's sign
            assert ((p - (before - 1e-3)).abs() <= 4 * U * before).all()


def test_attack_adamw_needs_an_eps(tmp_path, monkeypatch):
    """A cell that is all 0 has no gradient: without eps its step would be 0 / 0."""
    monkeypatch.chdir(tmp_path)
    for eps in (0.0, 1e-60, -1e-8, float("nan")):       # (1e-60: 0 in the kernel's 32 bits)
        with pytest.raises(ValueError, match="eps"):
            attack(update="adamw", adamw=dict(eps=eps))


@pytest.mark.parametrize("V", [300, 2520, 9001, 40003])
def test_logits_on_both_sides_of_the_far_border(V):
    """References of 2^22 and more take differences, smaller ones do not: rows whose lanes hold the one and the other are joined."""
    spread = rand(6, V, seed=V, scale=4.0)
    x = torch.stack([s * 2.0 ** 22 + spread[k] for k, s in enumerate((1.0, -1.0, 1.0, -1.0, 1.0, -1.0))])
    x[2:4, ::2] = spread[2:4, ::2]                  # ordinary ones, far below or above
    x[4, V // 2:] += 16.0                           # ascending and descending borders
    x[5, :V // 2] -= 16.0
    y = x.argmax(1)
    y[1] = 0
    p, want, entropy, _ = softmax64(x, y)
    xd, yd = x.to(DEV), y.to(DEV)
    logp, ent, stats = ops.label_logprob(xd, yd, want_entropy=True)
    check_logp(logp, want), check_logp(ent, entropy)
    one = torch.ones(6)
    check_grad(ops.label_logprob_bwd(xd, yd, stats, one.to(DEV)), onehot(y, V) - p, one, p, y, "fp32")
    old, adv = want.float(), torch.ones(6)
    loss, d, lp, h = ops.policy_loss(xd, yd, old.to(DEV), adv.to(DEV), 0.2, 0.2, 1.0, entropy_coef=0.1)
    wl, wd, wlp, wh, slope, _ = policy64(x, y, old, adv, 0.2, 0.2, 1.0, None, 0.0, 0.1, None)
    check_logp(lp, wlp), check_logp(h, wh)
    check_grad(d, wd, slope, p, y, "fp32", g_err=LOG_S + 4 * U, entropy=0.1)


def test_preference_loss_of_nothing_writes_zeroes_into_a_leaf():
    """No pairs: the gradient is zeroes, written over logits that require one as any other is, and no operation of their graph."""
    y, cu = torch.tensor([1, 2]).to(DEV), torch.zeros(1, dtype=torch.int32).to(DEV)
    leaf = rand(2, 9, seed=1).to(DEV).requires_grad_(True)
    before = leaf._version
    loss, d, seq = ops.preference_loss(leaf, y, cu, None, 0.3, 1.0, out=leaf)
    assert d is leaf and (d == 0).all() and loss.numel() == seq.numel() == 0 and leaf.is_leaf and leaf._version > before
    inner = torch.tanh(rand(2, 9, seed=2).to(DEV).requires_grad_(True))
    node = inner.grad_fn
    ops.preference_loss(inner, y, cu, None, 0.3, 1.0, out=inner)
    assert inner.grad_fn is node and (inner == 0).all()
    none, ref = torch.zeros(0, 9).to(DEV), torch.tensor([0.5, -1.0]).to(DEV).requires_grad_(True)
    loss, d, seq = ops.preference_loss(none, y[:0], torch.zeros(3, dtype=torch.int32).to(DEV), ref, 0.3, 1.0)
    assert not loss.requires_grad and abs(float(loss) - float(torch.nn.functional.softplus(torch.tensor(0.45)))) <= 4 * U
