"""The training operators as a program runs them on the device: captured and replayed, on streams of their own, on tensors whose offsets
pass 32 bits."""
import pytest
import torch

from dorpatch_amd import ops, optim

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


class Step(object):
    """One training step on buffers of its own; `run` may be captured."""

    def __init__(self, bits, max_norm, seed=0, R=40, V=3001, dtype=torch.bfloat16):
        self.x = rand(R, V, seed=seed, scale=3).to(DEV, dtype)
        g = torch.Generator().manual_seed(seed)
        self.y = torch.randint(0, V, (R,), generator=g).to(DEV)
        self.y[::7] = -100
        self.old = ops.label_logprob(self.x, self.y)[0] + 0.1
        self.adv = rand(R, seed=seed + 1).to(DEV)
        self.cu = torch.tensor([0, 11, 20, 33, R], dtype=torch.int32, device=DEV)
        self.p = [rand(R, V, seed=seed + 2).to(DEV), rand(V, seed=seed + 3).to(DEV, torch.bfloat16)]
        self.opt = optim.AdamW(self.p, lr=1e-2, weight_decay=0.01, state_bits=bits, max_norm=max_norm, capturable=True, seed=3)

    def run(self):
        lp, ent, stats = ops.label_logprob(self.x, self.y, want_entropy=True)
        one = ops.label_logprob_bwd(self.x, self.y, stats, self.adv)
        loss, dl, _, _ = ops.policy_loss(self.x, self.y, self.old, self.adv, 0.2, 0.2, 0.1, ref_logp=lp, kl_coef=0.1, entropy_coef=0.01)
        pref, dp, seq = ops.preference_loss(self.x, self.y, self.cu, None, 0.01, 1.0)
        g = (one + dl + dp).float()
        norm = self.opt.step([g, g[3].bfloat16()])
        return [lp, ent, one, loss, dl, pref, dp, seq] + ([norm] if norm is not None else [])

    def all(self):
        o = self.opt
        return [t.clone() for t in self.p + [o.exp_avg.view(torch.uint8), o.exp_avg_sq.view(torch.uint8), o._counter]]


def same(a, b):
    return len(a) == len(b) and all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("bits,max_norm", [(32, None), (32, 1.0), (8, 1.0), (8, None)])
def test_a_captured_step_replays_as_the_eager_one(bits, max_norm):
    """Two steps captured into graphs of their own, replayed in turn with eager work between: every replay as the eager run."""
    eager = [Step(bits, max_norm, seed=s) for s in (0, 10)]
    caught = [Step(bits, max_norm, seed=s) for s in (0, 10)]
    for e, c in zip(eager, caught):
        e.run(), c.run()                            # before a capture everything has run once
    graphs, outs = [], []
    torch.cuda.synchronize()
    for c in caught:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(c.run())
        graphs.append(graph)
    for turn in range(4):
        for e, c, graph, out in zip(eager, caught, graphs, outs):
            e.x.add_(0.01 * turn)
            c.x.add_(0.01 * turn)
            graph.replay()
            junk = torch.randn(1 << 20, device=DEV).sum()
            want = e.run()
            assert same(out, want), turn
            assert same(c.all(), e.all()), turn
            assert torch.isfinite(junk)
        torch.cuda.synchronize()
    assert eager[0].opt.steps == caught[0].opt.steps == 5


def test_an_optimiser_that_counts_on_the_host_is_not_captured():
    p = torch.zeros(100, device=DEV)
    opt = optim.AdamW([p])
    g = torch.ones(100, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(graph):
            opt.step([g])
    torch.cuda.synchronize()
    assert opt.steps == 0 and (p == 0).all()


def test_steps_on_streams_of_their_own():
    want, got = [Step(8, 1.0, seed=s) for s in (0, 10)], [Step(8, 1.0, seed=s) for s in (0, 10)]
    streams = [torch.cuda.Stream() for _ in got]
    first = [w.run() for w in want]
    second = [w.run() for w in want]
    torch.cuda.synchronize()
    mine = []
    for turn in range(2):                           # both streams at once
        for s, g in zip(streams, got):
            with torch.cuda.stream(s):
                mine.append(g.run())
    torch.cuda.synchronize()
    assert same(mine[0], first[0]) and same(mine[1], first[1]) and same(mine[2], second[0]) and same(mine[3], second[1])
    assert all(same(w.all(), g.all()) for w, g in zip(want, got))


def test_offsets_past_32_bits():
    """2.2e9 elements of logits (4.4 GB): the last rows as the same rows by themselves, forward and gradients; bits and all, but for the
    number of slices, which goes by the number of rows."""
    R, V = 17000, 131072
    x = torch.empty(R, V, dtype=torch.bfloat16, device=DEV)
    block = rand(500, V, seed=1, scale=3).to(DEV, torch.bfloat16)
    for r in range(0, R, 500):
        x[r:r + 500] = block
    y = torch.randint(0, V, (500,), generator=torch.Generator().manual_seed(2)).to(DEV).repeat(R // 500)
    adv = rand(500, seed=3).to(DEV).repeat(R // 500)
    logp, ent, stats = ops.label_logprob(x, y, want_entropy=True)
    assert same([t.view(R // 500, -1)[-1] for t in (logp, ent, stats)], [t.view(R // 500, -1)[0] for t in (logp, ent, stats)])
    lp64 = torch.log_softmax(block[-8:].double(), 1).gather(1, y[-8:, None])[:, 0]
    assert (logp[-8:].double() - lp64).abs().max() <= 6e-6 + 2 ** -23 * 30
    d = ops.label_logprob_bwd(x, y, stats, adv)
    assert torch.equal(d[-500:], d[:500])
    loss, d, _, _ = ops.policy_loss(x, y, logp, adv, 0.2, 0.2, 1.0, entropy_coef=0.01, out=d)
    assert torch.equal(d[-500:], d[:500]) and torch.equal(loss[-500:], loss[:500])
    cu = torch.arange(0, R + 1, 250, dtype=torch.int32, device=DEV)
    loss, d, seq = ops.preference_loss(x, y, cu, None, 1e-3, 1.0, out=d)
    assert torch.equal(d[-500:], d[:500]) and torch.equal(loss[-1:], loss[:1])
    # a (B, T, V) tensor whose batches lie further apart than 2^31 elements
    far = x.as_strided((2, 3, V), ((R - 500) * V, V, 1))
    a, _, _ = ops.label_logprob(far, torch.stack([y[:3], y[:3]]))
    assert torch.equal(a[0], a[1])


@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_past_32_bits(bits):
    n = 2 ** 31 + 5000
    p = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    g = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    part = rand(4000, seed=1).to(DEV, torch.bfloat16)
    for at in (0, 2 ** 31 - 2000, n - 4000):        # (the last two share 1000 elements)
        g[at:at + 4000] = part
    written = [g[:4000], g[2 ** 31 - 2000:]]
    opt = optim.AdamW([p], lr=1e-2, weight_decay=0.0, state_bits=bits, max_norm=1e6)
    norm = opt.step([g])
    want = sum(float(w.double().square().sum()) for w in written) ** 0.5
    assert abs(float(norm) - want) <= 1e-5 * want
    for q, w in zip((p[:4000], p[2 ** 31 - 2000:]), written):
        # the first step moves by lr against the sign, where the gradient is far over eps
        assert ((q.float() + 1e-2 * torch.sign(w.float())).abs() <= 1e-2 * 2 ** -7).all()
    assert p[10000:20000].abs().max() == 0 and opt.steps == 1


def test_many_short_rows():
    R, V = 300001, 5
    x, y = rand(R, V, seed=1).to(DEV), torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(2)).to(DEV)
    logp, _, stats = ops.label_logprob(x, y)
    want = torch.log_softmax(x.double(), 1).gather(1, y[:, None])[:, 0]
    assert (logp.double() - want).abs().max() <= 6e-6
    loss, d, _, _ = ops.policy_loss(x, y, logp, torch.ones(R, device=DEV), 0.2, 0.2, 1.0)
    w = torch.softmax(x.double(), 1) - torch.nn.functional.one_hot(y, V)
    assert (d.double() - w).abs().max() <= 2e-5


def test_rows_of_4_to_6_kb():
    """A wave a row from 4096 rows on, a workgroup a row below: the same rows both ways, and against 64 bits."""
    R, V = 4096, 1400
    x, y = rand(R, V, seed=1, scale=3).to(DEV), torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(2)).to(DEV)
    x[:, 3] = -float("inf")
    y[y == 3] = 4
    y[::9] = -1
    logp, ent, stats = ops.label_logprob(x, y, want_entropy=True)
    few, e, st = ops.label_logprob(x[:200], y[:200], want_entropy=True)
    p = torch.softmax(x.double(), 1)
    want = torch.log_softmax(x.double(), 1).gather(1, y.clamp(min=0)[:, None])[:, 0] * (y >= 0)
    h = -torch.xlogy(p, p).sum(1) * (y >= 0)
    for a, b, n in ((logp, ent, R), (few, e, 200)):
        assert (a.double() - want[:n]).abs().max() <= 6e-6 and (b.double() - h[:n]).abs().max() <= 6e-6
    w = (torch.nn.functional.one_hot(y.clamp(min=0), V) - p) * (y >= 0)[:, None]
    one = torch.ones(R, device=DEV)
    for d, n in ((ops.label_logprob_bwd(x, y, stats, one), R), (ops.label_logprob_bwd(x[:200], y[:200], st, one[:200]), 200)):
        assert (d.double() - w[:n]).abs().max() <= 2e-5


def test_tensors_of_the_host_are_refused_and_mixed_ones():
    x, y = torch.randn(4, 9, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    r = torch.zeros(4, device=DEV)
    for call in (lambda: ops.label_logprob(x.cpu(), y.cpu()), lambda: ops.label_logprob(x.cpu(), y), lambda: ops.label_logprob(x, y.cpu()),
                 lambda: ops.policy_loss(x, y, r.cpu(), r, 0.2, 0.2, 1.0), lambda: ops.policy_loss(x, y, r, r, 0.2, 0.2, 1.0, weight=r.cpu()),
                 lambda: ops.preference_loss(x, y, torch.zeros(3, dtype=torch.int32), None, 0.1, 1.0), lambda: optim.AdamW([torch.zeros(4)])):
        with pytest.raises(RuntimeError):
            call()
    opt = optim.AdamW([r])
    with pytest.raises(RuntimeError):
        opt.step([torch.zeros(4)])
    with pytest.raises(ValueError):
        ops.label_logprob_bwd(x, y, ops.label_logprob(x, y)[2], r, out=x.cpu())
