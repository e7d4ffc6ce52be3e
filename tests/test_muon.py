"""The Muon optimizer: its passes and whole steps against 64-bit arithmetic, what it takes for a matrix, training with it."""
import math

import pytest
import torch

from tests.test_newton_schulz import BOUND, exact, matrices
from tnn_b200.models import zoo
from tnn_b200.nn.graph import Graph
from tnn_b200.nn.layers import BatchNorm, Conv2D, Dense, Flatten, ReLU
from tnn_b200.nn.optim import Muon, OverlappedUpdate, create_optimizer
from tnn_b200.ops import functional as F
from tnn_b200.ops import raw
from tnn_b200.trainer import Trainer
from tnn_b200.utils.config import TrainingConfig

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("m,n,offsets", [(8, 12, (0, 200, 400)), (5, 7, (3, 40)), (1, 1, (2,)), (64, 96, tuple(range(0, 6144 * 9, 6144)))])
@pytest.mark.parametrize("nesterov", [True, False])
def test_passes(dev, m, n, offsets, nesterov):
    total, count = max(offsets) + m * n + 5, len(offsets)
    gen = torch.Generator().manual_seed(m)
    grads, master, buf = (torch.randn(s, generator=gen) for s in ((total,), (total,), (count, m, n)))
    low = master.to(torch.bfloat16)
    group = raw.MatrixGroup(m, n, offsets, dev)
    b2, g64 = buf.clone().to(dev), torch.stack([grads[o:o + m * n] for o in offsets]).view(count, m, n).double() * 0.5
    u = raw.muon_momentum(grads.to(dev), group, b2, 0.9, nesterov, 0.5)
    want = 0.9 * buf.double() + 0.1 * g64
    size = buf.double().abs() + g64.abs()
    # a handful of fp32 roundings (and those of 0.9 and 0.1 themselves)
    assert bool(((b2.cpu().double() - want).abs() <= 6 * 2.0 ** -24 * size).all())
    want_u = 0.9 * want + 0.1 * g64 if nesterov else want
    assert bool(((u.cpu().double() - want_u).abs() <= 12 * 2.0 ** -24 * size).all())
    o = torch.randn(count, m, n, generator=gen).to(torch.bfloat16)
    w, l = master.clone().to(dev), low.clone().to(dev)
    raw.muon_apply(w, l, group, o.to(dev), 0.02, 1.5, 0.1)
    ref = master.double()
    touched = torch.zeros(total, dtype=torch.bool)
    for k, at in enumerate(offsets):
        x = ref[at:at + m * n]
        ref[at:at + m * n] = x - 0.02 * (1.5 * o[k].double().reshape(-1) + 0.1 * x)
        touched[at:at + m * n] = True
    assert bool(((w.cpu().double() - ref).abs() <= 8 * 2.0 ** -24 * (ref.abs() + 0.1)).all())
    assert torch.equal(w.cpu()[~touched], master[~touched]) and torch.equal(l.cpu()[~touched], low[~touched])
    assert torch.equal(l.cpu()[touched], w.cpu()[touched].to(torch.bfloat16))


@pytest.mark.parametrize("dev", DEVICES)
def test_adam_on_pieces(dev):
    total = 5000
    gen = torch.Generator().manual_seed(1)
    master, grads = torch.randn(total, generator=gen), torch.randn(total, generator=gen)
    pieces = torch.tensor([[3, 1, 0], [100, 700, 1], [4000, 1000, 701]], dtype=torch.int64)
    where = torch.cat([torch.arange(a, a + n) for a, n, _ in pieces.tolist()])
    w, m, v = master.clone().to(dev), torch.zeros(1701, device=dev), torch.zeros(1701, device=dev)
    w2, m2, v2 = master[where].clone(), torch.zeros(1701), torch.zeros(1701)
    for step in (1, 2, 3):
        raw.adam_pieces(w, None, grads.to(dev), m, v, pieces.to(dev), 0.01, 0.9, 0.95, 1e-8, 0.1, step, 0.5, 0.25)
        raw.adam_step(w2, None, grads[where], m2, v2, 0.0025, 0.9, 0.95, 1e-8, 0.1, step, 0.5)
    assert torch.allclose(w.cpu()[where], w2, rtol=1e-5, atol=1e-6) and torch.allclose(v.cpu(), v2, rtol=1e-5, atol=1e-9)
    rest = torch.ones(total, dtype=torch.bool)
    rest[where] = False
    assert torch.equal(w.cpu()[rest], master[rest])


def test_what_counts_as_a_matrix():
    g = zoo.gpt2(64, 1, 2, "t", seq_len=16, vocab=50).compile(device="cpu", seed=0)
    opt = create_optimizer({"type": "muon", "learning_rate": 0.01, "momentum": 0.9}).attach(g)
    assert isinstance(opt, Muon) and opt.momentum == 0.9
    assert {(x.m, x.n): len(x.offsets) for x in opt.groups} == {(192, 64): 2, (64, 64): 2, (256, 64): 2, (64, 256): 2}
    matrices_, others = sum(x.size * len(x.offsets) for x in opt.groups), int(opt.pieces[:, 1].sum())
    assert matrices_ + others == g.num_parameters() and opt.m.numel() == others
    h = Graph()
    x = ReLU()(BatchNorm(8)(Conv2D(3, 8, 3, 3, pad_h=1, pad_w=1)(h.input("input"))))
    y = Dense(8 * 16, 10)(Flatten()(x))
    y.set_uid("output")
    h.set_output(y)
    h.compile(device="cpu", seed=0)
    opt = Muon().attach(h)
    assert [(x.m, x.n) for x in opt.groups] == [(8, 27)]
    assert int(opt.pieces[:, 1].sum()) == 8 + 16 + 1280 + 10  # filter bias, the norm's weights (not its statistics), the output layer


@pytest.mark.parametrize("dev", DEVICES)
def test_step_of_a_graph(dev):
    """One update of every parameter against the formulas, from the gradients of a real backward pass."""
    g = zoo.gpt2(64, 1, 2, "t", seq_len=16, vocab=50, drop=0.0).compile(device=dev, seed=0)
    opt = create_optimizer({"type": "muon", "learning_rate": 0.02, "weight_decay": 0.1, "adam_learning_rate": 0.001}).attach(g)
    ids = torch.randint(0, 50, (2, 16), generator=torch.Generator().manual_seed(3)).to(dev)
    out = g.forward({"input": ids})["output"]
    _, grad = __import__("tnn_b200.nn.loss", fromlist=["x"]).CrossEntropyLoss().compute(out, ids, 1.0)
    g.backward({"output": grad})
    before, grads = g.master_flat.cpu().double(), g.grads_flat.cpu().double()
    opt.update()
    after = g.master_flat.cpu().double()
    for group in opt.groups:
        for at in group.offsets:
            gm = grads[at:at + group.size].view(group.m, group.n)
            u = 0.95 * 0.05 * gm + 0.05 * gm
            step = 0.02 * (max(1.0, group.m / group.n) ** 0.5 * exact(u) + 0.1 * before[at:at + group.size].view(group.m, group.n))
            got = before[at:at + group.size].view(group.m, group.n) - after[at:at + group.size].view(group.m, group.n)
            assert float((got - step).norm() / step.norm()) < BOUND + 1e-3  # and the weights' own fp32 rounding
    for at, n, _ in opt.pieces.tolist():
        gp = grads[at:at + n]
        want = before[at:at + n] - 0.001 * gp / (gp.abs() + 1e-8)  # Adam's first step
        assert bool(((after[at:at + n] - want).abs() <= 2e-5 * 0.001 + 4 * 2.0 ** -24 * want.abs() + 0.001 * 1e-6).all())
    if dev == "cuda":
        assert torch.equal(g.params_flat, g.master_flat.to(torch.bfloat16))


def test_state_can_be_saved():
    def make():
        g = zoo.gpt2(64, 1, 1, "t", seq_len=8, vocab=20).compile(device="cpu", seed=0)
        return g, Muon(0.01).attach(g)

    (g1, o1), (g2, o2) = make(), make()
    for k in range(3):
        g1.grads_flat.copy_(torch.randn(g1.total_elems, generator=torch.Generator().manual_seed(k)))
        o1.update()
    saved = {k: v.clone() for k, v in o1.state_dict().items()}
    g2.master_flat.copy_(g1.master_flat)
    o2.load_state_dict(saved)
    for g, o in ((g1, o1), (g2, o2)):
        g.grads_flat.copy_(torch.randn(g.total_elems, generator=torch.Generator().manual_seed(9)))
        o.update()
    assert torch.equal(g1.master_flat, g2.master_flat)


def test_refusals():
    with pytest.raises(ValueError):
        Muon(0.0)
    with pytest.raises(ValueError):
        Muon(ns_steps=0)
    g = zoo.gpt2(64, 1, 1, "t", seq_len=8, vocab=20).compile(device="cpu", seed=0)
    opt = Muon().attach(g)
    with pytest.raises(ValueError):
        opt.update(sl=slice(0, 8))
    assert not OverlappedUpdate.usable(opt, g)
    group = raw.MatrixGroup(4, 6, [10], "cpu")
    flat, buf = torch.zeros(33), torch.zeros(1, 4, 6)
    for call in (lambda: raw.muon_momentum(flat, group, buf, 0.9),  # 34 elements needed
                 lambda: raw.muon_momentum(torch.zeros(34), group, buf[0], 0.9),
                 lambda: raw.muon_momentum(torch.zeros(34), group, buf.double(), 0.9),
                 lambda: raw.muon_apply(flat, None, group, buf.to(torch.bfloat16), 0.1, 1.0),
                 lambda: raw.muon_apply(torch.zeros(34), None, group, buf, 0.1, 1.0),
                 lambda: raw.muon_apply(torch.zeros(34), torch.zeros(34), group, buf.to(torch.bfloat16), 0.1, 1.0),
                 lambda: raw.MatrixGroup(0, 4, [0], "cpu"), lambda: raw.MatrixGroup(2, 4, [], "cpu")):
        with pytest.raises(ValueError):
            call()
    from tnn_b200.parallel import dp
    with pytest.raises(ValueError, match="whole matrices"):
        dp.FusedDPOptimizer(opt, g, None, [], 1.0)


@gpu
def test_captured_training_steps_equal_eager_ones():
    cfg = {"model_name": "t", "batch_size": 4, "optimizer": {"type": "muon", "learning_rate": 0.02, "adam_learning_rate": 2e-3}}
    seq = torch.randint(0, 203, (4, 129), generator=torch.Generator().manual_seed(1))
    d, l = seq[:, :-1].contiguous(), seq[:, 1:].contiguous()
    weights = []
    for captured in (False, True):
        g = zoo.gpt2(128, 2, 2, "t", seq_len=128, vocab=203, drop=0.0).compile(device="cuda", seed=3)
        t = Trainer(TrainingConfig.from_dict(cfg), graph=g, log=False)
        if captured:
            t.enable_cuda_graph(d, l, warmup=2)  # two steps, and one on the capturing stream
        else:
            for _ in range(3):
                t.train_step(d, l)
        for _ in range(2):
            t.train_step(d, l)
        t.optimizer.set_learning_rate(0.01)
        loss = t.train_step(d, l)
        weights.append(g.master_flat.clone())
        assert math.isfinite(float(loss))
        t.close()
    # weight gradients and embeddings are added up by atomics in both, so that steps agree to their noise only
    assert float((weights[0] - weights[1]).norm() / weights[0].norm()) < 1e-2


@pytest.mark.parametrize("dev,dtype", [("cpu", torch.float32), pytest.param("cuda", torch.bfloat16, marks=gpu)])
def test_operators_together(dev, dtype):
    """Embedding, products, token log probabilities, their gradients and an orthogonalised update, as a training step uses them."""
    V, E, T = 301, 64, 48
    gen = torch.Generator().manual_seed(5)
    table0, w0, head0 = torch.randn(V, E, generator=gen) * 0.2, torch.randn(E, E, generator=gen) / 8, torch.randn(V, E, generator=gen) / 8
    ids, nxt = torch.randint(0, V, (2, T), generator=gen), torch.randint(0, V, (2, T), generator=gen)
    nxt[0, :5] = -100

    def step(dev, dtype, rounded):
        table, w, head = (t.to(dtype).to(rounded).to(dev).clone().requires_grad_() for t in (table0, w0, head0))
        x = F.embedding(ids.to(dev), table, scale=8.0, padding_idx=7)
        logits = F.linear(F.linear(x, w, None, gelu=True), head, None)
        r = F.token_log_probs(logits, nxt.to(dev), 3, 0.9)
        loss = -r.log_probs.mean() - 0.1 * r.entropy.mean()
        loss.backward()
        return [t.detach().double().cpu() for t in (r.log_probs, r.entropy, table.grad, w.grad, head.grad,
                                                    raw.newton_schulz(w.grad))], r.top_indices

    got, _ = step(dev, dtype, dtype)
    ref, _ = step("cpu", dtype, torch.float32)  # from the same (rounded) weights
    # bf16 activations: three roundings between table and logits of 2^-8 each, logits of size about 3 that are rounded once more
    tol = {torch.float32: 1e-5, torch.bfloat16: 0.03}[dtype]
    for a, b in zip(got[:5], ref[:5]):
        assert float((a - b).norm() / b.norm()) < tol
    own = got[3].to(torch.float32)
    assert float((got[5] - exact(own)).norm() / exact(own).norm()) < BOUND


def test_stages_of_a_pipeline_take_the_same_matrices():
    """The layer in front of a cut is not the model's last: all stages together orthogonalise what the whole model does."""
    from tnn_b200.nn.graph import partition_graph

    make = lambda: zoo.gpt2(64, 2, 2, "t", seq_len=16, vocab=50)  # noqa: E731
    count = lambda opt: {(x.m, x.n): len(x.offsets) for x in opt.groups}  # noqa: E731
    whole = count(Muon().attach(make().compile(device="cpu", seed=0)))
    for cuts in ([1.0, 1.0], [1.0, 1.0, 1.0, 1.0, 1.0]):
        parts = {}
        for stage in partition_graph(make(), cuts):
            for k, v in count(Muon().attach(stage.compile(device="cpu", seed=0))).items():
                parts[k] = parts.get(k, 0) + v
        assert parts == whole


def test_refusals_of_places():
    flat = torch.zeros(64)
    for offsets in ([0, 0], [0, 23], [30, 8]):
        with pytest.raises(ValueError, match="overlap"):
            raw.MatrixGroup(4, 6, offsets, "cpu")
    pieces = torch.tensor([[0, 8, 0]])
    m, v = torch.zeros(8), torch.zeros(8)
    bad = [dict(pieces=pieces.int()), dict(pieces=pieces[0]), dict(m=m.double()), dict(v=torch.zeros(9)), dict(grads=torch.zeros(63)),
           dict(low=torch.zeros(63)), dict(master=flat.bfloat16())]
    for change in bad:
        args = dict(master=flat, low=None, grads=torch.zeros(64), m=m, v=v, pieces=pieces)
        args.update(change)
        with pytest.raises(ValueError):
            raw.adam_pieces(*args.values(), 0.1, 0.9, 0.95, 1e-8, 0.0, 1)


@gpu
def test_places_on_another_device_are_refused():
    group = raw.MatrixGroup(4, 6, [0], "cpu")
    with pytest.raises(ValueError):
        raw.muon_momentum(torch.zeros(24, device="cuda"), group, torch.zeros(1, 4, 6, device="cuda"), 0.9)
    with pytest.raises(ValueError):
        raw.muon_apply(torch.zeros(24, device="cuda"), None, group, torch.zeros(1, 4, 6, device="cuda", dtype=torch.bfloat16), 0.1, 1.0)


def test_replicas_reduced_by_the_library():
    """The update of data-parallel replicas that all-reduce their gradients: scaled by a power of two, the same bits."""
    from tnn_b200.parallel import dp

    g1, g2 = (zoo.gpt2(64, 1, 1, "t", seq_len=8, vocab=20).compile(device="cpu", seed=0) for _ in range(2))
    one = dp.NcclDPOptimizer(Muon(0.01), g1, [dp.Region(0, g1.total_elems, [0], None)], 0.5)
    two = Muon(0.01).attach(g2)
    for k in range(2):
        grads = torch.randn(g1.total_elems, generator=torch.Generator().manual_seed(k))
        g1.grads_flat.copy_(grads)
        g2.grads_flat.copy_(grads * 0.5)
        one.update()
        two.update()
    assert torch.equal(g1.master_flat, g2.master_flat)


BAD_PIECES = [(60, 5, 0), (-1, 3, 0), (0, 3, 18), (5, 4, -2), (5, -4, 2), (2 ** 62, 2 ** 62, 0), (0, 2 ** 63 - 1, 2 ** 63 - 1)]


@pytest.mark.parametrize("bad", BAD_PIECES)
def test_pieces_outside_of_the_buffers_on_the_cpu(bad):
    w = torch.ones(64)
    m, v = torch.zeros(20), torch.zeros(20)
    with pytest.raises(ValueError):
        raw.adam_pieces(w, None, torch.ones(64), m, v, torch.tensor([(3, 4, 0), bad]), 0.1, 0.9, 0.95, 1e-8, 0.0, 1)
    assert torch.equal(w, torch.ones(64)) and not bool(m.any())


@gpu
@pytest.mark.parametrize("bad", BAD_PIECES)
def test_pieces_outside_of_the_buffers_on_the_gpu(bad):
    """Left out and recorded; the others are worked on."""
    from tnn_b200.ops import _lib

    w, ref, grads = (torch.ones(64, device="cuda") for _ in range(3))
    state, state_ref = torch.zeros(2, 20, device="cuda"), torch.zeros(2, 20, device="cuda")
    good = torch.tensor([(3, 4, 0), (48, 16, 4)], device="cuda")
    both = torch.cat([good[:1], torch.tensor([bad], device="cuda"), good[1:]])
    _lib.check_status()
    raw.adam_pieces(ref, None, grads, *state_ref, good, 0.1, 0.9, 0.95, 1e-8, 0.0, 1)
    _lib.check_status()
    raw.adam_pieces(w, None, grads, *state, both, 0.1, 0.9, 0.95, 1e-8, 0.0, 1)
    with pytest.raises(RuntimeError):
        _lib.check_status()
    assert torch.equal(w, ref) and torch.equal(state, state_ref)
    _lib.check_status()
