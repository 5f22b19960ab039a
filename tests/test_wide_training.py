"""Networks with a wide softmax head (train_labels, score, RandomModel past 64 classes) and networks that keep their
activations in 8 bits (keep8): the operators of one training step together."""
import math

import pytest
import torch

from distributeddeeplearning_amd import config
from distributeddeeplearning_amd.models import ir, search
from distributeddeeplearning_amd.models.classifier import RandomModel
from distributeddeeplearning_amd.models.network import ConvOp, Network
from distributeddeeplearning_amd.models.optim import OptimConfig
from distributeddeeplearning_amd.ops import functional as F
from distributeddeeplearning_amd.utils.data import Data


def spec(*layers, shape=(6, 6, 2)):
    m = ir.ModelSpec("m", [ir.Input("in", shape)])
    for l in layers:
        m.append(l)
    return m


def mlp(classes=90):
    return spec(ir.Flatten("f"), ir.Dense("d1", 20, "relu"), ir.Dense("d2", 33, "tanh"), ir.Dense("d3", 16, "softplus"),
                ir.Dense("o", classes, "softmax"))


def convnet(classes=70):
    return spec(ir.Conv2D("c1", 5, (3, 3), 1, 1, "same", "relu"), ir.Conv2D("c2", 9, (3, 3), 2, 1, "same", "sigmoid"),
                ir.Flatten("f"), ir.Dense("d1", 24, "relu"), ir.Dense("o", classes, "softmax"))


def bn_net(classes=80):
    return spec(ir.Conv2D("c1", 8, (3, 3), 1, 1, "same", "relu"), ir.BatchNorm("b1"), ir.Flatten("f"),
                ir.Dense("d1", 24, "softsign"), ir.BatchNorm("b2"), ir.Dense("d2", 17, "relu"), ir.LeakyReLU("l2"),
                ir.Dense("o", classes, "softmax"))


SPECS = {"mlp": mlp, "conv": convnet, "bn": bn_net}


def batch(n, classes, seed=0, shape=(6, 6, 2)):
    g = torch.Generator().manual_seed(seed)
    lab = torch.randint(0, classes, (n,), generator=g)
    lab[n // 3] = -1
    return torch.rand(n, *shape, generator=g).bfloat16().float(), lab


def saved(net):
    """[(op, attribute, value)] of what the last training forward kept."""
    return [(op, a, getattr(op, a, None)) for op in net.ops for a in ("x", "y") if getattr(op, a, None) is not None]


def grads(net):
    return {(p.layer, p.wname): net.G[p.offset:p.offset + p.numel].view(p.shape)[p.corner()].float().cpu().clone()
            for p in net.param_table() if p.trainable}


def rel(a, b):
    return float((a - b).norm() / (b.norm() + 1e-12))


# ------------------------------------------------------------------------------------------------ wide head, CPU path
def test_train_labels_matches_autograd():
    net = Network(mlp(), "cpu", seed=3)
    x, lab = batch(13, 90)
    loss, rows = net.train_labels(net.prepare_input(x), lab)
    w = {k: v.double().requires_grad_() for k, v in net.logical_state().items()}
    h = x.double().reshape(13, -1)
    for name, act in (("d1", torch.relu), ("d2", torch.tanh), ("d3", torch.nn.functional.softplus)):
        h = act(h @ w[(name, "kernel")].t() + w[(name, "bias")])
    z = h @ w[("o", "kernel")].t() + w[("o", "bias")]
    live = lab >= 0
    ref = torch.nn.functional.cross_entropy(z[live], lab[live])
    ref.backward()
    assert abs(float(loss) - float(ref)) < 1e-5 and float(rows[13 // 3]) == 0
    for k, g in grads(net).items():
        assert rel(g.reshape(w[k].shape), w[k].grad.float()) < 1e-5, k     # fp32 sums of up to 72 terms
    s, rows_s = net.score(net.prepare_input(x), lab)
    assert abs(float(s) - float(ref)) < 1e-5 and torch.allclose(rows_s, rows, atol=1e-5)


def test_label_head_refusals():
    net = Network(spec(ir.Flatten("f"), ir.Dense("o", 5, "relu")), "cpu")
    x, lab = batch(4, 5)
    with pytest.raises(ValueError):
        net.train_labels(net.prepare_input(x), lab)
    with pytest.raises(ValueError):
        net.score(net.prepare_input(x), lab)


# ------------------------------------------------------------------------------------------------ keep8
def check_keep8(device, name, n=11):
    """keep8 against the same network whose kept tensors were replaced by what their checkpoints stand for: everything
    else of the two backward passes is the same arithmetic (on the device up to the summation order of the weight
    gradients and one bf16 rounding of a dY where the input-gradient kernel would have multiplied by act')."""
    classes = {"mlp": 90, "conv": 70, "bn": 80}[name]
    x, lab = batch(n, classes)
    nets = [Network(SPECS[name](classes), device, seed=5) for _ in range(2)]
    a, b = nets
    b.keep8 = True
    labels = lab.to(device)
    ha = a.forward(a.prepare_input(x), training=True, stop=-1)
    hb = b.forward(b.prepare_input(x), training=True, stop=-1)
    assert torch.equal(ha, hb)
    kept = [(op.name, at) for op, at, t in saved(b) if isinstance(t, F.Packed8)]
    assert kept, "nothing was kept in 8 bits"
    swap = {(op.name, at): F.unpack8(t) for op, at, t in saved(b) if isinstance(t, F.Packed8)}
    for op in a.ops:
        for at in ("x", "y"):
            if (op.name, at) in swap:
                t = getattr(op, at)
                setattr(op, at, swap[(op.name, at)].reshape(t.shape).to(t.dtype))
    for net, h in ((a, ha), (b, hb)):
        op = net.ops[-1]
        loss, dh, _, _, _ = F.dense_softmax_ce(h, op.w_main, op.bias, labels, out_dw=op.gkernel, out_db=op.gbias)
        net.backward(dh, start=-1)
    ga, gb = grads(a), grads(b)
    tol = 1e-5 if device == "cpu" else 2.0 ** -8
    for k in ga:
        assert rel(gb[k], ga[k]) <= tol, (k, rel(gb[k], ga[k]))
    b.release()
    assert not saved(b)
    return kept


@pytest.mark.parametrize("name", list(SPECS))
def test_keep8_is_the_backward_of_the_checkpoints_cpu(name):
    kept = check_keep8("cpu", name)
    if name == "mlp":       # the first layer's input is the network's: kept as it is; a layer's y is the next one's x
        assert ("d1", "x") not in kept and {("d1", "y"), ("d2", "x"), ("d2", "y"), ("d3", "x"), ("d3", "y")} <= set(kept)


def test_keep8_shares_a_checkpoint_between_layers():
    net = Network(mlp(), "cpu", seed=1)
    net.keep8 = True
    x, _ = batch(6, 90)
    net.forward(net.prepare_input(x), training=True)
    ops = [op for op in net.ops if isinstance(op, ConvOp)]
    assert ops[0].y is ops[1].x and ops[1].y is ops[2].x and ops[2].y is ops[3].x
    assert ops[3].y is None and isinstance(ops[0].x, torch.Tensor)
    net.forward(net.prepare_input(x), training=False)          # inference keeps nothing and packs nothing
    with pytest.raises(ValueError):
        net.narrow_saved(0, 3)


def test_keep8_error_is_the_quantisation():
    """The gradients move by no more than what half a step (2^-7 of a block's largest value, 2^-6 with the kept signs)
    can do to them: far inside 2 % here."""
    x, lab = batch(40, 90)
    nets = [Network(mlp(), "cpu", seed=2) for _ in range(2)]
    nets[1].keep8 = True
    for net in nets:
        net.train_labels(net.prepare_input(x), lab)
    ga, gb = (grads(n) for n in nets)
    for k in ga:
        assert rel(gb[k], ga[k]) < 2e-2, k


# ------------------------------------------------------------------------------------------------ RandomModel
def member(device, classes=100, over=(), n=300, seed=0, loss="categorical_crossentropy", **kw):
    sp = config.get_space("ddl_ray", [f"data_train_size={n - 50}", *over])
    data = Data(device, channels=1, n_train=n, n_test=40, synthetic=True)
    data.train_labels = data.train_labels * (classes // 10)
    data.test_labels = data.test_labels * (classes // 10)
    m = spec(ir.Flatten("f"), ir.Dense("d1", 24, "relu"), ir.Dense("d2", 40, "tanh"), ir.Dense("o", classes, "softmax"),
             shape=data.input_shape)
    cs = search.CompiledSpec(m, OptimConfig.keras("adam", 1e-3), loss)
    return RandomModel(data, data.get_random_sample(n - 50, seed=seed), sp, cs, device, 0, seed=seed, verbose=False, **kw)


def test_wide_member_trains_scores_and_predicts_cpu():
    m = member("cpu", over=["keep8=1"])
    assert m.net.keep8
    loss = m.train_step(m.sample.train_idx[:32])
    assert math.isfinite(float(loss))
    p = m.predict(m.data.test_x)
    assert p.shape == (40, 100) and torch.allclose(p.sum(1), torch.ones(40), atol=1e-4)
    assert 0.0 <= m.get_accuracy() <= 1.0 and 0.0 <= m.get_accuracy((m.data.test_x, m.data.test_labels)) <= 1.0
    with pytest.raises(ValueError):
        member("cpu", loss="mean_squared_error")


def test_narrow_member_keeps_its_losses():
    m = member("cpu", classes=10)
    assert not m._wide and not m.net.keep8
    m.train_step(m.sample.train_idx[:32])


# ------------------------------------------------------------------------------------------------ device
@pytest.mark.gpu
@pytest.mark.parametrize("name", list(SPECS))
@pytest.mark.parametrize("n", [11, 130])
def test_keep8_is_the_backward_of_the_checkpoints(name, n):
    check_keep8("cuda", name, n)


@pytest.mark.gpu
@pytest.mark.parametrize("keep8", [False, True])
@pytest.mark.parametrize("name", ["mlp", "conv"])
def test_train_labels_against_the_oracle(name, keep8):
    """Against the bf16-emulating oracle with the same checkpoints: 3 % per kernel, 6 % per bias (test_network_gpu.py)."""
    classes = {"mlp": 90, "conv": 70}[name]
    c, g = Network(SPECS[name](classes), "cpu", 7), Network(SPECS[name](classes), "cuda", 7)
    st = {k: v.bfloat16().float() for k, v in c.logical_state().items()}
    c.load_logical_state(st)
    g.load_logical_state(st)
    c.emulate_bf16 = True
    c.keep8 = g.keep8 = keep8
    x, lab = batch(64, classes)
    lc, rc = c.train_labels(c.prepare_input(x), lab)
    lg, rg = g.train_labels(g.prepare_input(x), lab.cuda())
    assert abs(float(lc) - float(lg)) < 1e-2 * abs(float(lc)) and float(rg[64 // 3]) == 0
    gc, gg = grads(c), grads(g)
    for k in gc:
        assert float((gg[k].reshape(gc[k].shape) - gc[k]).norm() / (gc[k].norm() + 1e-2)) < (3e-2 if k[1] == "kernel" else 6e-2), k
    sc, _ = c.score(c.prepare_input(x), lab)
    sg, _ = g.score(g.prepare_input(x), lab.cuda())
    assert abs(float(sc) - float(sg)) < 1e-2 * abs(float(sc))


@pytest.mark.gpu
def test_keep8_halves_what_a_step_keeps():
    m = spec(ir.Flatten("f"), *[ir.Dense(f"d{i}", 512, "tanh") for i in range(5)], ir.Dense("o", 300, "softmax"))
    held = []
    for keep8 in (False, True):
        net = Network(m, "cuda", 0)
        net.keep8 = keep8
        x, _ = batch(4096, 300)
        xd = net.prepare_input(x)
        net.forward(xd, training=True, stop=-1)                # autotunes; frees its temporaries
        net.release()
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        h = net.forward(xd, training=True, stop=-1)
        del h
        torch.cuda.synchronize()
        held.append(torch.cuda.memory_allocated() - base)
        net.release()
    # five [4096][512] activations: 64 bytes of bf16 per 32 elements against 33 (allocator blocks of 512 bytes on top)
    assert held[0] >= 5 * 4096 * 512 * 2 and held[1] <= held[0] * 33 / 64 + 5 * 2 * 512 + (1 << 20)


@pytest.mark.gpu
@pytest.mark.parametrize("keep8", [0, 1])
def test_wide_member_graph_steps_equal_eager_steps(keep8):
    a = member("cuda", over=[f"keep8={keep8}"], use_graph=False)
    b = member("cuda", over=[f"keep8={keep8}"], use_graph=True)
    idx = a.sample.train_idx
    for i in range(6):
        la = a.train_step(idx[i * 32:(i + 1) * 32])
        lb = b.train_step(idx[i * 32:(i + 1) * 32])
        torch.cuda.synchronize()
        assert torch.equal(la, lb), i
    assert torch.equal(a.net.P, b.net.P)
    p = b.predict(b.data.test_x)
    assert p.shape == (40, 100) and torch.allclose(p.sum(1).cpu(), torch.ones(40), atol=1e-4)
    assert 0.0 <= b.get_accuracy() <= 1.0 and 0.0 <= b.get_accuracy((b.data.test_x, b.data.test_labels)) <= 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("B,N", [(1, 65), (3, 1000), (7, 4099), (2, 50021)])
def test_softmax_of_wide_rows(B, N):
    g = torch.Generator().manual_seed(N)
    z = torch.zeros(B, (N + 7) // 8 * 8)
    z[:, :N] = torch.randn(B, N, generator=g) * 4
    z[0, 3] = -math.inf
    z[-1, :N] += 200.0
    z = z.bfloat16()
    got = F.softmax(z.cuda(), N).double().cpu()
    ref = torch.softmax(z[:, :N].double(), 1)
    # exponentials good to 2^-22 relative of |z - max| < 64 and a sum of N of them in pieces of 256: 2^-15 is generous
    assert got.shape == ref.shape and ((got - ref).abs() <= 2.0 ** -15 * ref + 1e-30).all()
    with pytest.raises(ValueError):
        F.softmax_ce(z.cuda(), torch.zeros(B, N, device="cuda"))


@pytest.mark.gpu
def test_softmax_of_more_wide_rows_than_a_launch_holds():
    """2^24 blocks of 256 threads and more are taken modulo 2^32 threads, without an error: 64 rows repeated have the bits of their first copies."""
    g = torch.Generator().manual_seed(1)
    z = torch.zeros(64, 72)
    z[:, :65] = torch.randn(64, 65, generator=g) * 4
    z = z.bfloat16().cuda()
    B = (1 << 24) + 64
    one, all_ = F.softmax(z, 65), F.softmax(z.expand(B // 64, 64, 72).reshape(B, 72), 65)
    assert torch.equal(all_.view(-1, 64, 65), one.expand(B // 64, 64, 65))
    ref = torch.softmax(z[:, :65].double(), 1)
    assert ((one.double() - ref).abs() <= 2.0 ** -15 * ref).all()


def mlp_member(device, keep8, seed=0):
    """A member inside the persistent MLP kernel's limits (32 units, batches of 32)."""
    sp = config.get_space("ddl_ray", ["data_train_size=250", f"keep8={keep8}", "epochs=2", "mini_epochs=2"])
    data = Data(device, channels=1, n_train=300, n_test=40, synthetic=True)
    m = spec(ir.Flatten("f"), ir.Dense("d1", 24, "relu"), ir.Dense("d2", 32, "tanh"), ir.Dense("o", 10, "softmax"),
             shape=data.input_shape)
    cs = search.CompiledSpec(m, OptimConfig.keras("adam", 1e-3), "categorical_crossentropy")
    return RandomModel(data, data.get_random_sample(250, seed=seed), sp, cs, device, 0, seed=seed, verbose=False)


def test_persistent_kernel_leaves_keep8_members_alone(monkeypatch):
    """Its activations are fp32 in LDS: a member that keeps 8 bits would train differently in a group than alone."""
    from distributeddeeplearning_amd.models import mlp_fast
    for keep8 in (0, 1):
        m = mlp_member("cpu", keep8)
        monkeypatch.setattr(m.net, "on_gpu", True)
        monkeypatch.setattr(next(op for op in m.net.ops if isinstance(op, ConvOp)), "kstruct", (28, 28, 1))
        assert mlp_fast.eligible(m) == (not keep8)


@pytest.mark.gpu
def test_keep8_members_train_alike_alone_and_side_by_side():
    from distributeddeeplearning_amd.models import mlp_fast
    from distributeddeeplearning_amd.models.classifier import train_concurrently
    alone, a, b = (mlp_member("cuda", 1, s) for s in (0, 0, 1))
    assert mlp_fast.eligible(mlp_member("cuda", 0)) and not mlp_fast.eligible(a)
    alone.train()
    train_concurrently([a, b])
    assert a.history == alone.history and torch.equal(a.net.P, alone.net.P)


def actor(device, classes):
    from distributeddeeplearning_amd.parallel.ensemble import MemberActor
    sp = config.get_space("ddl_ray", ["data_train_size=250", "channels=1"])
    m = spec(ir.Flatten("f"), ir.Dense("d1", 24, "relu"), ir.Dense("o", classes, "softmax"), shape=(28, 28, 1))
    cs = search.CompiledSpec(m, OptimConfig.keras("adam", 1e-3), "categorical_crossentropy")
    return MemberActor(sp, cs, 0, 0, 0, data_kw=dict(n_train=300, n_test=40, synthetic=True), device=device, verbose=False)


def check_actor(device):
    """The test accuracy of a hosted member, against its own predictions: wide heads by class numbers, the others by their
    one-hot rows."""
    for classes in (10, 100):
        a = actor(device, classes)
        want = int((torch.from_numpy(a.predict_test()).argmax(1) == a.data.test_labels.cpu()).sum()) / 40
        assert a.get_accuracy(True) == want
        assert a.model.test_data()[1].dim() == (1 if classes > 64 else 2)


def test_hosted_member_of_any_width_is_tested_cpu():
    check_actor("cpu")


@pytest.mark.gpu
def test_hosted_member_of_any_width_is_tested():
    check_actor("cuda")
