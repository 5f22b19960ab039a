"""dense_softmax_ce against its definition in 64 bits, on the CPU path and on the device.

Bounds.  u = 2^-8 is the largest relative error of a rounding to bf16, 2^-24 to fp32.  With dl the exact gradient of the
logits and sums of absolute values in 64 bits:
  rows   the logits carry K fp32 additions, (K + 2) 2^-24 sum |x||w| at the row's largest; it enters the label's logit and
         the log-sum, hence twice; the exponential, the sum and the logarithm add 2^-20 (1 + |lse| + |z_label|).
  dx     E is rounded to bf16 once, the result once: u sum_v |dl||w| + u |dx|, plus the logits' error in p (2 relative terms
         of it) and V fp32 additions
  dw     E once, the scaled x once, the result once (bf16 output): (2 u + u^2) sum_r |dl||x| + u |dw|
  db     E once, the result once: u sum_r |dl| + u |db|"""
import math

import pytest
import torch

from distributeddeeplearning_amd.ops import functional as F

U16, U32 = 2.0 ** -8, 2.0 ** -24


def make(N, K, V, seed=0, scale=1.0, bias=True, drop=0.0, mask=0.0):
    g = torch.Generator().manual_seed(seed)
    Kp = (K + 7) // 8 * 8
    x, w = torch.zeros(N, Kp), torch.zeros(V, Kp)
    x[:, :K] = torch.randn(N, K, generator=g) * scale
    w[:, :K] = torch.randn(V, K, generator=g) * (1.5 / math.sqrt(K))
    b = torch.randn(V, generator=g) * 0.3 if bias else None
    labels = torch.randint(0, V, (N,), generator=g)
    if mask and b is not None:
        off = torch.rand(V, generator=g) < mask
        off[labels] = False
        b[off] = -math.inf
    if drop:
        labels[torch.rand(N, generator=g) < drop] = -1
    return x.bfloat16(), w.bfloat16(), b, labels


def exact(x, w, b, labels):
    """The definition in 64 bits with the sums of absolute values its error bounds need."""
    live = labels >= 0
    x, w = torch.where(live[:, None], x.double(), 0.0), w.double()
    z = x @ w.t() + (0 if b is None else b.double())
    at = labels.clamp_min(0)[:, None]
    lse = torch.logsumexp(z, 1)
    zt = z.gather(1, at)[:, 0]
    rows = torch.where(live, lse - zt, 0.0)
    cnt = max(int(live.sum()), 1)
    dl = torch.exp(z - lse[:, None])
    dl.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float64))
    dl = torch.where(live[:, None], dl / cnt, 0.0)
    K, V = x.shape[1], w.shape[0]
    az = (x.abs() @ w.abs().t()).amax(1) + (0 if b is None else b[torch.isfinite(b)].abs().max().double())
    ez = (K + 4) * U32 * az                                     # error of a logit
    p = dl.abs()
    dp = p * (2 * ez[:, None] + 2.0 ** -20) + (2 * ez[:, None] + 2.0 ** -20) * torch.where(live[:, None], torch.exp(z - lse[:, None]) / cnt, 0.0)
    return dict(rows=rows, loss=rows.sum() / cnt, dx=dl @ w, dw=dl.t() @ x, db=dl.sum(0),
                t_rows=2 * ez + 2.0 ** -20 * (1 + lse.abs() + zt.abs()),
                a_dx=p @ w.abs(), a_dw=p.t() @ x.abs(), a_db=p.sum(0),
                e_dx=dp @ w.abs(), e_dw=dp.t() @ x.abs(), e_db=dp.sum(0), n=x.shape[0], V=V)


def check(out, ref, dtype=torch.float32, x_dtype=torch.bfloat16, device=True):
    loss, dx, dw, db, rows = out
    u = U16 if device else 0.0
    uo = U16 if dtype == torch.bfloat16 else U32
    ux = U16 if x_dtype == torch.bfloat16 else U32
    err = (rows.double().cpu() - ref["rows"]).abs()
    assert (err <= ref["t_rows"]).all(), f"rows off by {err.max():.3g}"
    assert abs(float(loss) - float(ref["loss"])) <= float(ref["t_rows"].max()) + U32 * abs(float(ref["loss"]))
    if dx is None:
        return
    for name, got, lim in (
            ("dx", dx, (u + ref["V"] * U32) * ref["a_dx"] + ref["e_dx"] + ux * ref["dx"].abs()),
            ("dw", dw, (2 * u + u * u + ref["n"] * U32) * ref["a_dw"] + ref["e_dw"] + uo * ref["dw"].abs()),
            ("db", db, (u + ref["n"] * U32 + 2.0 ** -16) * ref["a_db"] + ref["e_db"] + uo * ref["db"].abs())):
        if got is None:
            continue
        err = (got.double().cpu() - ref[name]).abs()
        lim = lim * 1.01 + 1e-30                               # second-order terms
        assert torch.isfinite(got).all(), name
        assert (err <= lim).all(), f"{name}: {float((err / lim).max()):.3g} of its bound"


# ------------------------------------------------------------------------------------------------ CPU path
@pytest.mark.parametrize("N,K,V", [(1, 8, 1), (3, 5, 70), (17, 30, 333)])
@pytest.mark.parametrize("bias", [False, True])
def test_cpu_matches_definition(N, K, V, bias):
    x, w, b, lab = make(N, K, V, bias=bias, drop=0.2)
    ref = exact(x, w, b, lab)
    check(F.dense_softmax_ce(x.float(), w.float(), b, lab), ref, x_dtype=torch.float32, device=False)
    loss, dx, dw, db, rows = F.dense_softmax_ce(x.float(), w.float(), b, lab, want_grad=False)
    assert dx is None and dw is None and db is None


def test_cpu_gradients_match_differences():
    x, w, b, lab = make(5, 8, 70, drop=0.3)
    x, w = x.double(), w.double()
    _, dx, dw, db, _ = F.dense_softmax_ce(x, w, b, lab)

    def loss(x, w, b):
        z = x @ w.t() + b
        live = lab >= 0
        return -(torch.log_softmax(z, 1).gather(1, lab.clamp_min(0)[:, None])[:, 0][live]).sum() / live.sum()
    h = 1e-5
    for t, g, k in ((x, dx, 0), (w, dw, 1), (b.double(), db, 2)):
        for i in (0, 3, t.numel() - 1):
            args = [x, w, b.double()]
            lo, hi = t.clone(), t.clone()
            lo.view(-1)[i] -= h
            hi.view(-1)[i] += h
            args[k] = hi
            up = loss(*args)
            args[k] = lo
            d = (up - loss(*args)) / (2 * h)
            # central difference: h^2 / 6 times a third derivative below 10, and the fp32 of the CPU path
            assert abs(float(d) - float(g.reshape(-1)[i])) < 1e-5


def test_cpu_rows_without_label_and_bad_labels():
    x, w, b, lab = make(6, 16, 80)
    lab[2] = -1
    lab[4] = -100
    xn = x.float().clone()
    xn[2] = math.nan
    xn[4] = math.inf
    loss, dx, dw, db, rows = F.dense_softmax_ce(xn, w.float(), b, lab)
    check((loss, dx, dw, db, rows), exact(x, w, b, lab), x_dtype=torch.float32, device=False)
    assert (dx[[2, 4]] == 0).all() and (rows[[2, 4]] == 0).all()
    none = F.dense_softmax_ce(xn, w.float(), b, torch.full((6,), -1))
    assert float(none[0]) == 0 and all((t == 0).all() for t in none[1:])
    lab2 = lab.clone()
    lab2[0] = 80
    loss, dx, dw, db, rows = F.dense_softmax_ce(x.float(), w.float(), b, lab2)
    assert math.isnan(float(loss)) and math.isnan(float(rows[0])) and torch.isfinite(rows[1:]).all()
    assert (dx[0] == 0).all() and torch.isfinite(dw).all()


def check_label_column(x, w, b, lab):
    one, two = F.dense_softmax_ce(x, w, b, lab), F.dense_softmax_ce(x, w, b, lab[:, None])
    assert all(p.shape == q.shape and torch.equal(p, q) for p, q in zip(one, two))


def test_cpu_labels_in_a_column():
    x, w, b, lab = make(7, 16, 80, drop=0.3)
    check_label_column(x.float(), w.float(), b, lab)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_cpu_input_gradient_has_the_inputs_type(dtype):
    x, w, b, lab = make(5, 16, 80)
    a, ref = F.dense_softmax_ce(x.to(dtype), w.float(), b, lab)[1], F.dense_softmax_ce(x.float(), w.float(), b, lab)[1]
    assert a.dtype == dtype and torch.equal(a, ref.to(dtype))


def test_cpu_refusals():
    x, w, b, lab = make(4, 16, 80)
    x, w = x.float(), w.float()
    for bad in (dict(w=w[:, :8]), dict(labels=lab[:3]), dict(labels=lab.int()), dict(bias=b[:79])):
        a = dict(x=x, w=w, bias=b, labels=lab)
        a.update(bad)
        with pytest.raises(ValueError):
            F.dense_softmax_ce(**a)
    with pytest.raises(ValueError):
        F.dense_softmax_ce(x, w, b, lab, want_grad=False, out_dw=torch.empty(80, 16))
    with pytest.raises(ValueError):
        F.dense_softmax_ce(x, w, b, lab, out_dw=torch.empty(80, 8))
    with pytest.raises(ValueError):
        F.dense_softmax_ce(x, w, None, lab, out_db=torch.empty(80))


def overlaps(x, w, b, lab):
    """Calls whose gradients would land in an input or in one another."""
    V, K = w.shape
    flat = torch.zeros(V * K + V, dtype=b.dtype, device=b.device)
    ints = torch.zeros(2 * V, dtype=torch.int64, device=b.device)
    ints[:lab.numel()] = lab
    for args in (dict(out_db=b), dict(bias=flat[8:8 + V], out_db=flat[16:16 + V]), dict(bias=flat[8:8 + V], out_dw=flat[:V * K].view(V, K)),
                 dict(out_dw=flat[:V * K].view(V, K), out_db=flat[V * K - 8:V * K - 8 + V]),
                 dict(labels=ints[:lab.numel()], out_db=ints.view(torch.float32)[8:8 + V])):
        with pytest.raises(ValueError):
            F.dense_softmax_ce(**{**dict(x=x, w=w, bias=b, labels=lab), **args})
    dw, db = flat[:V * K].view(V, K), flat[V * K:]            # neighbours are apart, and so is a batch of no rows inside one
    F.dense_softmax_ce(x, w, b, lab, out_dw=dw, out_db=db)
    none = flat.view(x.dtype)[64:64].view(0, K)
    F.dense_softmax_ce(none, w, b, lab[:0], out_dw=dw, out_db=db)


def test_cpu_overlapping_gradients_are_refused():
    x, w, b, lab = make(8, 16, 80)
    overlaps(x.float(), w.float(), b, lab)


def test_scored_rows_come_in_pieces_a_launch_can_hold():
    """A piece's launches hold less than 2^32 threads (256 per row, 256 per 128 statistics of 8 bytes), so its workspace stops
    growing: at 2^20 rows, and at 4 GiB of statistics however much the caller allows."""
    from distributeddeeplearning_amd.ops import hip
    for K, V in ((520, 100), (8, 100), (1024, 5000)):
        most = hip._dense_ce_ws(1 << 20, V, K, 0, 0, 4 << 30, -1)
        assert 0 < hip._dense_ce_ws(1 << 19, V, K, 0, 0, 4 << 30, -1) < most
        for n in ((1 << 20) + 1, 1 << 24, (1 << 28) - 1):
            assert hip._dense_ce_ws(n, V, K, 0, 0, 4 << 30, -1) == most
    assert hip._dense_ce_ws(1 << 20, 1 << 21, 64, 0, 0, 1 << 40, -1) <= (4 << 30) + (8 << 20)


# ------------------------------------------------------------------------------------------------ device
def cuda(x, w, b, lab):
    return x.cuda(), w.cuda(), None if b is None else b.cuda(), lab.cuda()


SHAPES = [(1, 8, 1), (1, 16, 65), (2, 24, 1000), (5, 8, 128), (16, 64, 64), (31, 40, 333), (33, 136, 4099), (64, 120, 64),
          (130, 200, 777), (257, 72, 2051), (300, 520, 515), (513, 264, 769), (1100, 64, 65), (2500, 40, 70)]


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,V", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_train(N, K, V, dtype):
    a = make(N, K, V, seed=N + V, drop=0.1 if N > 4 else 0.0)
    out = F.dense_softmax_ce(*cuda(*a), grad_dtype=dtype)
    assert out[1].dtype == torch.bfloat16 and out[2].dtype == dtype and out[3].dtype == dtype
    check(out, exact(*a), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,V", SHAPES)
def test_score(N, K, V):
    a = make(N, K, V, seed=7, drop=0.1 if N > 4 else 0.0)
    out = F.dense_softmax_ce(*cuda(*a), want_grad=False)
    assert out[1] is None and out[2] is None and out[3] is None
    check(out, exact(*a))


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [0, 1, 2, 3, 109, 119, 129, 9, 19, 29])
@pytest.mark.parametrize("N,K,V", [(37, 72, 1030), (64, 328, 500), (128, 136, 333), (190, 136, 400), (260, 136, 600)])
def test_every_tile(tile, N, K, V, monkeypatch):
    from distributeddeeplearning_amd.ops import hip
    monkeypatch.setattr(hip, "CE_TILE", tile)
    a = make(N, K, V, seed=tile, drop=0.1)
    check(F.dense_softmax_ce(*cuda(*a)), exact(*a))


@pytest.mark.gpu
@pytest.mark.parametrize("bias,mask", [(False, 0.0), (True, 0.5), (True, 0.97)])
def test_bias_and_classes_switched_off(bias, mask):
    a = make(70, 40, 900, seed=3, bias=bias, mask=mask)
    out = F.dense_softmax_ce(*cuda(*a))
    assert (out[3] is None) == (not bias)
    check(out, exact(*a))


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [-3000.0, -100.0, 60.0, 300.0, 3000.0])
@pytest.mark.parametrize("part", [False, True])
def test_logits_far_from_zero(shift, part):
    """References other than 0: all classes far away, or one stretch of them (tiles of one row disagree)."""
    x, w, b, lab = make(40, 64, 1500, seed=5)
    if part:
        b[300:700] += shift
        lab[lab % 3 == 0] = 500
    else:
        b += shift
    a = (x, w, b, lab)
    check(F.dense_softmax_ce(*cuda(*a)), exact(*a))


@pytest.mark.gpu
def test_large_logits_saturate():
    a = make(64, 64, 700, seed=6, scale=40.0)
    check(F.dense_softmax_ce(*cuda(*a)), exact(*a))


@pytest.mark.gpu
@pytest.mark.parametrize("N", [2, 40, 300])
def test_rows_without_label_hold_anything(N):
    x, w, b, lab = make(N, 48, 520, seed=8)
    lab[1::2] = -1
    xb = x.clone()
    xb[1::4], xb[3::4] = math.nan, math.inf
    out = F.dense_softmax_ce(*cuda(xb, w, b, lab))
    check(out, exact(x, w, b, lab))
    assert (out[1][1::2] == 0).all() and (out[4][1::2] == 0).all()
    none = F.dense_softmax_ce(*cuda(xb, w, b, torch.full((N,), -1)))
    assert float(none[0]) == 0 and all((t == 0).all() for t in none[1:])


@pytest.mark.gpu
def test_bad_label_nan_row_and_no_class_left():
    x, w, b, lab = make(9, 16, 300, seed=9)
    lab2 = lab.clone()
    lab2[4] = 300
    loss, dx, dw, db, rows = F.dense_softmax_ce(*cuda(x, w, b, lab2))
    assert math.isnan(float(loss)) and math.isnan(float(rows[4])) and int(torch.isnan(rows).sum()) == 1
    assert (dx[4] == 0).all() and torch.isfinite(dw).all() and torch.isfinite(db).all()
    xn = x.clone()
    xn[2, 3] = math.nan
    loss, dx, dw, db, rows = F.dense_softmax_ce(*cuda(xn, w, b, lab))
    assert math.isnan(float(rows[2])) and int(torch.isnan(rows).sum()) == 1 and torch.isnan(dx[2]).all()
    assert torch.isfinite(dx[:2]).all() and torch.isfinite(dx[3:]).all() and torch.isnan(dw).all()
    off = torch.full_like(b, -math.inf)
    loss, dx, dw, db, rows = F.dense_softmax_ce(*cuda(x, w, off, lab))
    assert torch.isnan(rows).all() and torch.isnan(dx).all()
    b2 = b.clone()                                            # the label's own class switched off: loss inf, gradient exists
    b2[lab[0]] = -math.inf
    loss, dx, dw, db, rows = F.dense_softmax_ce(*cuda(x[:1], w, b2, lab[:1]))
    assert float(rows[0]) == math.inf
    p = torch.softmax(x[:1].double() @ w.double().t() + b2.double(), 1)
    p[0, lab[0]] -= 1
    lim = U16 * (p.abs() @ w.double().abs()) + U16 * (p @ w.double()).abs() + 1e-5
    assert ((dx.double().cpu() - p @ w.double()).abs() <= lim).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [512, 600, 777])
def test_row_pieces(N, dtype, monkeypatch):
    from distributeddeeplearning_amd.ops import hip
    a = make(N, 72, 700, seed=N, drop=0.1)
    d = cuda(*a)
    for piece in (256, 64):
        monkeypatch.setattr(hip, "CE_PIECE_BYTES", piece * 704 * 2)
        out = F.dense_softmax_ce(*d, grad_dtype=dtype)
        check(out, exact(*a), dtype)


@pytest.mark.gpu
def test_offsets_past_32_bits(monkeypatch):
    """8192 rows x 270001 classes in one piece: the exponentials end 4.4 GB behind their start."""
    from distributeddeeplearning_amd.ops import hip
    monkeypatch.setattr(hip, "CE_PIECE_BYTES", 8 << 30)
    N, K, V = 8192, 64, 270001
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(N, K, generator=g, device="cuda").bfloat16()
    w = (torch.randn(V, K, generator=g, device="cuda") / 8).bfloat16()
    b = torch.randn(V, generator=g, device="cuda") * 0.1
    lab = torch.randint(0, V, (N,), generator=g, device="cuda")
    lab[-1] = V - 1
    loss, dx, dw, db, rows = F.dense_softmax_ce(x, w, b, lab)
    lse = torch.empty(N, dtype=torch.float64, device="cuda")
    p_last = torch.empty(N, 8, dtype=torch.float64, device="cuda")          # the last eight classes' gradients
    for r in range(0, N, 1024):
        z = x[r:r + 1024].double() @ w.double().t() + b.double()
        lse[r:r + 1024] = torch.logsumexp(z, 1)
        p_last[r:r + 1024] = torch.exp(z[:, -8:] - lse[r:r + 1024, None])
    zt = (x.double() * w[lab].double()).sum(1) + b[lab].double()
    assert ((rows.double() - (lse - zt)).abs() <= 2.0 ** -18 * (1 + lse.abs() + zt.abs())).all()
    p_last -= torch.nn.functional.one_hot((lab - (V - 8)).clamp_min(-1) + 1, 9)[:, 1:].double()
    p_last /= N
    ref = p_last.t() @ x.double()
    lim = 2 * U16 * 1.01 * (p_last.abs().t() @ x.double().abs()) + 1e-9
    assert ((dw[-8:].double() - ref).abs() <= lim).all()
    assert ((db[-8:].double() - p_last.sum(0)).abs() <= 1.01 * U16 * p_last.abs().sum(0) + 1e-9).all()
    last = slice(N - 4, N)
    p = torch.exp(x[last].double() @ w.double().t() + b.double() - lse[last, None])
    p[torch.arange(4, device="cuda"), lab[last]] -= 1
    ref = p @ w.double() / N
    assert ((dx[last].double() - ref).abs() <= 1.01 * (U16 * (p.abs() @ w.double().abs()) / N + U16 * ref.abs())).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_out_tensors_and_empty_batch(dtype):
    a = make(20, 40, 130, seed=2)
    d = cuda(*a)
    flat = torch.full((130 * 40 + 136,), 7.0, dtype=dtype, device="cuda")
    dw, db = flat[:130 * 40].view(130, 40), flat[130 * 40:130 * 40 + 130]
    out = F.dense_softmax_ce(*d, out_dw=dw, out_db=db)
    assert out[2] is dw and out[3] is db and (flat[-6:] == 7).all()
    check(out, exact(*a), dtype)
    out = F.dense_softmax_ce(d[0][:0], d[1], d[2], d[3][:0], out_dw=dw, out_db=db)
    assert float(out[0]) == 0 and (dw == 0).all() and (db == 0).all() and out[4].numel() == 0 and (flat[-6:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N,V,classes", [(200, 500, 1), (700, 300, 3), (1500, 4000, 40), (3000, 100, 14)])
def test_many_rows_of_one_class_and_label_terms(N, V, classes):
    """Labels repeat; the label terms are exact, so a class that only its own rows' label terms reach (p ~ 0 elsewhere) has
    its dw row to the output's rounding."""
    x, w, b, lab = make(N, 64, V, seed=N, drop=0.05)
    lab = torch.where(lab >= 0, lab % classes * 7, lab)
    a = (x, w, b, lab)
    ref = exact(*a)
    out = F.dense_softmax_ce(*cuda(*a))
    check(out, ref)
    # the label entries carry no bf16 rounding: what is left is u times the other entries of each sum
    live = lab >= 0
    oh = torch.zeros(N, V, dtype=torch.float64)
    oh[live.nonzero()[:, 0], lab[live]] = 1.0
    xd = torch.where(live[:, None], x.double(), 0.0)
    z = xd @ w.double().t() + b.double()
    other = torch.softmax(z, 1) * (1 - oh) * live[:, None] / int(live.sum())
    lim = (2 * U16 + U16 ** 2) * (other.t() @ xd.abs()) + N * U32 * ref["a_dw"] + ref["e_dw"] + 2 * U32 * ref["a_dw"]
    assert ((out[2].double().cpu() - ref["dw"]).abs() <= 1.01 * lim + 1e-30).all()


@pytest.mark.gpu
def test_same_bits_twice_and_on_another_stream():
    a = make(150, 200, 3001, seed=4)
    d = cuda(*a)
    one = F.dense_softmax_ce(*d)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        two = F.dense_softmax_ce(*d)
    torch.cuda.current_stream().wait_stream(s)
    for p, q in zip(one, two):
        assert torch.equal(p, q)


@pytest.mark.gpu
def test_captured_and_replayed():
    from distributeddeeplearning_amd.utils import hipgraph
    a = make(100, 64, 900, seed=1, drop=0.1)
    d = cuda(*a)
    x, lab = d[0].clone(), d[3].clone()
    F.dense_softmax_ce(x, d[1], d[2], lab)
    hipgraph.quiesce()
    g, out = hipgraph.capture(lambda: F.dense_softmax_ce(x, d[1], d[2], lab))
    for seed in (11, 12, 13):
        b = make(100, 64, 900, seed=seed, drop=0.1)
        x.copy_(b[0])
        lab.copy_(b[3])
        g.replay()
        torch.cuda.synchronize()
        want = F.dense_softmax_ce(x, d[1], d[2], lab)
        for p, q in zip(out, want):
            assert torch.equal(p, q)


@pytest.mark.gpu
def test_refusals():
    x, w, b, lab = cuda(*make(8, 16, 80))
    ok = dict(x=x, w=w, bias=b, labels=lab)
    wide = torch.zeros(8, 32, dtype=torch.bfloat16, device="cuda")
    for bad in (dict(w=w[:, :8]), dict(w=w.float()), dict(x=wide[:, ::2]), dict(x=x[:, :15].contiguous()), dict(x=x[0]),
                dict(labels=lab[:7]), dict(labels=lab.int()), dict(labels=lab.cpu()), dict(bias=b[:79].contiguous()),
                dict(bias=b.double()), dict(bias=b.cpu()), dict(out_dw=torch.empty(80, 8, device="cuda")),
                dict(out_dw=torch.empty(80, 16, device="cuda", dtype=torch.float16)), dict(grad_dtype=torch.float16),
                dict(out_db=torch.empty(79, device="cuda")), dict(want_grad=False, out_dw=torch.empty(80, 16, device="cuda")),
                dict(out_dw=torch.empty(80, 16, device="cuda"), out_db=torch.empty(80, device="cuda", dtype=torch.bfloat16)),
                dict(bias=None, out_db=torch.empty(80, device="cuda")), dict(out_dw=torch.empty(80, 16))):
        with pytest.raises(ValueError):
            F.dense_softmax_ce(**{**ok, **bad})


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,V", [(3, 24, 65), (20, 40, 97), (31, 72, 1030), (40, 64, 130)])
def test_padding_classes_are_zero_in_a_dirty_workspace(N, K, V):
    """The exponentials' columns behind the last class enter the products: they have to be written, not found zero."""
    a = make(N, K, V, seed=V)
    d = cuda(*a)
    for _ in range(3):
        dirty = [torch.full((1 << s,), 255, dtype=torch.uint8, device="cuda") for s in (14, 16, 18, 20, 20, 21, 22)]
        del dirty                                              # NaN bits in the allocator's free blocks
        check(F.dense_softmax_ce(*d), exact(*a))


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,V", [(64, 1024, 300), (64, 1032, 300), (1, 1032, 70), (9, 2048, 515), (65, 1024, 200), (128, 1032, 333)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_few_rows_of_both_widths(N, K, V, dtype):
    """Both sides of the rule that picks the weight gradient's kernel for few rows."""
    a = make(N, K, V, seed=N + K, drop=0.1 if N > 4 else 0.0)
    check(F.dense_softmax_ce(*cuda(*a), grad_dtype=dtype), exact(*a), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,V", [(5, 1024, 150001), (100, 1024, 150001), (200, 1024, 150001), (7, 4800, 30011)])
def test_weights_larger_than_the_cache(N, K, V):
    """More than 256 MiB of weights, read past the caches where one row tile is all there is.  Most classes are switched off, so
    the definition needs only the others; what is switched off has gradients of exactly 0."""
    g = torch.Generator(device="cuda").manual_seed(K)
    x = torch.randn(N, K, generator=g, device="cuda").bfloat16()
    w = torch.randn(V, K, generator=g, device="cuda", dtype=torch.bfloat16) * (1.5 / math.sqrt(K))
    assert w.numel() * 2 > 256 << 20
    on = torch.cat([torch.randperm(V, generator=g, device="cuda")[:500], torch.tensor([0, V - 1], device="cuda")]).unique()
    b = torch.full((V,), -math.inf, device="cuda")
    b[on] = torch.randn(on.numel(), generator=g, device="cuda") * 0.3
    pick = torch.randint(0, on.numel(), (N,), generator=g, device="cuda")
    loss, dx, dw, db, rows = F.dense_softmax_ce(x, w, b, on[pick])
    ref = exact(x.cpu(), w[on].cpu(), b[on].cpu(), pick.cpu())
    ref["V"] = V
    check((loss, dx, dw[on], db[on], rows), ref)
    off = torch.ones(V, dtype=torch.bool, device="cuda")
    off[on] = False
    assert int((dw[off] != 0).sum()) == 0 and int((db[off] != 0).sum()) == 0
    score = F.dense_softmax_ce(x, w, b, on[pick], want_grad=False)
    check((score[0], None, None, None, score[4]), ref)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [257, 600, 1024])
def test_scored_row_pieces(N, monkeypatch):
    """A workspace that holds the statistics of 256 rows at a time: the same row losses, and the mean over all of them."""
    from distributeddeeplearning_amd.ops import hip
    a = make(N, 72, 700, seed=N, drop=0.1)
    d = cuda(*a)
    whole = F.dense_softmax_ce(*d, want_grad=False)
    monkeypatch.setattr(hip, "CE_PIECE_BYTES", 1024)
    out = F.dense_softmax_ce(*d, want_grad=False)
    check(out, exact(*a))
    assert torch.equal(out[4], whole[4]) and torch.equal(out[0], whole[0])


@pytest.mark.gpu
def test_gradient_over_the_weights_is_refused():
    x, w, b, lab = cuda(*make(8, 16, 80))
    both = torch.zeros(88, 16, dtype=torch.bfloat16, device="cuda")
    both[:80] = w
    for args in (dict(w=w, out_dw=w), dict(w=both[:80], out_dw=both[8:]), dict(x=both[80:], w=w, out_dw=both[8:])):
        with pytest.raises(ValueError):
            F.dense_softmax_ce(**{**dict(x=x, bias=b, labels=lab), **args})


@pytest.mark.gpu
@pytest.mark.parametrize("N,V", [(9, 300), (200, 1500)])
def test_lowest_value_switches_a_class_off(N, V):
    """A mask of the type's lowest value: the same bits as one of -inf (the labels' own classes stay on)."""
    x, w, b, lab = make(N, 40, V, seed=N, mask=0.5)
    low = torch.where(torch.isfinite(b), b, torch.full_like(b, torch.finfo(torch.float32).min))
    for p, q in zip(F.dense_softmax_ce(*cuda(x, w, b, lab)), F.dense_softmax_ce(*cuda(x, w, low, lab))):
        assert torch.equal(p, q)


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,V", [(9, 1960, 156), (40, 4096, 500)])
def test_row_losses_are_not_the_long_sums_error(N, K, V):
    """The label's logit has the error of a tree of additions (log2 K + 6 of them, the logit and the logarithm rounded at their own
    size) instead of a chain's; the other classes' errors enter the logarithm by their probabilities, which average them: a
    quarter of the chain's bound."""
    x, w, b, lab = make(N, K, V, seed=K)
    ref = exact(x, w, b, lab)
    az = (x.double().abs() * w[lab].double().abs()).sum(1) + b[lab].abs().double()
    own = (math.log2(K) + 6) * U32 * az + 2.0 ** -21 * (1 + ref["rows"].abs())
    out = F.dense_softmax_ce(*cuda(x, w, b, lab), want_grad=False)
    err = (out[4].double().cpu() - ref["rows"]).abs()
    assert (err <= own + ref["t_rows"] / 8).all(), f"{float((err / (own + ref['t_rows'] / 8)).max()):.3g} of its bound"


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", [((1 << 24) + 64, 520), ((1 << 26) + 64, 8)])
def test_scoring_more_rows_than_a_launch_holds(N, K):
    """Blocks of 256 and of 64 threads per row, 2^32 threads and more over all the rows.  64 rows repeated: each has the bits of
    its first copy, and those are right."""
    a = make(64, K, 100, seed=K)
    x, w, b, lab = cuda(*a)
    x, lab = (t.expand(N // 64, *t.shape).reshape(N, *t.shape[1:]).contiguous() for t in (x, lab))
    loss, _, _, _, rows = F.dense_softmax_ce(x, w, b, lab, want_grad=False)
    ref = exact(*a)
    check((loss, None, None, None, rows[:64]), ref)
    assert torch.equal(rows.view(-1, 64), rows[:64].expand(N // 64, 64))


@pytest.mark.gpu
def test_overlapping_gradients_are_refused():
    overlaps(*cuda(*make(8, 16, 80)))


@pytest.mark.gpu
def test_labels_in_a_column():
    check_label_column(*cuda(*make(7, 16, 80, drop=0.3)))
