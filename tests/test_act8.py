"""8-bit activation checkpoints: format, packing, and the backward operators that read them.

pack8 / unpack8 have no tolerance: scales are powers of two, so both are exact to the bit.  act_bwd8 is one rounding to bf16
(2^-8 relative) of an fp32 formula whose factor is good to 2^-18 of 1; dense_wgrad8 multiplies exact bf16 numbers and adds R
products in fp32: R 2^-24 sum |dy||x|."""
import math

import pytest
import torch

from distributeddeeplearning_amd.ops import cpu_ref
from distributeddeeplearning_amd.ops import functional as F

KINDS = ("relu", "sigmoid", "softplus", "tanh", "softsign", "leaky", "tanh01")


def values(rows, c, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, c, generator=g) * torch.exp(torch.randn(rows, 1, generator=g) * spread)
    return x.bfloat16()


def edge_rows():
    """Blocks with every special case, [9, 32]."""
    x = torch.zeros(9, 32)
    x[0] = torch.linspace(-1, 1, 32)
    x[1, 3] = 1.0e-40                                  # below the smallest scale
    x[1, 4] = -1.0e-39
    x[2] = 127.0                                       # exactly at the top of the code range
    x[2, 0] = 0.25
    x[3, 0], x[3, 1] = 127.5, -0.001                   # mantissa 255: the next scale; a small value keeps its sign
    x[4, 5] = math.inf
    x[5, 6] = math.nan
    x[6] = 3.0e38
    x[6, 1] = -3.3895e38
    x[7, 0], x[7, 1], x[7, 2] = 64.0, 0.5, 1.5         # ties: 0.5 -> 0 would be 0, kept as 1; 1.5 -> 2
    x[8, 7] = -0.0
    return x.bfloat16()


def definition(x):
    """Codes, scales and values by exact arithmetic on Python numbers."""
    flat = [float(v) for v in x.reshape(-1)]
    codes, scales, vals = [], [], []
    for i in range(0, len(flat), 32):
        blk = flat[i:i + 32]
        if not all(math.isfinite(v) for v in blk):
            codes += [0] * len(blk)
            scales.append(255)
            vals += [math.nan] * len(blk)
            continue
        top = max(abs(v) for v in blk)
        e = -119
        while e < 121 and top > 127 * 2.0 ** e:
            e += 1
        scales.append(e + 127)
        for v in blk:
            q = max(-127, min(127, round(v / 2.0 ** e)))       # Python rounds ties to even
            if q == 0 and v != 0:
                q = 1 if v > 0 else -1
            codes.append(q)
            vals.append(q * 2.0 ** e)
    return codes, scales, vals


def same(a, b):
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


@pytest.mark.parametrize("x", [edge_rows(), values(7, 40, 1), values(1, 8, 2), values(3, 24, 3, 40.0)],
                         ids=["edges", "ragged", "one_unit", "wide_range"])
def test_cpu_format(x):
    codes, scales, vals = definition(x)
    q = F.pack8(x.float())
    bad = (torch.tensor(scales) == 255).repeat_interleave(32)[:len(codes)]
    assert q.scales.tolist() == scales
    assert torch.equal(q.codes.reshape(-1)[~bad], torch.tensor(codes, dtype=torch.int8)[~bad])
    y = F.unpack8(q)
    assert same(y.reshape(-1).double(), torch.tensor(vals, dtype=torch.float64))
    assert same(y, y.bfloat16().float())               # every value is a bf16 number


def test_cpu_error_and_sign():
    x = values(200, 64, 5).float()
    y = F.unpack8(F.pack8(x))
    top = x.view(-1, 32).abs().amax(1, keepdim=True)
    err = (y - x).abs().view(-1, 32)
    # the scale s is the smallest power of two with top <= 127 s, so 127 s / 2 < top: s < top / 63.5 (not top / 64)
    assert (err <= top / 63.5).all()                                       # a whole step where a small value was kept
    assert ((err <= top / 127) | (x.view(-1, 32).abs() < top / 127)).all()                  # half a step elsewhere
    assert torch.equal(torch.sign(y), torch.sign(x))


@pytest.mark.parametrize("kind", KINDS)
def test_cpu_act_bwd8(kind):
    y = cpu_ref.act_fwd(values(9, 40, 4, 0.5).float(), kind)
    dy = values(9, 40, 6, 0.0).float()
    q = F.pack8(y)
    assert torch.equal(F.act_bwd8(dy, q, kind), cpu_ref.act_bwd(dy, F.unpack8(q), kind))
    if kind in ("relu", "leaky"):                      # the sign survives: exact
        assert torch.equal(F.act_bwd8(dy, q, kind), cpu_ref.act_bwd(dy, y, kind))


def test_cpu_dense_wgrad8():
    x, dy = values(33, 24, 1, 1.0).float(), values(33, 16, 2, 0.0).float()
    q = F.pack8(x)
    dw, db = F.dense_wgrad8(q, dy, n_out=13)
    assert torch.equal(dw, dy[:, :13].t() @ F.unpack8(q)) and torch.equal(db, dy[:, :13].sum(0))


def test_cpu_refusals():
    x = values(4, 32).float()
    q = F.pack8(x)
    with pytest.raises(ValueError):
        F.Packed8(q.codes, q.scales[:-1])
    with pytest.raises(ValueError):
        F.Packed8(q.codes.float(), q.scales)
    with pytest.raises(ValueError):
        F.act_bwd8(x[:2], q, "relu")
    with pytest.raises(ValueError):
        F.dense_wgrad8(q, x[:3])
    with pytest.raises(ValueError):
        F.dense_wgrad8(q, x, n_out=33)
    with pytest.raises(ValueError):
        F.unpack8(q, out=torch.empty(5))


def test_cpu_codes_in_another_order_are_refused():
    """Scales belong to 32 neighbours in memory: transposed codes would be unpacked, or copied by a reshape, with the scales of
    other elements."""
    q = F.pack8(values(64, 40, 3, 20.0).float())
    for codes, scales in ((q.codes.t(), q.scales), (q.codes.view(64, 5, 8).transpose(1, 2), q.scales),
                          (q.codes, q.scales.repeat_interleave(2)[::2])):
        with pytest.raises(ValueError):
            F.Packed8(codes, scales)
    assert same(F.unpack8(q.reshape(40, 64)).reshape(-1), F.unpack8(q).reshape(-1))


def overlaps(x, dy):
    """Outputs over an input or over one another."""
    q = F.pack8(x)
    R, K, O = x.shape[0], x.shape[1], dy.shape[1]
    buf = torch.zeros(4 * R * max(K, O) + 4 * O * K + 64, dtype=torch.uint8, device=x.device)
    codes = buf[:R * K].view(torch.int8).view(R, K)
    codes.copy_(q.codes)
    p = F.Packed8(codes, q.scales)
    d = buf[:dy.numel() * dy.element_size()].view(dy.dtype).view(R, O)
    flat = buf[:4 * O * K].view(torch.float32)
    for call in (lambda: F.unpack8(p, out=buf[:R * K * x.element_size()].view(x.dtype).view(R, K)),
                 lambda: F.dense_wgrad8(p, dy, out_dw=flat.view(O, K)), lambda: F.dense_wgrad8(p, dy, out_db=flat[:O]),
                 lambda: F.dense_wgrad8(q, d, out_dw=flat.view(O, K)), lambda: F.dense_wgrad8(q, d, out_db=flat[:O]),
                 lambda: F.dense_wgrad8(q, dy, out_dw=flat.view(O, K), out_db=flat[8:8 + O])):
        with pytest.raises(ValueError):
            call()


def test_cpu_overlapping_outputs_are_refused():
    overlaps(values(40, 32, 1).float(), values(40, 16, 2).float())


# ------------------------------------------------------------------------------------------------ device
DEV_SHAPES = [(1, 8), (1, 16), (5, 24), (3, 1000), (257, 40), (1000, 264), (4099, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,c", DEV_SHAPES)
@pytest.mark.parametrize("spread", [0.0, 40.0])
def test_pack8(rows, c, spread):
    x = values(rows, c, rows + c, spread)
    q, d = F.pack8(x.float()), F.pack8(x.cuda())
    assert torch.equal(d.scales.cpu(), q.scales) and torch.equal(d.codes.cpu(), q.codes)
    y = F.unpack8(d)
    assert y.dtype == torch.bfloat16 and same(y.float().cpu(), F.unpack8(q))


@pytest.mark.gpu
def test_pack8_edges():
    x = edge_rows()
    q, d = F.pack8(x.float()), F.pack8(x.cuda())
    assert torch.equal(d.scales.cpu(), q.scales)
    ok = (q.scales != 255).repeat_interleave(32)
    assert torch.equal(d.codes.cpu().reshape(-1)[ok], q.codes.reshape(-1)[ok])
    assert same(F.unpack8(d).float().cpu(), F.unpack8(q))


@pytest.mark.gpu
def test_pack8_more_units_than_the_grid():
    x = torch.randn(1 << 20, 72, device="cuda").bfloat16()
    y = F.unpack8(F.pack8(x))
    top = x.view(-1, 32).abs().amax(1, keepdim=True).float()
    # one step: s < top / 63.5, see test_cpu_error_and_sign
    assert ((y.view(-1, 32).float() - x.view(-1, 32).float()).abs() <= top / 63.5).all()
    assert torch.equal(torch.sign(y), torch.sign(x))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,c", [(1, 8), (33, 40), (500, 264)])
def test_act_bwd8(kind, rows, c):
    y = cpu_ref.act_fwd(values(rows, c, 4, 0.5).float(), kind).bfloat16()
    dy = values(rows, c, 6, 0.0)
    got = F.act_bwd8(dy.cuda(), F.pack8(y.cuda()), kind)
    q = F.pack8(y.float())
    ref = dy.double() * cpu_ref.act_grad_from_y(F.unpack8(q).double(), kind)
    lim = 2.0 ** -8 * ref.abs() + 2.0 ** -18 * dy.double().abs()
    assert got.dtype == torch.bfloat16 and ((got.double().cpu() - ref).abs() <= lim).all()


@pytest.mark.gpu
def test_act_bwd8_bad_block_is_nan():
    y, dy = edge_rows(), torch.ones(9, 32).bfloat16()
    for kind in ("relu", "leaky", "tanh"):
        got = F.act_bwd8(dy.cuda(), F.pack8(y.cuda()), kind)
        assert torch.isnan(got[4:6]).all() and not torch.isnan(got[:4]).any()
        assert torch.isnan(F.act_bwd8(dy.float(), F.pack8(y.float()), kind)[4:6]).all()


WG = [(1, 8, 8, 8), (1, 40, 16, 13), (64, 64, 64, 64), (65, 72, 136, 129), (300, 1000, 48, 48), (1000, 264, 520, 517),
      (2051, 136, 256, 250), (129, 2056, 2048, 2048)]


@pytest.mark.gpu
@pytest.mark.parametrize("R,K,Op,O", WG)
def test_dense_wgrad8(R, K, Op, O):
    x, dy = values(R, K, R + K, 1.0), values(R, Op, Op, 0.0)
    q = F.pack8(x.cuda())
    dw, db = F.dense_wgrad8(q, dy.cuda(), n_out=O)
    xh, d = F.unpack8(F.pack8(x.float())).double(), dy.double()[:, :O]
    for got, ref, mag in ((dw, d.t() @ xh, d.abs().t() @ xh.abs()), (db, d.sum(0), d.abs().sum(0))):
        assert got.dtype == torch.float32 and got.shape == ref.shape
        assert ((got.double().cpu() - ref).abs() <= (R + 2) * 2.0 ** -24 * mag + 1e-30).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [0, 1, 2, 3])
@pytest.mark.parametrize("R,K,O", [(70, 72, 40), (640, 520, 264), (3000, 136, 72)])
def test_dense_wgrad8_every_tile(tile, R, K, O, monkeypatch):
    from distributeddeeplearning_amd.ops import hip
    monkeypatch.setattr(hip, "WGRAD8_TILE", tile)
    test_dense_wgrad8(R, K, O, O - 3)


@pytest.mark.gpu
def test_dense_wgrad8_bad_block():
    """A block that held a NaN or an infinity reads as NaN: its features' gradients, no others."""
    x, dy = values(130, 64, 1, 0.0), values(130, 16, 2, 0.0)
    x[77, 5] = math.inf
    dw, db = F.dense_wgrad8(F.pack8(x.cuda()), dy.cuda())
    assert torch.isnan(dw[:, :32]).all() and torch.isfinite(dw[:, 32:]).all() and torch.isfinite(db).all()


@pytest.mark.gpu
def test_dense_wgrad8_outputs_streams_and_empty():
    x, dy = values(130, 40, 1, 1.0).cuda(), values(130, 24, 2, 0.0).cuda()
    q = F.pack8(x)
    flat = torch.full((24 * 40 + 32,), 5.0, device="cuda")
    dw, db = flat[:960].view(24, 40), flat[960:984]
    a = F.dense_wgrad8(q, dy, out_dw=dw, out_db=db)
    assert a[0] is dw and a[1] is db and (flat[984:] == 5).all()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = F.dense_wgrad8(F.pack8(x), dy)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(b[0], dw) and torch.equal(b[1], db)
    e = F.dense_wgrad8(F.pack8(x[:0]), dy[:0])
    assert (e[0] == 0).all() and (e[1] == 0).all()


@pytest.mark.gpu
def test_more_than_2_to_31_elements():
    n = (1 << 31) + 8 * 40
    x = torch.empty(n // 8, 8, dtype=torch.bfloat16, device="cuda").normal_()
    q = F.pack8(x)
    y = F.unpack8(q)
    d = F.act_bwd8(x, q, "relu")
    for rows in (slice(0, 512), slice((1 << 28) - 256, None)):       # around the start and past 2^31 elements
        part = x[rows].cpu()
        ref = F.unpack8(F.pack8(part.float()))
        assert torch.equal(y[rows].float().cpu(), ref)
        assert torch.equal(d[rows].cpu(), torch.where(part > 0, part, torch.zeros_like(part)))


@pytest.mark.gpu
def test_captured_checkpoint_round_trip():
    from distributeddeeplearning_amd.utils import hipgraph
    x, dy = values(70, 72, 1, 1.0).cuda(), values(70, 72, 2, 0.0).cuda()

    def step():
        q = F.pack8(x)
        d = F.act_bwd8(dy, q, "tanh")
        return (F.unpack8(q), d) + F.dense_wgrad8(q, d)
    step()
    hipgraph.quiesce()
    g, out = hipgraph.capture(step)
    for seed in (3, 4, 5):
        x.copy_(values(70, 72, seed, 1.0))
        g.replay()
        torch.cuda.synchronize()
        for p, r in zip(out, step()):
            assert torch.equal(p, r)


@pytest.mark.gpu
def test_refusals():
    x = values(8, 32).cuda()
    q = F.pack8(x)
    for call in (lambda: F.pack8(x.float()), lambda: F.pack8(x[:, :12].contiguous()), lambda: F.pack8(x[:, ::2]),
                 lambda: F.act_bwd8(x[:4], q, "relu"), lambda: F.act_bwd8(x, F.Packed8(q.codes, q.scales.cpu()), "relu"),
                 lambda: F.act_bwd8(x, F.Packed8(q.codes.cpu(), q.scales.cpu()), "relu"),
                 lambda: F.dense_wgrad8(q, x[:4]), lambda: F.dense_wgrad8(q, x, n_out=33), lambda: F.dense_wgrad8(q, x, n_out=0),
                 lambda: F.dense_wgrad8(q, x, out_dw=torch.empty(32, 31, device="cuda")),
                 lambda: F.dense_wgrad8(q, x, out_db=torch.empty(31, device="cuda")),
                 lambda: F.unpack8(q, out=torch.empty(8, 32, device="cuda")),
                 lambda: F.unpack8(F.Packed8(q.codes.t(), q.scales)),
                 lambda: F.dense_wgrad8(q.reshape(2, 4, 32), x), lambda: F.act_bwd8(x.cpu(), q, "relu"),
                 lambda: F.dense_wgrad8(q, x.cpu())):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [0, 1, 2, 3])
@pytest.mark.parametrize("R,K,O,col", [(65, 72, 24, 70), (65, 72, 24, 3), (129, 264, 40, 263), (33, 8, 16, 1), (64, 72, 8, 71)])
def test_dense_wgrad8_bad_last_block(tile, R, K, O, col, monkeypatch):
    """R K is no multiple of 32 in most of these, so the last block is a partial one: bad, it reaches the gradients of its own
    features and of no others, whatever the tile."""
    from distributeddeeplearning_amd.ops import hip
    monkeypatch.setattr(hip, "WGRAD8_TILE", tile)
    x, dy = values(R, K, 1, 0.0), values(R, O, 2, 0.0)
    x[R - 1, col] = math.inf
    dw, db = F.dense_wgrad8(F.pack8(x.cuda()), dy.cuda())
    nan = torch.zeros(R * K, dtype=torch.bool)
    first = ((R - 1) * K + col) // 32 * 32
    nan[first:first + 32] = True
    assert torch.equal(torch.isnan(dw).cpu(), nan.view(R, K).any(0).expand(O, K)) and torch.isfinite(db).all()


@pytest.mark.gpu
def test_overlapping_outputs_are_refused():
    overlaps(values(40, 32, 1).cuda(), values(40, 16, 2).cuda())
