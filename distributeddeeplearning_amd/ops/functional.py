"""Device dispatch for every framework op.

CPU tensors run the fp32 oracle (ops/cpu_ref.py); device tensors run the hand-written gfx950
kernels through ops/hip.py.  There is deliberately no third path: a device tensor with the HIP
extension missing raises instead of silently falling back to eager PyTorch.

Device tensors are bf16 with the channel (last) dimension physically padded to a multiple of 8
(zeros in the padding lanes), so every kernel access is a 16-byte vector and every reduction
dimension is MFMA-friendly; `c_true` arguments carry the logical channel count where an op must
keep the padding lanes at exactly zero.  CPU tensors are unpadded fp32.
"""
from __future__ import annotations

import torch

from . import cpu_ref

_hip = None


def hip_backend():
    global _hip
    if _hip is None:
        from . import hip as _h   # raises with a clear message if the .so is missing
        _hip = _h
    return _hip


def _b(t: torch.Tensor):
    return hip_backend() if t.is_cuda else cpu_ref


# conv family -------------------------------------------------------------------------------
def _cpu_mul(t, mul):
    if mul is None:
        return t
    y, act, alpha = mul
    return cpu_ref.act_bwd(t, y.reshape(t.shape), act, alpha)


def conv_fprop(x, wA, bias, g, act=None, alpha=0.3, mul=None, stats_out=None, bn_infer=None, in_affine=None,
               aff_sink=None):
    """`mul` = (y, act, alpha): result *= act'(y), the activation backward of the layer below (fused
    into the kernel epilogue on device).  `stats_out` (dict): on device, a kernel that can emit the
    output's per-channel partial sums for a following BatchNorm leaves them in stats_out["part"/"nb"];
    with `bn_infer` = (gamma, beta, moving_mean, moving_var, eps) a kernel that can fold that inference-phase
    BatchNorm into its epilogue does so and sets stats_out["affine"]."""
    if x.is_cuda:
        return hip_backend().conv_fprop(x, wA, bias, g, act, alpha, mul, stats_out, bn_infer, in_affine=in_affine,
                                        aff_sink=aff_sink)
    if in_affine is not None:
        raise ValueError("conv_fprop: in_affine exists on the device only")
    return _cpu_mul(cpu_ref.conv_fprop(x, wA, bias, g, act, alpha), mul)


def conv_dgrad(dy, wB, g, bias=None, act=None, alpha=0.3, mul=None, stats_out=None, bn_infer=None, in_affine=None,
               aff_sink=None):
    """`wB` is the core weight in [I][KH][KW][O] order (reduction channel contiguous);
    depthwise: [KH][KW][C].  `in_affine`: device only (a BatchNorm applied on load, ops/hip.py)."""
    if dy.is_cuda:
        return hip_backend().conv_dgrad(dy, wB, g, bias, act, alpha, mul, stats_out, bn_infer, in_affine=in_affine,
                                        aff_sink=aff_sink)
    if in_affine is not None:
        raise ValueError("conv_dgrad: in_affine exists on the device only")
    wA = wB if g.depthwise else wB.permute(3, 1, 2, 0)
    return _cpu_mul(cpu_ref.conv_dgrad(dy, wA, g, bias, act, alpha), mul)


def conv_wgrad(x, dy, g, layout="A", out=None, x_affine=None):
    """Weight gradient of the core correlation, written in layout A=[O][KH][KW][I] or
    B=[I][KH][KW][O] (depthwise: [KH][KW][C]), fp32.  `out` (a view into the flat gradient
    buffer) is overwritten."""
    if x.is_cuda:
        return hip_backend().conv_wgrad(x, dy, g, layout, out, x_affine=x_affine)
    if x_affine is not None:
        raise ValueError("conv_wgrad: x_affine exists on the device only")
    dw = cpu_ref.conv_wgrad(x, dy, g)
    if layout == "B" and not g.depthwise:
        dw = dw.permute(3, 1, 2, 0)
    if out is not None:
        out.copy_(dw.reshape(out.shape))
        return out
    return dw.contiguous()


def bias_grad(dy, out):
    if dy.is_cuda:
        return hip_backend().bias_grad(dy, out)
    out.copy_(cpu_ref.bias_grad(dy))
    return out


# activations -------------------------------------------------------------------------------
def act_fwd(x, kind, alpha=0.3, c_true=None):
    if x.is_cuda:
        return hip_backend().act_fwd(x, kind, alpha, c_true)
    return cpu_ref.act_fwd(x, kind, alpha)


def act_bwd(dy, y, kind, alpha=0.3):
    return _b(dy).act_bwd(dy, y, kind, alpha)


def affine(x, scale, shift, c_true=None):
    if x.is_cuda:
        return hip_backend().affine(x, scale, shift, c_true)
    return x * scale + shift


def spatial_pad(x, pt, pb, pl, pr):
    """ZeroPadding2D on NHWC (negative values crop: used for its backward)."""
    if x.is_cuda:
        return hip_backend().spatial_pad(x, pt, pb, pl, pr)
    return torch.nn.functional.pad(x, (0, 0, pl, pr, pt, pb))


# batch norm --------------------------------------------------------------------------------
def bn_train_affine(x, gamma, beta, mm, mv, momentum, eps, bessel, update_moving=True, groups=1):
    """Batch statistics of x -> (scale, shift, mean, invstd) with y = x*scale + shift, plus the
    Keras moving-average update  moving = moving*momentum + batch*(1-momentum)  (variance
    Bessel-corrected for 4-D inputs, as TF's fused batch norm does).

    `groups` > 1: the batch is `groups` equal contiguous parts, each normalised with its own
    statistics (results are [groups][C]); the moving statistics take one update per part, in order --
    what calling the layer once per part would do (a GAN discriminator on [real ; fake])."""
    if x.is_cuda:
        return hip_backend().bn_train_affine(x, gamma, beta, mm, mv, momentum, eps, bessel, update_moving, groups)
    outs = []
    for xs in x.chunk(groups, 0):
        mean, var = cpu_ref.bn_stats(xs)
        count = xs.numel() // xs.shape[-1]
        invstd = torch.rsqrt(var + eps)
        scale = gamma * invstd
        shift = beta - mean * scale
        if update_moving:
            mm.mul_(momentum).add_(mean, alpha=1 - momentum)
            v = var * (count / max(count - 1, 1)) if bessel else var
            mv.mul_(momentum).add_(v, alpha=1 - momentum)
        outs.append((scale, shift, mean, invstd))
    if groups == 1:
        return outs[0]
    return tuple(torch.stack([o[k] for o in outs], 0) for k in range(4))


def bn_train_affine_from_part(part, nb, rows, gamma, beta, mm, mv, momentum, eps, bessel, update_moving=True,
                              groups=1):
    """Device only: batch statistics from partial sums the producing conv kernel already wrote."""
    return hip_backend().bn_train_affine_from_part(part, nb, rows, gamma, beta, mm, mv, momentum, eps, bessel,
                                                   update_moving, groups)


def bn_infer_affine(gamma, beta, mm, mv, eps):
    """(scale, shift, invstd) from the moving statistics (inference-phase BN)."""
    if gamma.is_cuda:
        return hip_backend().bn_infer_affine(gamma, beta, mm, mv, eps)
    invstd = torch.rsqrt(mv + eps)
    scale = gamma * invstd
    return scale, beta - mm * scale, invstd


def bn_apply_infer(x, gamma, beta, mm, mv, eps, act=None, alpha=0.3, c_true=None):
    """y = act(BN(x)) with the moving statistics, nothing saved for a backward pass."""
    if x.is_cuda:
        return hip_backend().bn_apply_infer(x, gamma, beta, mm, mv, eps, act, alpha, c_true)
    scale, shift, _ = bn_infer_affine(gamma, beta, mm, mv, eps)
    return cpu_ref.bn_apply(x, scale, shift, act, alpha)


def bn_apply(x, scale, shift, act=None, alpha=0.3, c_true=None, groups=1):
    """`groups` > 1: scale / shift are [groups][C], one row per equal contiguous part of the batch."""
    if x.is_cuda:
        return hip_backend().bn_apply(x, scale, shift, act, alpha, c_true, groups)
    if groups == 1:
        return cpu_ref.bn_apply(x, scale, shift, act, alpha)
    return torch.cat([cpu_ref.bn_apply(xs, scale[i], shift[i], act, alpha)
                      for i, xs in enumerate(x.chunk(groups, 0))], 0)


def bn_bwd(dy, x, y, mean, invstd, gamma, act, alpha, train_stats, prev_act=None, prev_alpha=0.3,
           out_dgamma=None, out_dbeta=None, out_dbias=None, groups=1):
    """`out_dbias`: also write the bias gradient of the conv/dense layer feeding this BN (the column
    sums of dx) -- on device it comes out of the same reduction pass as dgamma/dbeta.
    `groups` > 1: per-part statistics (mean / invstd are [groups][C]); dgamma / dbeta / dbias sum over parts."""
    if dy.is_cuda:
        return hip_backend().bn_bwd(dy, x, y, mean, invstd, gamma, act, alpha, train_stats, prev_act,
                                    prev_alpha, out_dgamma, out_dbeta, out_dbias, groups)
    if groups == 1:
        dx, dgamma, dbeta = cpu_ref.bn_bwd(dy, x, y, mean, invstd, gamma, act, alpha, train_stats, prev_act,
                                           prev_alpha)
    else:
        ys = y.chunk(groups, 0) if y is not None else [None] * groups
        parts = [cpu_ref.bn_bwd(d, xx, yy, mean[i], invstd[i], gamma, act, alpha, train_stats, prev_act, prev_alpha)
                 for i, (d, xx, yy) in enumerate(zip(dy.chunk(groups, 0), x.chunk(groups, 0), ys))]
        dx = torch.cat([p[0] for p in parts], 0)
        dgamma, dbeta = sum(p[1] for p in parts), sum(p[2] for p in parts)
    if out_dgamma is not None:
        out_dgamma.copy_(dgamma)
        out_dbeta.copy_(dbeta)
    if out_dbias is not None:
        out_dbias.copy_(cpu_ref.bias_grad(dx)[:out_dbias.numel()])
    return dx, dgamma, dbeta


# losses ------------------------------------------------------------------------------------
def softmax(logits, n_true=None):
    if logits.is_cuda:
        return hip_backend().softmax(logits, n_true)
    return cpu_ref.softmax(logits)


def softmax_ce(logits, onehot, want_grad=True, index=None):
    """`index`: row r's target is onehot[index[r]] -- on device the gather happens inside the loss kernel."""
    if index is not None and not logits.is_cuda:
        onehot, index = onehot.index_select(0, index), None
    return _b(logits).softmax_ce(logits, onehot, want_grad, **({"index": index} if index is not None else {}))


def softmax_mse(logits, target, want_grad=True, index=None):
    if index is not None and not logits.is_cuda:
        target, index = target.index_select(0, index), None
    return _b(logits).softmax_mse(logits, target, want_grad, **({"index": index} if index is not None else {}))


def sigmoid_bce(logits, labels, want_grad=True):
    return _b(logits).sigmoid_bce(logits, labels, want_grad)


def dense1_bce_fwd_bwd(x, w, b, label_first, label_second, n_first, want_dx=True, want_dw=True,
                       out_dw=None, out_db=None, bn=None):
    """`bn`: device only -- the BatchNorm in front of the head fused into the kernel (ops/hip.py)."""
    if x.is_cuda:
        return hip_backend().dense1_bce_fwd_bwd(x, w, b, label_first, label_second, n_first, want_dx, want_dw,
                                                out_dw, out_db, bn)
    if bn is not None:
        raise ValueError("dense1_bce: the BatchNorm fusion exists on the device only")
    loss, dx, dw, db, logits = cpu_ref.dense1_bce_fwd_bwd(x, w, b, label_first, label_second, n_first,
                                                          want_dx, want_dw)
    if want_dw and out_dw is not None:
        out_dw.copy_(dw.reshape(out_dw.shape))
        out_db.copy_(db.reshape(out_db.shape))
    return loss, dx, dw, db, logits


def _apart(what, outs, ins):
    """Refuse outputs that share memory with an input or with one another: kernels write outputs while others still read (a
    gradient over the bias would be the next piece of rows' bias).  (name, tensor or None) each; contiguous ones, as the device
    wants them."""
    spans = []
    for name, t in ins:
        if t is not None:
            lo = t.data_ptr()
            spans.append((lo, lo + t.nbytes, name, t))
    for name, t in outs:
        if t is None:
            continue
        lo = t.data_ptr()
        hi = lo + t.nbytes
        for a, b, other, u in spans:
            if lo < b and a < hi and a < b and lo < hi and t.is_contiguous() and u.is_contiguous():
                raise ValueError(f"{what}: {name} overlaps {other}")
        spans.append((lo, hi, name, t))


def dense_softmax_ce(x, w, bias, labels, want_grad=True, out_dw=None, out_db=None, grad_dtype=torch.float32):
    """Dense(K -> V) + softmax cross entropy for any number of classes, forward and backward.  The logits are not kept; on the
    device a step keeps their exponentials, 2 bytes per row and class, at most DDL_CE_PIECE_BYTES (4 GiB) of them at a time.

    x [N][K], w [V][K] (device: bf16, K padded to a multiple of 8 with zero lanes), bias [V] fp32 or None (-inf switches
    a class off; on the device so does anything below -2.3e38, the type's lowest value among it), labels [N] int64.  A row
    whose label is negative takes no part, whatever its x holds: row loss 0, dx 0, not counted.  Returns (loss, dx, dw, db,
    rows): the mean over the labelled rows (0 if there are none), the gradients of that mean (None without `want_grad`; db
    None without a bias) and the row losses.  dx has x's type, dw [V][K] and db [V] `grad_dtype` (fp32 | bf16), or they
    overwrite `out_dw` / `out_db` in those tensors' type, which share no memory with each other or with an input.

    A label past the last class makes its row loss (and the mean) NaN and its row no gradient; a labelled row with a NaN
    or infinite logit, or with every class switched off, has NaN loss and gradients.  On the device the gradient of the
    logits is rounded to bf16 as every dY is, twice for dw (its scale is folded into x), the label's own entry excepted: fp32
    gradients are good to 5e-5 .. 4e-4 of their rms, not to fp32's 1e-7.  The losses are fp32 throughout."""
    if out_dw is not None or out_db is not None:
        _apart("dense_softmax_ce", (("out_dw", out_dw), ("out_db", out_db)),
               (("x", x), ("w", w), ("bias", bias), ("labels", labels)))
    if x.is_cuda:
        return hip_backend().dense_softmax_ce(x, w, bias, labels, want_grad, out_dw, out_db, grad_dtype)
    loss, dx, dw, db, rows = cpu_ref.dense_softmax_ce(x, w, bias, labels, want_grad)
    if want_grad:
        dw, db = (_cpu_out(t, o, grad_dtype) for t, o in ((dw, out_dw), (db, out_db)))
    elif out_dw is not None or out_db is not None:
        raise ValueError("dense_softmax_ce: out_dw / out_db need want_grad")
    return loss, dx, dw, db, rows


def _cpu_out(t, out, dtype):
    if out is None:
        return t if t is None else t.to(dtype)
    if t is None:
        raise ValueError("an output tensor for a gradient that is not computed")
    if out.numel() != t.numel():
        raise ValueError(f"output: {out.numel()} elements, need {t.numel()}")
    out.copy_(t.reshape(out.shape))
    return out


# 8-bit activation checkpoints ----------------------------------------------------------------
class Packed8:
    """An activation tensor in 8 bits: `codes` (int8, the tensor's shape) and `scales` (uint8, one per 32 consecutive
    codes in memory order, exponent + 127, 8 to 248; 255: the block held a NaN or an infinity and reads as NaN).  The value
    of a code is code * 2^(scale - 127), exact in bf16.  Both are contiguous: a block is 32 neighbours in memory, which a copy of
    a transposed view would take apart."""
    __slots__ = ("codes", "scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype != torch.int8 or scales.dtype != torch.uint8:
            raise ValueError(f"Packed8: int8 codes and uint8 scales, got {codes.dtype} and {scales.dtype}")
        if not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("Packed8: codes and scales have to be contiguous")
        if scales.numel() != (codes.numel() + 31) // 32:
            raise ValueError(f"Packed8: {codes.numel()} codes need {(codes.numel() + 31) // 32} scales, got {scales.numel()}")
        self.codes, self.scales = codes, scales

    @property
    def shape(self):
        return self.codes.shape

    def reshape(self, *shape):
        return Packed8(self.codes.reshape(*shape), self.scales)

    def nbytes(self):
        return self.codes.numel() + self.scales.numel()


def pack8(x):
    """Activation tensor -> Packed8 (33 bytes per 32 elements).  Per 32 elements the scale is the smallest power of two
    from 2^-119 to 2^121 with max |x| <= 127 scale; codes round to nearest even, except that no non-zero value becomes 0
    and the largest bf16 number stays finite."""
    return _b(x).pack8(x)


def unpack8(q, out=None):
    """Packed8 -> activation tensor (device: bf16, exact; CPU: fp32), into `out` (apart from the checkpoint) if given."""
    if out is not None:
        _apart("unpack8", (("out", out),), (("the codes", q.codes), ("the scales", q.scales)))
    return (hip_backend() if q.codes.is_cuda else cpu_ref).unpack8(q, out)


def _same_device(dy, q):
    if dy.device != q.codes.device or q.scales.device != q.codes.device:
        raise ValueError(f"dy is on {dy.device}, the checkpoint's codes on {q.codes.device}, its scales on {q.scales.device}")


def act_bwd8(dy, q, kind, alpha=0.3):
    """Activation backward dx = dy * act'(y) with y = act(x) read from its 8-bit checkpoint."""
    _same_device(dy, q)
    return _b(dy).act_bwd8(dy, q, kind, alpha)


def dense_wgrad8(q, dy, out_dw=None, out_db=None, n_out=None):
    """Gradients of a Dense layer's weights [O][K] and bias [O] (fp32) from its input's 8-bit checkpoint [R][K] and
    dy [R][Op]; `n_out`: O, when dy carries padding lanes behind it.  `out_dw` / `out_db` share no memory with each other or with
    an input."""
    _same_device(dy, q)
    if out_dw is not None or out_db is not None:
        _apart("dense_wgrad8", (("out_dw", out_dw), ("out_db", out_db)),
               (("dy", dy), ("the codes", q.codes), ("the scales", q.scales)))
    return _b(dy).dense_wgrad8(q, dy, out_dw, out_db, n_out)


def argmax_match_count(pred, onehot):
    return _b(pred).argmax_match_count(pred, onehot)
