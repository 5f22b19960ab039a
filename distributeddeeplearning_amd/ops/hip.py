"""ctypes bindings to libddl_hip.so (the gfx950 kernels in csrc/hip) for device tensors.

The kernels have a plain C ABI (raw pointers + hipStream_t) so the native library has no
PyTorch/pybind dependency: tensors are passed as `data_ptr()`, launches go to the *current*
torch stream (so they are captured by `torch.cuda.graph`).  Every wrapper validates shapes,
dtypes and contiguity on the host before launching -- a kernel is never started on operands
it was not written for.

Device tensor convention: bf16, channel (last) dim padded to a multiple of 8, padding lanes zero.
"""
from __future__ import annotations

import ctypes as C
import functools
import os
from pathlib import Path
from typing import Dict, Optional, Tuple

import numpy as np
import torch

from .geometry import ConvGeom

_LIB_PATH = Path(__file__).resolve().parent.parent / "_C" / "libddl_hip.so"
if not _LIB_PATH.exists():
    raise ImportError(
        f"{_LIB_PATH} is missing: the HIP kernels are not built.  Run `python build.py` "
        "(hipcc --offload-arch=gfx950).  Device tensors have no PyTorch fallback by design.")
_lib = C.CDLL(str(_LIB_PATH))

_SYNC_CHECK = os.environ.get("DDL_SYNC_CHECK", "0") == "1"

ACT_CODE = {None: 0, "linear": 0, "relu": 1, "sigmoid": 2, "softplus": 3, "tanh": 4, "softsign": 5,
            "leaky": 6, "tanh01": 7}

vp, ci, cl, cf = C.c_void_p, C.c_int, C.c_long, C.c_float


def _sig(name, restype, *argtypes):
    fn = getattr(_lib, name)
    fn.restype = restype
    fn.argtypes = list(argtypes)
    return fn


_act_fwd = _sig("ddl_act_fwd", None, vp, vp, cl, ci, ci, ci, cf, vp)
_act_bwd = _sig("ddl_act_bwd", None, vp, vp, vp, cl, ci, cf, vp)
_colreduce_blocks = _sig("ddl_colreduce_blocks", ci, cl, ci)
_bn_batch_stats = _sig("ddl_bn_batch_stats", None, vp, cl, ci, vp, vp, vp, vp, vp, cf, cf, ci, ci, vp, vp, vp, vp, ci, vp)
_bn_stats_from_part = _sig("ddl_bn_stats_from_part", None, vp, ci, cl, ci, vp, vp, vp, vp, cf, cf, ci, ci, vp, vp, vp, vp, ci, vp)
_fold_partials = _sig("ddl_fold_partials", None, vp, ci, ci, ci, ci, vp, vp)
_bn_infer_affine = _sig("ddl_bn_infer_affine", None, vp, vp, vp, vp, cf, ci, vp, vp, vp, vp)
_bn_apply = _sig("ddl_bn_apply", None, vp, vp, vp, vp, cl, ci, ci, ci, cf, ci, vp)
_bn_apply_infer = _sig("ddl_bn_apply_infer", None, vp, vp, vp, vp, vp, vp, cf, cl, ci, ci, ci, cf, vp)
_bn_bwd = _sig("ddl_bn_bwd", None, vp, vp, vp, vp, cl, ci, vp, vp, vp, ci, cf, ci, ci, cf, vp, vp, vp, vp, vp, vp, ci,
              ci, ci, vp)
_bias_grad = _sig("ddl_bias_grad", None, vp, cl, ci, ci, vp, vp, vp)
_cast = _sig("ddl_cast_f32_bf16", None, vp, vp, cl, vp)
_relayout = _sig("ddl_relayout_alt", None, vp, vp, vp, ci, cl, vp)
_pad_channels = _sig("ddl_pad_channels", None, vp, ci, vp, vp, cl, ci, ci, ci, ci, cf, vp)
_strip_channels = _sig("ddl_strip_channels", None, vp, vp, cl, ci, ci, vp)
_spatial_pad = _sig("ddl_spatial_pad", None, vp, vp, ci, ci, ci, ci, ci, ci, ci, ci, vp)
_affine = _sig("ddl_affine", None, vp, vp, cl, ci, ci, cf, cf, vp)
_softmax_loss = _sig("ddl_softmax_loss", None, vp, vp, vp, vp, vp, vp, vp, ci, ci, ci, ci, ci, vp)
_softmax_wide = _sig("ddl_softmax_wide", ci, vp, vp, ci, ci, ci, vp)
_sigmoid_bce = _sig("ddl_sigmoid_bce", None, vp, vp, vp, vp, vp, ci, vp)
_dense1_blocks = _sig("ddl_dense1_bce_blocks", ci, ci)
_dense1_bce = _sig("ddl_dense1_bce", ci, vp, vp, vp, cf, cf, ci, ci, ci, vp, vp, vp, vp, vp, vp, vp, vp, ci, ci,
                   vp, vp, vp, vp, vp, ci, ci, ci, cf, vp)
_argmax_match = _sig("ddl_argmax_match", None, vp, vp, ci, ci, vp, vp)
_optim_step = _sig("ddl_optim_step", None, vp, vp, vp, vp, vp, vp, cl, ci, cf, cf, cf, cf, cf, cf, vp, cf, vp)
_step_inc = _sig("ddl_step_inc", None, vp, vp)
_scale_emit = _sig("ddl_scale_emit", None, vp, vp, cl, cf, vp)
_add_f32 = _sig("ddl_add_f32", None, vp, vp, cl, vp)
_zero_bytes = _sig("ddl_zero_bytes", ci, vp, cl, vp)
_avg_delta = _sig("ddl_avg_delta", None, vp, vp, vp, vp, cl, cf, vp)
_im2col = _sig("ddl_im2col_1ch", ci, vp, vp, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, vp)
_col2im = _sig("ddl_col2im_1ch", ci, vp, vp, vp, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, cf, vp, ci,
               cf, vp)
_tapfold = _sig("ddl_tapfold_1ch", ci, vp, vp, vp, vp, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, cf, vp, ci,
                cf, vp, vp, ci, ci, ci, vp)
_tapconv = _sig("ddl_tapconv_1ch", ci, vp, vp, vp, vp, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci,
                cf, vp, vp, vp, vp, ci, ci, cf, vp)
_upconv_blocks = _sig("ddl_upconv_1ch_blocks", ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci)
_upconv = _sig("ddl_upconv_1ch", ci, vp, vp, vp, vp, vp, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci,
               ci, ci, ci, cf, ci, vp)
_upconv_wgrad = _sig("ddl_upconv_1ch_wgrad", ci, vp, vp, vp, vp, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci,
                     ci, ci, ci, vp, vp, vp, vp, vp, vp, ci, cf, ci, vp)
_s1_blocks = _sig("ddl_stream1_wgrad_blocks", ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci)
_s1_wgrad = _sig("ddl_stream1_wgrad", ci, vp, vp, vp, vp, vp, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci,
                 ci, cl, cl, ci, ci, vp, vp, ci, ci, ci, vp)
_gather = _sig("ddl_relayout_gather", None, vp, vp, vp, ci, cl, vp)
_relayout_both = _sig("ddl_relayout_both", None, vp, vp, vp, ci, vp, vp, ci, cl, vp)
_gemm_sk = _sig("ddl_gemm_sk", ci, vp, vp, vp, vp, cl, ci, ci, ci, ci, cf, vp, vp, ci, vp, ci, ci, vp)
_gemm_sk_cols = _sig("ddl_gemm_sk_stats_cols", ci, cl, ci, ci)
_philox = _sig("ddl_philox_uniform", None, vp, cl, vp, cf, cf, vp)
_igemm = _sig("ddl_igemm_conv", ci, vp, vp, vp, vp, vp, vp, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci,
              ci, ci, ci, ci, cf, ci, ci, vp, vp, cf, vp, ci, ci, vp)
_pconv = _sig("ddl_pconv", ci, vp, vp, vp, vp, vp, vp, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, cf,
              ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, vp, vp, vp, vp, vp, cf, vp, vp, ci, ci, vp, cf, ci, ci, vp)
_pconv_lds = _sig("ddl_pconv_lds_bytes", ci, ci, ci, cl, ci)
_wgrad_ksplit = _sig("ddl_wgrad_ksplit", ci, ci, ci, ci, ci)
_wgrad = _sig("ddl_conv_wgrad", ci, vp, vp, vp, vp, cl, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci,
              ci, ci, ci, ci, cl, cl, cl, vp, vp, ci, ci, cl, ci, vp)
_wgrad2 = _sig("ddl_conv_wgrad2", ci, vp, vp, vp, cl, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci,
               cl, cl, cl, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, vp, vp, ci, vp)
_wgrad2_frag_elems = _sig("ddl_wgrad2_frag_elems", cl, ci, ci, ci, ci, ci, ci, ci)
_slab_reduce_frag = _sig("ddl_slab_reduce_frag", ci, vp, vp, ci, ci, ci, ci, ci, ci, ci, ci, ci, cl, cl, cl, vp)
_wgrad2_lds = _sig("ddl_wgrad2_lds", ci, ci, ci, ci, ci, ci, ci, ci, ci, ci)
_wgrad2_lds_dma = _sig("ddl_wgrad2_lds_dma", ci, ci, ci, ci, ci, ci, ci, ci, ci, ci)
_slab_reduce = _sig("ddl_slab_reduce", None, vp, vp, cl, cl, ci, vp)
_dw_blocks = _sig("ddl_dw_wgrad_blocks", ci, cl, ci)
_dw_dgrad_bn = _sig("ddl_dw_dgrad_bn", ci, ci, vp, vp, vp, vp, vp, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci,
                    vp, vp, vp, vp, vp, ci, cf, ci, vp)
_dw_fwd_stats = _sig("ddl_depthwise_fwd_stats", ci, vp, vp, vp, vp, vp, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, cf,
                     vp, vp, ci, vp)
_depthwise = _sig("ddl_depthwise", ci, ci, vp, vp, vp, vp, vp, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci, ci,
                  ci, ci, ci, ci, cf, vp, vp, ci, vp)

IGEMM_TILE = int(os.environ.get("DDL_IGEMM_TILE", "0"))     # 0 = heuristic; tuning knob
CONV_IMPL = os.environ.get("DDL_CONV", "pconv")             # pconv (patch-resident, default) | igemm
PCONV_LDS = int(os.environ.get("DDL_PCONV_LDS", "0"))       # LDS budget per block in bytes (0 = 80 KiB)
PCONV_MIN_ROWS = int(os.environ.get("DDL_PCONV_MIN_ROWS", "150"))   # units with fewer output rows -> igemm
PCONV_FR = int(os.environ.get("DDL_PCONV_FR", "0"))         # fragments per wave (4 | 8; 0 = heuristic)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _done():
    if _SYNC_CHECK:
        torch.cuda.synchronize()


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def pad8(c: int) -> int:
    return (c + 7) // 8 * 8


def _chk_act(t: torch.Tensor, name="tensor"):
    if not (t.is_cuda and t.dtype == torch.bfloat16 and t.is_contiguous()):
        raise ValueError(f"{name}: device kernels need a contiguous bf16 cuda tensor, got "
                         f"{t.dtype} {t.device} contiguous={t.is_contiguous()}")
    if t.shape[-1] % 8:
        raise ValueError(f"{name}: channel dim {t.shape[-1]} is not padded to a multiple of 8")
    if t.data_ptr() % 16:
        raise ValueError(f"{name}: not 16-byte aligned")


def _chk_f32(t: torch.Tensor, n=None, name="tensor"):
    if not (t.is_cuda and t.dtype == torch.float32 and t.is_contiguous()):
        raise ValueError(f"{name}: need contiguous fp32 cuda tensor")
    if n is not None and t.numel() < n:
        raise ValueError(f"{name}: {t.numel()} elements, need >= {n}")


def _rows_c(t):
    return t.numel() // t.shape[-1], t.shape[-1]


# ------------------------------------------------------------------------------ activations
def act_fwd(x, kind, alpha=0.3, c_true=None):
    if kind in (None, "linear"):
        return x
    _chk_act(x, "x")
    y = torch.empty_like(x)
    rows, Cp = _rows_c(x)
    _act_fwd(x.data_ptr(), y.data_ptr(), rows, Cp, Cp if c_true is None else c_true, ACT_CODE[kind], alpha,
             _stream())
    _done()
    return y


def act_bwd(dy, y, kind, alpha=0.3):
    if kind in (None, "linear"):
        return dy
    _chk_act(dy, "dy")
    _chk_act(y, "y")
    if dy.shape != y.shape:
        raise ValueError("act_bwd shape mismatch")
    dx = torch.empty_like(dy)
    _act_bwd(dy.data_ptr(), y.data_ptr(), dx.data_ptr(), dy.numel(), ACT_CODE[kind], alpha, _stream())
    _done()
    return dx


def affine(x, scale, shift, c_true=None):
    _chk_act(x, "x")
    y = torch.empty_like(x)
    rows, Cp = _rows_c(x)
    _affine(x.data_ptr(), y.data_ptr(), rows, Cp, Cp if c_true is None else c_true, scale, shift, _stream())
    _done()
    return y


def spatial_pad(x, pt, pb, pl, pr):
    _chk_act(x, "x")
    B, H, W, Cp = x.shape
    Hd, Wd = H + pt + pb, W + pl + pr
    if Hd <= 0 or Wd <= 0:
        raise ValueError("spatial_pad produces an empty tensor")
    y = torch.empty(B, Hd, Wd, Cp, dtype=x.dtype, device=x.device)
    _spatial_pad(x.data_ptr(), y.data_ptr(), B, H, W, Hd, Wd, Cp, pt, pl, _stream())
    _done()
    return y


# ------------------------------------------------------------------------------ batch norm
def _part(rows, Cp, device, ns=2, groups=1):
    nb = _colreduce_blocks(rows, Cp)
    return torch.empty(nb * ns * Cp * groups, dtype=torch.float32, device=device)


def _group_rows(x, groups):
    """Rows per batch group: the batch (leading) dim splits into `groups` equal contiguous parts."""
    rows, Cp = _rows_c(x)
    if groups < 1 or x.shape[0] % groups:
        raise ValueError(f"batch {x.shape[0]} does not split into {groups} equal groups")
    return rows // groups, Cp


def bn_train_affine(x, gamma, beta, mm, mv, momentum, eps, bessel, update_moving=True, groups=1):
    """-> scale, shift, mean, invstd: [Cp] each, or [groups][Cp] with per-group batch statistics (`groups` > 1:
    the batch is `groups` equal contiguous parts, each normalised with its own statistics; the moving
    statistics take one momentum update per group, in order)."""
    _chk_act(x, "x")
    rows, Cp = _group_rows(x, groups)
    for t, n in ((gamma, "gamma"), (beta, "beta"), (mm, "moving_mean"), (mv, "moving_var")):
        _chk_f32(t, Cp, n)
    out = torch.empty(4, groups, Cp, dtype=torch.float32, device=x.device)
    part = _part(rows, Cp, x.device, 2, groups)
    _bn_batch_stats(x.data_ptr(), rows, Cp, part.data_ptr(), gamma.data_ptr(), beta.data_ptr(), mm.data_ptr(),
                    mv.data_ptr(), momentum, eps, int(bool(bessel)), int(bool(update_moving)),
                    out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), out[3].data_ptr(), groups, _stream())
    _done()
    if groups == 1:
        out = out.view(4, Cp)
    return out[0], out[1], out[2], out[3]


FOLD_PARTIALS_MIN = int(os.environ.get("DDL_FOLD_PARTIALS_MIN", "16384"))


def bn_train_affine_from_part(part, nb, rows, gamma, beta, mm, mv, momentum, eps, bessel, update_moving=True,
                              groups=1):
    """`bn_train_affine` when the producer kernel already left per-block partial sums part[2][Cp][nb].
    `rows` = rows of the whole batch; with `groups` > 1 both `nb` and `rows` must split evenly (the
    producer's blocks are batch-major and none straddles a group boundary -- the caller checks that)."""
    Cp = gamma.numel()
    _chk_f32(part, 2 * Cp * nb, "stats partials")
    if nb % groups or rows % groups:
        raise ValueError("partials / rows do not split into the batch groups")
    for t, n in ((gamma, "gamma"), (beta, "beta"), (mm, "moving_mean"), (mv, "moving_var")):
        _chk_f32(t, Cp, n)
    out = torch.empty(4, groups, Cp, dtype=torch.float32, device=gamma.device)
    if nb // groups >= FOLD_PARTIALS_MIN:          # very many columns: fold them 64-fold across the chip first
        S = 64
        folded = torch.empty(2 * Cp * groups * S, dtype=torch.float32, device=gamma.device)
        _fold_partials(part.data_ptr(), 2 * Cp, nb // groups, groups, S, folded.data_ptr(), _stream())
        part, nb = folded, groups * S
    _bn_stats_from_part(part.data_ptr(), nb // groups, rows // groups, Cp, gamma.data_ptr(), beta.data_ptr(),
                        mm.data_ptr(), mv.data_ptr(), momentum, eps, int(bool(bessel)), int(bool(update_moving)),
                        out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), out[3].data_ptr(), groups, _stream())
    _done()
    if groups == 1:
        out = out.view(4, Cp)
    return out[0], out[1], out[2], out[3]


def bn_infer_affine(gamma, beta, mm, mv, eps):
    Cp = gamma.numel()
    out = torch.empty(3, Cp, dtype=torch.float32, device=gamma.device)
    _bn_infer_affine(gamma.data_ptr(), beta.data_ptr(), mm.data_ptr(), mv.data_ptr(), eps, Cp,
                     out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), _stream())
    _done()
    return out[0], out[1], out[2]


def bn_apply(x, scale, shift, act=None, alpha=0.3, c_true=None, groups=1):
    _chk_act(x, "x")
    rows, Cp = _group_rows(x, groups)
    _chk_f32(scale, Cp * groups, "scale")
    _chk_f32(shift, Cp * groups, "shift")
    y = torch.empty_like(x)
    _bn_apply(x.data_ptr(), y.data_ptr(), scale.data_ptr(), shift.data_ptr(), rows, Cp,
              Cp if c_true is None else c_true, ACT_CODE[act], alpha, groups, _stream())
    _done()
    return y


def bn_apply_infer(x, gamma, beta, mm, mv, eps, act=None, alpha=0.3, c_true=None):
    """Inference-phase BN (moving statistics) + activation in ONE launch."""
    _chk_act(x, "x")
    rows, Cp = _rows_c(x)
    for t, n in ((gamma, "gamma"), (beta, "beta"), (mm, "moving_mean"), (mv, "moving_var")):
        _chk_f32(t, Cp, n)
    y = torch.empty_like(x)
    _bn_apply_infer(x.data_ptr(), y.data_ptr(), gamma.data_ptr(), beta.data_ptr(), mm.data_ptr(), mv.data_ptr(), eps,
                    rows, Cp, Cp if c_true is None else c_true, ACT_CODE[act], alpha, _stream())
    _done()
    return y


def bn_bwd(dy, x, y, mean, invstd, gamma, act, alpha, train_stats, prev_act=None, prev_alpha=0.3,
           out_dgamma=None, out_dbeta=None, out_dbias=None, groups=1, part=None, part_blocks=0):
    """`out_dbias` (fp32, <= C entries): also emit the bias gradient of the conv layer feeding this BN
    (= column sums of dx) from the same reduction pass (colreduce MODE 3).
    `part`, `part_blocks`: column sums of (dy, dy * xhat) already written by the producer of dy as
    [2][Cp][groups * part_blocks] (the fused discriminator head): the reduction pass is skipped."""
    _chk_act(dy, "dy")
    _chk_act(x, "x")
    if dy.shape != x.shape:
        raise ValueError(f"bn_bwd: dy {tuple(dy.shape)} vs x {tuple(x.shape)}")
    if ACT_CODE[act] != 0:
        _chk_act(y, "y")
    rows, Cp = _group_rows(x, groups)
    for t, n in ((mean, "mean"), (invstd, "invstd")):
        _chk_f32(t, Cp * groups, n)
    _chk_f32(gamma, Cp, "gamma")
    dev = x.device
    dx = torch.empty_like(x)
    if out_dbias is not None:
        _chk_f32(out_dbias, None, "dbias")
        if out_dbias.numel() > Cp:
            raise ValueError("bn_bwd: bias gradient longer than the channel dim")
    if part is not None:
        if part_blocks <= 0:
            raise ValueError("bn_bwd: precomputed partials need part_blocks")
        _chk_f32(part, (5 if out_dbias is not None else 2) * Cp * groups * part_blocks, "bn_bwd partials")
    else:
        part_blocks = 0
        part = _part(rows, Cp, dev, 5 if out_dbias is not None else 2, groups)
    coef = torch.empty(2, groups * Cp, dtype=torch.float32, device=dev)
    if out_dgamma is None:
        out_dgamma = torch.empty(Cp, dtype=torch.float32, device=dev)
        out_dbeta = torch.empty(Cp, dtype=torch.float32, device=dev)
    else:
        _chk_f32(out_dgamma, Cp, "dgamma")
        _chk_f32(out_dbeta, Cp, "dbeta")
    _bn_bwd(dy.data_ptr(), x.data_ptr(), _p(y), dx.data_ptr(), rows, Cp, mean.data_ptr(), invstd.data_ptr(),
            gamma.data_ptr(), ACT_CODE[act], alpha, int(bool(train_stats)), ACT_CODE[prev_act], prev_alpha,
            part.data_ptr(), out_dgamma.data_ptr(), out_dbeta.data_ptr(), coef[0].data_ptr(),
            coef[1].data_ptr(), _p(out_dbias), 0 if out_dbias is None else out_dbias.numel(), groups, part_blocks,
            _stream())
    _done()
    return dx, out_dgamma, out_dbeta


def dw_dgrad_bn_bwd(dy, w, g: "ConvGeom", x, mean, invstd, gamma, prev_act, prev_alpha, out_dgamma, out_dbeta,
                    out_dbias=None):
    """Depthwise input gradient fused with the backward of the batch-statistics BatchNorm in front of the layer
    (csrc/hip/wgrad.hip `dw_dgrad_bn_*`): dy [B][OH][OW][Cp] -> dx [B][H][W][Cp], the gradient at the BatchNorm's INPUT
    `x` (times prev_act'(x) of the conv in front of it), plus dgamma / dbeta (/ that conv's bias gradient).  The
    BatchNorm's dY -- the depthwise input gradient proper -- is recomputed in both passes and never stored.
    Returns None when the shape is outside the fused kernels' range."""
    _chk_act(dy, "dy")
    _chk_act(x, "x")
    B, Cp = x.shape[0], x.shape[-1]
    if tuple(x.shape[1:3]) != (g.H, g.W) or tuple(dy.shape) != (B, g.OH, g.OW, Cp) or g.KH != g.KW:
        return None
    cgn = Cp // 8
    if cgn > 64 or cgn & (cgn - 1) or g.KH > 3 or g.sh > 3 or g.sw > 3:
        return None
    _chk_w(w, (g.KH, g.KW, Cp), "depthwise kernel")
    for t, nme in ((mean, "mean"), (invstd, "invstd"), (gamma, "gamma"), (out_dgamma, "dgamma"), (out_dbeta, "dbeta")):
        _chk_f32(t, Cp, nme)
    ns = 5 if out_dbias is not None else 2
    dev = x.device
    classes = g.sh * g.sw
    nb_max = (-(-2048 // classes)) * classes
    part = torch.empty(ns * Cp * nb_max, dtype=torch.float32, device=dev)
    coef = torch.empty(2, Cp, dtype=torch.float32, device=dev)
    args = (B, g.H, g.W, Cp, g.OH, g.OW, g.KH, g.sh, g.sw, g.dh, g.dw, g.pt, g.pl, mean.data_ptr(), invstd.data_ptr(),
            gamma.data_ptr(), coef[0].data_ptr(), coef[1].data_ptr(), ACT_CODE[prev_act], prev_alpha, ns, _stream())
    nb = _dw_dgrad_bn(0, dy.data_ptr(), w.data_ptr(), x.data_ptr(), None, part.data_ptr(), *args)
    if nb <= 0:
        return None
    # the ordinary finalize (fp64, fixed order): c1, c2, dgamma, dbeta, dbias from part[ns][Cp][nb]
    _bn_bwd(None, None, None, None, B * g.H * g.W, Cp, mean.data_ptr(), invstd.data_ptr(), gamma.data_ptr(), 0, 0.3, 1,
            ACT_CODE[prev_act], prev_alpha, part.data_ptr(), out_dgamma.data_ptr(), out_dbeta.data_ptr(),
            coef[0].data_ptr(), coef[1].data_ptr(), _p(out_dbias), 0 if out_dbias is None else out_dbias.numel(), 1,
            nb, _stream())
    dx = torch.empty_like(x)
    rc = _dw_dgrad_bn(1, dy.data_ptr(), w.data_ptr(), x.data_ptr(), dx.data_ptr(), part.data_ptr(), *args)
    if rc < 0:
        raise ValueError("dw_dgrad_bn apply pass rejected a shape its reduce pass accepted")
    _done()
    return dx


def bias_grad(dy, out):
    _chk_act(dy, "dy")
    rows, Cp = _rows_c(dy)
    _chk_f32(out, None, "bias grad")
    if out.numel() > Cp:
        raise ValueError("bias grad longer than channel dim")
    part = _part(rows, Cp, dy.device)
    _bias_grad(dy.data_ptr(), rows, Cp, out.numel(), part.data_ptr(), out.data_ptr(), _stream())
    _done()
    return out


# ------------------------------------------------------------------------------ casts / layout
def cast_f32_to_bf16(src, dst):
    if src.numel() != dst.numel() or src.numel() % 8:
        raise ValueError("cast: flat buffers must match and be padded to 8")
    _cast(src.data_ptr(), dst.data_ptr(), src.numel(), _stream())
    _done()


def relayout_alt(net, launch=True):
    """Refresh every alternate-layout weight copy of `net` in one launch."""
    tab = getattr(net, "_relayout_tab", None)
    if tab is None:
        descs, mx = [], 0
        skip = net.first_param_op() if getattr(net, "no_input_grad", False) else None
        for op, alt_off in net._alt:
            if op is skip:              # its adjoint-direction copy only ever serves the network-input gradient
                continue
            R, T, Cc, Rp = op.relayout_dims()
            poff = net._pmap[(op.name, "kernel")].offset
            descs.append((poff, alt_off, R, T, Cc, Rp))
            mx = max(mx, Cc * T * Rp)
        arr = np.zeros(len(descs), dtype=[("s", "<i8"), ("d", "<i8"), ("R", "<i4"), ("T", "<i4"), ("C", "<i4"),
                                          ("Rp", "<i4")])
        for i, d in enumerate(descs):
            arr[i] = d
        dev = torch.from_numpy(arr.view(np.uint8).copy()).to(net.device) if len(descs) else None
        tab = net._relayout_tab = (dev, len(descs), mx)
    dev, n, mx = tab
    if n and launch:
        _relayout(net.P.data_ptr(), net.Palt.data_ptr(), dev.data_ptr(), n, mx, _stream())
        _done()


def relayout_all(net):
    """Alternate-layout and strided-gather weight copies of `net`, one launch when it has both kinds."""
    if not net._gather:
        return relayout_alt(net)
    relayout_alt(net, launch=False)
    relayout_gather(net, launch=False)
    adev, na, amx = net._relayout_tab
    gdev, ng, gmx = net._gather_tab
    if na == 0:
        return relayout_gather(net)
    _relayout_both(net.P.data_ptr(), net.Palt.data_ptr(), adev.data_ptr(), na, net.Pg.data_ptr(), gdev.data_ptr(), ng,
                   max(amx, gmx), _stream())
    _done()


def relayout_gather(net, launch=True):
    """Refresh the strided-gather weight copies (one-channel conv path) of `net` in one launch."""
    if not net._gather:
        return
    tab = getattr(net, "_gather_tab", None)
    if tab is None:
        arr = np.zeros(len(net._gather), dtype=[("s", "<i8"), ("d", "<i8"), ("R1", "<i4"), ("C1", "<i4"),
                                                ("R2", "<i4"), ("C2", "<i4"), ("sr", "<i8"), ("sc", "<i8")])
        for i, d in enumerate(net._gather):
            arr[i] = d
        mx = max(d[4] * d[5] for d in net._gather)
        tab = net._gather_tab = (torch.from_numpy(arr.view(np.uint8).copy()).to(net.device), len(net._gather), mx)
    dev, n, mx = tab
    if not launch:
        return
    _gather(net.P.data_ptr(), net.Pg.data_ptr(), dev.data_ptr(), n, mx, _stream())
    _done()


def im2col_1ch(img, g: ConvGeom, out=None, ones=False):
    """[B][g.H][g.W][Ci] (channel 0 is the image) -> taps-as-channels [B][g.OH][g.OW][pad8(KH*KW)].
    `ones`: the first padding tap (column KH*KW, needs KH*KW < pad8(KH*KW)) holds 1.0 instead of 0 -- the column the
    streaming weight gradient turns into the bias gradient (`conv_wgrad(bias_tail=...)`)."""
    _chk_act(img, "img")
    B = img.shape[0]
    if tuple(img.shape[1:3]) != (g.H, g.W):
        raise ValueError(f"im2col_1ch: image {tuple(img.shape)} vs geometry {g}")
    Tp = pad8(g.KH * g.KW)
    col = out if out is not None else torch.empty(B, g.OH, g.OW, Tp, dtype=torch.bfloat16, device=img.device)
    ranges = _batch_ranges(B, max(g.OH * g.OW * Tp, g.H * g.W * img.shape[-1]))
    if ranges is not None:
        for b0, b1 in ranges:
            im2col_1ch(img[b0:b1], g, col[b0:b1], ones)
        return col
    rc = _im2col(img.data_ptr(), col.data_ptr(), B, g.H, g.W, img.shape[-1], g.OH, g.OW, g.KH, g.KW, g.sh, g.sw,
                 g.dh, g.dw, g.pt, g.pl, Tp, 1 if ones else 0, _stream())
    if rc:
        raise ValueError("im2col_1ch rejected")
    _done()
    return col


def _mul_args(mul, like):
    """`mul` = (y, act, alpha): fused activation backward of the layer below, result *= act'(y).  -> ctypes args."""
    if mul is None:
        return None, 0, 0.0
    y, act, alpha = mul
    _chk_act(y, "mul y")
    if y.numel() != like.numel():
        raise ValueError(f"fused act backward: y has {y.numel()} elements, result {like.numel()}")
    return y.data_ptr(), ACT_CODE[act], alpha


def _mul_inplace(t, mul):
    """The unfused form of `mul` for kernels without that epilogue: t *= act'(y), in place."""
    if mul is not None:
        y, act, alpha = mul
        _act_bwd(t.data_ptr(), y.data_ptr(), t.data_ptr(), t.numel(), ACT_CODE[act], alpha, _stream())


def col2im_1ch(col, g: ConvGeom, bias=None, act=None, alpha=0.3, out=None, mul=None):
    """taps-as-channels [B][g.OH][g.OW][pad8(T)] -> single-channel image [B][g.H][g.W][8] = act(bias + fold).
    `out`: write into this (contiguous, same shape) tensor instead of a fresh one."""
    _chk_act(col, "col")
    B = col.shape[0]
    Tp = pad8(g.KH * g.KW)
    if tuple(col.shape[1:]) != (g.OH, g.OW, Tp):
        raise ValueError(f"col2im_1ch: col {tuple(col.shape)} vs geometry {g}")
    if bias is not None:
        _chk_f32(bias, 1, "bias")
    if out is not None:
        _chk_act(out, "out")
        if tuple(out.shape) != (B, g.H, g.W, 8):
            raise ValueError(f"col2im_1ch: out {tuple(out.shape)} != {(B, g.H, g.W, 8)}")
        img = out
    else:
        img = torch.empty(B, g.H, g.W, 8, dtype=torch.bfloat16, device=col.device)
    ranges = _batch_ranges(B, max(g.OH * g.OW * Tp, g.H * g.W * 8))
    if ranges is not None:
        for b0, b1 in ranges:
            col2im_1ch(col[b0:b1], g, bias, act, alpha, img[b0:b1], _mul_slice(mul, b0, b1))
        return img
    my, ma, mal = _mul_args(mul, img)
    rc = _col2im(col.data_ptr(), img.data_ptr(), _p(bias), B, g.H, g.W, g.OH, g.OW, g.KH, g.KW, g.sh, g.sw, g.dh,
                 g.dw, g.pt, g.pl, Tp, ACT_CODE[act], alpha, my, ma, mal, _stream())
    if rc:
        raise ValueError("col2im_1ch rejected")
    _done()
    return img


TAPFOLD = os.environ.get("DDL_TAPFOLD", "1") == "1"


def tapfold_1ch(x, w, g: ConvGeom, bias=None, act=None, alpha=0.3, out=None, mul=None, in_affine=None, _b_off=0):
    """Fused taps GEMM + fold (csrc/hip/onech_fused.hip): x [B][g.OH][g.OW][Cp], w [T][Cp] (bf16) ->
    single-channel image [B][g.H][g.W][8] = act(bias + fold_t(x . w[t])), optionally *= act'(mul y).
    `in_affine` = (scale, shift, groups, c_true): x is read as bf16(x * scale[grp] + shift[grp]) -- the
    BatchNorm in front of this layer applied on load instead of as a pass of its own ([groups][Cp] rows, the
    batch being `groups` equal contiguous parts).
    Returns None when the shape is outside the fused kernel's range (caller uses gemm + col2im_1ch)."""
    if not TAPFOLD:
        return None
    _chk_act(x, "x")
    B, Cp = x.shape[0], x.shape[-1]
    T = g.KH * g.KW
    if tuple(x.shape[1:3]) != (g.OH, g.OW):
        raise ValueError(f"tapfold_1ch: x {tuple(x.shape)} vs geometry {g}")
    if not (w.is_cuda and w.dtype == torch.bfloat16 and w.is_contiguous()) or w.numel() < T * Cp:
        raise ValueError("tapfold_1ch: weights must be contiguous bf16 [T][Cp]")
    if T > 32 or Cp > 128:
        return None
    if bias is not None:
        _chk_f32(bias, 1, "bias")
    if out is not None:
        _chk_act(out, "out")
        if tuple(out.shape) != (B, g.H, g.W, 8):
            raise ValueError(f"tapfold_1ch: out {tuple(out.shape)} != {(B, g.H, g.W, 8)}")
        img = out
    else:
        img = torch.empty(B, g.H, g.W, 8, dtype=torch.bfloat16, device=x.device)
    isc = ish = None
    grows, ctrue = 1, Cp
    if in_affine is not None:
        isc_t, ish_t, groups, ctrue = in_affine
        if isinstance(groups, tuple):           # (rows per group,) of the whole batch: a batch-split recursion
            grows = groups[0]
        else:
            if groups < 1 or B % groups:
                raise ValueError(f"tapfold_1ch: batch {B} does not split into {groups} groups")
            grows = B // groups
        ngroups = -(-(_b_off + B) // grows)
        _chk_f32(isc_t, None, "in_affine scale")
        _chk_f32(ish_t, None, "in_affine shift")
        if isc_t.numel() < ngroups * Cp or ish_t.numel() < ngroups * Cp:
            raise ValueError("tapfold_1ch: in_affine needs [groups][Cp] scale / shift rows")
        isc, ish = isc_t.data_ptr(), ish_t.data_ptr()
    ranges = _batch_ranges(B, max(g.OH * g.OW * Cp, g.H * g.W * 8))
    if ranges is not None:
        sub = None if in_affine is None else (in_affine[0], in_affine[1], (grows,), ctrue)
        for b0, b1 in ranges:
            if tapfold_1ch(x[b0:b1], w, g, bias, act, alpha, img[b0:b1], _mul_slice(mul, b0, b1), sub,
                           _b_off + b0) is None:
                return None
        return img
    my, ma, mal = _mul_args(mul, img)
    rc = _tapfold(x.data_ptr(), w.data_ptr(), _p(bias), img.data_ptr(), B, g.H, g.W, g.OH, g.OW, Cp, g.KH, g.KW,
                  g.sh, g.sw, g.dh, g.dw, g.pt, g.pl, ACT_CODE[act], alpha, my, ma, mal, isc, ish, grows, _b_off,
                  ctrue, _stream())
    if rc < 0:
        raise ValueError(f"tapfold_1ch rejected its arguments (rc={rc})")
    if rc > 0:
        return None
    _done()
    return img


TAPCONV = os.environ.get("DDL_TAPCONV", "1") == "1"


def tapconv_1ch(img, w, g: ConvGeom, bias=None, act=None, alpha=0.3, out=None, bn_red=None):
    """Direct convolution from a single-channel image (csrc/hip/onech_fused.hip: tapconv_1ch_kernel):
    img [B][g.H][g.W][8] (channel 0 real), w [N][1][1][Tp] bf16 (row n = the taps of output channel n) ->
    [B][g.OH][g.OW][pad8(N)] = act(bias + sum_t img[tap t of the pixel] * w[n][t]): im2col_1ch + the 1x1 GEMM in
    one kernel, bit-identical to them.  Returns None when the shape is outside the kernel's range.
    `bn_red` = dict(x, mean, invstd, sums (2 | 5), prev_act, prev_alpha): the result is the gradient at the output of
    a BatchNorm whose input is `x`; the kernel also emits that BatchNorm's backward column sums (what
    colreduce<1> / <3> would compute from the result and x in another pass) into bn_red["part"], bn_red["nb"]."""
    if not TAPCONV:
        return None
    _chk_act(img, "img")
    B = img.shape[0]
    T = g.KH * g.KW
    if tuple(img.shape[1:]) != (g.H, g.W, 8):
        raise ValueError(f"tapconv_1ch: image {tuple(img.shape)} vs geometry {g}")
    if not (w.is_cuda and w.dtype == torch.bfloat16 and w.is_contiguous()) or w.dim() != 4:
        raise ValueError("tapconv_1ch: weights must be contiguous bf16 [N][1][1][Tp]")
    N, Tp = w.shape[0], w.shape[-1]
    Np = pad8(N)
    if T > 32 or Tp > 32 or Tp < T or Np > 64:
        return None
    if bias is not None:
        _chk_f32(bias, N, "bias")
    if out is not None:
        _chk_act(out, "out")
        if tuple(out.shape) != (B, g.OH, g.OW, Np):
            raise ValueError(f"tapconv_1ch: out {tuple(out.shape)} != {(B, g.OH, g.OW, Np)}")
        y = out
    else:
        y = torch.empty(B, g.OH, g.OW, Np, dtype=torch.bfloat16, device=img.device)
    ranges = _batch_ranges(B, max(g.OH * g.OW * Np, g.H * g.W * 8))
    if ranges is not None:
        for b0, b1 in ranges:           # (no reduction fusion across split launches: bn_red stays untouched)
            if tapconv_1ch(img[b0:b1], w, g, bias, act, alpha, y[b0:b1]) is None:
                return None
        return y
    rx = rmu = ris = rpart = None
    rsums, ract, ralpha = 0, 0, 0.0
    if bn_red is not None and ACT_CODE[act] in (0, 1, 6):
        xr = bn_red["x"]
        _chk_act(xr, "bn_red x")
        if tuple(xr.shape) != tuple(y.shape):
            raise ValueError(f"tapconv_1ch: bn_red x {tuple(xr.shape)} vs output {tuple(y.shape)}")
        rsums = int(bn_red["sums"])
        _chk_f32(bn_red["mean"], Np, "bn_red mean")
        _chk_f32(bn_red["invstd"], Np, "bn_red invstd")
        part = torch.empty(rsums * Np * B, dtype=torch.float32, device=img.device)
        rx, rmu, ris, rpart = xr.data_ptr(), bn_red["mean"].data_ptr(), bn_red["invstd"].data_ptr(), part.data_ptr()
        ract, ralpha = ACT_CODE[bn_red.get("prev_act")], float(bn_red.get("prev_alpha", 0.3))
    rc = _tapconv(img.data_ptr(), w.data_ptr(), _p(bias), y.data_ptr(), B, g.H, g.W, g.OH, g.OW, g.KH, g.KW, g.sh,
                  g.sw, g.dh, g.dw, g.pt, g.pl, Tp, Np, N, ACT_CODE[act], alpha, rx, rmu, ris, rpart, rsums, ract,
                  ralpha, _stream())
    if rc == 0 and rx is not None:
        bn_red["part"], bn_red["nb"] = part, B
    if rc < 0:
        raise ValueError(f"tapconv_1ch rejected its arguments (rc={rc})")
    if rc > 0:
        return None
    _done()
    return y


UPCONV = os.environ.get("DDL_UPCONV", "1") == "1"
DW_STATS = os.environ.get("DDL_DW_STATS", "1") == "1"       # BatchNorm statistics out of the depthwise ring forward


def _upconv_shape(x, w, g: ConvGeom, name, wgrad=0, fwdconv=False):
    """Operands of a convolution from a one-channel image against its core geometry `g`.  Transposed (default): g is
    the forward conv whose input gradient the layer is (g.O = 1 layer input channel, g.I layer output channels,
    g.OH x g.OW the layer's input, g.H x g.W its output).  `fwdconv`: a Conv2D, g.I = 1, g.H x g.W -> g.OH x g.OW x g.O.
    Returns (B, Cs, Cw, Np, blocks of the launch, (IH, IW, H, W, N)) or None when outside the kernels' range."""
    _chk_act(x, "x")
    B, Cs = x.shape[0], x.shape[-1]
    IH, IW, H, W, N = (g.H, g.W, g.OH, g.OW, g.O) if fwdconv else (g.OH, g.OW, g.H, g.W, g.I)
    if (g.I if fwdconv else g.O) != 1 or g.depthwise or tuple(x.shape[1:3]) != (IH, IW):
        raise ValueError(f"{name}: x {tuple(x.shape)} vs geometry {g}")
    if not (w.is_cuda and w.dtype == torch.bfloat16 and w.is_contiguous()) or w.dim() != 4 \
            or tuple(w.shape[:3]) != (N, g.KH, g.KW):
        raise ValueError(f"{name}: weights must be contiguous bf16 [N][KH][KW][Cw], got {tuple(w.shape)} for {g}")
    Np = pad8(N)
    nby = _upconv_blocks(wgrad, B, H, W, Np, g.KH, g.KW, g.sh, g.sw, int(fwdconv))
    if nby <= 0 or _batch_ranges(B, max(H * W * Np, IH * IW * Cs)) is not None:
        return None
    return B, Cs, w.shape[-1], Np, nby, (IH, IW, H, W, N)


def upconv_1ch(x, w, g: ConvGeom, bias=None, act=None, alpha=0.3, stats_out=None, fwdconv=False):
    """Convolution from a single-channel image as a streaming kernel (csrc/hip/upconv_1ch.hip): transposed (default: x
    [B][g.OH][g.OW][Cs] -> [B][g.H][g.W][pad8(N)]) or forward (`fwdconv`: x [B][g.H][g.W][Cs] -> [B][g.OH][g.OW][pad8(N)]),
    w canonical [N][KH][KW][Cw] bf16 (channel 0 real), K <= 3.  One 16-byte store per lane, only live taps computed.
    `stats_out` (dict): receives the BatchNorm partials of the output ("part", "nb", "img") like the conv kernels'
    statistics epilogue.  Returns None when the shape is outside the kernel's range (nothing launched)."""
    if not UPCONV:
        return None
    shp = _upconv_shape(x, w, g, "upconv_1ch", 0, fwdconv)
    if shp is None:
        return None
    B, Cs, Cw, Np, nby, (IH, IW, H, W, N) = shp
    if bias is not None:
        _chk_f32(bias, N, "bias")
    y = torch.empty(B, H, W, Np, dtype=torch.bfloat16, device=x.device)
    part = None
    if stats_out is not None:
        part = torch.empty(2 * Np * nby, dtype=torch.float32, device=x.device)
    rc = _upconv(x.data_ptr(), w.data_ptr(), _p(bias), y.data_ptr(), _p(part), 0, 0, B, IH, IW, Cs, Cw, H, W,
                 Np, N, g.KH, g.KW, g.sh, g.sw, g.dh, g.dw, g.pt, g.pl, ACT_CODE[act], alpha, int(fwdconv), _stream())
    if rc < 0:
        raise ValueError(f"upconv_1ch rejected its arguments (rc={rc})")
    if rc > 0:
        return None
    if part is not None:
        stats_out["part"], stats_out["nb"], stats_out["img"] = part, nby, 1
    _done()
    return y


def upconv_1ch_wgrad(x, dy, w_like, g: ConvGeom, out, bn=None, fwdconv=False):
    """Weight gradient of `upconv_1ch`: out (fp32, canonical [N][KH][KW][Cw] like `w_like`) = sum over pixels of
    dY[b][h][w][n] * x[tap]; the padding channels of `out` are written as zeros.  Deterministic (per-block slabs summed
    in a fixed order).  `bn` = dict(x, mean, invstd, gamma, c1, c2, act, alpha): `dy` is the gradient at the OUTPUT of
    the batch-statistics BatchNorm behind the layer and bn["x"] that BatchNorm's input (the layer's own output); the
    BatchNorm's backward apply step -- act'(x) * (k0 dy + k1 x + k2) with the finalized coefficients c1, c2
    (`bn_bwd_sums`) -- happens on load and the gradient at the BatchNorm's input is never written.
    Returns False when the shape is outside the kernel's range (nothing launched)."""
    if not UPCONV:
        return False
    shp = _upconv_shape(x, w_like, g, "upconv_1ch_wgrad", 2 if bn is not None else 1, fwdconv)
    if shp is None:
        return False
    B, Cs, Cw, Np, nby, (IH, IW, H, W, N) = shp
    _chk_act(dy, "dy")
    if tuple(dy.shape) != (B, H, W, Np):
        raise ValueError(f"upconv_1ch_wgrad: dy {tuple(dy.shape)} != {(B, H, W, Np)}")
    _chk_f32(out, N * g.KH * g.KW * Cw, "out")
    if tuple(out.shape) != tuple(w_like.shape):
        raise ValueError(f"upconv_1ch_wgrad: out {tuple(out.shape)} != weights {tuple(w_like.shape)}")
    bargs = (None, None, None, None, None, None, 0, 0.0)
    if bn is not None:
        _chk_act(bn["x"], "bn x")
        if tuple(bn["x"].shape) != tuple(dy.shape):
            raise ValueError(f"upconv_1ch_wgrad: bn x {tuple(bn['x'].shape)} vs dy {tuple(dy.shape)}")
        for k_ in ("mean", "invstd", "gamma", "c1", "c2"):
            _chk_f32(bn[k_], N, f"bn {k_}")
        bargs = (bn["x"].data_ptr(), bn["mean"].data_ptr(), bn["invstd"].data_ptr(), bn["gamma"].data_ptr(),
                 bn["c1"].data_ptr(), bn["c2"].data_ptr(), ACT_CODE[bn.get("act")], float(bn.get("alpha", 0.3)))
    slab = torch.empty(nby * g.KH * g.KW * Np, dtype=torch.float32, device=x.device)
    rc = _upconv_wgrad(x.data_ptr(), dy.data_ptr(), slab.data_ptr(), out.data_ptr(), B, IH, IW, Cs, Cw, H, W, Np,
                       N, g.KH, g.KW, g.sh, g.sw, g.dh, g.dw, g.pt, g.pl, *bargs, int(fwdconv), _stream())
    if rc < 0:
        raise ValueError(f"upconv_1ch_wgrad rejected its arguments (rc={rc})")
    _done()
    return rc == 0


S1_WGRAD = os.environ.get("DDL_S1_WGRAD", "1") == "1"


def stream1_wgrad(img, t, g: ConvGeom, out, sn, st, zfill=1, n_out=None, bias=None, bias_mode=0, affine=None):
    """Weight gradient of a 4x4 / 5x5 convolution between a one-channel image and an N-channel tensor, as a streaming
    kernel (csrc/hip/upconv_1ch.hip, stream1_wgrad_kernel; no taps tensor, no split-K GEMM):

        out[n * sn + tap * st] = sum_{b,oh,ow} t[b][oh][ow][n] * img[b][oh*sh + kh*dh - pt][ow*sw + kw*dw - pl]   (n < n_out)

    with `zfill - 1` zeros written behind each element (the padding channels of a canonical [O][KH][KW][8] gradient).
    `g` is the forward core geometry image (g.H x g.W, 1 channel) -> tensor (g.OH x g.OW): the first Conv2D of the DCGAN
    discriminator (img = x, t = dY) and the last Conv2DTranspose of its generator (img = dY, t = x;
    /root/reference/DCGAN.py:22-66).  `affine` = (scale, shift, c_true): t is a BatchNorm's INPUT and the normalisation
    is applied on load (rounded to bf16 like the tensor it replaces).  bias_mode 1: bias[n] = column sums of t (a Conv2D's
    bias gradient); 2: bias[0] = sum of img's channel 0 (the C -> 1 layer's scalar bias gradient).  Deterministic.
    Returns False when the shape is outside the kernel's range (nothing launched)."""
    if not S1_WGRAD or g.depthwise or g.KH != g.KW or g.KH not in (4, 5):
        return False
    _chk_act(img, "img")
    _chk_act(t, "t")
    B, Cs, Np = img.shape[0], img.shape[-1], t.shape[-1]
    if img.dim() != 4 or t.dim() != 4 or tuple(img.shape[1:3]) != (g.H, g.W) or tuple(t.shape[:3]) != (B, g.OH, g.OW):
        raise ValueError(f"stream1_wgrad: img {tuple(img.shape)} / t {tuple(t.shape)} vs geometry {g}")
    N = Np if n_out is None else int(n_out)
    if not 0 < N <= Np:
        raise ValueError(f"stream1_wgrad: n_out {N} vs {Np} channels")
    # tensors of 2^31 elements and more go in batch slices: each writes its slabs, the last call sums them all
    rngs = _batch_ranges(B, max(g.OH * g.OW * Np, g.H * g.W * Cs)) or [(0, B)]
    nbys = [_s1_blocks(b1 - b0, g.H, g.W, Cs, g.OH, g.OW, Np, g.KH, g.KW, g.sh, g.sw, g.dh, g.dw, g.pt, g.pl)
            for b0, b1 in rngs]
    if min(nbys) <= 0:
        return False
    T = g.KH * g.KW
    _chk_f32(out, (N - 1) * sn + (T - 1) * st + zfill, "out")
    if sn < 0 or st < 0 or zfill < 1 or bias_mode not in (0, 1, 2):
        raise ValueError("stream1_wgrad: bad output layout")
    if bias_mode:
        _chk_f32(bias, N if bias_mode == 1 else 1, "bias")
    asc = ash = None
    actrue = 0
    if affine is not None:
        asc, ash, actrue = affine
        _chk_f32(asc, Np, "affine scale")
        _chk_f32(ash, Np, "affine shift")
    total = sum(nbys)
    slab = torch.empty(total * ((T + 1) * Np + 1), dtype=torch.float32, device=img.device)
    first = 0
    for k, (b0, b1) in enumerate(rngs):
        last = k + 1 == len(rngs)
        rc = _s1_wgrad(img[b0:b1].data_ptr(), t[b0:b1].data_ptr(), slab.data_ptr(), out.data_ptr(),
                       _p(bias) if bias_mode else None, b1 - b0, g.H, g.W, Cs, g.OH, g.OW, Np, N, g.KH, g.KW, g.sh, g.sw,
                       g.dh, g.dw, g.pt, g.pl, int(sn), int(st), int(zfill), int(bias_mode), _p(asc), _p(ash),
                       int(actrue), first, total if last else 0, _stream())
        if rc < 0:
            raise ValueError(f"stream1_wgrad rejected its arguments (rc={rc})")
        if rc != 0:
            if k:
                raise RuntimeError("stream1_wgrad: a later batch slice fell outside the kernel's range")
            return False
        first += nbys[k]
    _done()
    return True


def bn_bwd_sums(dy, x, mean, invstd, gamma, prev_act, prev_alpha, out_dgamma, out_dbeta, out_dbias=None):
    """The reduction + finalize half of `bn_bwd` for a BatchNorm without an activation of its own (one statistics
    group): dgamma, dbeta (and the bias gradient of the conv in front of it) are written, the coefficients (c1, c2) of
    the apply step are returned for a consumer that applies them on load (`upconv_1ch_wgrad(bn=...)`)."""
    _chk_act(dy, "dy")
    _chk_act(x, "x")
    if dy.shape != x.shape:
        raise ValueError(f"bn_bwd_sums: dy {tuple(dy.shape)} vs x {tuple(x.shape)}")
    rows, Cp = _group_rows(x, 1)
    for t, n in ((mean, "mean"), (invstd, "invstd"), (gamma, "gamma"), (out_dgamma, "dgamma"), (out_dbeta, "dbeta")):
        _chk_f32(t, Cp, n)
    dev = x.device
    part = _part(rows, Cp, dev, 5 if out_dbias is not None else 2, 1)
    coef = torch.empty(2, Cp, dtype=torch.float32, device=dev)
    _bn_bwd(dy.data_ptr(), x.data_ptr(), None, None, rows, Cp, mean.data_ptr(), invstd.data_ptr(), gamma.data_ptr(), 0,
            0.3, 1, ACT_CODE[prev_act], prev_alpha, part.data_ptr(), out_dgamma.data_ptr(), out_dbeta.data_ptr(),
            coef[0].data_ptr(), coef[1].data_ptr(), _p(out_dbias), 0 if out_dbias is None else out_dbias.numel(), 1, 0,
            _stream())
    _done()
    return coef[0], coef[1]


def pad_channels(x, c_phys, index=None, scale=1.0, c_true=None):
    """[N,...,c_in] fp32/u8/bf16 (or a row gather of it via `index`) -> bf16 [...,c_phys];
    a 1-channel source is replicated to `c_true` channels (DDL.py:119 stacks MNIST x3)."""
    if not x.is_cuda or not x.is_contiguous():
        raise ValueError("pad_channels: contiguous cuda tensor required")
    c_in = x.shape[-1]
    c_true = c_in if c_true is None else c_true
    code = {torch.float32: 0, torch.uint8: 1, torch.bfloat16: 2}.get(x.dtype)
    if code is None:
        raise ValueError(f"pad_channels: unsupported dtype {x.dtype}")
    if c_in != 1 and c_in != c_true:
        raise ValueError("pad_channels: c_true must equal source channels unless replicating 1 channel")
    pix = int(np.prod(x.shape[1:-1])) if x.dim() > 2 else 1
    n = x.shape[0] if index is None else index.numel()
    if index is not None:
        if index.dtype != torch.int64 or not index.is_cuda:
            raise ValueError("index must be int64 cuda")
    out = torch.empty((n,) + tuple(x.shape[1:-1]) + (c_phys,), dtype=torch.bfloat16, device=x.device)
    _pad_channels(x.data_ptr(), code, _p(index), out.data_ptr(), n * pix, pix, c_in, c_true, c_phys, scale,
                  _stream())
    _done()
    return out


def strip_channels(x, c_true):
    _chk_act(x, "x")
    rows, Cp = _rows_c(x)
    out = torch.empty(tuple(x.shape[:-1]) + (c_true,), dtype=torch.float32, device=x.device)
    _strip_channels(x.data_ptr(), out.data_ptr(), rows, Cp, c_true, _stream())
    _done()
    return out


# ------------------------------------------------------------------------------ losses
def _softmax_common(logits, target, mode, want_grad, want_probs=True, n_true=None, index=None):
    _chk_act(logits, "logits")
    B, Cs = logits.shape
    N = n_true if target is None else target.shape[1]
    dev = logits.device
    if mode == 0 and 64 < N <= Cs:
        probs = torch.empty(B, N, dtype=torch.float32, device=dev)
        if B:
            with _on_device(logits):
                _rc(_softmax_wide(logits.data_ptr(), probs.data_ptr(), B, Cs, N, _stream_of(logits)), "softmax")
        _done()
        return None, None, probs
    if N > 64 or N > Cs:
        raise ValueError("softmax losses support up to 64 classes (wider heads: dense_softmax_ce)")
    probs = torch.empty(B, N, dtype=torch.float32, device=dev) if want_probs else None
    if mode == 0:
        _softmax_loss(logits.data_ptr(), None, None, probs.data_ptr(), None, None, None, B, Cs, N, 0, 0, _stream())
        _done()
        return None, None, probs
    if not (target.is_cuda and target.dtype == torch.float32 and target.is_contiguous()
            and target.shape[0] == (B if index is None else target.shape[0]) and target.shape[1] == N):
        raise ValueError("target must be contiguous fp32 cuda [B,N] ([rows,N] with `index`)")
    if index is not None and not (index.is_cuda and index.dtype == torch.int64 and index.is_contiguous()
                                  and index.numel() == B):
        raise ValueError("index must be a contiguous cuda int64 vector of B row numbers")
    dl = torch.empty_like(logits) if want_grad else None
    rowloss = torch.empty(B, dtype=torch.float32, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    _softmax_loss(logits.data_ptr(), target.data_ptr(), _p(index), _p(probs), _p(dl), rowloss.data_ptr(),
                  loss.data_ptr(), B, Cs, N, mode, int(want_grad), _stream())
    _done()
    return loss, dl, probs


def softmax(logits, n_true=None):
    return _softmax_common(logits, None, 0, False, True, n_true or logits.shape[1])[2]


def softmax_ce(logits, onehot, want_grad=True, index=None):
    """`index`: row r's target is onehot[index[r]] (label gather fused into the loss kernel)."""
    return _softmax_common(logits, onehot, 1, want_grad, index=index)


def softmax_mse(logits, target, want_grad=True, index=None):
    return _softmax_common(logits, target, 2, want_grad, index=index)


def sigmoid_bce(logits, labels, want_grad=True):
    x = logits.float().reshape(-1).contiguous()
    z = labels.float().reshape(-1).contiguous()
    n = x.numel()
    rowloss = torch.empty(n, dtype=torch.float32, device=x.device)
    dl = torch.empty(n, dtype=torch.float32, device=x.device) if want_grad else None
    loss = torch.empty((), dtype=torch.float32, device=x.device)
    _sigmoid_bce(x.data_ptr(), z.data_ptr(), rowloss.data_ptr(), _p(dl), loss.data_ptr(), n, _stream())
    _done()
    return loss, (dl.reshape(logits.shape) if want_grad else None)


def dense1_bce_fwd_bwd(x, w, b, label_first, label_second, n_first, want_dx=True, want_dw=True,
                       out_dw=None, out_db=None, bn=None):
    """Dense(K -> 1) + sigmoid-BCE forward and backward in one kernel.
    `bn` = dict(scale, shift, mean, invstd ([groups][C] fp32), C, groups, act, alpha): `x` is the tensor in FRONT
    of a BatchNorm(+activation) that is applied on load; the returned dx is then the gradient with respect to the
    BatchNorm's pre-activation output and bn["part"], bn["nb"] receive the column sums of (dx, dx * xhat) for
    `bn_bwd(..., part=, part_blocks=)` -- no bn_apply pass, no reduction pass (csrc/hip/loss_optim.hip HeadBn)."""
    _chk_act(x, "x")
    M = x.shape[0]
    K = x.numel() // M
    if w.numel() != K or w.dtype != torch.bfloat16 or not w.is_contiguous():
        raise ValueError(f"dense1_bce: weight must be bf16 with {K} elements")
    _chk_f32(b, 1, "bias")
    dev = x.device
    groups = 1
    bsc = bsh = bmu = bis = bpart = None
    bC, bact, balpha = 0, 0, 0.0
    if bn is not None:
        bC, groups = int(bn["C"]), int(bn["groups"])
        if M % groups or K % bC or 512 % bC or K > 2048 or (bC // 8) * 64 > K:
            raise ValueError(f"dense1_bce: BatchNorm fusion does not support M={M} K={K} C={bC} groups={groups}")
        for k_ in ("scale", "shift", "mean", "invstd"):
            _chk_f32(bn[k_], groups * bC, f"bn {k_}")
        bact, balpha = ACT_CODE[bn.get("act")], float(bn.get("alpha", 0.3))
    dx = torch.empty_like(x) if want_dx else None
    nb = _dense1_blocks(M // groups)
    dw_part = torch.empty(nb * groups * K, dtype=torch.float32, device=dev) if want_dw else None
    aux = torch.empty(3, M, dtype=torch.float32, device=dev)       # logits, rowloss, dlogit
    # With a weight gradient the mean loss rides in head_finalize; without one (the generator phase) it would be a
    # single-block launch of its own on every step, for a number that is only read when somebody logs it: the row
    # losses stay on the device and the mean is taken when asked for (DeferredMean; a replayed graph rewrites `aux`)
    loss = torch.empty((), dtype=torch.float32, device=dev) if (want_dw or not DEFER_MEAN) else None
    if bn is not None:
        part = torch.empty(2 * bC * groups * nb, dtype=torch.float32, device=dev)
        bn["part"], bn["nb"] = part, nb
        bsc, bsh, bmu, bis, bpart = (bn["scale"].data_ptr(), bn["shift"].data_ptr(), bn["mean"].data_ptr(),
                                     bn["invstd"].data_ptr(), part.data_ptr())
    if want_dw and out_dw is None:
        out_dw = torch.empty(K, dtype=torch.float32, device=dev)
        out_db = torch.empty(1, dtype=torch.float32, device=dev)
    if want_dw:
        _chk_f32(out_dw, K, "dw")
        _chk_f32(out_db, 1, "db")
    rc = _dense1_bce(x.data_ptr(), w.data_ptr(), b.data_ptr(), label_first, label_second, n_first, M, K,
                     _p(dx), _p(dw_part), aux[0].data_ptr(), aux[1].data_ptr(), aux[2].data_ptr(),
                     _p(loss), _p(out_dw) if want_dw else None, _p(out_db) if want_dw else None,
                     int(want_dx), int(want_dw), bsc, bsh, bmu, bis, bpart, bC, groups, bact, balpha, _stream())
    if rc != 0:
        raise ValueError(f"dense1_bce: unsupported K={K} (rc={rc})")
    _done()
    return (loss if loss is not None else DeferredMean(aux[1])), dx, out_dw, out_db, aux[0]


DEFER_MEAN = os.environ.get("DDL_DEFER_MEAN", "1") == "1"


class DeferredMean:
    """Mean of a device vector, computed when read (`float(x)` / `x.item()`): in fp64 over the row order, as the
    single-block mean kernel does.  Holds the (static, under graph replay) buffer, not a value."""
    __slots__ = ("rows",)

    def __init__(self, rows: torch.Tensor):
        self.rows = rows

    def item(self) -> float:
        return float(self.rows.double().sum().item() / self.rows.numel())

    __float__ = item

    def detach(self):
        return self

    def __repr__(self):
        return f"DeferredMean({self.item():.6g})"


def argmax_match_count(pred, onehot):
    pred = pred.float().contiguous()
    onehot = onehot.float().contiguous()
    if pred.shape != onehot.shape:
        raise ValueError("argmax_match_count shape mismatch")
    cnt = torch.zeros(1, dtype=torch.int32, device=pred.device)
    _argmax_match(pred.data_ptr(), onehot.data_ptr(), pred.shape[0], pred.shape[1], cnt.data_ptr(), _stream())
    _done()
    return cnt[0]


# ------------------------------------------------------------------------------ optimizer / rng
_OPT_KIND = {"adam": 0, "sgd": 1, "rmsprop": 2, "adam_fresh_double": 3}


def optimizer_step(opt, grad_scale=1.0):
    net, c = opt.net, opt.cfg
    n = net.P.numel()
    if opt.step_dev.numel() < 2:
        raise ValueError("step_dev must hold [steps, scratch]")
    _optim_step(net.P.data_ptr(), net.G.data_ptr(), _p(opt.m), _p(opt.v), net.Pc.data_ptr(),
                opt.step_dev.data_ptr(), n, _OPT_KIND[c.kind], c.lr, c.beta1, c.beta2, c.eps, c.rho, grad_scale,
                None, 0.0, _stream())
    _done()


def step_inc(step_dev):
    """Advance a device-side optimizer step counter (one-thread kernel on the current stream)."""
    _step_inc(step_dev.data_ptr(), _stream())


def optimizer_step_flat(P, G, m, v, Pc, step_dev, c, grad_scale=1.0):
    """The fused update on explicit flat tensors (a shard of a network's buffers: ZeRO-1 mode)."""
    n = P.numel()
    if step_dev.numel() < 2:
        raise ValueError("step_dev must hold [steps, scratch]")
    _chk_f32(G, n, "grad shard")
    _optim_step(P.data_ptr(), G.data_ptr(), _p(m), _p(v), _p(Pc), step_dev.data_ptr(), n, _OPT_KIND[c.kind],
                c.lr, c.beta1, c.beta2, c.eps, c.rho, grad_scale, None, 0.0, _stream())
    _done()


def add_f32_(dst, src):
    """dst += src (flat fp32, same size)."""
    n = dst.numel()
    _chk_f32(dst, n, "dst")
    _chk_f32(src, n, "src")
    _add_f32(dst.data_ptr(), src.data_ptr(), n, _stream())
    _done()
    return dst


def zero_(t):
    """t = 0 for a contiguous device tensor (hipMemsetAsync on the current stream; capturable)."""
    if not (t.is_cuda and t.is_contiguous()):
        return t.zero_()
    if _zero_bytes(t.data_ptr(), t.numel() * t.element_size(), _stream()) != 0:
        raise RuntimeError("hipMemsetAsync failed")
    return t


def scale_emit(P, Pc, scale):
    _scale_emit(P.data_ptr(), _p(Pc), P.numel(), scale, _stream())
    _done()


def avg_delta(P, Pc, total, snap, inv_world):
    """P += total*inv_world - snap (delayed weight averaging), bf16 copy re-emitted."""
    n = P.numel()
    _chk_f32(total, n, "sum")
    _chk_f32(snap, n, "snapshot")
    _avg_delta(P.data_ptr(), _p(Pc), total.data_ptr(), snap.data_ptr(), n, inv_world, _stream())
    _done()


def philox_uniform(shape, dtype, state, lo=-1.0, hi=1.0):
    if dtype != torch.bfloat16:
        raise ValueError("device noise is generated in bf16")
    if state.dtype != torch.int64 or state.numel() < 3 or not state.is_cuda:
        raise ValueError("philox state must be a cuda int64 tensor [seed, offset, scratch]")
    out = torch.empty(shape, dtype=dtype, device=state.device)
    _philox(out.data_ptr(), out.numel(), state.data_ptr(), lo, hi, _stream())
    _done()
    return out


# ------------------------------------------------------------------------------ conv family
_TAB_CACHE: Dict[Tuple, Tuple] = {}


def _class_taps(g: ConvGeom, mode: str):
    """Python-side class / tap lists of the class-grid formulation (see igemm_conv.hip):
    classes [(ph, pw, Hc, Wc, ntaps, tap_off)], taps [(offh, offw, wtap)]."""
    classes, taps = [], []
    if mode == "fprop":
        tl = [(kh * g.dh - g.pt, kw * g.dw - g.pl, kh * g.KW + kw) for kh in range(g.KH) for kw in range(g.KW)]
        classes.append((0, 0, g.OH, g.OW, len(tl), 0))
        taps += tl
    else:
        for ph in range(g.sh):
            for pw in range(g.sw):
                Hc = (g.H - ph + g.sh - 1) // g.sh
                Wc = (g.W - pw + g.sw - 1) // g.sw
                if Hc <= 0 or Wc <= 0:
                    continue
                tl = []
                for kh in range(g.KH):
                    th = ph + g.pt - kh * g.dh
                    if th % g.sh:
                        continue
                    for kw in range(g.KW):
                        tw = pw + g.pl - kw * g.dw
                        if tw % g.sw:
                            continue
                        tl.append((th // g.sh, tw // g.sw, kh * g.KW + kw))
                classes.append((ph, pw, Hc, Wc, len(tl), len(taps)))
                taps += tl
    return classes, taps


IGEMM_UT = os.environ.get("DDL_IGEMM_UT", "1") == "1"      # uniform-tap gather in the implicit-GEMM kernels


def _tables(g: ConvGeom, mode: str, B: int, device):
    """Class descriptors + tap tables for the implicit-GEMM kernel (see igemm_conv.hip)."""
    key = (g, mode, B, str(device))
    hit = _TAB_CACHE.get(key)
    if hit is not None:
        return hit
    cl_, tp_ = _class_taps(g, mode)
    # uniform-tap gather (igemm_conv.hip): per class the box of its taps' (offh, offw); when the box has at most 32
    # cells every gathered row keeps one validity bit per cell, and a tap's fourth word is its cell
    classes, taps = [], [(t[0], t[1], t[2], 0) for t in tp_] or [(0, 0, 0, 0)]
    for c in cl_:
        pad = 0
        tl = tp_[c[5]:c[5] + c[4]]
        if tl and IGEMM_UT:
            minh, minw = min(t[0] for t in tl), min(t[1] for t in tl)
            rh, rw = max(t[0] for t in tl) - minh + 1, max(t[1] for t in tl) - minw + 1
            if rh * rw <= 32 and -64 <= minh < 64 and -64 <= minw < 64:
                pad = 1 | (minh + 64) << 1 | (minw + 64) << 8 | rw << 15 | rh << 21
                for k in range(c[5], c[5] + c[4]):
                    t = tp_[k]
                    taps[k] = (t[0], t[1], t[2], (t[0] - minh) * rw + (t[1] - minw))
        classes.append((c[0], c[1], c[2], c[3], c[4], c[5], B * c[2] * c[3], pad))
    ct = torch.tensor(classes, dtype=torch.int32).to(device)
    tt = torch.tensor(taps + [(0, 0, 0, 0)], dtype=torch.int32).to(device)   # spare entry: a tap-less class reads it
    res = (ct, tt, len(classes), max(c[6] for c in classes), max(max(c[4] for c in classes), 1),
           all(c[7] != 0 or c[4] == 0 for c in classes))
    _TAB_CACHE[key] = res
    return res


_PLAN_CACHE: Dict[Tuple, Optional[dict]] = {}


def _pick_pitch(Cs: int, stride: int) -> int:
    """Smallest patch pixel pitch (bytes) whose ds_read_b128 lane groups are conflict-free for pixels
    `stride` apart: (stride * pitch/16) % 4 == 2 (see pconv.hip)."""
    p0 = Cs // 8
    for p in range(p0, p0 + 4):
        if (stride * p) % 4 == 2:
            return p * 16
    return (p0 | 1) * 16


def _pconv_plan(g: ConvGeom, mode: str, B: int, Cs: int, Nd: int, ss, device, budget=None, img=None, fr=None,
                min_rows=None, nw=4):
    """Unit decomposition + patch geometry + k-unit table for the patch-resident kernel, or None when
    the problem does not fit the scheme (Dense, patch too big for LDS, too few rows per unit).
    `budget` = LDS bytes per block (80 KiB -> two blocks per CU), `img` = images per unit (default:
    as many as fit, capped), `fr` = 16-row fragments per wave (4 | 8)."""
    budget = budget or PCONV_LDS or 80 * 1024
    min_rows = PCONV_MIN_ROWS if min_rows is None else min_rows
    key = (g, mode, B, Cs, Nd, str(device), budget, img, fr, min_rows, nw)
    if key in _PLAN_CACHE:
        return _PLAN_CACHE[key]
    plan = None
    classes, taps = _class_taps(g, mode)
    live = [t for c in classes for t in taps[c[5]:c[5] + c[4]]]
    Hs, Ws = (g.H, g.W) if mode == "fprop" else (g.OH, g.OW)
    if live and Hs * Ws > 1:
        ssh, ssw = ss
        omin_h, omax_h = min(t[0] for t in live), max(t[0] for t in live)
        omin_w, omax_w = min(t[1] for t in live), max(t[1] for t in live)
        maxHc, maxWc = max(c[2] for c in classes), max(c[3] for c in classes)
        BN = 16 if Nd <= 16 else (32 if Nd <= 32 else (64 if Nd <= 64 else 128))
        ntile = (Nd + BN - 1) // BN
        pitch = _pick_pitch(Cs, ssw)
        PW = (maxWc - 1) * ssw + (omax_w - omin_w) + 1
        nst = [((c[4] * Cs + 63) // 64 + 1) // 2 * 2 for c in classes]       # even: the kernel works in stage pairs
        total_stages = sum(nst)
        if nw == 8 and BN not in (32, 64):
            _PLAN_CACHE[key] = None
            return None
        fixed = _pconv_lds(BN, total_stages, 0, nw)
        rows_of = lambda br: (br - 1) * ssh + (omax_h - omin_h) + 1
        img_full = rows_of(maxHc) * PW * pitch
        IMG, BR = 0, maxHc
        if img_full <= budget - fixed:
            rows_per_img = maxHc * maxWc
            n = min((budget - fixed) // img_full, B)
            if img is not None:
                IMG = min(img, n)
            else:
                n = min(n, -(-1024 // rows_per_img))
                while n > 1 and -(-B // n) * ntile < 256:       # keep every CU busy
                    n -= 1
                best, best_eff = n, 0.0
                for c in range(n, max((n + 1) // 2, 1) - 1, -1):
                    rows = c * rows_per_img
                    eff = rows / (-(-rows // 256) * 256)
                    if eff > best_eff + 1e-9:
                        best, best_eff = c, eff
                IMG = best
        elif img in (None, 1):
            br = maxHc
            while br > 1 and rows_of(br) * PW * pitch > budget - fixed:
                br -= 1
            if rows_of(br) * PW * pitch <= budget - fixed:
                IMG, BR = 1, br
        if IMG and IMG * min(BR, maxHc) * maxWc >= min_rows:
            bands = -(-maxHc // BR)
            PH = rows_of(BR)
            rows_unit = IMG * BR * maxWc
            FR = fr or PCONV_FR or (8 if (BN <= 32 and rows_unit >= 320) else 4)
            if BN == 128:
                FR = 4
            elif not (fr or PCONV_FR) and 32 <= Nd <= 64 and rows_unit <= 128:
                FR = 2                  # a 256-row pass over <= 128 rows wastes half the MFMAs (what the autotuner picks)
            if nw == 8 and FR not in (2, 4):
                FR = 2                  # eight-wave blocks: 256- or 512-row passes
            ktab = np.zeros((total_stages * 8, 2), dtype=np.int32)
            cdesc = np.zeros(len(classes), dtype=[("ph", "<i4"), ("pw", "<i4"), ("Hc", "<i4"), ("Wc", "<i4"),
                                                  ("nst", "<i4"), ("soff", "<i4"), ("invWc", "<f4"), ("pad", "<f4")])
            soff = 0
            for ci_, c in enumerate(classes):
                cdesc[ci_] = (c[0], c[1], c[2], c[3], nst[ci_], soff, 1.0 / c[3], 0.0)
                for st in range(nst[ci_]):
                    for u in range(8):
                        k = st * 64 + u * 8
                        tap, ch = divmod(k, Cs)
                        row = (soff + st) * 8 + u
                        if tap < c[4]:
                            oh, ow, wt = taps[c[5] + tap]
                            ktab[row] = (((oh - omin_h) * PW + (ow - omin_w)) * pitch + ch * 2, wt * Cs + ch)
                        else:
                            ktab[row] = (0, -1)
                soff += nst[ci_]
            if _pconv_lds(BN, total_stages, IMG * PH * PW * pitch, nw) <= 160 * 1024:
                plan = dict(classes=torch.from_numpy(cdesc.view(np.uint8).copy()).to(device),
                            ktab=torch.from_numpy(ktab).to(device), ncls=len(classes), nst=total_stages,
                            IMG=IMG, BR=BR, bands=bands, omin_h=omin_h, omin_w=omin_w, PH=PH, PW=PW, pitch=pitch,
                            BN=BN, FR=FR, budget=budget, NW=nw)
    _PLAN_CACHE[key] = plan
    return plan


def _pconv_candidates(g, mode, B, Cs, Nd, ss, device):
    """Distinct plans worth timing: two LDS budgets (2 or 1 blocks per CU) x image counts x FR."""
    out, seen = [], set()
    for budget in (40 * 1024, 53 * 1024, 80 * 1024, 160 * 1024):      # 4 / 3 / 2 / 1 blocks per CU
        base = _pconv_plan(g, mode, B, Cs, Nd, ss, device, budget=budget, min_rows=64)
        if base is None:
            continue
        imgs = {base["IMG"]}
        if base["bands"] == 1:
            imgs |= {max(1, base["IMG"] // 2), base["IMG"] * 2}
            # unit counts that fill whole rounds of the chip at one to four blocks per CU (2000 images in units of
            # five are 400 blocks: 1.56 rounds of 256 one-block CUs, the second round 56 % full; units of four are 1.95)
            imgs |= {-(-B // (256 * k)) for k in (1, 2, 3, 4)}
        for im in sorted(imgs):
            shapes = [(fr, 4) for fr in ((2, 4, 8) if 32 <= Nd <= 64 else (4, 8))]      # FR 2: 128-row passes for small units
            if PCONV_NW8 and 16 < Nd <= 64:
                shapes += [(2, 8), (4, 8)]      # eight waves on one patch: twice the waves per CU at the same LDS
            for fr, nw in shapes:
                pl = _pconv_plan(g, mode, B, Cs, Nd, ss, device, budget=budget, img=im, fr=fr, min_rows=64, nw=nw)
                if pl is None:
                    continue
                sig = (pl["IMG"], pl["BR"], pl["FR"], pl["budget"] if pl["bands"] > 1 else 0, pl["NW"])
                if sig not in seen:
                    seen.add(sig)
                    out.append(pl)
    return out


PCONV_NW8 = os.environ.get("DDL_PCONV_NW8", "1") == "1"
_CONV_CHOICE: Dict[Tuple, object] = {}
AUTOTUNE = os.environ.get("DDL_AUTOTUNE", "1") == "1"

# ---- plan choices are portable: export / import / persist --------------------------------------------------
# A tuned choice is recorded as plain data under a device-independent key string, so that (a) data-parallel ranks
# can all run rank 0's plans instead of eight independently (and noisily) tuned sets -- `sync_choices(dp)` between
# the warm-up step and graph capture -- and (b) a later process on the same machine skips tuning: the table is
# persisted to DDL_AUTOTUNE_CACHE (default ~/.cache/distributeddeeplearning_amd/autotune.json), keyed by the problem
# and stamped with the kernel library's identity so a rebuilt libddl_hip.so never reuses stale plans.
_CHOICE_SPEC: Dict[str, object] = {}        # key string -> ["igemm", tile] | ["pconv", budget, IMG, FR] | ["wgrad", index]
_CHOICE_DIRTY = False


def _lib_stamp() -> str:
    st = _LIB_PATH.stat()
    # PLAN_SCHEMA: bumped whenever the Python side changes what a recorded choice means (candidate order, plan fields)
    return f"{st.st_size}-{int(st.st_mtime)}-s{PLAN_SCHEMA}"


PLAN_SCHEMA = 3


def _cache_path() -> Optional[Path]:
    p = os.environ.get("DDL_AUTOTUNE_CACHE")
    if p == "":
        return None
    return Path(p) if p else Path.home() / ".cache" / "distributeddeeplearning_amd" / "autotune.json"


def _kstr(*parts) -> str:
    out = []
    for x in parts:
        out.append(",".join(str(int(v)) for v in vars(x).values()) if isinstance(x, ConvGeom) else str(x))
    return "|".join(out)


def _load_choice_cache():
    import json
    p = _cache_path()
    try:
        if p is not None and p.exists():
            blob = json.loads(p.read_text())
            if blob.get("lib") == _lib_stamp():
                _CHOICE_SPEC.update(blob.get("choices", {}))
    except Exception:       # noqa: BLE001 - a broken cache file only costs a re-tune
        pass


def save_choice_cache():
    """Persist the tuned plans (called by the benchmark / CLIs after warm-up; cheap, atomic)."""
    import json
    global _CHOICE_DIRTY
    p = _cache_path()
    if p is None or not _CHOICE_DIRTY:
        return
    try:
        p.parent.mkdir(parents=True, exist_ok=True)
        tmp = p.with_suffix(f".tmp{os.getpid()}")
        tmp.write_text(json.dumps({"lib": _lib_stamp(), "choices": _CHOICE_SPEC}))
        os.replace(tmp, p)
        _CHOICE_DIRTY = False
    except Exception:       # noqa: BLE001
        pass


def export_choices() -> Dict[str, object]:
    return dict(_CHOICE_SPEC)


def import_choices(table: Dict[str, object], overwrite: bool = True):
    """Adopt another process's tuned plans; already-resolved in-memory choices for those keys are dropped so the
    next launch of each problem rebuilds its plan from the imported record."""
    global _CHOICE_DIRTY
    for k, v in table.items():
        if overwrite or k not in _CHOICE_SPEC:
            if _CHOICE_SPEC.get(k) != v:
                _CHOICE_SPEC[k] = v
                _CHOICE_DIRTY = True
    if overwrite:
        _CONV_CHOICE.clear()


def sync_choices(dp, src: int = 0):
    """Every rank adopts rank `src`'s plan table (a collective over the default process group)."""
    import torch.distributed as dist
    if dp is None or getattr(dp, "world", 1) <= 1 or not (dist.is_available() and dist.is_initialized()):
        return
    box = [export_choices() if dp.rank == src else None]
    dist.broadcast_object_list(box, src=src)
    if dp.rank != src:
        import_choices(box[0], overwrite=True)


def _record_choice(kstr: str, spec):
    global _CHOICE_DIRTY
    if _CHOICE_SPEC.get(kstr) != spec:
        _CHOICE_SPEC[kstr] = spec
        _CHOICE_DIRTY = True


_load_choice_cache()


def _pconv_units(pl, B):
    return -(-B // pl["IMG"]) * pl["bands"]


PCONV_MULY = os.environ.get("DDL_PCONV_MULY", "1") == "1"
IGEMM_MULY = os.environ.get("DDL_IGEMM_MULY", "1") == "1"


def _run_pconv(pl, src, wgt, bias, dst, g, B, Hs, Ws, Cs, Hd, Wd, Nd, Nw, ss, sd, act, alpha, mul=None, stats=None,
               bn_infer=None, in_affine=None, stats_at=(0, 0)):
    """`stats`: fp32 tensor of 2 * Nd * units elements that receives per-block column sums / sums of squares
    of the output (layout [2][Nd][units]) for the BatchNorm that follows; `stats_at` = (row pitch, first column) when
    the partials of several launches (batch slices) share one [2][Nd][pitch] array.
    `bn_infer` = (gamma, beta, moving_mean, moving_var, eps): fold an inference-phase BatchNorm into the epilogue."""
    bg = bb = bm = bvv = None
    beps = 0.0
    if bn_infer is not None:
        gamma, beta, mm, mv, beps = bn_infer
        for t, n in ((gamma, "gamma"), (beta, "beta"), (mm, "moving_mean"), (mv, "moving_var")):
            _chk_f32(t, Nw, n)
        bg, bb, bm, bvv = gamma.data_ptr(), beta.data_ptr(), mm.data_ptr(), mv.data_ptr()
    # act'(y) of the layer below for linear / relu / leaky: its own epilogue instantiation, y prefetched ahead of the
    # transposes (fetched inside the store loop, and with a run-time activation switch per element, the fusion once
    # cost as much as the separate pass it replaced); other activations, or a statistics / BatchNorm epilogue: own pass
    my, ms = None, 0.0
    if (PCONV_MULY and mul is not None and stats is None and bn_infer is None and mul[1] in (None, "linear", "relu", "leaky")
            and ACT_CODE[act] in (0, 1, 6) and tuple(mul[0].shape) == tuple(dst.shape) and mul[0].is_contiguous()):
        my = mul[0].data_ptr()
        ms = 1.0 if mul[1] in (None, "linear") else (0.0 if mul[1] == "relu" else float(mul[2]))
    isc = ish = None
    igr, ict = 1, Cs
    if in_affine is not None:           # (scale, shift, (images per group,), c_true): [groups][Cs] fp32 rows
        sc_t, sh_t, (igr,), ict = in_affine
        ngr = -(-B // igr)
        _chk_f32(sc_t, ngr * Cs, "in_affine scale")
        _chk_f32(sh_t, ngr * Cs, "in_affine shift")
        isc, ish = sc_t.data_ptr(), sh_t.data_ptr()
    rc = _pconv(src.data_ptr(), wgt.data_ptr(), _p(bias), dst.data_ptr(), pl["classes"].data_ptr(),
                pl["ktab"].data_ptr(), pl["ncls"], pl["nst"], B, Hs, Ws, Cs, Hd, Wd, Nd, Nw, ss[0], ss[1],
                sd[0], sd[1], g.KH * g.KW, ACT_CODE[act], alpha, pl["IMG"], pl["BR"], pl["bands"],
                pl["omin_h"], pl["omin_w"], pl["PH"], pl["PW"], pl["pitch"], pl["BN"], pl["FR"], pl.get("NW", 4), _p(stats),
                bg, bb, bm,
                bvv, beps, isc, ish, igr, ict, my, ms, stats_at[0], stats_at[1], _stream())
    if rc != 0:
        raise ValueError(f"pconv rejected its plan (rc={rc}): {g} B={B} "
                         f"{ {k: v for k, v in pl.items() if k not in ('classes', 'ktab')} }")
    if my is None:
        _mul_inplace(dst, mul)


def _mul_slope(mul, dst):
    """(y pointer, slope) when `mul` = act'(y) of a linear / relu / leaky layer can ride in a conv epilogue, else None."""
    if (IGEMM_MULY and mul is not None and mul[1] in (None, "linear", "relu", "leaky")
            and tuple(mul[0].shape) == tuple(dst.shape) and mul[0].is_contiguous()):
        return mul[0].data_ptr(), (1.0 if mul[1] in (None, "linear") else (0.0 if mul[1] == "relu" else float(mul[2])))
    return None


_IGEMM_BM = {1: 256, 2: 64, 3: 256, 4: 128, 5: 256, 6: 128, 8: 64, 33: 128, 34: 256, 35: 128, 36: 256, 37: 256, 38: 128,
             39: 256, 40: 128, 41: 256}
_IGEMM_NO_STATS = ()


def _igemm_ksplit(g, mode, Cs, Nd, maxM, ncls, tile):
    """Split-K factor of the implicit-GEMM launch: a Dense / 1x1 fprop with few output tiles and a very long reduction
    (model0's 86528 -> 10 head at batch 512 is TWO 256-row blocks walking 2704 k-steps each) is spread over K."""
    if mode == "fprop" and ncls == 1 and _is_1x1(g) and (tile or 0) < 32:
        nsteps = (g.KH * g.KW * Cs + 63) // 64
        blocks = -(-maxM // 256) * -(-Nd // 128)
        if blocks < 128 and nsteps >= 32:
            return max(1, min(nsteps // 8, 512 // blocks))
    return 1


def _igemm_stats_cols(tile, g, mode, B, device):
    """(partial columns, images per column) of the implicit-GEMM kernels' statistics epilogue for this tile, or None
    when the tile has none (heuristic tile, classes of different sizes).  A column is one pixel tile of one class
    (pixel-tile-major = batch-major); `images per column` is what a consumer with per-group statistics checks the
    group size against -- B + 1 when pixel tiles do not line up with images at all."""
    if tile is None:
        return None
    t = tile - 16 if 16 < tile < 32 else tile
    if t not in _IGEMM_BM or t in _IGEMM_NO_STATS:
        return None
    cl_, _ = _class_taps(g, mode)
    hw = {c[2] * c[3] for c in cl_}
    if len(hw) != 1:
        return None
    hw, BM = hw.pop(), _IGEMM_BM[t]
    if _igemm_ksplit(g, mode, pad8(g.I), pad8(g.O), B * hw, len(cl_), tile) > 1:
        return None                     # the split-K path finishes in its own kernel: no statistics epilogue
    img = BM // hw if BM % hw == 0 else (1 if hw % BM == 0 else B + 1)
    return -(-(B * hw) // BM) * len(cl_), img


def _run_igemm(src, wgt, bias, dst, g, mode, B, Hs, Ws, Cs, Hd, Wd, Nd, Nw, ss, sd, act, alpha, tile=None, mul=None,
               stats=None):
    """`mul` = (y, act, alpha): result *= act'(y) -- in the kernel's epilogue for linear / relu / leaky, else as a pass.
    `stats` = (fp32 tensor, row pitch, first column): per-block column sums / sums of squares of the stored output,
    [2][Nd][pitch] (see _igemm_stats_cols)."""
    ct, tt, ncls, maxM, maxT, ut_all = _tables(g, mode, B, src.device)
    tile = IGEMM_TILE if tile is None else tile
    if tile >= 32 and not (ut_all and Cs % 32 == 0):
        raise ValueError(f"igemm tile {tile} (LDS-DMA staging) needs uniform-tap tables and Cs % 32 == 0: {g} Cs={Cs}")
    ksplit, slab = _igemm_ksplit(g, mode, Cs, Nd, maxM, ncls, tile), None
    if ksplit > 1:
        slab = torch.empty(ksplit * maxM * Nd, dtype=torch.float32, device=src.device)
    _ms = _mul_slope(mul, dst) if ACT_CODE[act] in (0, 1, 6) else None
    if stats is not None:
        if mul is not None or slab is not None:
            raise ValueError("igemm statistics epilogue: not with a fused multiply or split-K")
        _chk_f32(stats[0], 2 * Nd * stats[1], "stats partials")
    st = (None, 0, 0) if stats is None else (stats[0].data_ptr(), stats[1], stats[2])
    rc = _igemm(src.data_ptr(), wgt.data_ptr(), _p(bias), dst.data_ptr(), ct.data_ptr(), tt.data_ptr(), ncls,
                maxM, maxT, B, Hs, Ws, Cs, Hd, Wd, Nd, Nw, ss[0], ss[1], sd[0], sd[1], g.KH * g.KW,
                ACT_CODE[act], alpha, tile, ksplit if slab is not None else 1,
                _p(slab), *( (None, 0.0) if _ms is None else _ms ), *st, _stream())
    if rc == -5:                        # no fused multiply for this shape: plain launch, separate pass
        _ms = None
        rc = _igemm(src.data_ptr(), wgt.data_ptr(), _p(bias), dst.data_ptr(), ct.data_ptr(), tt.data_ptr(), ncls,
                    maxM, maxT, B, Hs, Ws, Cs, Hd, Wd, Nd, Nw, ss[0], ss[1], sd[0], sd[1], g.KH * g.KW,
                    ACT_CODE[act], alpha, tile, ksplit if slab is not None else 1,
                    _p(slab), None, 0.0, *st, _stream())
    if rc != 0:
        raise ValueError(f"igemm_conv rejected the problem (rc={rc}): {g} mode={mode} B={B}")
    if _ms is None:
        _mul_inplace(dst, mul)


AUTOTUNE_COLD = os.environ.get("DDL_AUTOTUNE_COLD", "0") == "1"
_FLUSH = {}


def _flush_caches(device):
    """Overwrite a buffer larger than L2 + Infinity Cache so the next launch finds its operands in HBM."""
    buf = _FLUSH.get(device)
    if buf is None:
        buf = _FLUSH[device] = torch.empty(384 << 20, dtype=torch.uint8, device=device)
    buf.zero_()


def _time_us(fn, reps=4, inner=4):
    """Best-of-`reps` device time of one call; `inner` back-to-back launches per measurement keep the
    launch latency of a ~20 us kernel out of the comparison.  DDL_AUTOTUNE_COLD=1 times single launches
    behind a cache flush instead (operands in HBM, as inside a training step, not hot from the last try)."""
    fn()
    torch.cuda.synchronize()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    best = float("inf")
    if AUTOTUNE_COLD:
        dev = torch.cuda.current_device()
        ts = []
        for _ in range(reps + 1):
            _flush_caches(dev)
            e0.record()
            fn()
            e1.record()
            e1.synchronize()
            ts.append(e0.elapsed_time(e1) * 1e3)
        ts.sort()
        return ts[len(ts) // 2]
    for _ in range(reps):
        e0.record()
        for _ in range(inner):
            fn()
        e1.record()
        e1.synchronize()
        best = min(best, e0.elapsed_time(e1) * 1e3 / inner)
    return best


PCONV_STATS = os.environ.get("DDL_PCONV_STATS", "1") == "1"


IGEMM_DMA = os.environ.get("DDL_IGEMM_DMA", "1") == "1"
IGEMM_DMA_MIN_ROWS = int(os.environ.get("DDL_IGEMM_DMA_MIN_ROWS", "65536"))


def _dma_tiles(g, mode, B, Cs, Nd, device):
    """LDS-DMA staged tile candidates (igemm_conv.hip, ids 32+): uniform-tap tables, whole 32-channel K stages, and a
    problem large enough (rows x classes) that the staging path, not launch latency, is what bounds it."""
    if not IGEMM_DMA or Cs % 32:
        return []
    _, _, ncls, maxM, _, ut_all = _tables(g, mode, B, device)
    if not ut_all or maxM * ncls < IGEMM_DMA_MIN_ROWS:
        return []
    if Nd <= 32:
        return [39]
    if Nd <= 64:
        return [35, 36, 37]
    if Nd <= 128:
        return [33, 34, 35, 40]
    return [33, 34, 38, 40, 41]


def _conv_choice(src, wgt, bias, dst, g, mode, B, Hs, Ws, Cs, Hd, Wd, Nd, Nw, ss, sd, act, alpha, mul=None,
                 want_stats=False):
    """("pconv", plan) | ("igemm", tile) for one class-grid convolution.  The first (non-captured) call of each
    problem times the candidates on the real operands and caches the winner -- these shapes are static for a whole
    training run."""
    tail = (B, Hs, Ws, Cs, Hd, Wd, Nd, Nw, ss, sd, act, alpha)
    slow = ACT_CODE[act] not in (0, 1, 6)
    key = (g, mode, B, Cs, Nd, slow, str(src.device))
    kstr = _kstr("conv", g, mode, B, Cs, Nd, int(slow))
    choice = _CONV_CHOICE.get(key)
    if choice is None and kstr in _CHOICE_SPEC:          # imported from rank 0 / the on-disk cache
        spec = _CHOICE_SPEC[kstr]
        if spec[0] == "igemm":
            choice = ("igemm", spec[1])
        else:
            pl = _pconv_plan(g, mode, B, Cs, Nd, ss, src.device, budget=spec[1], img=spec[2], fr=spec[3], min_rows=64,
                             nw=spec[4] if len(spec) > 4 else 4)
            choice = ("pconv", pl) if pl is not None else None
        if choice is not None:
            _CONV_CHOICE[key] = choice
    if choice is None:
        if AUTOTUNE and not torch.cuda.is_current_stream_capturing():
            tiles = [1] if Nd <= 16 else ([3] if Nd <= 32 else ([4, 5, 2] if Nd <= 64 else [6, 8]))
            if 64 < Nd <= 256:
                tiles += [2, 4]          # 64-wide N tiles over a z-grid: more, smaller blocks for short pixel dims
            tiles = tiles + [t + 16 for t in tiles]          # deep (64-wide, 3 stages in flight) and shallow variants
            tiles += _dma_tiles(g, mode, B, Cs, Nd, src.device)
            cands = [("igemm", t) for t in tiles] + \
                    [("pconv", pl) for pl in _pconv_candidates(g, mode, B, Cs, Nd, ss, src.device)]
            timed = []
            for kind, pl in cands:
                fn = (lambda pl=pl: _run_igemm(src, wgt, bias, dst, g, mode, *tail, tile=pl, mul=mul)) \
                    if kind == "igemm" else (lambda pl=pl: _run_pconv(pl, src, wgt, bias, dst, g, *tail, mul=mul))
                t_us = _time_us(fn)
                if (kind == "igemm" and want_stats and PCONV_STATS and mul is None
                        and _igemm_stats_cols(pl, g, mode, B, src.device) is None):
                    # a BatchNorm behind this layer and a tile without the statistics epilogue: it leaves them to a
                    # pass over the output (launch + streaming read)
                    t_us += 4.0 + B * Hd * Wd * Nd * 2 / 3.0e6
                timed.append((t_us, kind, pl))
            timed.sort(key=lambda t: t[0])
            choice = (timed[0][1], timed[0][2])
            _record_choice(kstr, ["igemm", choice[1]] if choice[0] == "igemm" else
                           ["pconv", choice[1]["budget"], choice[1]["IMG"], choice[1]["FR"], choice[1]["NW"]])
            if os.environ.get("DDL_AUTOTUNE_VERBOSE"):
                desc = [(round(t, 1), k, p if k == "igemm" else (p["IMG"], p["BR"], p["FR"], p["budget"] // 1024, p["NW"]))
                        for t, k, p in timed]
                print(f"[autotune] {mode} B={B} {g.H}x{g.W}x{g.I}->{g.OH}x{g.OW}x{g.O} k{g.KH} s{g.sh}: {desc}",
                      flush=True)
        else:
            pl = _pconv_plan(g, mode, B, Cs, Nd, ss, src.device)
            choice = ("pconv", pl) if pl is not None else ("igemm", None)
        _CONV_CHOICE[key] = choice
    return choice


def _choice_stats_cols(choice, g, mode, B, device):
    """(partial columns, images per column) of the chosen kernel's statistics epilogue, or None."""
    if choice[0] == "pconv":
        return _pconv_units(choice[1], B), choice[1]["IMG"]
    return _igemm_stats_cols(choice[1], g, mode, B, device)


def _igemm_call(src, wgt, bias, dst, g, mode, B, Hs, Ws, Cs, Hd, Wd, Nd, Nw, ss, sd, act, alpha, mul=None,
                stats_out=None, bn_infer=None, in_affine=None, aff_sink=None, stats_into=None):
    """Dispatch one class-grid convolution: the patch-resident kernel with a tuned plan, or the global-gather kernel
    (_conv_choice).  `stats_out`: dict that receives the BatchNorm partials the kernel's epilogue leaves ("part", "nb",
    "img"); `stats_into` = (tensor, row pitch, first column): write them there instead (one slice of a batch-split
    layer: the caller made sure this slice's kernel has the epilogue)."""
    def materialise():                  # the global-gather kernel has no affine on load: apply the BatchNorm first
        sc_t, sh_t, (igr,), ict = in_affine
        m = bn_apply(src, sc_t, sh_t, None, 0.3, ict, B // igr)
        if aff_sink is not None:        # the caller keeps it (weight gradient) instead of rebuilding it
            aff_sink["x"] = m
        return m
    args = (src, wgt, bias, dst, g)
    tail = (B, Hs, Ws, Cs, Hd, Wd, Nd, Nw, ss, sd, act, alpha)
    if CONV_IMPL != "pconv":
        if in_affine is not None:
            src = materialise()
        _run_igemm(src, wgt, bias, dst, g, mode, *tail, mul=mul)
        _done()
        return
    want_stats = (stats_out is not None or stats_into is not None) and PCONV_STATS and mul is None
    choice = _conv_choice(*args, mode, *tail, mul=mul, want_stats=want_stats)
    stats = stats_into
    if choice[0] == "pconv":
        if bn_infer is not None and (stats_out is None or mul is not None or not PCONV_STATS):
            bn_infer = None
        if bn_infer is not None:
            stats_out["affine"] = True                   # the caller skips its BatchNorm pass
            stats = None
    if stats is None and want_stats and stats_out is not None and not stats_out.get("affine"):
        cols = _choice_stats_cols(choice, g, mode, B, src.device)
        if cols is not None:
            part = torch.empty(2 * Nd * cols[0], dtype=torch.float32, device=src.device)
            stats = (part, cols[0], 0)
            stats_out["part"], stats_out["nb"], stats_out["img"] = part, cols[0], cols[1]
    if choice[0] == "pconv":
        _run_pconv(choice[1], *args, *tail, mul=mul, stats=None if stats is None else stats[0], bn_infer=bn_infer,
                   in_affine=in_affine, stats_at=(0, 0) if stats is None else (stats[1], stats[2]))
    else:
        if in_affine is not None:
            src = materialise()
        _run_igemm(src, wgt, bias, dst, g, mode, *tail, tile=choice[1], mul=mul, stats=stats)
    _done()


def _chk_w(w, shape, name):
    if not (w.is_cuda and w.dtype == torch.bfloat16 and w.is_contiguous()):
        raise ValueError(f"{name}: weights must be contiguous bf16 cuda")
    if tuple(w.shape) != tuple(shape):
        raise ValueError(f"{name}: weight shape {tuple(w.shape)} != expected {tuple(shape)}")


GEMM_SK = os.environ.get("DDL_GEMM_SK", "1") == "1"


SK_AFFINE = os.environ.get("DDL_SK_AFFINE", "1") == "1"     # BatchNorm in front of a 1x1 layer applied on load by gemm_sk
# BatchNorm statistics from gemm_sk's store loop for problems with at least this many rows (below, the separate
# column reduction over a cache-sized output is as cheap as the epilogue; model0's 57x57x128 layer at batch 512 is
# 1.66 M rows and 426 MB: the reduction pass alone was 104 us)
SK_STATS_MIN_ROWS = int(os.environ.get("DDL_SK_STATS_MIN_ROWS", "262144"))


def _gemm_sk_call(x, w, bias, y, M, K, Nd, Nw, act, alpha, in_affine=None, stats_out=None):
    """One launch of the skinny-K GEMM (csrc/hip/gemm_sk.hip).  `in_affine` = (scale, shift, c_true): fp32 rows applied
    to x as it is loaded; `stats_out`: receives the BatchNorm partials of y ("part", "nb", "img" = 2^30: pixel tiles
    straddle images, one statistics group only).  Returns False when the problem is outside the kernel's range
    (nothing launched)."""
    isc = ish = part = None
    ict = cols = 0
    if in_affine is not None:
        _chk_f32(in_affine[0], K, "in_affine scale")
        _chk_f32(in_affine[1], K, "in_affine shift")
        isc, ish, ict = in_affine[0].data_ptr(), in_affine[1].data_ptr(), int(in_affine[2])
    if stats_out is not None and PCONV_STATS and M >= SK_STATS_MIN_ROWS and int(stats_out.get("groups", 1)) == 1:
        cols = _gemm_sk_cols(M, K, Nd)
        if cols > 0:
            part = torch.empty(2 * Nd * cols, dtype=torch.float32, device=x.device)
    rc = _gemm_sk(x.data_ptr(), w.data_ptr(), _p(bias), y.data_ptr(), M, K, Nd, Nw, ACT_CODE[act], alpha, isc, ish, ict,
                  _p(part), cols, 0, _stream())
    if rc < 0:
        raise ValueError(f"gemm_sk rejected the problem (rc={rc}): M={M} K={K} N={Nd}")
    if rc == 0 and part is not None:
        stats_out["part"], stats_out["nb"], stats_out["img"] = part, cols, 1 << 30
    return rc == 0


def _is_1x1(g: ConvGeom) -> bool:
    """A 1x1 / stride-1 / unpadded correlation: a row-major GEMM over pixels (also Dense)."""
    return (g.KH == g.KW == 1 and g.sh == g.sw == 1 and g.pt == g.pl == 0 and g.OH == g.H and g.OW == g.W
            and not g.depthwise)


# The conv kernels address their operands through 32-bit buffer descriptors / element offsets: one launch handles
# tensors below 2^31 elements.  Larger batches ("per-GPU batch sized to 288 GB HBM") are split
# along the batch dimension into several launches on contiguous slices -- fprop / dgrad write their slice of the
# output, wgrad sums the per-slice gradients in fp32.
ELEM_LIMIT = int(os.environ.get("DDL_CONV_ELEM_LIMIT", str((1 << 31) - 1)))


def _batch_ranges(B: int, per_image: int, align: int = 0):
    """[(b0, b1)] so that no slice has more than ELEM_LIMIT elements in its largest operand (None: no split).
    `align` > 0: no slice crosses a multiple of `align` images (batch groups with their own BatchNorm statistics)."""
    if B * per_image <= ELEM_LIMIT:
        return None
    step = max(1, ELEM_LIMIT // per_image)
    if step >= 8:
        step -= step % 8
    segs = [(a, min(a + align, B)) for a in range(0, B, align)] if align > 0 else [(0, B)]
    out = []
    for a0, a1 in segs:                 # equal slices (one tuned plan serves them all), not full ones + a sliver
        n = -(-(a1 - a0) // step)
        sz = -(-(a1 - a0) // n)
        if sz % 8 and sz + 8 - sz % 8 <= step:
            sz += 8 - sz % 8
        out += [(b, min(b + sz, a1)) for b in range(a0, a1, sz)]
    return out


GROUP_SPLIT = os.environ.get("DDL_CONV_GROUP_SPLIT", "1") == "1"


def _group_split(kind, x, w, bias, y, g, act, alpha, mul, stats_out, groups):
    """Ranges that run ONE launch per batch group -- when the BatchNorm behind the layer keeps statistics per group and
    the kernel chosen for the whole batch is an implicit-GEMM tile whose pixel tiles straddle images (its partial
    columns then cannot be split by group, and the consumer would fall back to a pass over the output).  None: the
    single launch is fine."""
    if not (GROUP_SPLIT and CONV_IMPL == "pconv" and PCONV_STATS and stats_out is not None and mul is None
            and groups > 1 and x.shape[0] % groups == 0):
        return None
    B, Ip, Op = x.shape[0], pad8(g.I), pad8(g.O)
    if kind == "fprop":
        ga = (x, w, bias, y, g, "fprop", B, g.H, g.W, Ip, g.OH, g.OW, Op, min(w.shape[0], g.O), (g.sh, g.sw), (1, 1),
              act, alpha)
    else:
        ga = (x, w, bias, y, g, "dgrad", B, g.OH, g.OW, Op, g.H, g.W, Ip, min(w.shape[0], g.I), (1, 1), (g.sh, g.sw),
              act, alpha)
    ch = _conv_choice(*ga, mul=None, want_stats=True)
    if ch[0] != "igemm":
        return None
    cols = _igemm_stats_cols(ch[1], g, ga[5], B, x.device)
    if cols is None or B % (cols[1] * groups) == 0:
        return None
    step = B // groups
    return [(b, b + step) for b in range(0, B, step)]


def _conv_slices(kind, x, w, bias, y, g, act, alpha, mul, stats_out, ranges, groups, in_affine=None, aff_sink=None):
    """A convolution whose operands exceed the 32-bit element offsets of one launch, as batch slices -- with the
    fusions of the unsliced path kept: every slice's kernel is chosen first (tuning it if this is its first call), then
      * the BatchNorm statistics epilogue runs in every slice, all writing their partial columns side by side into
        one [2][Nd][columns] array (when every chosen kernel has the epilogue), and
      * a BatchNorm applied on load stays on load (when every chosen kernel is the patch-resident one), each slice
        with the (scale, shift) row of the batch group it lies in; otherwise the operand is materialised once.
    `ranges` never cross a batch-group boundary (`groups` equal parts).  `in_affine` = (scale, shift, groups, c_true)
    as given to conv_dgrad."""
    B = x.shape[0]
    Ip, Op = pad8(g.I), pad8(g.O)

    def grid_args(b0, b1):
        xs, ys = x[b0:b1], y[b0:b1]
        if kind == "fprop":
            return (xs, w, bias, ys, g, "fprop", b1 - b0, g.H, g.W, Ip, g.OH, g.OW, Op, min(w.shape[0], g.O),
                    (g.sh, g.sw), (1, 1), act, alpha)
        return (xs, w, bias, ys, g, "dgrad", b1 - b0, g.OH, g.OW, Op, g.H, g.W, Ip, min(w.shape[0], g.I),
                (1, 1), (g.sh, g.sw), act, alpha)

    want_stats = stats_out is not None and PCONV_STATS and mul is None and CONV_IMPL == "pconv"
    choices, cols = [], []
    if CONV_IMPL == "pconv":
        for b0, b1 in ranges:
            ga = grid_args(b0, b1)
            ch = _conv_choice(*ga, mul=_mul_slice(mul, b0, b1), want_stats=want_stats)
            choices.append(ch)
            cols.append(_choice_stats_cols(ch, g, ga[5], b1 - b0, x.device))
    if in_affine is not None:
        sc_t, sh_t, agr, ict = in_affine
        on_load = bool(choices) and all(c[0] == "pconv" for c in choices) and groups % agr == 0
        if not on_load:
            x = bn_apply(x, sc_t, sh_t, None, 0.3, ict, agr)
            if aff_sink is not None:
                aff_sink["x"] = x
            in_affine = None
    part, nb = None, 0
    if want_stats and all(c is not None for c in cols):
        nb = sum(c[0] for c in cols)
        Nd = Op if kind == "fprop" else Ip
        part = torch.empty(2 * Nd * nb, dtype=torch.float32, device=x.device)
        # every slice, and so every partial column, lies inside one of the `groups` aligned batch parts: that is all
        # a consumer with per-group statistics may assume ("img" = images per indivisible run of columns)
        stats_out["part"], stats_out["nb"], stats_out["img"] = part, nb, B // max(groups, 1)
    off = 0
    for k, (b0, b1) in enumerate(ranges):
        aff = None
        if in_affine is not None:
            z = b0 // (B // agr)
            aff = (sc_t.view(agr, -1)[z], sh_t.view(agr, -1)[z], (b1 - b0,), ict)
        _igemm_call(*grid_args(b0, b1), _mul_slice(mul, b0, b1), None, None, aff, None,
                    None if part is None else (part, nb, off))
        if part is not None:
            off += cols[k][0]
    return y




def _mul_slice(mul, b0, b1):
    return None if mul is None else (mul[0][b0:b1], mul[1], mul[2])


def conv_fprop(x, wA, bias, g: ConvGeom, act=None, alpha=0.3, mul=None, stats_out=None, bn_infer=None, out=None,
               in_affine=None, aff_sink=None):
    """`mul` = (y, act, alpha): multiply the (bf16) result by act'(y) -- the activation backward of the layer
    below, fused into the epilogue when this runs as a transposed conv's input gradient.
    `out`: write into this contiguous [B, OH, OW, Op] tensor (a batch slice of a larger one).
    `in_affine` = (scale, shift, groups, c_true): x is read as bf16(x * scale + shift) -- a BatchNorm in front of
    the layer applied on load by the depthwise stencil (one statistics group; everything else gets it materialised)."""
    _chk_act(x, "x")
    if in_affine is not None and not (g.depthwise and in_affine[2] == 1):
        x = bn_apply(x, in_affine[0], in_affine[1], None, 0.3, in_affine[3], in_affine[2])
        in_affine = None
        if aff_sink is not None:        # materialised: the caller keeps it for the weight gradient
            aff_sink["x"] = x
    B = x.shape[0]
    Ip, Op = pad8(g.I), pad8(g.O)
    if tuple(x.shape[1:]) != (g.H, g.W, Ip):
        raise ValueError(f"conv_fprop: x {tuple(x.shape)} does not match geometry {g} (padded I={Ip})")
    if bias is not None:
        _chk_f32(bias, g.O, "bias")
    if out is not None:
        _chk_act(out, "out")
        if tuple(out.shape) != (B, g.OH, g.OW, Op):
            raise ValueError(f"conv_fprop: out {tuple(out.shape)} != {(B, g.OH, g.OW, Op)}")
    y = out if out is not None else torch.empty(B, g.OH, g.OW, Op, dtype=torch.bfloat16, device=x.device)
    sgroups = int(stats_out.get("groups", 1)) if stats_out is not None else 1
    ranges = _batch_ranges(B, max(g.H * g.W * Ip, g.OH * g.OW * Op), B // sgroups if sgroups > 1 and B % sgroups == 0 else 0)
    if ranges is not None:
        if g.depthwise or (_is_1x1(g) and GEMM_SK) or wA.dim() != 4:
            for b0, b1 in ranges:       # no BN statistics / folded BN across slices: the caller runs its own pass
                conv_fprop(x[b0:b1], wA, bias, g, act, alpha, _mul_slice(mul, b0, b1), None, None, y[b0:b1], in_affine)
            return y
        if wA.shape[1:] != (g.KH, g.KW, Ip) or wA.shape[0] > Op:
            raise ValueError(f"conv_fprop: weight {tuple(wA.shape)} vs geometry {g}")
        _chk_w(wA, wA.shape, "kernel")
        return _conv_slices("fprop", x, wA, bias, y, g, act, alpha, mul, stats_out, ranges, sgroups)
    if not (g.depthwise or (_is_1x1(g) and GEMM_SK)) and wA.dim() == 4 and wA.shape[1:] == (g.KH, g.KW, Ip) \
            and wA.shape[0] <= Op and in_affine is None and bn_infer is None:
        gr = _group_split("fprop", x, wA, bias, y, g, act, alpha, mul, stats_out, sgroups)
        if gr is not None:
            _chk_w(wA, wA.shape, "kernel")
            return _conv_slices("fprop", x, wA, bias, y, g, act, alpha, mul, stats_out, gr, sgroups)
    if g.depthwise:
        _chk_w(wA, (g.KH, g.KW, Ip), "depthwise kernel")
        isc = ish = None
        ict = 0
        if in_affine is not None:
            _chk_f32(in_affine[0], Ip, "in_affine scale")
            _chk_f32(in_affine[1], Ip, "in_affine shift")
            isc, ish, ict = in_affine[0].data_ptr(), in_affine[1].data_ptr(), int(in_affine[3])
        if (stats_out is not None and PCONV_STATS and DW_STATS and mul is None and bn_infer is None and sgroups == 1
                and g.KH == g.KW and g.dh == g.dw == 1 and g.pt == g.pl == 0):
            # the row-ring kernel also leaves the statistics of the BatchNorm behind the layer (one column per image)
            part = torch.empty(2 * Ip * B, dtype=torch.float32, device=x.device)
            if _dw_fwd_stats(x.data_ptr(), wA.data_ptr(), _p(bias), y.data_ptr(), part.data_ptr(), B, g.H, g.W, Ip,
                             g.OH, g.OW, g.KH, g.sh, g.sw, g.O, ACT_CODE[act], alpha, isc, ish, ict, _stream()) == 0:
                stats_out["part"], stats_out["nb"], stats_out["img"] = part, B, 1
                _done()
                return y
        rc = _depthwise(0, x.data_ptr(), wA.data_ptr(), _p(bias), y.data_ptr(), None, B, g.H, g.W, Ip, g.OH, g.OW,
                        g.KH, g.KW, g.sh, g.sw, g.dh, g.dw, g.pt, g.pl, g.O, ACT_CODE[act], alpha, isc, ish, ict,
                        _stream())
        if rc == -5:                    # outside the fast stencil's range: materialise the BatchNorm output after all
            xm = bn_apply(x, in_affine[0], in_affine[1], None, 0.3, in_affine[3], 1)
            if aff_sink is not None:
                aff_sink["x"] = xm
            rc = _depthwise(0, xm.data_ptr(), wA.data_ptr(), _p(bias), y.data_ptr(), None, B, g.H, g.W, Ip, g.OH,
                            g.OW, g.KH, g.KW, g.sh, g.sw, g.dh, g.dw, g.pt, g.pl, g.O, ACT_CODE[act], alpha, None,
                            None, 0, _stream())
        if rc:
            raise ValueError("depthwise fprop rejected")
        _mul_inplace(y, mul)
        _done()
        return y
    if wA.dim() != 4 or wA.shape[1:] != (g.KH, g.KW, Ip) or wA.shape[0] > Op:
        raise ValueError(f"conv_fprop: weight {tuple(wA.shape)} vs geometry {g}")
    _chk_w(wA, wA.shape, "kernel")
    if _is_1x1(g) and GEMM_SK:
        if _gemm_sk_call(x, wA, bias, y, B * g.H * g.W, Ip, Op, min(wA.shape[0], g.O), act, alpha,
                         stats_out=stats_out if (mul is None and bn_infer is None) else None):
            _mul_inplace(y, mul)
            _done()
            return y
    _igemm_call(x, wA, bias, y, g, "fprop", B, g.H, g.W, Ip, g.OH, g.OW, Op, min(wA.shape[0], g.O),
                (g.sh, g.sw), (1, 1), act, alpha, mul, stats_out, bn_infer)
    return y


def conv_dgrad(dy, wB, g: ConvGeom, bias=None, act=None, alpha=0.3, mul=None, stats_out=None, bn_infer=None,
               out=None, in_affine=None, aff_sink=None):
    """`in_affine` = (scale, shift, groups, c_true): dy is read as bf16(dy * scale[grp] + shift[grp]) -- a BatchNorm
    in front of a transposed convolution (which runs as this dgrad) applied on load by the patch-resident kernel
    ([groups][Op] fp32 rows, the batch being `groups` equal parts; other kernels get it materialised first)."""
    _chk_act(dy, "dy")
    B = dy.shape[0]
    Ip, Op = pad8(g.I), pad8(g.O)
    if tuple(dy.shape[1:]) != (g.OH, g.OW, Op):
        raise ValueError(f"conv_dgrad: dy {tuple(dy.shape)} does not match geometry {g} (padded O={Op})")
    if bias is not None:
        _chk_f32(bias, g.I, "bias")
    if out is not None:
        _chk_act(out, "out")
        if tuple(out.shape) != (B, g.H, g.W, Ip):
            raise ValueError(f"conv_dgrad: out {tuple(out.shape)} != {(B, g.H, g.W, Ip)}")
    dx = out if out is not None else torch.empty(B, g.H, g.W, Ip, dtype=torch.bfloat16, device=dy.device)
    sgroups = int(stats_out.get("groups", 1)) if stats_out is not None else 1
    agroups = in_affine[2] if in_affine is not None else 1
    if B % agroups:
        raise ValueError(f"conv_dgrad: batch {B} does not split into {agroups} groups")
    # slices (operands beyond one launch's 32-bit offsets) never cross a batch-group boundary
    ngr = max(sgroups, agroups) if (B % sgroups == 0 and max(sgroups, agroups) % min(sgroups, agroups) == 0) else agroups
    ranges = _batch_ranges(B, max(g.H * g.W * Ip, g.OH * g.OW * Op), B // ngr if ngr > 1 else 0)
    plain = g.depthwise or (_is_1x1(g) and GEMM_SK)
    sk_aff = None
    if in_affine is not None:
        sc_t, sh_t, groups, ictrue = in_affine
        if (plain and not g.depthwise and SK_AFFINE and groups == 1 and ranges is None and wB.dim() == 4
                and _gemm_sk_cols(B * g.H * g.W, Op, Ip) > 0):
            sk_aff, in_affine = (sc_t.reshape(-1), sh_t.reshape(-1), ictrue), None      # gemm_sk applies it on load
        elif plain:
            dy = bn_apply(dy, sc_t, sh_t, None, 0.3, ictrue, groups)        # no on-load path there
            in_affine = None
            if aff_sink is not None:    # `aff_sink["x"]`: the materialised operand, kept by the caller
                aff_sink["x"] = dy
        elif ranges is None:
            in_affine = (sc_t, sh_t, (B // groups,), ictrue)
    if ranges is not None:
        if plain or wB.dim() != 4:
            for b0, b1 in ranges:
                conv_dgrad(dy[b0:b1], wB, g, bias, act, alpha, _mul_slice(mul, b0, b1), None, None, dx[b0:b1])
            return dx
        if wB.shape[1:] != (g.KH, g.KW, Op) or wB.shape[0] > Ip:
            raise ValueError(f"conv_dgrad: weight {tuple(wB.shape)} vs geometry {g}")
        _chk_w(wB, wB.shape, "kernel")
        return _conv_slices("dgrad", dy, wB, bias, dx, g, act, alpha, mul, stats_out, ranges, ngr, in_affine, aff_sink)
    if not plain and wB.dim() == 4 and wB.shape[1:] == (g.KH, g.KW, Op) and wB.shape[0] <= Ip and bn_infer is None \
            and ngr == sgroups:
        gr = _group_split("dgrad", dy, wB, bias, dx, g, act, alpha, mul, stats_out, sgroups)
        if gr is not None:
            _chk_w(wB, wB.shape, "kernel")
            aff0 = None if in_affine is None else (in_affine[0], in_affine[1], B // in_affine[2][0], in_affine[3])
            return _conv_slices("dgrad", dy, wB, bias, dx, g, act, alpha, mul, stats_out, gr, ngr, aff0, aff_sink)
    if g.depthwise:
        _chk_w(wB, (g.KH, g.KW, Ip), "depthwise kernel")
        if bias is not None or act not in (None, "linear"):
            raise ValueError("depthwise dgrad has no fused epilogue")
        rc = _depthwise(1, dy.data_ptr(), wB.data_ptr(), None, dx.data_ptr(), None, B, g.H, g.W, Ip, g.OH, g.OW,
                        g.KH, g.KW, g.sh, g.sw, g.dh, g.dw, g.pt, g.pl, g.O, 0, 0.0, None, None, 0, _stream())
        if rc:
            raise ValueError("depthwise dgrad rejected")
        _mul_inplace(dx, mul)
        _done()
        return dx
    if wB.dim() != 4 or wB.shape[1:] != (g.KH, g.KW, Op) or wB.shape[0] > Ip:
        raise ValueError(f"conv_dgrad: weight {tuple(wB.shape)} vs geometry {g}")
    _chk_w(wB, wB.shape, "kernel")
    if _is_1x1(g) and GEMM_SK:
        if _gemm_sk_call(dy, wB, bias, dx, B * g.H * g.W, Op, Ip, min(wB.shape[0], g.I), act, alpha, in_affine=sk_aff,
                         stats_out=stats_out if (mul is None and bn_infer is None) else None):
            _mul_inplace(dx, mul)
            _done()
            return dx
        if sk_aff is not None:          # (not reached: the range was checked above) materialise for the generic kernels
            dy = bn_apply(dy, sk_aff[0], sk_aff[1], None, 0.3, sk_aff[2], 1)
            if aff_sink is not None:
                aff_sink["x"] = dy
    _igemm_call(dy, wB, bias, dx, g, "dgrad", B, g.OH, g.OW, Op, g.H, g.W, Ip, min(wB.shape[0], g.I),
                (1, 1), (g.sh, g.sw), act, alpha, mul, stats_out, bn_infer, in_affine, aff_sink)
    return dx


WGRAD_IMPL = os.environ.get("DDL_WGRAD", "wgrad2")          # wgrad2 (patch-resident, persistent) | wgrad
_W2_COMBOS = {(64, 64): (2, 3), (64, 32): (4, 7), (32, 64): (4, 7), (32, 32): (4, 7), (64, 16): (7,), (16, 64): (7,),
              (32, 16): (7,), (16, 32): (7,), (16, 16): (7,)}
# eight-wave blocks (one 512-thread block per CU sharing a staged unit): tile -> taps per wave
_W2_COMBOS8 = {(64, 64): 2, (64, 32): 4, (32, 64): 4, (32, 32): 4}
W2_NW8 = os.environ.get("DDL_W2_NW8", "1") == "1"
W2_DMA = os.environ.get("DDL_W2_DMA", "1") == "1"
_W2_DMA4 = {(64, 32): (7, 4), (32, 32): (7, 4)}           # four-wave DMA instantiations: tile -> taps per wave
_W2_PLANS: Dict[Tuple, Optional[dict]] = {}


def _tr_pitch(nbytes: int) -> int:
    """Pixel pitch for ds_read_b64_tr_b16 operands: an odd multiple of 32 B >= nbytes, so the 8 pixel
    rows a half-wave reads fall in 8 distinct 32-byte bank groups."""
    p = (nbytes + 31) // 32
    return (p if p % 2 else p + 1) * 32


W2_XPITCH_SKEW = os.environ.get("DDL_W2_XPITCH_SKEW", "1") == "1"
W2_FRAG_SLAB = os.environ.get("DDL_W2_FRAG_SLAB", "1") == "1"


def _tr_pitch_x(nbytes: int, sw: int) -> int:
    """Pixel pitch of wgrad2's X patch.  Consecutive output pixels read patch pixels `sw` apart, so it is
    sw * pitch that has to be an odd multiple of 32 B: for stride 2 an odd multiple of 16 B (16 B keeps the
    staging stores aligned).  With the plain pitch every stride-2 layer read X through 2-way bank conflicts
    (44 % of the kernel's LDS cycles, profiles/r1_dcgan28_pmc_counters.md)."""
    if sw == 2 and W2_XPITCH_SKEW:
        p = (nbytes + 15) // 16
        return (p if p % 2 else p + 1) * 16
    return _tr_pitch(nbytes)


def _wgrad2_one_plan(g, B, Cx, Ny, n_lim, c_lim, tn, tc, TPW, budget_kb=None, NW=4, dma=False):
    """One wgrad2 launch plan for an output tile (tn x tc), TPW taps per wave and an LDS budget (which
    sets how many images / rows a unit holds and with it how many blocks share a CU).  `dma`: LDS-DMA staging into two
    buffers (the budget covers both), the next unit's transfer under the current unit's MFMA phase."""
    T = g.KH * g.KW
    ngroups = -(-T // (NW * TPW))
    tiles = -(-n_lim // tn) * -(-c_lim // tc)
    one_block = NW == 8 or TPW * (tn // 16) * (tc // 16) * 4 > 160
    if budget_kb is None:
        budget_kb = 150 if one_block else 76
    budget = budget_kb * 1024
    # only the output tile's channels are staged: pitches follow the tile, not the tensor
    xp, yp = _tr_pitch_x(min(Cx, tc) * 2, g.sw), _tr_pitch(min(Ny, tn) * 2)
    PW = (g.OW - 1) * g.sw + (g.KW - 1) * g.dw + 1
    if dma:
        lds = lambda img, br: _wgrad2_lds_dma(img, br, g.OW, (br - 1) * g.sh + (g.KH - 1) * g.dh + 1, PW, xp, yp, T, NW)
    else:
        lds = lambda img, br: _wgrad2_lds(img, br, g.OW, Ny, (br - 1) * g.sh + (g.KH - 1) * g.dh + 1, PW, xp, yp, T)
    IMG, BR = 0, g.OH
    if lds(1, g.OH) <= budget:
        IMG = 1
        while IMG < B and IMG * g.OH * g.OW < 512 and lds(IMG + 1, g.OH) <= budget:
            IMG += 1
    else:
        br = g.OH
        while br > 1 and lds(1, br) > budget:
            br -= 1
        if lds(1, br) <= budget:
            IMG, BR = 1, br
    if not IMG:
        return None
    n_units = -(-B // IMG) * -(-g.OH // BR)
    per_cu = 1 if one_block else max(1, min(2, (160 * 1024) // max(lds(IMG, BR), 1)))
    target = 256 * per_cu
    nsplit = max(1, min(n_units, target // (ngroups * tiles)))
    pl = dict(IMG=IMG, BR=BR, xp=xp, yp=yp, TN=tn, TC=tc, TPW=TPW, NW=NW, ngroups=ngroups, nsplit=nsplit,
              budget=budget_kb)
    if dma:
        pl["DMA"] = 1
    return pl


def _wgrad2_plans(g: ConvGeom, B: int, Cx: int, Ny: int, n_lim: int, c_lim: int):
    """Candidate plans, the heuristic default first (the autotuner times them all against wgrad.hip)."""
    key = (g, B, Cx, Ny, n_lim, c_lim)
    if key in _W2_PLANS:
        return _W2_PLANS[key]
    plans = []
    T = g.KH * g.KW
    if T >= 4 and not g.depthwise:
        tn = 64 if n_lim > 32 else (32 if n_lim > 16 else 16)
        tc = 64 if c_lim > 32 else (32 if c_lim > 16 else 16)
        opts = _W2_COMBOS[(tn, tc)]
        ngroups = -(-T // (4 * max(opts)))
        need = -(-T // (4 * ngroups))
        first = None
        if W2_NW8 and (tn, tc) in _W2_COMBOS8:      # the autotuner's usual winner first: it is the untuned default
            first = _wgrad2_one_plan(g, B, Cx, Ny, n_lim, c_lim, tn, tc, _W2_COMBOS8[(tn, tc)], 150, NW=8)
        if first is None:
            first = _wgrad2_one_plan(g, B, Cx, Ny, n_lim, c_lim, tn, tc, min(o for o in opts if o >= need))
        if first is not None:
            plans.append(first)
        tiles = {(tn, tc)}
        if tn == 64 and tc == 64:
            tiles |= {(64, 32), (32, 64)}
        elif tn == 64 and tc == 32:
            tiles.add((32, 32))
        elif tn == 32 and tc == 64:
            tiles.add((32, 32))
        seen = {tuple(sorted((k, v) for k, v in first.items() if k != "budget"))} if first else set()
        for (a_, b_) in sorted(tiles):
            for tpw in _W2_COMBOS[(a_, b_)]:
                for kb in (150, 76, 50, 36):
                    pl = _wgrad2_one_plan(g, B, Cx, Ny, n_lim, c_lim, a_, b_, tpw, kb)
                    if pl is None:
                        continue
                    sig = tuple(sorted((k, v) for k, v in pl.items() if k != "budget"))
                    if sig in seen:
                        continue
                    seen.add(sig)
                    plans.append(pl)
            if W2_NW8 and (a_, b_) in _W2_COMBOS8:
                for kb in (150, 100, 76):
                    pl = _wgrad2_one_plan(g, B, Cx, Ny, n_lim, c_lim, a_, b_, _W2_COMBOS8[(a_, b_)], kb, NW=8)
                    if pl is None:
                        continue
                    sig = tuple(sorted((k, v) for k, v in pl.items() if k != "budget"))
                    if sig not in seen:
                        seen.add(sig)
                        plans.append(pl)
        # LDS-DMA staged, double-buffered forms (appended: the indices of the plans above are what recorded choices
        # name).  Two unit sizes each: the buffers halve what a unit can hold, and the transfer only hides behind the
        # MFMA phase when a block walks several units
        if W2_DMA:
            for (a_, b_) in sorted(tiles):
                forms = [(8, _W2_COMBOS8[(a_, b_)])] if (a_, b_) in _W2_COMBOS8 else []
                forms += [(4, t) for t in _W2_DMA4.get((a_, b_), ())]
                for nw, tpw in forms:
                    for kb in (150, 76):
                        pl = _wgrad2_one_plan(g, B, Cx, Ny, n_lim, c_lim, a_, b_, tpw, kb, NW=nw, dma=True)
                        if pl is None:
                            continue
                        sig = tuple(sorted((k, v) for k, v in pl.items() if k != "budget"))
                        if sig not in seen:
                            seen.add(sig)
                            plans.append(pl)
    _W2_PLANS[key] = plans
    return plans


def _box_slab(holder, n, box, device):
    """Split-K slab of a custom-box weight gradient.  The kernel writes box elements only and the slab reduce sweeps
    every element, so the rest must read as zero -- but nothing ever writes it: a zeroed slab kept by the caller
    (`holder`, a dict owned by the layer; filled on the first, uncaptured call) stays valid for the layer's life
    instead of a 6 MB fill per step.  Without a holder the slab is zero-filled per call."""
    if holder is None:
        return torch.zeros(n, dtype=torch.float32, device=device)
    key = (n, tuple(box))
    slab = holder.get(key)
    if slab is None:
        slab = torch.zeros(n, dtype=torch.float32, device=device)
        if not torch.cuda.is_current_stream_capturing():
            holder[key] = slab
    return slab


W2_DY_AFFINE = os.environ.get("DDL_W2_DY_AFFINE", "1") == "1"


def conv_wgrad(x, dy, g: ConvGeom, layout="A", out=None, box=None, x_affine=None, slab_holder=None, bias_tail=None,
               dy_affine=None):
    """`box` = (n_lim, c_lim, sn, st, sc, numel): write dW[n][t][c] at out[n*sn + t*st + c*sc] instead of one of
    the two standard layouts (the caller guarantees `out` has `numel` elements and is zero elsewhere).
    `x_affine` = (scale, shift, c_true), fp32 [Ip]: X is read as bf16(X * scale + shift) on real pixels (a
    BatchNorm in front of the layer applied on load); only the streaming kernel (1x1 / few-tap problems) has it.
    `bias_tail` = (col, off), 1x1 problems with a custom box on the streaming kernel: column `col` >= c_lim of X is a
    column of ones (`im2col_1ch(ones=True)`) and sum_m dY[m][n] -- the bias gradient -- is written at out[off + n].
    `bias_tail` = ("row", row, off): sum_m dY[m][row] (one row of the dY operand summed over all pixels, from one more
    MFMA against a fragment of ones) is written at out[off] -- the scalar bias gradient of a one-channel transposed
    conv, whose dY operand is the taps tensor of the image gradient (row = the centre tap).
    `bias_tail` = ("rows", off): the same for every row n < n_lim, at out[off + n] (a Dense layer's bias gradient).
    `dy_affine` = (scale, shift, c_true), fp32 [Op]: the dY OPERAND is read as bf16(dY * scale + shift) on real pixels
    (channels >= c_true as zero) -- the weight gradient of a transposed convolution, whose input plays dY here, behind a
    BatchNorm that was applied on load.  The register-staged persistent kernel applies it as it stages the tile; where
    no such plan exists the operand is materialised first."""
    _chk_act(x, "x")
    _chk_act(dy, "dy")
    B = x.shape[0]
    Ip, Op = pad8(g.I), pad8(g.O)
    if tuple(x.shape) != (B, g.H, g.W, Ip) or tuple(dy.shape) != (B, g.OH, g.OW, Op):
        raise ValueError(f"conv_wgrad: x {tuple(x.shape)} / dy {tuple(dy.shape)} vs geometry {g}")
    if dy_affine is not None:
        _chk_f32(dy_affine[0], Op, "dy_affine scale")
        _chk_f32(dy_affine[1], Op, "dy_affine shift")
        usable = W2_DY_AFFINE and WGRAD_IMPL == "wgrad2" and bias_tail is None and x_affine is None and not g.depthwise
        if not usable:
            dy = bn_apply(dy, dy_affine[0], dy_affine[1], None, 0.3, int(dy_affine[2]), 1)
            dy_affine = None
    ranges = _batch_ranges(B, max(g.H * g.W * Ip, g.OH * g.OW * Op))
    if ranges is not None:                      # sum of the per-slice gradients (fp32)
        total = None
        for b0, b1 in ranges:
            if total is None:
                total = conv_wgrad(x[b0:b1], dy[b0:b1], g, layout, out, box, x_affine, slab_holder, bias_tail, dy_affine)
            else:
                part = torch.empty_like(total)
                if box is not None:
                    zero_(part)
                add_f32_(total.reshape(-1), conv_wgrad(x[b0:b1], dy[b0:b1], g, layout, part, box, x_affine,
                                                       slab_holder, bias_tail, dy_affine).reshape(-1))
        return total
    dev = x.device
    T = g.KH * g.KW
    if g.depthwise:
        if out is None:
            out = torch.empty(g.KH, g.KW, Ip, dtype=torch.float32, device=dev)
        _chk_f32(out, T * Ip, "dW")
        nb = _dw_blocks(B * g.OH * g.OW, Ip)
        part = torch.empty(nb * T * Ip, dtype=torch.float32, device=dev)
        xs = xh = None
        xct = 0
        if x_affine is not None:
            _chk_f32(x_affine[0], Ip, "x_affine scale")
            _chk_f32(x_affine[1], Ip, "x_affine shift")
            xs, xh, xct = x_affine[0].data_ptr(), x_affine[1].data_ptr(), int(x_affine[2])
        rc = _depthwise(2, dy.data_ptr(), x.data_ptr(), None, out.data_ptr(), part.data_ptr(), B, g.H, g.W, Ip,
                        g.OH, g.OW, g.KH, g.KW, g.sh, g.sw, g.dh, g.dw, g.pt, g.pl, g.O, 0, 0.0, xs, xh, xct,
                        _stream())
        if rc == -5:                    # generic stencil: no on-load affine
            xm = bn_apply(x, x_affine[0], x_affine[1], None, 0.3, x_affine[2], 1)
            rc = _depthwise(2, dy.data_ptr(), xm.data_ptr(), None, out.data_ptr(), part.data_ptr(), B, g.H, g.W, Ip,
                            g.OH, g.OW, g.KH, g.KW, g.sh, g.sw, g.dh, g.dw, g.pt, g.pl, g.O, 0, 0.0, None, None, 0,
                            _stream())
        if rc:
            raise ValueError("depthwise wgrad rejected")
        _done()
        return out
    if layout == "A":            # [O][T][Ip]
        shape = (g.O, g.KH, g.KW, Ip)
        n_lim, c_lim, sn, st, sc = g.O, Ip, T * Ip, Ip, 1
    else:                        # [I][T][Op]
        shape = (g.I, g.KH, g.KW, Op)
        n_lim, c_lim, sn, st, sc = Op, g.I, 1, Op, T * Op
    numel = int(np.prod(shape))
    if box is not None:
        n_lim, c_lim, sn, st, sc, numel = box
        if out is None or n_lim > Op or c_lim > Ip:
            raise ValueError("conv_wgrad: a custom box needs `out` and limits inside the operands")
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=dev)
    if out.numel() != numel:
        raise ValueError(f"conv_wgrad: out has {out.numel()} elements, expected {numel} for layout {layout}")
    _chk_f32(out, numel, "dW")
    plans = _wgrad2_plans(g, B, Ip, Op, n_lim, c_lim) \
        if (WGRAD_IMPL == "wgrad2" and bias_tail is None and x_affine is None) else []
    if dy_affine is not None:
        # only the register-staged forms touch the operand (plans are filtered, so their indices -- what a recorded
        # choice holds -- are those of this filtered list: the choice key below carries the affine flag)
        plans = [pl for pl in plans if not pl.get("DMA")]
        if not plans:
            dy = bn_apply(dy, dy_affine[0], dy_affine[1], None, 0.3, int(dy_affine[2]), 1)
            dy_affine = None
            plans = _wgrad2_plans(g, B, Ip, Op, n_lim, c_lim)
    if bias_tail is not None and box is None:
        raise ValueError("conv_wgrad: bias_tail needs a custom box")
    bcol, boff, brow = -1, 0, -1
    if bias_tail is not None:
        if bias_tail[0] == "row":
            brow, boff = int(bias_tail[1]), int(bias_tail[2])
        elif bias_tail[0] == "rows":           # every row: sum_m dY[m][n] at out[off + n]
            brow, boff = -2, int(bias_tail[1])
        else:
            bcol, boff = int(bias_tail[0]), int(bias_tail[1])
    xs = xh = None
    xct = Ip
    if x_affine is not None:
        if plans:
            raise ValueError("conv_wgrad: x_affine is only available on the streaming weight-gradient kernel")
        _chk_f32(x_affine[0], Ip, "x_affine scale")
        _chk_f32(x_affine[1], Ip, "x_affine shift")
        xs, xh, xct = x_affine[0].data_ptr(), x_affine[1].data_ptr(), int(x_affine[2])

    def run_w2(pl):
        ns = pl["nsplit"]
        if W2_FRAG_SLAB:
            # slabs in the kernel's fragment order (fully coalesced stores); the reduce scatters the final gradient
            # and writes the box only, so whatever lies outside a custom box is zeroed here
            per = _wgrad2_frag_elems(pl["TN"], pl["TC"], pl["TPW"], pl["NW"], pl["ngroups"], n_lim, c_lim)
            slab = torch.empty(ns * per, dtype=torch.float32, device=dev)
            if box is not None:
                zero_(out)
        else:
            slab = (torch.zeros if box is not None else torch.empty)(ns * numel, dtype=torch.float32, device=dev)
        rc = _wgrad2(dy.data_ptr(), x.data_ptr(), slab.data_ptr(), numel, ns, B, g.OH, g.OW, Op, g.H, g.W, Ip,
                     g.KH, g.KW, g.sh, g.sw, g.dh, g.dw, g.pt, g.pl, n_lim, c_lim, sn, st, sc, pl["IMG"], pl["BR"],
                     pl["xp"], pl["yp"], pl["TN"], pl["TC"], pl["TPW"], pl["NW"], pl["ngroups"],
                     (1 if W2_FRAG_SLAB else 0) | (2 if pl.get("DMA") else 0),
                     None if dy_affine is None else dy_affine[0].data_ptr(),
                     None if dy_affine is None else dy_affine[1].data_ptr(),
                     0 if dy_affine is None else int(dy_affine[2]), _stream())
        if rc:
            raise ValueError(f"conv_wgrad2 rejected its plan (rc={rc}): {g} {pl}")
        if W2_FRAG_SLAB:
            rc = _slab_reduce_frag(slab.data_ptr(), out.data_ptr(), ns, pl["TN"], pl["TC"], pl["TPW"], pl["NW"],
                                   pl["ngroups"], T, n_lim, c_lim, sn, st, sc, _stream())
            if rc:
                raise ValueError(f"slab_reduce_frag rejected its arguments (rc={rc})")
        else:
            _slab_reduce(slab.data_ptr(), out.data_ptr(), numel, numel, ns, _stream())

    def run_w1():
        M = B * g.OH * g.OW
        ksplit = _wgrad_ksplit(M, T, n_lim, c_lim)
        slab = None
        if ksplit > 1:
            slab = _box_slab(slab_holder, ksplit * numel, box, dev) if box is not None else \
                torch.empty(ksplit * numel, dtype=torch.float32, device=dev)
        rc = _wgrad(dy.data_ptr(), x.data_ptr(), out.data_ptr(), _p(slab), numel, ksplit, B, g.OH, g.OW, Op, g.H,
                    g.W, Ip, g.KH, g.KW, g.sh, g.sw, g.dh, g.dw, g.pt, g.pl, n_lim, c_lim, sn, st, sc, xs, xh, xct,
                    bcol, boff, brow, _stream())
        if rc:
            raise ValueError(f"conv_wgrad rejected the problem (rc={rc}): {g}")

    if plans:
        aff = 0 if dy_affine is None else 1
        key = ("wgrad", g, B, Ip, Op, n_lim, c_lim, sn, st, sc, aff)
        kstr = _kstr("wgrad", g, B, Ip, Op, n_lim, c_lim, sn, st, sc, len(plans), aff)
        choice = _CONV_CHOICE.get(key)
        if choice is None and kstr in _CHOICE_SPEC and (-1 if dy_affine is None else 0) <= int(_CHOICE_SPEC[kstr][1]) < len(plans):
            choice = _CONV_CHOICE[key] = int(_CHOICE_SPEC[kstr][1])
        if choice is None:
            if AUTOTUNE and not torch.cuda.is_current_stream_capturing():
                timed = [(_time_us(lambda pl=pl: run_w2(pl)), i) for i, pl in enumerate(plans)]
                if dy_affine is None:       # (the streaming kernel has no affine on this operand)
                    timed.append((_time_us(run_w1), -1))
                timed.sort()
                choice = timed[0][1]
                _record_choice(kstr, ["wgrad", choice])
                if os.environ.get("DDL_AUTOTUNE_VERBOSE"):
                    desc = [(round(t, 1), "wgrad" if i < 0 else
                             tuple(plans[i][k] for k in ("TN", "TC", "TPW", "NW", "IMG", "BR", "ngroups", "nsplit")) +
                             (("dma",) if plans[i].get("DMA") else ()))
                            for t, i in timed[:6]]
                    print(f"[autotune] wgrad B={B} {g.H}x{g.W}x{g.I}->{g.OH}x{g.OW}x{g.O}: {desc}", flush=True)
            else:
                choice = 0
            _CONV_CHOICE[key] = choice
        if choice >= 0:
            run_w2(plans[choice])
        else:
            run_w1()
        _done()
        return out
    M = B * g.OH * g.OW
    ksplit = _wgrad_ksplit(M, T, n_lim, c_lim)
    # with a custom box the slab reduce also sweeps elements the kernel never writes: they must read as 0
    slab = None
    if ksplit > 1:
        slab = _box_slab(slab_holder, ksplit * numel, box, dev) if box is not None else \
            torch.empty(ksplit * numel, dtype=torch.float32, device=dev)
    rc = _wgrad(dy.data_ptr(), x.data_ptr(), out.data_ptr(), _p(slab), numel, ksplit, B, g.OH, g.OW, Op, g.H,
                g.W, Ip, g.KH, g.KW, g.sh, g.sw, g.dh, g.dw, g.pt, g.pl, n_lim, c_lim, sn, st, sc, xs, xh, xct,
                bcol, boff, brow, _stream())
    if rc:
        raise ValueError(f"conv_wgrad rejected the problem (rc={rc}): {g}")
    _done()
    return out


# ------------------------------------------------------------------------------ wide softmax head
_dense_ce_ws = functools.lru_cache(maxsize=4096)(_sig("ddl_dense_ce_workspace", cl, ci, ci, ci, ci, ci, cl, ci))
_dense_ce = _sig("ddl_dense_ce", ci, vp, vp, vp, vp, ci, ci, ci, vp, vp, vp, vp, vp, ci, vp, cl, cl, ci, vp)

# Bound on the exponentials a training call keeps at a time, 2 bytes per row and class; a batch that needs more goes
# through in pieces of rows (at most 8192), each of which reads and writes the fp32 weight gradient once more.  4 GiB,
# 1.4 % of the card's memory, is 8192 rows of 262144 classes.
CE_PIECE_BYTES = int(os.environ.get("DDL_CE_PIECE_BYTES", str(4 << 30)))
CE_TILE = -1                # tiles of the products: -1 = by the sizes, else digits dw, dx, logits (csrc/hip/dense_ce.hip)


def _rc(rc, what):
    if rc != 0:
        raise RuntimeError(f"{what}: kernel launch refused (code {rc})")


class _Here:
    def __enter__(self):
        pass

    def __exit__(self, *exc):
        pass


_HERE = _Here()


def _on_device(t):
    """Launches go to the current device: make the tensors' device the current one (no cost where it already is)."""
    return _HERE if torch._C._cuda_getDevice() == t.get_device() else torch.cuda.device(t.device)


def _stream_of(t):
    """The current stream of the tensors' device (the raw handle: torch.cuda.current_stream() builds an object first, 3 us)."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _chk_out(t, n, dtypes, like, name):
    if not (t.device == like.device and t.dtype in dtypes and t.is_contiguous() and t.numel() == n):
        raise ValueError(f"{name}: need a contiguous tensor of {n} elements, {' / '.join(map(str, dtypes))} on {like.device}, "
                         f"got {tuple(t.shape)} {t.dtype} {t.device} contiguous={t.is_contiguous()}")
    if t.data_ptr() % 16:
        raise ValueError(f"{name}: not 16-byte aligned")


def ceil_div(a, b):
    return -(-a // b)


def dense_softmax_ce(x, w, bias, labels, want_grad=True, out_dw=None, out_db=None, grad_dtype=torch.float32):
    """Dense(K -> V) + softmax cross entropy (csrc/hip/dense_ce.hip).  x [N][Kp] bf16, w [V][Kp] bf16, bias [V] fp32
    or None, labels [N] int64 (negative: row left out).  Returns (loss, dx, dw, db, rows)."""
    _chk_act(x, "x")
    _chk_act(w, "w")
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"dense_softmax_ce: x {tuple(x.shape)} and w {tuple(w.shape)} must be [N][K] and [V][K]")
    N, K = x.shape
    V = w.shape[0]
    dev = x.device
    if V < 1 or K < 8 or N >= 1 << 28 or max(V, K) >= (1 << 22) - 64:
        raise ValueError(f"dense_softmax_ce: N={N} K={K} V={V} outside the supported range")
    for t, name in ((w, "w"), (bias, "bias"), (labels, "labels"), (out_dw, "out_dw"), (out_db, "out_db")):
        if t is not None and t.device != dev:
            raise ValueError(f"dense_softmax_ce: {name} is on {t.device}, x on {dev}")
    if bias is not None:
        _chk_f32(bias, V, "bias")
        if bias.numel() != V:
            raise ValueError(f"bias: {bias.numel()} elements, need {V}")
    if labels.dtype != torch.int64 or not labels.is_contiguous() or labels.numel() != N:
        raise ValueError(f"labels must be a contiguous int64 vector of {N} class numbers")
    dw = db = dx = None
    if want_grad:
        if out_dw is not None:
            grad_dtype = out_dw.dtype
        elif out_db is not None:
            grad_dtype = out_db.dtype
        if grad_dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"dense_softmax_ce: gradients are fp32 or bf16, not {grad_dtype}")
        dw = torch.empty(V, K, dtype=grad_dtype, device=dev) if out_dw is None else out_dw
        _chk_out(dw, V * K, (grad_dtype,), x, "out_dw")
        if bias is not None:
            db = torch.empty(V, dtype=grad_dtype, device=dev) if out_db is None else out_db
            _chk_out(db, V, (grad_dtype,), x, "out_db")
        elif out_db is not None:
            raise ValueError("dense_softmax_ce: out_db without a bias")
        dx = torch.empty_like(x)
    elif out_dw is not None or out_db is not None:
        raise ValueError("dense_softmax_ce: out_dw / out_db need want_grad")
    with _on_device(x):
        if N == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
            return torch.zeros((), dtype=torch.float32, device=dev), dx, dw, db, torch.empty(0, dtype=torch.float32, device=dev)
        loss, rows = torch.empty((), dtype=torch.float32, device=dev), torch.empty(N, dtype=torch.float32, device=dev)
        bf = int(want_grad and dw.dtype == torch.bfloat16)
        nws = _dense_ce_ws(N, V, K, int(want_grad), bf, CE_PIECE_BYTES, CE_TILE)
        if nws < 0:
            raise ValueError(f"dense_softmax_ce: N={N} K={K} V={V} outside the kernels' range")
        ws = torch.empty(nws, dtype=torch.uint8, device=dev)
        _rc(_dense_ce(x.data_ptr(), w.data_ptr(), _p(bias), labels.data_ptr(), N, V, K, loss.data_ptr(), rows.data_ptr(),
                      _p(dx), _p(dw), _p(db), bf, ws.data_ptr(), nws, CE_PIECE_BYTES, CE_TILE, _stream_of(x)),
            "dense_softmax_ce")
        _done()
    return loss, dx, dw, db, rows


# ------------------------------------------------------------------------------ 8-bit activation checkpoints
from .functional import Packed8  # noqa: E402  (functional imports this module when it is first called)

_pack8 = _sig("ddl_pack8", ci, vp, vp, vp, cl, vp)
_unpack8 = _sig("ddl_unpack8", ci, vp, vp, vp, cl, vp)
_act_bwd8 = _sig("ddl_act_bwd8", ci, vp, vp, vp, vp, cl, ci, cf, vp)
_wgrad8_ws = functools.lru_cache(maxsize=4096)(_sig("ddl_dense_wgrad8_workspace", cl, ci, ci, ci, ci, ci))
_wgrad8 = _sig("ddl_dense_wgrad8", ci, vp, vp, vp, ci, ci, ci, ci, vp, vp, vp, cl, ci, vp)
WGRAD8_TILE = -1            # tile of dense_wgrad8: -1 = by the sizes (csrc/hip/act8.hip wg8_plan)


def _chk_packed(q, name="q"):
    c, s = q.codes, q.scales
    n = c.numel()
    if not (c.is_cuda and c.dtype == torch.int8 and c.is_contiguous() and s.device == c.device and s.dtype == torch.uint8
            and s.is_contiguous() and s.numel() == ceil_div(n, 32)):
        raise ValueError(f"{name}: codes must be contiguous int8 and scales uint8, one per 32 codes, on one device")
    if c.dim() < 1 or c.shape[-1] % 8 or c.data_ptr() % 8:
        raise ValueError(f"{name}: channel dim must be a multiple of 8 and the codes 8-byte aligned")
    return n


def pack8(x):
    _chk_act(x, "x")
    n = x.numel()
    codes = torch.empty_like(x, dtype=torch.int8)             # (torch.empty of a shape and a device: 1 us more)
    scales = torch.empty(ceil_div(n, 32), dtype=torch.uint8, device=x.device)
    if n:
        with _on_device(x):
            _rc(_pack8(x.data_ptr(), codes.data_ptr(), scales.data_ptr(), n, _stream_of(x)), "pack8")
            _done()
    return Packed8(codes, scales)


def unpack8(q, out=None):
    n = _chk_packed(q)
    y = torch.empty_like(q.codes, dtype=torch.bfloat16) if out is None else out
    if out is not None:
        _chk_out(out, n, (torch.bfloat16,), q.codes, "out")
    if n:
        with _on_device(y):
            _rc(_unpack8(q.codes.data_ptr(), q.scales.data_ptr(), y.data_ptr(), n, _stream_of(y)), "unpack8")
            _done()
    return y


def act_bwd8(dy, q, kind, alpha=0.3):
    if kind in (None, "linear"):
        return dy
    _chk_act(dy, "dy")
    n = _chk_packed(q)
    if dy.shape != q.codes.shape or dy.device != q.codes.device:
        raise ValueError(f"act_bwd8: dy {tuple(dy.shape)} on {dy.device}, checkpoint {tuple(q.codes.shape)} on {q.codes.device}")
    dx = torch.empty_like(dy)
    if n:
        with _on_device(dy):
            _rc(_act_bwd8(dy.data_ptr(), q.codes.data_ptr(), q.scales.data_ptr(), dx.data_ptr(), n, ACT_CODE[kind], alpha,
                          _stream_of(dy)), "act_bwd8")
            _done()
    return dx


def dense_wgrad8(q, dy, out_dw=None, out_db=None, n_out=None):
    """dw [O][Kp] = dy^T x, db [O] = column sums of dy, x [R][Kp] read from its 8-bit checkpoint; fp32."""
    _chk_act(dy, "dy")
    _chk_packed(q)
    x = q.codes
    if x.dim() != 2 or dy.dim() != 2 or x.shape[0] != dy.shape[0] or x.device != dy.device:
        raise ValueError(f"dense_wgrad8: checkpoint {tuple(x.shape)} and dy {tuple(dy.shape)} must be [R][K] and [R][O] on one "
                         "device")
    R, K = x.shape
    Op = dy.shape[1]
    O = Op if n_out is None else int(n_out)
    if not 0 < O <= Op or K < 8 or max(R, K, Op) >= 1 << 24:
        raise ValueError(f"dense_wgrad8: R={R} K={K} O={O} of {Op} outside the supported range")
    dev = dy.device
    dw = torch.empty(O, K, dtype=torch.float32, device=dev) if out_dw is None else out_dw
    db = torch.empty(O, dtype=torch.float32, device=dev) if out_db is None else out_db
    _chk_out(dw, O * K, (torch.float32,), dy, "out_dw")
    if not (db.device == dev and db.dtype == torch.float32 and db.is_contiguous() and db.numel() == O):
        raise ValueError(f"out_db: need a contiguous fp32 vector of {O} elements on {dev}")
    with _on_device(dy):
        if R == 0:
            dw.zero_()
            db.zero_()
            return dw, db
        nws = _wgrad8_ws(R, K, Op, O, WGRAD8_TILE)
        if nws < 0:
            raise ValueError(f"dense_wgrad8: R={R} K={K} O={O} of {Op} outside the kernels' range")
        ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws else None
        _rc(_wgrad8(x.data_ptr(), q.scales.data_ptr(), dy.data_ptr(), R, K, Op, O, dw.data_ptr(), db.data_ptr(), _p(ws), nws,
                    WGRAD8_TILE, _stream_of(dy)), "dense_wgrad8")
        _done()
    return dw, db
