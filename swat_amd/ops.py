"""Path A device ops: thin tensor-level wrappers over the C ABI (include/swat_hip.h).

Every function launches hand-written gfx950 kernels on torch's current stream and allocates only
outputs; there is no PyTorch fallback.  bf16 tensors are torch.bfloat16, everything else fp32/int64.
"""
import functools
from collections import namedtuple

import torch

from . import _lib
from ._lib import ptr as _p

NT, NN, TN = 0, 1, 2
ACT = {None: 0, "none": 0, "quick_gelu": 1, "gelu": 2}
_BF, _F32 = torch.bfloat16, torch.float32


def _chk(rc, what):
    _lib.check(rc, what)


def gemm(layout, A, B, M, N, K, lda, ldb, C, ldc, batch=1, inner=1, sA=(0, 0), sB=(0, 0), sC=(0, 0),
         bias=None, residual=None, actin=None, ldact=0, act=None, C2=None, alpha=1.0):
    """Raw GEMM entry on explicit pointers/strides; A, B bf16 tensors (any shape), C bf16 or fp32 (None with a C2: only the
    activated output is stored)."""
    rc = _lib.lib().swat_gemm_bf16(layout, _p(A), _p(B), _p(C), M, N, K, lda, ldb, ldc, batch, inner,
                                   sA[0], sA[1], sB[0], sB[1], sC[0], sC[1], _p(bias), _p(residual), _p(actin),
                                   ldact, ACT[act], _p(C2), int(C is not None and C.dtype == _F32), float(alpha), _lib.stream())
    _chk(rc, "swat_gemm_bf16")
    return C


def linear_fwd(x, w, bias=None, residual=None, act=None, out_dtype=_BF, want_act=False):
    """y = x @ w.T (+bias) (+residual); x [M,K] bf16, w [N,K] bf16.  want_act -> (pre, act(pre))."""
    M, K = x.shape
    N = w.shape[0]
    y = torch.empty((M, N), dtype=out_dtype, device=x.device)
    y2 = torch.empty((M, N), dtype=_BF, device=x.device) if want_act else None
    gemm(NT, x, w, M, N, K, K, K, y, N, bias=bias, residual=residual, act=act, C2=y2)
    return (y, y2) if want_act else y


def linear_dgrad(dy, w, actin=None, act=None, out_dtype=_BF):
    """dx = dy @ w (* act'(actin)); dy [M,N] bf16, w [N,K] bf16."""
    M, N = dy.shape
    K = w.shape[1]
    dx = torch.empty((M, K), dtype=out_dtype, device=dy.device)
    gemm(NN, dy, w, M, K, N, N, K, dx, K, actin=actin, ldact=K if actin is not None else 0, act=act)
    return dx


def linear_wgrad(dy, x, out=None):
    """dw = dy.T @ x  -> [N,K] fp32; dy [M,N] bf16, x [M,K] bf16."""
    M, N = dy.shape
    K = x.shape[1]
    if out is None:
        out = torch.empty((N, K), dtype=_F32, device=dy.device)
    gemm(TN, dy, x, N, K, M, N, K, out, K)
    return out


def layernorm_fwd(x, gamma, beta, eps=1e-5, rows=None, row_stride=None, out_bf16=True, out_f32=False):
    d = gamma.numel()
    if rows is None:
        rows = x.numel() // d
        row_stride = d
    dev = x.device
    y_bf = torch.empty((rows, d), dtype=_BF, device=dev) if out_bf16 else None
    y_f = torch.empty((rows, d), dtype=_F32, device=dev) if out_f32 else None
    mean = torch.empty(rows, dtype=_F32, device=dev)
    rstd = torch.empty(rows, dtype=_F32, device=dev)
    rc = _lib.lib().swat_layernorm_fwd(_p(x), row_stride, _p(gamma), _p(beta), _p(y_bf), _p(y_f), _p(mean), _p(rstd),
                                       rows, d, float(eps), _lib.stream())
    _chk(rc, "swat_layernorm_fwd")
    return y_bf, y_f, mean, rstd


def layernorm_bwd(dy, x, gamma, mean, rstd, dx_add=None, want_bf16=False, rows=None, dy_stride=None, x_stride=None,
                  dx_out=None, dxo_stride=None, dxa_stride=None, want_colsum=False):
    d = gamma.numel()
    if rows is None:
        rows = dy.numel() // d
    dy_stride = dy_stride or d
    x_stride = x_stride or d
    dev = dy.device
    if dx_out is None:
        dx_out = torch.empty((rows, d), dtype=_F32, device=dev)
        dxo_stride = d
    dx_bf = torch.empty((rows, d), dtype=_BF, device=dev) if want_bf16 else None
    dg = torch.empty(d, dtype=_F32, device=dev)
    db = torch.empty(d, dtype=_F32, device=dev)
    dcs = torch.empty(d, dtype=_F32, device=dev) if want_bf16 else None
    ws = torch.empty(_lib.lib().swat_layernorm_bwd_workspace_bytes(rows, d), dtype=torch.uint8, device=dev)
    rc = _lib.lib().swat_layernorm_bwd(_p(dy), dy_stride, _p(x), x_stride, _p(gamma), _p(mean), _p(rstd), _p(dx_add),
                                       dxa_stride or d, _p(dx_out), dxo_stride, _p(dx_bf), d, _p(dg), _p(db), _p(dcs), _p(ws),
                                       rows, d, _lib.stream())
    _chk(rc, "swat_layernorm_bwd")
    if want_colsum:
        return dx_out, dx_bf, dg, db, dcs
    return dx_out, dx_bf, dg, db


ResidualNorm = namedtuple("ResidualNorm", "y z stats z8")


def _seam(what, rows, d, post, pre, gate, scale, norm):
    """The checked pointers of what both directions of the seam take: post w, b, gate, groups, per channel, scale, pre w, b, rms."""
    if norm != "layer" and norm != "rms":
        raise _lib.SwatHipError(f"{what}: norm {norm!r} ('layer' or 'rms')")
    if rows >= 1 << 31:
        raise _lib.SwatHipError(f"{what}: {rows} rows (under 2^31)")
    for wb in (post, pre):
        if wb is not None and (not isinstance(wb, (tuple, list)) or len(wb) != 2 or wb[0] is None):
            raise _lib.SwatHipError(f"{what}: post, pre = (weight, bias or None)")
    pw, pb = post if post is not None else (None, None)
    qw, qb = pre if pre is not None else (None, None)
    vec = _lib.vec_ptr
    g, groups, channels = None, 0, 0
    if gate is not None:
        if not isinstance(gate, torch.Tensor) or gate.dim() not in (1, 2):
            raise _lib.SwatHipError(f"{what}: gate is a tensor [groups] or [groups, d], got {tuple(gate.shape) if isinstance(gate, torch.Tensor) else gate!r:.80}")
        groups, channels = gate.shape[0], int(gate.dim() == 2)
        g = vec(gate, what, groups, d) if channels else vec(gate, what, groups)
        if groups < 1 or rows % groups:
            raise _lib.SwatHipError(f"{what}: {groups} gates do not divide {rows} rows")
    return (vec(pw, what, d), vec(pb, what, d), g, groups, channels, vec(scale, what, d), vec(qw, what, d), vec(qb, what, d),
            int(norm == "rms"))


def residual_norm_fwd(x, h, post=None, pre=None, gate=None, scale=None, alpha=1.0, norm="layer", eps=1e-5, z_dtype=_BF, pack=False):
    """The seam between two sublayers: y = alpha x + gate * scale * Norm_post(h), z = Norm_pre(y) -> (y, z, stats, z8).

    x [rows, d] the residual stream and h [rows, d] what the sublayer returned, bf16 or fp32 each (rows may be strided); post, pre:
    (weight, bias or None) fp32 [d], or None for no such norm (no pre: z is None); norm 'layer' | 'rms'; scale fp32 [d]; gate fp32
    [groups] or [groups, d], for rows / groups neighbouring rows each (stochastic depth: 0 or 1 / keep per image).  Where gate * scale is
    zero nothing of the branch is taken: without post h may hold anything there (NaN), with post in rows where all of it is zero.  y has x's type, z z_dtype; stats fp32 [4, rows] is for residual_norm_bwd; pack: z8 = z as an 8-bit
    microscaled matrix (mx.MX), the checkpoint of the next linear layer's input or an operand of mx.matmul."""
    px, sx = _lib.rows_ptr(x, "residual_norm_fwd: x", (_BF, _F32))
    rows, d = x.shape
    ph, sh = _lib.rows_ptr(h, "residual_norm_fwd: h", (_BF, _F32), d)
    if h.shape[0] != rows or not 1 <= d <= 8192 or z_dtype not in (_BF, _F32) or (pack and pre is None):
        raise _lib.SwatHipError(f"residual_norm_fwd: x {tuple(x.shape)}, h {tuple(h.shape)} (the same rows, 1 to 8192 columns), z in bf16 or "
                                "fp32, pack goes with pre")
    v = _seam("residual_norm_fwd", rows, d, post, pre, gate, scale, norm)
    y = x.new_empty((rows, d))
    z = x.new_empty((rows, d), dtype=z_dtype) if pre is not None else None
    stats = x.new_empty((4, rows), dtype=_F32)
    z8 = None
    if pack:
        from . import mx
        z8 = mx._empty(x, rows, d, 8)
    rc = _lib.lib().swat_residual_norm_fwd(px, sx, x.dtype == _BF, ph, sh, h.dtype == _BF, *v[:8], float(alpha), v[8], float(eps), y.data_ptr(),
                                           z.data_ptr() if z is not None else None, z_dtype == _BF, z8.codes.data_ptr() if pack else None,
                                           z8.scale.data_ptr() if pack else None, stats.data_ptr(), rows, d, _lib.stream())
    _chk(rc, "swat_residual_norm_fwd")
    return ResidualNorm(y, z, stats, z8)


@functools.lru_cache(maxsize=256)
def _seam_workspace(rows, d, groups, channels):
    return _lib.lib().swat_residual_norm_bwd_workspace_bytes(rows, d, groups, channels)


def residual_norm_bwd(dy, dz, h, y, stats, post=None, pre=None, gate=None, scale=None, alpha=1.0, norm="layer"):
    """Backward of residual_norm_fwd: dy (stream, may be None) and dz (None without pre) -> dict of gradients: 'x', 'h', and of what was
    given 'post_w', 'post_b', 'gate', 'scale', 'pre_w', 'pre_b'.  y, stats: the forward's (y may be None without pre).  Sums in a fixed order."""
    ph, sh = _lib.rows_ptr(h, "residual_norm_bwd: h", (_BF, _F32))
    rows, d = h.shape
    if (dz is None) != (pre is None) or (dy is None and dz is None) or (pre is not None and y is None) or not 1 <= d <= 8192:
        raise _lib.SwatHipError(f"residual_norm_bwd: dz and y go with pre, dy or dz is needed, 1 to 8192 columns (d = {d})")
    py, sy = _lib.rows_ptr(y, "residual_norm_bwd: y", (_BF, _F32), d) if y is not None else (None, d)
    xt = y.dtype if y is not None else getattr(dy, "dtype", _F32)
    pdy, sdy = _lib.rows_ptr(dy, "residual_norm_bwd: dy", (xt,), d) if dy is not None else (None, d)
    pdz, sdz = _lib.rows_ptr(dz, "residual_norm_bwd: dz", (_BF, _F32), d) if dz is not None else (None, d)
    if (xt != _BF and xt != _F32) or any(t is not None and t.shape[0] != rows for t in (dy, dz, y)):
        raise _lib.SwatHipError("residual_norm_bwd: dy, dz, h and y have the same rows; the stream is bf16 or fp32")
    pst = _lib.vec_ptr(stats, "residual_norm_bwd: stats", 4, rows)
    v = _seam("residual_norm_bwd", rows, d, post, pre, gate, scale, norm)
    pw, pb, g, groups, channels, sc, qw, qb, rms = v
    out = {"x": h.new_empty((rows, d), dtype=xt), "h": h.new_empty((rows, d))}
    names = [n for n, t in (("post_w", pw), ("post_b", pb), ("scale", sc), ("pre_w", qw), ("pre_b", qb)) if t is not None]
    cols = {}
    if names:  # (one allocation: a row each)
        flat = h.new_empty((len(names), d), dtype=_F32)
        base = flat.data_ptr()
        for i, (n, t) in enumerate(zip(names, flat.unbind(0))):
            out[n] = t
            cols[n] = base + 4 * d * i
    dgate = None
    if g is not None:
        out["gate"] = torch.empty_like(gate)
        dgate = out["gate"].data_ptr()
    nbytes = _seam_workspace(rows, d, groups, channels)
    ws = h.new_empty(nbytes, dtype=torch.uint8)
    rc = _lib.lib().swat_residual_norm_bwd(pdy, sdy, pdz, sdz, dz is not None and dz.dtype == _BF, ph, sh, h.dtype == _BF, py, sy, xt == _BF, pst,
                                   *v[:8], float(alpha), rms, out["x"].data_ptr(), out["h"].data_ptr(), cols.get("post_w"), cols.get("post_b"),
                                   dgate, cols.get("scale"), cols.get("pre_w"), cols.get("pre_b"), ws.data_ptr(), nbytes, rows, d, _lib.stream())
    _chk(rc, "swat_residual_norm_bwd")
    return out


def softmax_fwd(S, Tq, T, scale, causal=False):
    """S fp32 [..., Tq, ld] -> P bf16 same shape (pad columns zero)."""
    ld = S.shape[-1]
    rows = S.numel() // ld
    P = torch.empty(S.shape, dtype=_BF, device=S.device)
    rc = _lib.lib().swat_softmax_fwd(_p(S), _p(P), rows, Tq, T, ld, float(scale), int(causal), _lib.stream())
    _chk(rc, "swat_softmax_fwd")
    return P


def softmax_bwd(P, dP, T, scale):
    ld = P.shape[-1]
    rows = P.numel() // ld
    dS = torch.empty(P.shape, dtype=_BF, device=P.device)
    rc = _lib.lib().swat_softmax_bwd(_p(P), _p(dP), _p(dS), rows, T, ld, float(scale), _lib.stream())
    _chk(rc, "swat_softmax_bwd")
    return dS


def patchify_cutmix(images, patch, perm=None, box=None, ldp=None):
    """images fp32 [B,3,H,W] -> patches bf16 [B*g*g, ldp]; box = (bbx1, bby1, bbx2, bby2) as rand_bbox returns."""
    B, _, H, W = images.shape
    K = 3 * patch * patch
    ldp = ldp or (K + 7) // 8 * 8
    out = torch.empty((B * (H // patch) * (W // patch), ldp), dtype=_BF, device=images.device)
    x1 = x2 = y1 = y2 = 0
    if perm is not None and box is not None:
        x1, y1, x2, y2 = [int(v) for v in box]
    rc = _lib.lib().swat_patchify_cutmix(_p(images), _p(perm) if perm is not None else None, _p(out), B, H, W, patch,
                                         ldp, x1, x2, y1, y2, _lib.stream())
    _chk(rc, "swat_patchify_cutmix")
    return out


def cutmix_paste(images, perm, box):
    """Out-of-place images[:, :, x1:x2, y1:y2] = images[perm, :, x1:x2, y1:y2] (ref utils/training.py:1466)."""
    B, _, H, W = images.shape
    x1, y1, x2, y2 = [int(v) for v in box]
    out = torch.empty_like(images)
    rc = _lib.lib().swat_cutmix_paste(_p(images), _p(perm), _p(out), B, H, W, x1, x2, y1, y2, _lib.stream())
    _chk(rc, "swat_cutmix_paste")
    return out


def colsum(X, rows=None, n=None, ld=None, group=(0, 0, 0)):
    if rows is None:
        rows, n = X.shape
        ld = n
    out = torch.empty(n, dtype=_F32, device=X.device)
    rc = _lib.lib().swat_colsum(_p(X), 1 if X.dtype == _BF else 0, rows, n, ld, _p(out), group[0], group[1], group[2],
                                _lib.stream())
    _chk(rc, "swat_colsum")
    return out


def cast_bf16(x, out=None):
    if out is None:
        out = torch.empty(x.shape, dtype=_BF, device=x.device)
    rc = _lib.lib().swat_cast_bf16(_p(x), _p(out), x.numel(), _lib.stream())
    _chk(rc, "swat_cast_bf16")
    return out


def widen_bf16(x, out):
    """bf16 -> fp32 into `out` (same number of elements, a multiple of 4)."""
    rc = _lib.lib().swat_widen_bf16(_p(x), _p(out), x.numel(), _lib.stream())
    _chk(rc, "swat_widen_bf16")
    return out


def l2norm_fwd(x):
    rows, d = x.shape
    y = torch.empty_like(x)
    nrm = torch.empty(rows, dtype=_F32, device=x.device)
    _chk(_lib.lib().swat_l2norm_fwd(_p(x), _p(y), _p(nrm), rows, d, _lib.stream()), "swat_l2norm_fwd")
    return y, nrm


def l2norm_bwd(y, nrm, dy):
    rows, d = y.shape
    dx = torch.empty_like(y)
    _chk(_lib.lib().swat_l2norm_bwd(_p(y), _p(nrm), _p(dy), _p(dx), rows, d, _lib.stream()), "swat_l2norm_bwd")
    return dx


def sgemm_small(A, B, M, N, K, sam, sak, sbk, sbn, out=None, alpha=1.0, accumulate=False):
    if out is None:
        out = torch.empty((M, N), dtype=_F32, device=A.device)
    rc = _lib.lib().swat_sgemm_small(_p(A), _p(B), _p(out), M, N, K, sam, sak, sbk, sbn, out.shape[-1], float(alpha),
                                     int(accumulate), _lib.stream())
    _chk(rc, "swat_sgemm_small")
    return out


def ce_mixed(z, logit_scale, ya, yb, lam, want_grad=True, want_logits=False, loss_accum=None):
    """loss / dz / dlogit_scale of lam*CE(z*e^ls, ya) + (1-lam)*CE(z*e^ls, yb) (mean over the batch)."""
    B, C = z.shape
    dev = z.device
    ws = torch.empty(2 * B, dtype=_F32, device=dev)
    loss = torch.empty(1, dtype=_F32, device=dev)
    dls = torch.empty(1, dtype=_F32, device=dev)
    dz = torch.empty_like(z) if want_grad else None
    logits = torch.empty_like(z) if want_logits else None
    rc = _lib.lib().swat_ce_mixed(_p(z), _p(logit_scale), _p(ya), _p(yb), float(lam), _p(ws), _p(loss), _p(dls), _p(dz),
                                  _p(logits), _p(loss_accum), B, C, _lib.stream())
    _chk(rc, "swat_ce_mixed")
    return loss, dz, dls, logits


def adamw_step(params, grads, exp_avg, exp_avg_sq, shadow, seg_begin, lrs_dev, bias_corr_dev, beta1=0.9, beta2=0.999,
               eps=1e-8, weight_decay=1e-2, grad_scale=1.0):
    import ctypes
    n = params.numel()
    arr = (ctypes.c_int64 * len(seg_begin))(*seg_begin)
    rc = _lib.lib().swat_adamw(_p(params), _p(grads), _p(exp_avg), _p(exp_avg_sq), _p(shadow), n,
                               ctypes.cast(arr, ctypes.c_void_p), len(seg_begin), _p(lrs_dev), float(beta1), float(beta2),
                               float(eps), float(weight_decay), _p(bias_corr_dev), float(grad_scale), _lib.stream())
    _chk(rc, "swat_adamw")
