"""Thin torch-tensor wrappers over the C ABI (include/gpsr.h).

PyTorch is plumbing here: it owns device memory and the HIP stream; all
arithmetic on the path happens in libgpsr.so.  Every function requires CUDA
(ROCm) tensors and raises otherwise -- there is no CPU path.
"""
import ctypes
from typing import NamedTuple

import numpy as np
import torch

from . import _lib

RBF, MATERN12, MATERN32, MATERN52, LINEAR = 0, 1, 2, 3, 4
AVERAGE, BILINEAR = 0, 1
BLOCK = 112


def _stream():
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _p(t, dtype=None):
    if t is None:
        return None
    if not t.is_cuda:
        raise _lib.GpsrError("gpsr ops need device tensors (no CPU fallback)")
    if t.device.index != torch.cuda.current_device():
        # launches go on the current device's stream (_stream): a buffer of another GPU would fault there
        raise _lib.GpsrError(f"tensor on {t.device}, current device is cuda:{torch.cuda.current_device()} "
                             "(one process per GPU: torch.cuda.set_device(LOCAL_RANK) first)")
    if dtype is not None and t.dtype != dtype:
        raise _lib.GpsrError(f"expected {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise _lib.GpsrError("tensor must be contiguous")
    return t.data_ptr()


def padded_n(n):
    return ((n + BLOCK - 1) // BLOCK) * BLOCK


def block(A):
    """[B,N,N] row-major -> the library's tile-blocked layout [B][N/112][N/112][112][112] (same shape, a copy)."""
    B, N, _ = A.shape
    nb = N // BLOCK
    return A.view(B, nb, BLOCK, nb, BLOCK).permute(0, 1, 3, 2, 4).contiguous().view(B, N, N)


def unblock(Ab):
    """Inverse of block(): tile-blocked -> [B,N,N] row-major (a copy)."""
    B, N, _ = Ab.shape
    nb = N // BLOCK
    return Ab.view(B, nb, nb, BLOCK, BLOCK).permute(0, 1, 3, 2, 4).contiguous().view(B, N, N)


def gather(train_in, train_tgt, test_in, s, p, locs, tidx, out=None):
    """-> X [B,n,8], y [B,n], Xs [B,m,8]   (gpsr_gather).  out = (X, y, Xs): write into these (contiguous row slices of
    a batch buffer) instead of allocating."""
    lib = _lib.load()
    H, W = train_in.shape
    B, nt = locs.shape[0], tidx.shape[0]
    n, m = nt * nt, (p * s - 2) ** 2
    dev = train_in.device
    if out is None:
        X = torch.empty((B, n, 8), dtype=torch.float64, device=dev)
        y = torch.empty((B, n), dtype=torch.float64, device=dev)
        Xs = torch.empty((B, m, 8), dtype=torch.float64, device=dev)
    else:
        X, y, Xs = out
        if X.shape != (B, n, 8) or y.shape != (B, n) or Xs.shape != (B, m, 8):
            raise _lib.GpsrError(f"gather: out shapes {tuple(X.shape)}, {tuple(y.shape)}, {tuple(Xs.shape)} do not fit B={B}, n={n}, m={m}")
    _lib.check(lib.gpsr_gather(_p(train_in, torch.float64), _p(train_tgt, torch.float64),
                               _p(test_in, torch.float64), H, W, s, p, _p(locs, torch.int32), B,
                               _p(tidx, torch.int32), nt, _p(X, torch.float64), _p(y, torch.float64),
                               _p(Xs, torch.float64), _stream()), "gpsr_gather")
    return X, y, Xs


def init_hypers(y, kernel_id, init_raw_os=0.0, init_raw_ls=0.0, carry=None):
    """carry: None | [4] (every GP continues that one chain link) | [B,4] (GP b continues chain b)."""
    lib = _lib.load()
    B, n = y.shape
    raw = torch.empty((B, 4), dtype=torch.float32, device=y.device)
    stride = 0
    if carry is not None and carry.dim() == 2:
        if carry.shape != (B, 4):
            raise _lib.GpsrError(f"carry must be [4] or [{B},4], got {tuple(carry.shape)}")
        stride = 4
    _lib.check(lib.gpsr_init_hypers(_p(y, torch.float64), B, n, kernel_id, float(init_raw_os), float(init_raw_ls),
                                    _p(carry, torch.float32), stride, _p(raw), _stream()), "gpsr_init_hypers")
    return raw


def covariance(X, kernel_id, raw):
    lib = _lib.load()
    B, n, d = X.shape
    N = padded_n(n)
    K = torch.zeros((B, N, N), dtype=torch.float64, device=X.device)
    _lib.check(lib.gpsr_covariance(_p(X, torch.float64), B, n, d, kernel_id, _p(raw, torch.float32), _p(K),
                                   _stream()), "gpsr_covariance")
    return unblock(K)      # row-major for Python callers; the library's layout is tile-blocked (include/gpsr.h)


def covariance_grad(X, kernel_id, raw):
    """-> K, dK/dlengthscale (x outputscale), both [B,N,N] row-major, lower block-triangle valid (gpsr_covariance_grad)."""
    lib = _lib.load()
    B, n, d = X.shape
    N = padded_n(n)
    K = torch.zeros((B, N, N), dtype=torch.float64, device=X.device)
    dK = torch.zeros((B, N, N), dtype=torch.float64, device=X.device)
    _lib.check(lib.gpsr_covariance_grad(_p(X, torch.float64), B, n, d, kernel_id, _p(raw, torch.float32), _p(K),
                                        _p(dK), _stream()), "gpsr_covariance_grad")
    return unblock(K), unblock(dK)


def invert_(A):
    """In-place on a row-major [B,N,N] tensor: A[b] <- -inv(A[b]) (lower block-triangle).  Returns logdet, flags.
    (The library works on the tile-blocked layout: converted on the way in and out.)"""
    lib = _lib.load()
    B, N, _ = A.shape
    nbytes = lib.gpsr_invert_workspace_bytes(B, N)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=A.device)
    logdet = torch.empty(B, dtype=torch.float64, device=A.device)
    flags = torch.empty(B, dtype=torch.int32, device=A.device)
    Ab = block(A)
    _lib.check(lib.gpsr_invert(_p(Ab, torch.float64), B, N, _p(logdet), _p(flags), _p(ws), nbytes, _stream()),
               "gpsr_invert")
    A.copy_(unblock(Ab))
    return logdet, flags


def fit_workspace(B, n, d, device):
    lib = _lib.load()
    nbytes = lib.gpsr_fit_workspace_bytes(B, n, d)
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def fit(X, y, kernel_id, raw, iters=50, lr=0.1, workspace=None, want_loss=False):
    """Adam fit in place on raw [B,4]; returns alpha [B,N], flags [B] (, loss [B])."""
    lib = _lib.load()
    B, n, d = X.shape
    N = padded_n(n)
    if workspace is None:
        workspace = fit_workspace(B, n, d, X.device)
    alpha = torch.empty((B, N), dtype=torch.float64, device=X.device)
    flags = torch.empty(B, dtype=torch.int32, device=X.device)
    loss = torch.empty(B, dtype=torch.float64, device=X.device) if want_loss else None
    _lib.check(lib.gpsr_fit(_p(X, torch.float64), _p(y, torch.float64), B, n, d, kernel_id, _p(raw, torch.float32),
                            iters, float(lr), _p(alpha), _p(loss), _p(flags), _p(workspace), workspace.numel(),
                            _stream()), "gpsr_fit")
    return (alpha, flags, loss) if want_loss else (alpha, flags)


def set_dual_stream(on):
    """gpsr_set_dual_stream: two half-batches on two streams inside gpsr_fit (opt-in). Returns the previous setting."""
    return bool(_lib.load().gpsr_set_dual_stream(1 if on else 0))


def set_split_small(on):
    """gpsr_set_split_small: the small launches of a big batch as two halves on two streams (default on). Returns the previous setting."""
    return bool(_lib.load().gpsr_set_split_small(1 if on else 0))


def set_fused(on):
    """gpsr_set_fused: the one-launch per-GP route of gpsr_fit (opt-in, bit-identical, measured slower). Returns the previous setting."""
    return bool(_lib.load().gpsr_set_fused(1 if on else 0))


def loss_grad(X, y, kernel_id, raw, workspace=None):
    lib = _lib.load()
    B, n, d = X.shape
    if workspace is None:
        workspace = fit_workspace(B, n, d, X.device)
    loss = torch.empty(B, dtype=torch.float64, device=X.device)
    grad = torch.empty((B, 4), dtype=torch.float32, device=X.device)
    flags = torch.empty(B, dtype=torch.int32, device=X.device)
    _lib.check(lib.gpsr_loss_grad(_p(X, torch.float64), _p(y, torch.float64), B, n, d, kernel_id,
                                  _p(raw, torch.float32), _p(loss), _p(grad), _p(flags), _p(workspace),
                                  workspace.numel(), _stream()), "gpsr_loss_grad")
    return loss, grad, flags


def predict(X, Xs, alpha, raw, kernel_id):
    lib = _lib.load()
    B, n, d = X.shape
    if d != 8:
        raise _lib.GpsrError("gpsr_predict needs d == 8")
    m = Xs.shape[1]
    out = torch.empty((B, m), dtype=torch.float64, device=X.device)
    _lib.check(lib.gpsr_predict(_p(X, torch.float64), _p(Xs, torch.float64), _p(alpha, torch.float64),
                                _p(raw, torch.float32), B, n, m, kernel_id, _p(out), _stream()), "gpsr_predict")
    return out


def combine(pred, test_in, H, W, s, p, rows, cols, mode=AVERAGE, clip=True):
    """test_in=None: pred holds whole [B,P,P] patches (PatchHandler.combine_patches)."""
    lib = _lib.load()
    out = torch.empty((H * s, W * s), dtype=torch.float64, device=pred.device)
    _lib.check(lib.gpsr_combine(_p(pred, torch.float64), _p(test_in, torch.float64), H, W, s, p,
                                _p(rows, torch.int32), rows.numel(), _p(cols, torch.int32), cols.numel(), mode,
                                int(clip), _p(out), _stream()), "gpsr_combine")
    return out


def predict_pixels_fused(train_in, train_tgt, test_in, s, p, rows, cols, tidx, kernel_id, init_raw_os=0.0,
                         init_raw_ls=0.0, iters=50, lr=0.1, mode=AVERAGE, chunk=0):
    """One-call GPRSR.predict_pixels for one image (gpsr_predict_pixels) -> out [H*s,W*s], raw [B,4], flags [B]."""
    lib = _lib.load()
    H, W = train_in.shape
    nr, nc, nt = rows.numel(), cols.numel(), tidx.numel()
    B = nr * nc
    dev = train_in.device
    nbytes = lib.gpsr_predict_pixels_workspace_bytes(s, p, nt, B, chunk)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    out = torch.empty((H * s, W * s), dtype=torch.float64, device=dev)
    raw = torch.empty((B, 4), dtype=torch.float32, device=dev)
    flags = torch.empty(B, dtype=torch.int32, device=dev)
    _lib.check(lib.gpsr_predict_pixels(_p(train_in, torch.float64), _p(train_tgt, torch.float64),
                                       _p(test_in, torch.float64), H, W, s, p, _p(rows, torch.int32), nr,
                                       _p(cols, torch.int32), nc, _p(tidx, torch.int32), nt, kernel_id,
                                       float(init_raw_os), float(init_raw_ls), iters, float(lr), mode, chunk,
                                       _p(out), _p(raw), _p(flags), _p(ws), nbytes, _stream()), "gpsr_predict_pixels")
    return out, raw, flags


def agpr_weights(X, alpha, raw):
    lib = _lib.load()
    n, d = X.shape
    w = torch.empty(d, dtype=torch.float64, device=X.device)
    _lib.check(lib.gpsr_agpr_weights(_p(X, torch.float64), _p(alpha, torch.float64), _p(raw, torch.float32), n, d,
                                     _p(w), _stream()), "gpsr_agpr_weights")
    return w


def agpr_filter(img, L, w, raw):
    lib = _lib.load()
    Hs, Ws = img.shape
    out = torch.empty_like(img)
    _lib.check(lib.gpsr_agpr_filter(_p(img, torch.float64), Hs, Ws, L, _p(w, torch.float64), _p(raw, torch.float32),
                                    _p(out), _stream()), "gpsr_agpr_filter")
    return out


def selftest_mfma(A, Bm):
    lib = _lib.load()
    D = torch.empty((16, 16), dtype=torch.float64, device=A.device)
    _lib.check(lib.gpsr_selftest_mfma(_p(A, torch.float64), _p(Bm, torch.float64), _p(D), _stream()),
               "gpsr_selftest_mfma")
    return D


# ------------------------------------------------------------ image stages
def u8_to_unit(img_u8):
    lib = _lib.load()
    out = torch.empty(img_u8.shape, dtype=torch.float64, device=img_u8.device)
    _lib.check(lib.gpsr_u8_to_unit(_p(img_u8, torch.uint8), _p(out), img_u8.numel(), _stream()), "gpsr_u8_to_unit")
    return out


def unit_to_u8(img, scale=255.0):
    lib = _lib.load()
    out = torch.empty(img.shape, dtype=torch.uint8, device=img.device)
    _lib.check(lib.gpsr_unit_to_u8(_p(img, torch.float64), _p(out), img.numel(), float(scale), _stream()),
               "gpsr_unit_to_u8")
    return out


def resample(img, Hd, Wd, xi, xw, yi, yw):
    lib = _lib.load()
    Hs, Ws = img.shape
    taps = xi.shape[1]
    out = torch.empty((Hd, Wd), dtype=torch.float64, device=img.device)
    _lib.check(lib.gpsr_resample(_p(img, torch.float64), Hs, Ws, _p(out), Hd, Wd, _p(xi, torch.int32),
                                 _p(xw, torch.float64), _p(yi, torch.int32), _p(yw, torch.float64), taps,
                                 _stream()), "gpsr_resample")
    return out


def decimate2(img):
    lib = _lib.load()
    Hs, Ws = img.shape
    out = torch.empty((Hs // 2, Ws // 2), dtype=torch.float64, device=img.device)
    _lib.check(lib.gpsr_decimate2(_p(img, torch.float64), Hs, Ws, _p(out), _stream()), "gpsr_decimate2")
    return out


def sepfilter_sym(img, kern):
    lib = _lib.load()
    H, W = img.shape
    out = torch.empty_like(img)
    _lib.check(lib.gpsr_sepfilter_sym(_p(img, torch.float64), H, W, _p(out), _p(kern, torch.float64), kern.numel(),
                                      _stream()), "gpsr_sepfilter_sym")
    return out


def filter3x3(img, kern):
    lib = _lib.load()
    H, W = img.shape
    out = torch.empty_like(img)
    _lib.check(lib.gpsr_filter3x3(_p(img, torch.float64), H, W, _p(out), _p(kern, torch.float64), _stream()),
               "gpsr_filter3x3")
    return out


def axpy(a, b, alpha):
    lib = _lib.load()
    out = torch.empty_like(a)
    _lib.check(lib.gpsr_axpy(_p(a, torch.float64), _p(b, torch.float64), float(alpha), _p(out), a.numel(), _stream()),
               "gpsr_axpy")
    return out


# ------------------------------------------------------------ uint8 colour stages + metrics
def bgr2gray(bgr):
    """[H,W,3] uint8 device (cv.imread layout) -> [H,W] uint8   (gpsr_bgr2gray)."""
    lib = _lib.load()
    H, W, _ = bgr.shape
    out = torch.empty((H, W), dtype=torch.uint8, device=bgr.device)
    _lib.check(lib.gpsr_bgr2gray(_p(bgr, torch.uint8), _p(out), H * W, _stream()), "gpsr_bgr2gray")
    return out


def _split3(fn, name, bgr):
    H, W, _ = bgr.shape
    planes = [torch.empty((H, W), dtype=torch.uint8, device=bgr.device) for _ in range(3)]
    _lib.check(fn(_p(bgr, torch.uint8), _p(planes[0]), _p(planes[1]), _p(planes[2]), H * W, _stream()), name)
    return planes


def _merge3(fn, name, a, b, c):
    H, W = a.shape
    out = torch.empty((H, W, 3), dtype=torch.uint8, device=a.device)
    _lib.check(fn(_p(a, torch.uint8), _p(b, torch.uint8), _p(c, torch.uint8), _p(out), H * W, _stream()), name)
    return out


def bgr2yuv(bgr):
    return _split3(_lib.load().gpsr_bgr2yuv, "gpsr_bgr2yuv", bgr)


def yuv2bgr(y, u, v):
    return _merge3(_lib.load().gpsr_yuv2bgr, "gpsr_yuv2bgr", y, u, v)


def bgr2ycrcb(bgr):
    return _split3(_lib.load().gpsr_bgr2ycrcb, "gpsr_bgr2ycrcb", bgr)


def ycrcb2bgr(y, cr, cb):
    return _merge3(_lib.load().gpsr_ycrcb2bgr, "gpsr_ycrcb2bgr", y, cr, cb)


def resample_u8(img, Hd, Wd, xi, xw, yi, yw):
    lib = _lib.load()
    Hs, Ws = img.shape
    out = torch.empty((Hd, Wd), dtype=torch.uint8, device=img.device)
    _lib.check(lib.gpsr_resample_u8(_p(img, torch.uint8), Hs, Ws, _p(out), Hd, Wd, _p(xi, torch.int32),
                                    _p(xw, torch.float32), _p(yi, torch.int32), _p(yw, torch.float32), _stream()),
               "gpsr_resample_u8")
    return out


def sepfilter_u8(img, kern):
    """uint8 device plane [H,W], int32 fixed-point taps (sum 256) -> blurred uint8 plane (gpsr_sepfilter_u8)."""
    lib = _lib.load()
    H, W = img.shape
    out = torch.empty_like(img)
    _lib.check(lib.gpsr_sepfilter_u8(_p(img, torch.uint8), H, W, _p(out), _p(kern, torch.int32), kern.numel(), _stream()),
               "gpsr_sepfilter_u8")
    return out


def metrics(a, b, crop):
    """Two [H,W] uint8 device images -> device float64 [3] = (PSNR dB, SSIM, MSE) after cropping (gpsr_metrics)."""
    lib = _lib.load()
    H, W = a.shape
    if b.shape != a.shape:
        raise _lib.GpsrError(f"metrics: shapes differ {tuple(a.shape)} vs {tuple(b.shape)}")
    nbytes = lib.gpsr_metrics_workspace_bytes(H, W, crop)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=a.device)
    out = torch.empty(3, dtype=torch.float64, device=a.device)
    _lib.check(lib.gpsr_metrics(_p(a, torch.uint8), _p(b, torch.uint8), H, W, crop, _p(out), _p(ws), nbytes, _stream()),
               "gpsr_metrics")
    return out


def active_sample(data, K, n_pick, bandwidth, w_rep, w_div):
    """[N,D] float64 device rows -> (int32 [n_pick] chosen row indices in the order chosen, float64 [N]
    representativeness scores): the training-set selection of agpr.py:120-137 (gpsr_active_sample)."""
    lib = _lib.load()
    N, D = data.shape
    nbytes = lib.gpsr_active_sample_workspace_bytes(N)
    ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=data.device)
    idx = torch.empty(n_pick, dtype=torch.int32, device=data.device)
    rep = torch.empty(N, dtype=torch.float64, device=data.device)
    _lib.check(lib.gpsr_active_sample(_p(data, torch.float64), N, D, int(K), int(n_pick), float(bandwidth), float(w_rep), float(w_div),
                                      _p(idx, torch.int32), _p(rep), _p(ws), nbytes, _stream()), "gpsr_active_sample")
    return idx, rep


# ------------------------------------------------------------ example bank
BANK_GROUP = 32                              # columns that share a scale byte
BANK_DIMS = (32, 64, 96, 128, 192, 256)
BANK_PAGE_ROWS = (16, 32, 64, 128, 256)
_BANK_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_I64x3 = ctypes.c_int64 * 3


class Bank(NamedTuple):
    """Example windows in 4 or 8 bits (gpsr_bank of include/gpsr.h): the arrays of a bank, which bank_write fills and the
    other bank_* functions read.  codes [pages,H,P,D*bits/8] uint8, scales [pages,H,P,D/32] uint8, offset [pages,H,P]
    and centroid [pages,H,D] float32; kernel_id RBF or LINEAR.  bank_alloc makes an empty one.
    There are no gradients through a bank: rows and queries that ask for one are refused."""
    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor
    offset: torch.Tensor
    centroid: torch.Tensor
    bits: int = 4
    kernel_id: int = RBF


def bank_alloc(pages, heads, dim, page_rows=64, bits=4, kernel_id=RBF, device=None):
    """An empty Bank: `pages` pages of `page_rows` rows for each of `heads` heads, `dim` columns for keys and for values."""
    if bits not in (4, 8) or dim not in BANK_DIMS or page_rows not in BANK_PAGE_ROWS or pages < 1 or heads < 1:
        raise _lib.GpsrError(f"bank_alloc: pages={pages}, heads={heads}, dim={dim} (one of {BANK_DIMS}), page_rows={page_rows} "
                             f"(one of {BANK_PAGE_ROWS}), bits={bits} (4 or 8)")
    if kernel_id not in (RBF, LINEAR):
        raise _lib.GpsrError("bank_alloc: kernel_id must be RBF or LINEAR")
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    u8 = lambda n: torch.zeros((pages, heads, page_rows, n), dtype=torch.uint8, device=device)
    f32 = lambda n: torch.zeros((pages, heads, n), dtype=torch.float32, device=device)
    width, groups = dim * bits // 8, dim // BANK_GROUP
    return Bank(u8(width), u8(groups), u8(width), u8(groups), f32(page_rows), f32(dim), bits, kernel_id)


# The bank_* calls take a dozen tensors and some of them run for a few microseconds: the checks below ask torch as little as
# they can and leave the words of a refusal to _p.
def _ptr(t, dtype, dev):
    if t.get_device() != dev or t.dtype is not dtype or not t.is_contiguous():
        return _p(t, dtype)
    return t.data_ptr()


def _no_grad(t, what):
    if t.requires_grad and torch.is_grad_enabled():
        raise _lib.GpsrError(f"{what}: there are no gradients through an example bank (detach it, or call under torch.no_grad())")


def _bank_device(t):
    dev = t.get_device()
    if dev < 0 or dev != torch.cuda.current_device():
        _p(t)                            # says what is wrong
    return dev


def _bank(bank, dev):
    """The checked gpsr_bank of a Bank, and its heads and dim."""
    kc, ks, vc, vs, off, cent, bits, kernel_id = bank
    if kc.dim() != 4 or bits not in (4, 8):
        raise _lib.GpsrError(f"bank: bits must be 4 or 8 and codes [pages,H,P,width], got {bits}, {tuple(kc.shape)}")
    pages, H, P, width = shape = kc.shape
    if H < 1:
        raise _lib.GpsrError("bank: no heads")
    D = width * 8 // bits
    groups = (pages, H, P, D // BANK_GROUP)
    if vc.shape != shape or ks.shape != groups or vs.shape != groups or off.shape != (pages, H, P) or cent.shape != (pages, H, D):
        raise _lib.GpsrError(f"bank: array shapes {[tuple(t.shape) for t in bank[:6]]} do not belong together")
    u8, f32 = torch.uint8, torch.float32
    return ctypes.byref(_lib.Bank(_ptr(kc, u8, dev), _ptr(ks, u8, dev), _ptr(vc, u8, dev), _ptr(vs, u8, dev), _ptr(off, f32, dev),
                                  _ptr(cent, f32, dev), pages, H, P, D, bits, kernel_id)), H, D


def _rows_fit(n, what):
    if not 0 <= n < 2 ** 31:      # ctypes would pass the low 32 bits on
        raise _lib.GpsrError(f"{what}: from 0 to 2^31 - 1 rows in one call, got {n}")


def _strided(t, B, H, D, dev, what):
    """Pointer, dtype code and (first three) element strides of a [B,T,H,D] tensor whose columns are contiguous (H None: any)."""
    shape = t.shape
    if len(shape) != 4 or shape[0] != B or shape[3] != D or (H is not None and shape[2] != H):
        raise _lib.GpsrError(f"{what}: expected [{B},T,{'heads' if H is None else H},{D}], got {tuple(shape)}")
    code = _BANK_TYPES.get(t.dtype)
    if code is None:
        raise _lib.GpsrError(f"{what}: expected bfloat16, float16 or float32, got {t.dtype}")
    _rows_fit(shape[1], what)
    sb, st, sh, sd = t.stride()
    if sd != 1:
        raise _lib.GpsrError(f"{what}: the columns must be contiguous")
    if t.get_device() != dev:
        _p(t.as_strided((0,), (1,)))     # says what is wrong
    _no_grad(t, what)
    return t.data_ptr(), code, _I64x3(sb, st, sh)


def _bank_index(table, per_entry, dev, what):
    """Pointers of table [B,J] and of one int32 per entry."""
    shape = table.shape
    if len(shape) == 2:
        B = shape[:1]
        fits = True
        for t in per_entry:
            fits = fits and t.shape == B
    if len(shape) != 2 or not fits:
        raise _lib.GpsrError(f"{what}: expected a [B,J] table and [B] integers, got {tuple(table.shape)}, "
                             f"{[tuple(t.shape) for t in per_entry]}")
    if shape[1] >= 2 ** 31:
        raise _lib.GpsrError(f"{what}: a table of at most 2^31 - 1 pages an entry, got {shape[1]}")
    i32 = torch.int32
    return (_ptr(table, i32, dev), *[_ptr(t, i32, dev) for t in per_entry])


def bank_write(bank, table, start, count, k, v):
    """Rounds rows k, v [B,T,H,D] (bfloat16 / float16 / float32, any strides with contiguous columns) into the bank, in place:
    row t < count[b] goes to position start[b] + t of entry b, whose pages table [B,J] (int32) names; refreshes offsets and
    centroids (gpsr_bank_write).  A page may be written by one entry of a call only."""
    lib, dev = _lib.load(), _bank_device(table)
    ref, H, D = _bank(bank, dev)
    tp, sp, cp = _bank_index(table, (start, count), dev, "bank_write")
    B, J = table.shape
    kp, code, kst = _strided(k, B, H, D, dev, "bank_write: k")
    if v.shape != k.shape or v.dtype is not k.dtype:
        raise _lib.GpsrError(f"bank_write: v {tuple(v.shape)} {v.dtype} does not fit k {tuple(k.shape)} {k.dtype}")
    vp, _, vst = _strided(v, B, H, D, dev, "bank_write: v")
    _lib.check(lib.gpsr_bank_write(ref, tp, B, J, sp, cp, kp, vp, code, k.shape[1], kst, vst, _stream()), "gpsr_bank_write")


def bank_read(bank, table, start, count, rows, dtype=torch.float32):
    """-> k, v [B,rows,H,D]: the values that positions start[b] .. start[b] + count[b] - 1 hold, zeros behind them (gpsr_bank_read)."""
    lib, dev = _lib.load(), _bank_device(table)
    ref, H, D = _bank(bank, dev)
    tp, sp, cp = _bank_index(table, (start, count), dev, "bank_read")
    code = _BANK_TYPES.get(dtype)
    if code is None:
        raise _lib.GpsrError(f"bank_read: expected bfloat16, float16 or float32, got {dtype}")
    _rows_fit(rows, "bank_read")
    B, J = table.shape
    k = table.new_empty((B, rows, H, D), dtype=dtype)
    v = torch.empty_like(k)
    _lib.check(lib.gpsr_bank_read(ref, tp, B, J, sp, cp, k.data_ptr(), v.data_ptr(), code, rows, _stream()), "gpsr_bank_read")
    return k, v


def _bank_query(bank, table, length, q, skip, what):
    """(the arguments up to q's strides, q's sizes, pointer of skip, the library, the device)."""
    lib, dev = _lib.load(), _bank_device(table)
    ref, H, D = _bank(bank, dev)
    tp, lp = _bank_index(table, (length,), dev, what)
    B, J = table.shape
    qp, code, qst = _strided(q, B, None, D, dev, what + ": q")
    T, Hq = q.shape[1], q.shape[2]
    if Hq < 1 or Hq % H:
        raise _lib.GpsrError(f"{what}: {Hq} query heads are no multiple of the bank's {H}")
    if skip is not None and skip.shape != (B, T, 2):
        raise _lib.GpsrError(f"{what}: skip must be [{B},{T},2], got {tuple(skip.shape)}")
    sk = None if skip is None else _ptr(skip, torch.int32, dev)
    return (ref, tp, B, J, lp, qp, code, T, Hq, qst), (ref, B, J, T, Hq), (B, T, H, Hq, D), code, sk, lib, dev


def _bank_out(q, want_lse, B, T, Hq):
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((B, Hq, T), dtype=torch.float32) if want_lse else None
    return out, lse, None if lse is None else lse.data_ptr()


def _bank_workspace(nbytes, q):
    if not nbytes:
        return None, None
    ws = q.new_empty(nbytes, dtype=torch.uint8)
    return ws, ws.data_ptr()


def bank_attend(bank, table, length, q, scale, skip=None, want_lse=False):
    """q [B,T,Hq,D] -> out [B,T,Hq,D]: the mean of the values of entry b's first length[b] rows, weighted by
    exp(-scale |q - k|^2 / 2) (RBF) or exp(scale q.k) (LINEAR); with want_lse also the log of the sum of the weights
    [B,Hq,T] (RBF: without its factor exp(-scale |q|^2 / 2)).  skip [B,T,2] int32: positions lo <= r < hi that a query does
    not see; one that sees none gets zeros and -inf (gpsr_bank_attend)."""
    args, sizes, (B, T, H, Hq, D), code, sk, lib, dev = _bank_query(bank, table, length, q, skip, "bank_attend")
    out, lse, lse_p = _bank_out(q, want_lse, B, T, Hq)
    nbytes = lib.gpsr_bank_attend_workspace_bytes(*sizes, code)
    ws, ws_p = _bank_workspace(nbytes, q)
    _lib.check(lib.gpsr_bank_attend(*args, scale, sk, out.data_ptr(), lse_p, ws_p, nbytes, _stream()), "gpsr_bank_attend")
    return (out, lse) if want_lse else out


def bank_select(bank, table, length, q, n_sel, skip=None):
    """-> int32 [B,T,H,n_sel]: the n_sel (1..64) pages of entry b (columns of its table row) whose centroids suit the query
    best, ascending, -1 behind the last; the heads that share a bank head choose together (gpsr_bank_select)."""
    args, sizes, (B, T, H, Hq, D), code, sk, lib, dev = _bank_query(bank, table, length, q, skip, "bank_select")
    if not 1 <= n_sel <= 64:
        raise _lib.GpsrError(f"bank_select: n_sel must be in 1..64, got {n_sel}")
    sel = q.new_empty((B, T, H, n_sel), dtype=torch.int32)
    nbytes = lib.gpsr_bank_select_workspace_bytes(*sizes, n_sel, code)
    ws, ws_p = _bank_workspace(nbytes, q)
    _lib.check(lib.gpsr_bank_select(*args, n_sel, sk, sel.data_ptr(), ws_p, nbytes, _stream()), "gpsr_bank_select")
    return sel


def bank_attend_pages(bank, table, length, q, pages, scale, skip=None, want_lse=False):
    """bank_attend over the rows of each query's own pages [B,T,H,S] (S in 1..64; bank_select gives them) only.  Numbers outside the
    table and repeats are passed over (gpsr_bank_attend_pages)."""
    args, sizes, (B, T, H, Hq, D), code, sk, lib, dev = _bank_query(bank, table, length, q, skip, "bank_attend_pages")
    if pages.dim() != 4 or pages.shape[:3] != (B, T, H) or not 1 <= pages.shape[3] <= 64:
        raise _lib.GpsrError(f"bank_attend_pages: pages must be [{B},{T},{H},1..64], got {tuple(pages.shape)}")
    pp, n_sel = _ptr(pages, torch.int32, dev), pages.shape[3]
    out, lse, lse_p = _bank_out(q, want_lse, B, T, Hq)
    nbytes = lib.gpsr_bank_attend_pages_workspace_bytes(*sizes, n_sel, code)
    ws, ws_p = _bank_workspace(nbytes, q)
    _lib.check(lib.gpsr_bank_attend_pages(*args, pp, n_sel, scale, sk, out.data_ptr(), lse_p, ws_p, nbytes, _stream()),
               "gpsr_bank_attend_pages")
    return (out, lse) if want_lse else out


def bank_windows(img, side, dim, dtype=torch.bfloat16, centre=False):
    """float64 [H,W] -> [1,(H-side+1)*(W-side+1),1,dim]: the side x side window of every pixel that has a whole one, zeros behind
    its side*side columns; centre: less its own mean (gpsr_bank_windows)."""
    lib = _lib.load()
    H, W = img.shape
    if dtype not in _BANK_TYPES:
        raise _lib.GpsrError(f"bank_windows: expected bfloat16, float16 or float32, got {dtype}")
    _no_grad(img, "bank_windows: img")
    n = max(H - side + 1, 0) * max(W - side + 1, 0)
    out = torch.empty((1, n, 1, dim), dtype=dtype, device=img.device)
    _lib.check(lib.gpsr_bank_windows(_p(img, torch.float64), H, W, side, int(centre), out.data_ptr(), _BANK_TYPES[dtype], dim, _stream()),
               "gpsr_bank_windows")
    return out


def bank_blend(img, detail, side):
    """img [H,W] + the mean of what the windows that hold a pixel say about it; detail as bank_windows lays windows out (gpsr_bank_blend)."""
    lib = _lib.load()
    H, W = img.shape
    n = max(H - side + 1, 0) * max(W - side + 1, 0)
    dim = detail.shape[-1]
    if detail.numel() != n * dim or detail.dtype not in _BANK_TYPES:
        raise _lib.GpsrError(f"bank_blend: detail {tuple(detail.shape)} {detail.dtype} does not fit {H} x {W} and side {side}")
    _no_grad(img, "bank_blend: img")
    _no_grad(detail, "bank_blend: detail")
    out = torch.empty_like(img)
    _lib.check(lib.gpsr_bank_blend(_p(img, torch.float64), H, W, side, _p(detail), _BANK_TYPES[detail.dtype], dim, out.data_ptr(),
                                   _stream()), "gpsr_bank_blend")
    return out


# ------------------------------------------------------------ kernel timing
PROF_TAGS = ("update", "panel", "pivot", "build", "grad1", "grad2", "predict", "update_last", "update2", "update_sel", "fused")


def profile_begin(max_records=65536, tags=None):
    """tags: names out of PROF_TAGS to bracket (None: all).  Two event records per bracketed launch."""
    lib = _lib.load()
    mask = 0xFFFFFFFF if tags is None else sum(1 << PROF_TAGS.index(t) for t in tags)
    _lib.check(lib.gpsr_profile_select(mask), "gpsr_profile_select")
    _lib.check(lib.gpsr_profile_begin(int(max_records)), "gpsr_profile_begin")


def profile_end():
    """-> {tag: (launch_count, total_ms)} measured with HIP events on the launch stream."""
    import ctypes
    n = len(PROF_TAGS)
    counts = (ctypes.c_int32 * n)()
    ms = (ctypes.c_double * n)()
    _lib.check(_lib.load().gpsr_profile_end(ctypes.cast(counts, ctypes.c_void_p), ctypes.cast(ms, ctypes.c_void_p)),
               "gpsr_profile_end")
    return {t: (int(counts[i]), float(ms[i])) for i, t in enumerate(PROF_TAGS)}
