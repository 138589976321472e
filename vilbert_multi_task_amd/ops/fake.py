"""What the block-scaled operators and the root-mean-square norm return, by sizes and
types alone: for fake tensors, tracing and shape inference. Registered when the
extension is loaded; the checks are those of the plain forms.
"""

from __future__ import annotations

import torch

from . import functional as F_ops


def _rows8(x, sizes):
    """8-bit rows that begin at multiples of 16 bytes."""
    *lead, k = sizes
    pitch = (k + 15) // 16 * 16
    y = x.new_empty((*lead, pitch), dtype=torch.float8_e4m3fn)
    return y if pitch == k else y.narrow(-1, 0, k)


def _scales(x, sizes, f32):
    *lead, k = sizes
    dtype = torch.float32 if f32 else torch.bfloat16
    return x.new_empty((*lead, -(-k // F_ops.FP8_BLOCK)), dtype=dtype)


def _like(x):
    return x.new_empty(x.shape)


def _check_rms(x, w, res):
    F_ops._check_rows("rms_norm", x)  # its plain form takes 64 bits too
    F_ops._check_norm("rms_norm", x, w, res)


def _rms_norm(x, w, eps):
    _check_rms(x, w, None)
    return _like(x)


def _rms_norm_residual(x, res, w, eps):
    _check_rms(x, w, res)
    return _like(x), _like(x)


def _rms_fwd_train(x, res, w, eps):
    _check_rms(x, w, res)
    total = x.new_empty((0,)) if res is None else _like(x)
    return _like(x), total, x.new_empty((x.numel() // x.shape[-1],), dtype=torch.float32)


def _rms_bwd(gy, gsum, t, rstd, w):
    F_ops._check_norm("rms_bwd", t, w, gy)
    F_ops._check_norm("rms_bwd", t, w, gsum)
    return _like(t), _like(w)


def _rms_norm_fp8_block(x, res, w, eps, f32_scales=False):
    F_ops._check_norm("rms_norm_fp8_block", x, w, res)
    total = x.new_empty((0,)) if res is None else _like(x)
    return _rows8(x, x.shape), _scales(x, x.shape, f32_scales), total


def _layer_norm_fp8_block(x, res, w, b, eps, f32_scales=False):
    F_ops._check_norm("layer_norm_fp8_block", x, w, res, b)
    return _like(x), _rows8(x, x.shape), _scales(x, x.shape, f32_scales)


def _quantize_fp8_block(x, f32_scales=False):
    F_ops._check_rows("quantize_fp8_block", x)
    return _rows8(x, x.shape), _scales(x, x.shape, f32_scales)


def _quantize_fp8_block_weight(w, f32_scales=False):
    F_ops._check_weight(w)
    n, k = w.shape
    return _rows8(w, w.shape), _scales(w, (-(-n // F_ops.FP8_BLOCK), k), f32_scales)


def _fp8_block_linear(x8, x_scales, w8, w_scales, bias, gelu, f32_out=False):
    F_ops._check_product("fp8_block_linear", x8, x_scales, w8, w_scales, bias)
    dtype = torch.float32 if f32_out else torch.bfloat16
    return x8.new_empty((*x8.shape[:-1], w8.shape[0]), dtype=dtype)


def _fp8_block_linear_fp8(x8, x_scales, w8, w_scales, bias, gelu):
    F_ops._check_product("fp8_block_linear_fp8", x8, x_scales, w8, w_scales, bias)
    sizes = (*x8.shape[:-1], w8.shape[0])
    return _rows8(x8, sizes), _scales(x8, sizes, x_scales.dtype == torch.float32)


_REGISTERED = False


def register() -> None:
    global _REGISTERED
    if _REGISTERED:
        return
    for f in (
        _rms_norm, _rms_norm_residual, _rms_fwd_train, _rms_bwd, _rms_norm_fp8_block,
        _layer_norm_fp8_block, _quantize_fp8_block, _quantize_fp8_block_weight,
        _fp8_block_linear, _fp8_block_linear_fp8,
    ):
        torch.library.register_fake(f"vilbert_amd::{f.__name__[1:]}", f)
    _REGISTERED = True
