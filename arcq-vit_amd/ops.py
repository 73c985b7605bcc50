"""Operator layer: the reference extension's eight functions, same names, argument order and
returns, on top of ``libarcq_hip.so``.

Reference binding table: FQ/arcq_infer_cuda/arcq_infer_bind.cpp:57-66 (``FQ`` =
``methods/fair_qat_framework/fair_qat``).  Also here: the two launchers of
FQ/arcq_packed_triton.py (``unpack_weight_triton`` :77-120, ``dequant_activation_triton``
:181-215) under HIP names, and the fused entry points that have no counterpart in the
reference (``linear_fused``, ``linear_otf``).

All tensors must live on the GPU; outputs are allocated with torch on the same device and the
kernels are enqueued on torch's current stream.  Nothing here synchronises.
"""
from __future__ import annotations

import ctypes
import math
from typing import List, NamedTuple, Optional, Sequence

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import ARCQ_F16, ARCQ_F32


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _check(cond: bool, msg: str) -> None:
    # TORCH_CHECK raises c10::Error, which Python sees as RuntimeError.
    if not cond:
        raise RuntimeError(msg)


def _dtype_code(t: torch.Tensor, name: str) -> int:
    if t.dtype == torch.float32:
        return ARCQ_F32
    if t.dtype == torch.float16:
        return ARCQ_F16
    raise RuntimeError(f"{name} must be float32 or float16")


def _check_bits(bits: int) -> None:
    _check(bits in (2, 3, 4), "bits must be 2, 3, or 4")


def _f32c(t: torch.Tensor) -> torch.Tensor:
    return t.to(torch.float32).contiguous()


def _check_weights(n: int, k: int, group_size: int, center: torch.Tensor, scale: torch.Tensor, code_sum: torch.Tensor,
                   bias: Optional[torch.Tensor]) -> None:
    """The per-group metadata and the bias are on a GPU and hold at least what the kernels read for ``[n, k]`` weights."""
    need = n * (k // max(int(group_size), 1))
    for name, t in (("w_center", center), ("w_scale", scale), ("w_code_sum", code_sum)):
        _check(t.is_cuda, f"{name} must be CUDA tensor")
        _check(t.numel() >= need, f"{name} has {t.numel()} entries, {need} needed for [out_features, groups]")
    if bias is not None and bias.numel() > 0:
        _check(bias.is_cuda, "bias must be CUDA tensor")
        _check(bias.numel() >= n, "bias must have out_features entries")


def _check_codebooks(bits: int, w_codebook: Optional[torch.Tensor], a_thresholds: Optional[torch.Tensor] = None,
                     a_codebook: Optional[torch.Tensor] = None) -> None:
    for name, t, need in (("w_codebook", w_codebook, 1 << bits), ("a_thresholds", a_thresholds, (1 << bits) - 1),
                          ("a_codebook", a_codebook, 1 << bits)):
        _check(t is None or t.is_cuda, f"{name} must be CUDA tensor")
        _check(t is None or t.numel() >= need, f"{name} must have {need} entries for {bits}-bit codes")


# ---------------------------------------------------------------------------------------------
# bit packing -- EXT/arcq_pack_kernel.cu:94-158
# ---------------------------------------------------------------------------------------------
def pack_codes(codes: torch.Tensor, bits: int) -> torch.Tensor:
    """int codes ``[rows, length]`` -> ``uint8 [rows, ceil(length*bits/8)]`` (LSB-first bitstream)."""
    _check(codes.is_cuda, "codes must be CUDA tensor")
    _check_bits(bits)
    _check(codes.dim() == 2, "codes must have shape [rows, length]")
    c = codes.to(torch.int64).contiguous()
    rows, length = c.shape
    packed = torch.empty((rows, (length * bits + 7) // 8), dtype=torch.uint8, device=c.device)
    with torch.cuda.device(c.device):
        _lib.check(_lib.load().arcq_pack_codes(_ptr(c), _ptr(packed), rows, length, bits, _stream()))
    return packed


def _unpack(packed: torch.Tensor, bits: int, length: int, out_dtype: torch.dtype) -> torch.Tensor:
    _check(packed.is_cuda, "packed must be CUDA tensor")
    _check(packed.dtype == torch.uint8, "packed must be uint8")
    _check_bits(bits)
    _check(packed.dim() == 2, "packed must have shape [rows, packed_cols]")
    length = int(length)
    _check(length >= 0 and (length * bits + 7) // 8 <= packed.shape[1], "length exceeds the packed row")
    p = packed.contiguous()
    rows = p.shape[0]
    # The kernels index rows by ceil(length*bits/8); hand them exactly that row pitch.
    pc = (length * bits + 7) // 8
    if p.shape[1] != pc:
        p = p[:, :pc].contiguous()
    codes = torch.empty((rows, length), dtype=out_dtype, device=p.device)
    fn = _lib.load().arcq_unpack_codes if out_dtype == torch.int64 else _lib.load().arcq_unpack_codes_u8
    with torch.cuda.device(p.device):
        _lib.check(fn(_ptr(p), _ptr(codes), rows, length, bits, _stream()))
    return codes


def unpack_codes(packed: torch.Tensor, bits: int, length: int) -> torch.Tensor:
    """Inverse of :func:`pack_codes`, int64 out (EXT/arcq_pack_kernel.cu:116-136)."""
    return _unpack(packed, bits, length, torch.int64)


def unpack_codes_u8(packed: torch.Tensor, bits: int, length: int) -> torch.Tensor:
    """Inverse of :func:`pack_codes`, uint8 out (EXT/arcq_pack_kernel.cu:138-158)."""
    return _unpack(packed, bits, length, torch.uint8)


# ---------------------------------------------------------------------------------------------
# stage 1 -- EXT/arcq_activation_kernel.cu:188-326
# ---------------------------------------------------------------------------------------------
def _act_quant(x: torch.Tensor, thresholds: torch.Tensor, codebook: torch.Tensor, bits: int, group_size: int,
               want_packed: bool = False, want_u8: bool = False, want_meta: bool = False,
               x_hat: Optional[torch.Tensor] = None, strict_f32: bool = True, eps: float = 1.0e-6):
    _check(x.is_cuda, "x must be CUDA tensor")
    _check(thresholds.is_cuda, "thresholds must be CUDA tensor")
    _check(codebook.is_cuda, "codebook must be CUDA tensor")
    _check_bits(bits)
    _check(x.dim() == 2, "x must have shape [rows, cols]")
    if strict_f32:
        _check(x.dtype == torch.float32, "x must be float32")
    _check(thresholds.dtype == torch.float32, "thresholds must be float32")
    _check(codebook.dtype == torch.float32, "codebook must be float32")
    group_size = int(group_size)
    _check(group_size > 0 and x.shape[1] % group_size == 0, "in_features must be divisible by group_size")
    _check(codebook.numel() == (1 << bits), f"codebook must have {1 << bits} entries for {bits}-bit codes")
    _check(thresholds.numel() == codebook.numel() - 1, "thresholds must have one entry fewer than the codebook")
    x = x.contiguous()
    thresholds = thresholds.contiguous()
    codebook = codebook.contiguous()
    rows, cols = x.shape
    groups = cols // group_size
    dev = x.device
    packed = torch.empty((rows, (cols * bits + 7) // 8), dtype=torch.uint8, device=dev) if want_packed else None
    codes = torch.empty((rows, cols), dtype=torch.uint8, device=dev) if want_u8 else None
    center = torch.empty((rows, groups), dtype=torch.float32, device=dev) if want_meta else None
    scale = torch.empty((rows, groups), dtype=torch.float32, device=dev) if want_meta else None
    code_sum = torch.empty((rows, groups), dtype=torch.float32, device=dev) if want_meta else None
    with torch.cuda.device(dev):
        _lib.check(_lib.load().arcq_act_quant(
            _ptr(x), _dtype_code(x, "x"), _ptr(thresholds), _ptr(codebook), _ptr(packed), _ptr(codes), _ptr(center),
            _ptr(scale), _ptr(code_sum), _ptr(x_hat), _dtype_code(x_hat, "x_hat") if x_hat is not None else ARCQ_F32,
            rows, cols, bits, group_size, float(eps), _stream()))
    return packed, codes, center, scale, code_sum


def quantize_activation(x: torch.Tensor, thresholds: torch.Tensor, codebook: torch.Tensor, bits: int,
                        group_size: int) -> List[torch.Tensor]:
    """-> ``[packed u8 [rows, cols*bits/8], center, scale, code_sum f32 [rows, groups]]``
    (EXT/arcq_activation_kernel.cu:188-237)."""
    out = _lib.host().quantize(x, thresholds, codebook, bits, group_size, False)
    if out is not None:
        return out
    packed, _, center, scale, code_sum = _act_quant(x, thresholds, codebook, bits, group_size, want_packed=True,
                                                    want_meta=True)
    return [packed, center, scale, code_sum]


def quantize_activation_u8(x: torch.Tensor, thresholds: torch.Tensor, codebook: torch.Tensor, bits: int,
                           group_size: int) -> List[torch.Tensor]:
    """-> ``[codes u8 [rows, cols], center, scale, code_sum]`` (EXT/arcq_activation_kernel.cu:239-285)."""
    out = _lib.host().quantize(x, thresholds, codebook, bits, group_size, True)
    if out is not None:
        return out
    _, codes, center, scale, code_sum = _act_quant(x, thresholds, codebook, bits, group_size, want_u8=True,
                                                   want_meta=True)
    return [codes, center, scale, code_sum]


def quantize_activation_dequant(x: torch.Tensor, thresholds: torch.Tensor, codebook: torch.Tensor, bits: int,
                                group_size: int) -> torch.Tensor:
    """-> ``x_hat f32 [rows, cols]`` (EXT/arcq_activation_kernel.cu:287-326)."""
    _check(x.is_cuda, "x must be CUDA tensor")
    _check(x.dim() == 2, "x must have shape [rows, cols]")
    _check(x.dtype == torch.float32, "x must be float32")
    x = x.contiguous()
    x_hat = torch.empty_like(x)
    _act_quant(x, thresholds, codebook, bits, group_size, x_hat=x_hat)
    return x_hat


def dequant_activation_hip(x: torch.Tensor, thresholds: torch.Tensor, codebook: torch.Tensor, group_size: int,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Fused quantize+reconstruct, fp16 or fp32, optionally in place (``out=x``).

    Same contract as ``dequant_activation_triton`` (FQ/arcq_packed_triton.py:181-215), including its
    ``out`` checks; statistics are always taken in fp32, also for fp16 input.
    """
    _check(x.dim() == 2, "x must have shape [rows, cols]")
    x = x.contiguous()
    thresholds = thresholds.contiguous().float()
    codebook = codebook.contiguous().float()
    levels = codebook.numel()
    bits = levels.bit_length() - 1
    if out is None:
        out = torch.empty_like(x)
    else:
        if out.shape != x.shape:
            raise ValueError(f"dequant_activation out shape {tuple(out.shape)} != input shape {tuple(x.shape)}")
        if out.dtype != x.dtype:
            raise ValueError(f"dequant_activation out dtype {out.dtype} != input dtype {x.dtype}")
        if not out.is_contiguous():
            raise ValueError("dequant_activation out must be contiguous")
    _act_quant(x, thresholds, codebook, bits, group_size, x_hat=out, strict_f32=False)
    return out


# ---------------------------------------------------------------------------------------------
# stage 2 -- FQ/arcq_packed_triton.py:77-120
# ---------------------------------------------------------------------------------------------
def unpack_weight_hip(packed: torch.Tensor, codebook: torch.Tensor, center: torch.Tensor, scale: torch.Tensor,
                      code_sum: torch.Tensor, bits: int, group_size: int,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """packed codes + metadata -> fp16 weight ``[out_f, in_f]``.

    Same contract as ``unpack_weight_triton``: ``out`` may be a larger flat fp16 buffer shared by all
    layers (FQ/arcq_packed_on_the_fly.py:149-157); the first ``out_f*in_f`` elements are written and the
    buffer itself is returned.
    """
    _check(packed.is_cuda, "packed must be CUDA tensor")
    _check(packed.dtype == torch.uint8, "packed must be uint8")
    _check_bits(bits)
    out_f = packed.shape[0]
    groups = center.shape[1]
    in_f = groups * int(group_size)
    _check(packed.shape[1] == (in_f * bits + 7) // 8, "packed row length does not match in_features*bits/8")
    _check_weights(out_f, in_f, group_size, center, scale, code_sum, None)
    _check_codebooks(bits, codebook)
    packed = packed.contiguous()
    codebook, center, scale, code_sum = _f32c(codebook), _f32c(center), _f32c(scale), _f32c(code_sum)
    if out is None:
        out = torch.empty((out_f, in_f), dtype=torch.float16, device=packed.device)
    else:
        _check(out.is_cuda and out.is_contiguous() and out.numel() >= out_f * in_f, "out buffer too small")
        _check(out.dtype in (torch.float16, torch.float32), "out must be float16 or float32")
    with torch.cuda.device(packed.device):
        _lib.check(_lib.load().arcq_weight_dequant(
            _ptr(packed), _ptr(codebook), _ptr(center), _ptr(scale), _ptr(code_sum), _ptr(out),
            _dtype_code(out, "out"), out_f, in_f, bits, int(group_size), _stream()))
    return out


# Import-compatible aliases for code written against FQ/arcq_packed_triton.py.
dequant_activation_triton = dequant_activation_hip
unpack_weight_triton = unpack_weight_hip


# ---------------------------------------------------------------------------------------------
# stages 2+3 fused / whole layer -- no counterpart function in the reference; they replace the
# unpack + F.linear pair at FQ/arcq_packed_on_the_fly.py:148-160
# ---------------------------------------------------------------------------------------------
def linear_fused(x_hat: torch.Tensor, packed_w: torch.Tensor, w_codebook: torch.Tensor, w_center: torch.Tensor,
                 w_scale: torch.Tensor, w_code_sum: torch.Tensor, bias: Optional[torch.Tensor], bits: int,
                 group_size: int, out_dtype: torch.dtype = torch.float16,
                 w_hat_ws: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y = x_hat @ w_hat.T + bias`` with ``w_hat`` rebuilt from packed codes inside the GEMM.  ``w_hat_ws``
    (fp16, at least N*K elements; the role of the reference module's ``_weight_buffer``) lets shapes that would
    repeat the reconstruction in many workgroups rebuild the weights once instead; ``y`` is the same either way."""
    _check(x_hat.is_cuda and packed_w.is_cuda, "x_hat and packed_w must be CUDA tensors")
    _check(x_hat.dim() == 2 and x_hat.dtype == torch.float16, "x_hat must be float16 [M, K]")
    _check(packed_w.dtype == torch.uint8 and packed_w.dim() == 2, "packed_w must be uint8 [N, K*bits/8]")
    _check_bits(bits)
    x_hat = x_hat.contiguous()
    m, k = x_hat.shape
    n = packed_w.shape[0]
    _check(packed_w.shape[1] == (k * bits + 7) // 8, "packed_w row length does not match K*bits/8")
    _check_weights(n, k, group_size, w_center, w_scale, w_code_sum, bias)
    _check_codebooks(bits, w_codebook)
    y = torch.empty((m, n), dtype=out_dtype, device=x_hat.device)
    b = None if bias is None or bias.numel() == 0 else _f32c(bias)
    w = [packed_w.contiguous(), _f32c(w_codebook), _f32c(w_center), _f32c(w_scale), _f32c(w_code_sum)]
    _check_w_ws(w_hat_ws, n, k)
    with torch.cuda.device(x_hat.device):
        _lib.check(_lib.load().arcq_linear_fused_ws(
            _ptr(x_hat), *[_ptr(t) for t in w], _ptr(b), _ptr(w_hat_ws), _ptr(y), _dtype_code(y, "y"),
            m, n, k, bits, int(group_size), _stream()))
    return y


def _check_w_ws(w_hat_ws: Optional[torch.Tensor], n: int, k: int) -> None:
    if w_hat_ws is not None:
        _check(w_hat_ws.is_cuda and w_hat_ws.dtype == torch.float16 and w_hat_ws.is_contiguous()
               and w_hat_ws.numel() >= n * k, "w_hat_ws must be a contiguous float16 CUDA buffer of at least N*K elements")


def linear_otf(x: torch.Tensor, a_thresholds: torch.Tensor, a_codebook: torch.Tensor, packed_w: torch.Tensor,
               w_codebook: torch.Tensor, w_center: torch.Tensor, w_scale: torch.Tensor, w_code_sum: torch.Tensor,
               bias: Optional[torch.Tensor], bits: int, group_size: int, out_dtype: torch.dtype = torch.float16,
               x_hat_ws: Optional[torch.Tensor] = None, w_hat_ws: Optional[torch.Tensor] = None,
               scratch: bool = False) -> torch.Tensor:
    """Whole packed on-the-fly layer on ``x [M, K]`` (fp16 or fp32): stage 1 into ``x_hat_ws`` (fp16
    ``[M, K]``, allocated if not given), then the fused GEMM (``w_hat_ws``: see ``linear_fused``).

    With ``scratch=True`` or a ``w_hat_ws`` both workspaces are scratch only: ``y`` is the same bit for bit, but
    ``x_hat_ws`` may afterwards hold ``x_hat`` in the library's 32-row block layout instead of row-major (the
    faster path from 512 rows on).  Otherwise ``x_hat_ws`` holds ``x_hat`` row-major after the call."""
    _check(x.is_cuda and packed_w.is_cuda, "x and packed_w must be CUDA tensors")
    _check(x.dim() == 2, "x must have shape [M, K]")
    _check_bits(bits)
    x = x.contiguous()
    m, k = x.shape
    n = packed_w.shape[0]
    _check(packed_w.shape[1] == (k * bits + 7) // 8, "packed_w row length does not match K*bits/8")
    _check_weights(n, k, group_size, w_center, w_scale, w_code_sum, bias)
    _check_codebooks(bits, w_codebook, a_thresholds, a_codebook)
    if x_hat_ws is None:
        x_hat_ws = torch.empty((m, k), dtype=torch.float16, device=x.device)
    else:
        _check(x_hat_ws.dtype == torch.float16 and x_hat_ws.is_contiguous() and x_hat_ws.numel() >= m * k,
               "x_hat_ws must be a contiguous float16 buffer of at least M*K elements")
    y = torch.empty((m, n), dtype=out_dtype, device=x.device)
    b = None if bias is None or bias.numel() == 0 else _f32c(bias)
    a = [_f32c(a_thresholds), _f32c(a_codebook)]
    w = [packed_w.contiguous(), _f32c(w_codebook), _f32c(w_center), _f32c(w_scale), _f32c(w_code_sum)]
    _check_w_ws(w_hat_ws, n, k)
    with torch.cuda.device(x.device):
        if scratch or w_hat_ws is not None:
            _lib.check(_lib.load().arcq_linear_otf_ws(
                _ptr(x), _dtype_code(x, "x"), *[_ptr(t) for t in a], *[_ptr(t) for t in w], _ptr(b), _ptr(x_hat_ws),
                _ptr(w_hat_ws), _ptr(y), _dtype_code(y, "y"), m, n, k, bits, int(group_size), _stream()))
        else:
            _lib.check(_lib.load().arcq_linear_otf(
                _ptr(x), _dtype_code(x, "x"), *[_ptr(t) for t in a], *[_ptr(t) for t in w], _ptr(b), _ptr(x_hat_ws),
                _ptr(y), _dtype_code(y, "y"), m, n, k, bits, int(group_size), _stream()))
    return y


def quantize_activation_blocked(x: torch.Tensor, thresholds: torch.Tensor, codebook: torch.Tensor, bits: int,
                                out: Optional[torch.Tensor] = None, weights=None,
                                w_hat: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Stage 1 (group size 64) with ``x_hat`` written as fp16 in the 32-row block layout
    ``[M/32, K/8, 32, 8]`` that ``linear_fused_blocked`` reads (a last block of ``r = M % 32`` rows follows as
    ``[K/8, r, 8]``); same values as ``dequant_activation_hip``.

    ``weights=(packed_w, w_codebook, w_center, w_scale, w_code_sum)`` with ``w_hat`` (fp16, N*K elements): the same
    launch also reconstructs the layer's weights into ``w_hat`` (what ``unpack_weight_hip`` would write)."""
    _check(x.is_cuda and x.dim() == 2, "x must be a CUDA tensor [M, K]")
    _check_bits(bits)
    x = x.contiguous()
    m, k = x.shape
    _check(k % 64 == 0, "the block layout needs K divisible by 64")
    _check_codebooks(bits, None, thresholds, codebook)
    if out is None:      # whole blocks: [M/32, K/8, 32, 8]; a ragged last block is stored compactly behind them: flat
        shape = (m // 32, k // 8, 32, 8) if m % 32 == 0 else (m * k,)
        out = torch.empty(shape, dtype=torch.float16, device=x.device)
    else:
        _check(out.is_cuda and out.dtype == torch.float16 and out.is_contiguous() and out.numel() >= m * k,
               "out must be a contiguous float16 CUDA buffer of at least M*K elements")
    thr, cbk = _f32c(thresholds), _f32c(codebook)
    with torch.cuda.device(x.device):
        if weights is None:
            _lib.check(_lib.load().arcq_act_quant_blocked(
                _ptr(x), _dtype_code(x, "x"), _ptr(thr), _ptr(cbk), _ptr(out), m, k, bits, 1.0e-6, _stream()))
        else:
            packed_w = weights[0].contiguous()
            n = packed_w.shape[0]
            _check(packed_w.is_cuda and packed_w.dtype == torch.uint8 and packed_w.dim() == 2
                   and packed_w.shape[1] == (k * bits + 7) // 8, "packed_w must be uint8 [N, K*bits/8]")
            _check(w_hat is not None, "weights need a w_hat buffer")
            _check_weights(n, k, 64, *weights[2:], None)
            _check_codebooks(bits, weights[1])
            _check_w_ws(w_hat, n, k)
            meta = [_f32c(t) for t in weights[1:]]
            _lib.check(_lib.load().arcq_act_quant_blocked_with_weights(
                _ptr(x), _dtype_code(x, "x"), _ptr(thr), _ptr(cbk), _ptr(out), m, k, bits, 1.0e-6,
                _ptr(packed_w), *[_ptr(t) for t in meta], _ptr(w_hat), n, _stream()))
    return out


def quantize_activation_blocked_ln(x: torch.Tensor, ln_weight: torch.Tensor, ln_bias: torch.Tensor, ln_eps: float,
                                   thresholds: torch.Tensor, codebook: torch.Tensor, bits: int,
                                   out: Optional[torch.Tensor] = None, weights=None,
                                   w_hat: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``quantize_activation_blocked`` of ``LayerNorm(x)`` (over the last dimension, result rounded to ``x``'s
    dtype) in one launch; ``64 <= K <= 1024``.  ``weights`` / ``w_hat`` as there."""
    _check(x.is_cuda and x.dim() == 2, "x must be a CUDA tensor [M, K]")
    _check_bits(bits)
    x = x.contiguous()
    m, k = x.shape
    _check(k % 64 == 0 and 64 <= k <= 1024, "the fused LayerNorm needs K divisible by 64 and at most 1024")
    _check_codebooks(bits, None, thresholds, codebook)
    if out is None:
        shape = (m // 32, k // 8, 32, 8) if m % 32 == 0 else (m * k,)
        out = torch.empty(shape, dtype=torch.float16, device=x.device)
    else:
        _check(out.is_cuda and out.dtype == torch.float16 and out.is_contiguous() and out.numel() >= m * k,
               "out must be a contiguous float16 CUDA buffer of at least M*K elements")
    thr, cbk, g, b = _f32c(thresholds), _f32c(codebook), _f32c(ln_weight), _f32c(ln_bias)
    _check(g.numel() == k and b.numel() == k, "ln_weight and ln_bias must have K elements")
    wp = [0, 0, 0, 0, 0, 0, 0]
    keep = None
    if weights is not None:
        packed_w = weights[0].contiguous()
        n = packed_w.shape[0]
        _check(packed_w.is_cuda and packed_w.dtype == torch.uint8 and packed_w.dim() == 2
               and packed_w.shape[1] == (k * bits + 7) // 8, "packed_w must be uint8 [N, K*bits/8]")
        _check(w_hat is not None, "weights need a w_hat buffer")
        _check_weights(n, k, 64, *weights[2:], None)
        _check_codebooks(bits, weights[1])
        _check_w_ws(w_hat, n, k)
        keep = [packed_w] + [_f32c(t) for t in weights[1:]]
        wp = [_ptr(t) for t in keep] + [_ptr(w_hat), n]
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().arcq_act_quant_blocked_ln(
            _ptr(x), _dtype_code(x, "x"), _ptr(g), _ptr(b), float(ln_eps), _ptr(thr), _ptr(cbk), _ptr(out), m, k, bits,
            1.0e-6, *wp, _stream()))
    return out


def quantize_patches(img: torch.Tensor, thresholds: torch.Tensor, codebook: torch.Tensor, bits: int,
                     blocked: bool = False) -> torch.Tensor:
    """Stage 1 of a quantized 16 x 16 patch convolution on three channels (``arcq_act_quant_patches``): every pixel's
    channels are one group; returns the reconstructed patch rows ``[B * patches, 768]`` fp16 (column order ``(c, i, j)``
    of ``conv.weight.reshape``), or with ``blocked`` the flat 32-row block layout ``linear_fused_blocked`` reads."""
    _check(img.is_cuda and img.dim() == 4 and img.shape[1] == 3 and img.dtype in (torch.float16, torch.float32),
           "img must be a CUDA fp16 or fp32 tensor [B, 3, H, W]")
    _check_bits(bits)
    b, _, h, w = img.shape
    _check(h % 16 == 0 and w % 16 == 0, "image sides must be multiples of 16")
    _check_codebooks(bits, None, thresholds, codebook)
    img = img.contiguous()
    m = b * (h // 16) * (w // 16)
    out = torch.empty(m * 768 if blocked else (m, 768), dtype=torch.float16, device=img.device)
    with torch.cuda.device(img.device):
        _lib.check(_lib.load().arcq_act_quant_patches(_ptr(img), _dtype_code(img, "img"), _ptr(_f32c(thresholds)),
                                                      _ptr(_f32c(codebook)), _ptr(out), b, 3, h, w, 16, bits, 1.0e-6,
                                                      int(bool(blocked)), _stream()))
    return out


def patch_embed_fwd(img: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], cls_token: torch.Tensor,
                    pos_embed: torch.Tensor) -> torch.Tensor:
    """Front end of a ViT in one launch (``arcq_patch_embed_fwd``): 16 x 16 stride-16 patch convolution of ``img``
    ``[B, 3, H, W]`` with ``weight`` ``[N, 3, 16, 16]`` and ``bias``, the class token in front, ``pos_embed`` added ->
    ``[B, 1 + patches, N]``; everything fp16, fp32 accumulation, rounded as the separate torch operations round."""
    out = _lib.host().patch_embed(img, weight, bias, cls_token, pos_embed)
    if out is not None:
        return out
    _check(img.is_cuda and img.dtype == torch.float16 and img.dim() == 4 and img.shape[1] == 3,
           "img must be a CUDA fp16 tensor [B, 3, H, W]")
    _check(weight.is_cuda and weight.dtype == torch.float16 and weight.dim() == 4 and tuple(weight.shape[1:]) == (3, 16, 16),
           "weight must be a CUDA fp16 tensor [N, 3, 16, 16]")
    _check(weight.shape[0] % 32 == 0, "the embedding width must be a multiple of 32")
    b, _, h, w_ = img.shape
    n = weight.shape[0]
    tokens = 1 + (h // 16) * (w_ // 16)
    _check(h % 16 == 0 and w_ % 16 == 0, "image sides must be multiples of 16")
    _check(cls_token.numel() == n and pos_embed.numel() == tokens * n, "cls_token / pos_embed do not match the patch grid")
    for t in (cls_token, pos_embed, bias):
        _check(t is None or (t.is_cuda and t.dtype == torch.float16), "bias, cls_token and pos_embed must be CUDA fp16 tensors")
    img, weight = img.contiguous(), weight.contiguous()
    cls_c, pos_c = cls_token.contiguous(), pos_embed.contiguous()
    bias_c = None if bias is None else bias.contiguous()
    out = torch.empty((b, tokens, n), dtype=torch.float16, device=img.device)
    with torch.cuda.device(img.device):
        _lib.check(_lib.load().arcq_patch_embed_fwd(_ptr(img), _ptr(weight), _ptr(bias_c), _ptr(cls_c), _ptr(pos_c), _ptr(out),
                                                    b, h, w_, 16, n, _stream()))
    return out


def attention_fwd(qkv: torch.Tensor, heads: int, scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Softmax attention on the qkv layer's output ``[B, n, 3 C]`` fp16 (q, k, v of head h at columns
    ``(0|1|2) C + 64 h``) -> ``[B, n, C]`` fp16, the proj layer's input, in one launch with no reshaping copies
    (``arcq_attention_fwd``: head dimension 64, at most 256 tokens).  ``scale`` defaults to ``1 / sqrt(64)``."""
    if out is None:
        y = _lib.host().attention(qkv, heads, 0.125 if scale is None else float(scale))
        if y is not None:
            return y
    _check(qkv.is_cuda and qkv.dtype == torch.float16 and qkv.dim() == 3, "qkv must be a CUDA fp16 tensor [B, n, 3 C]")
    _check(qkv.is_contiguous(), "qkv must be contiguous")
    b, n, c3 = qkv.shape
    _check(c3 % 3 == 0 and (c3 // 3) == heads * 64, f"head dimension must be 64 (C={c3 // 3}, heads={heads})")
    c = c3 // 3
    if out is None:
        out = torch.empty((b, n, c), dtype=torch.float16, device=qkv.device)
    else:
        _check(out.is_cuda and out.dtype == torch.float16 and out.is_contiguous() and out.numel() == b * n * c,
               "out must be a contiguous CUDA fp16 tensor of B * n * C elements")
    with torch.cuda.device(qkv.device):
        _lib.check(_lib.load().arcq_attention_fwd(_ptr(qkv), _ptr(out), b, n, heads, 64,
                                                  0.125 if scale is None else float(scale), _stream()))
    return out.view(b, n, c)


def xhat_layout(m: int) -> int:
    """Layout of an ``x_hat`` passed between two chained layers (``linear_otf_ex`` with ``next_quant`` / ``x_is_xhat``):
    0 = row-major, 1 = the 32-row block layout."""
    return int(_lib.load().arcq_xhat_layout(int(m)))


def linear_otf_ex(x: torch.Tensor, a_thresholds: torch.Tensor, a_codebook: torch.Tensor, packed_w: torch.Tensor,
                  w_codebook: torch.Tensor, w_center: torch.Tensor, w_scale: torch.Tensor, w_code_sum: torch.Tensor,
                  bias: Optional[torch.Tensor], bits: int, group_size: int, out_dtype: torch.dtype = torch.float16,
                  layernorm=None, gelu: bool = False, residual: Optional[torch.Tensor] = None,
                  x_hat_ws: Optional[torch.Tensor] = None, w_hat_ws: Optional[torch.Tensor] = None,
                  next_quant=None, x_is_xhat: bool = False) -> torch.Tensor:
    """``residual + gelu(linear(stage1(LayerNorm(x))))`` with the optional parts fused into the layer's two launches
    (``arcq_linear_otf_ex``): ``layernorm = (weight, bias, eps)`` or None, ``residual`` ``[M, N]`` of ``out_dtype`` or
    None.  Below 512 rows the whole layer with its options is one launch (or stage 1 + the split-K kernel with the
    GELU / residual in its epilogue); from 512 rows on the block-layout path.  Raises ``RuntimeError`` where the
    library does not fuse (LayerNorm with K > 1024 from 512 rows on, K > 1536 below).
    ``next_quant = (thresholds, codebook)`` of the layer that consumes the output: the result is that layer's ``x_hat``
    (stage 1 applied to the rounded output) in the layout ``xhat_layout(M)`` instead of the output itself; that layer is
    then called with ``x_is_xhat=True`` (its own stage 1 is skipped)."""
    _check(x.is_cuda and packed_w.is_cuda, "x and packed_w must be CUDA tensors")
    _check(x.dim() == 2, "x must have shape [M, K]")
    _check_bits(bits)
    x = x.contiguous()
    m, k = x.shape
    n = packed_w.shape[0]
    _check(packed_w.shape[1] == (k * bits + 7) // 8, "packed_w row length does not match K*bits/8")
    _check_weights(n, k, group_size, w_center, w_scale, w_code_sum, bias)
    _check_codebooks(bits, w_codebook, a_thresholds, a_codebook)
    if x_hat_ws is None:
        x_hat_ws = torch.empty(m * k, dtype=torch.float16, device=x.device)
    y = torch.empty((m, n), dtype=out_dtype, device=x.device)
    keep = [_f32c(a_thresholds), _f32c(a_codebook), packed_w.contiguous(), _f32c(w_codebook), _f32c(w_center),
            _f32c(w_scale), _f32c(w_code_sum), None if bias is None or bias.numel() == 0 else _f32c(bias)]
    a = _lib.LinearExArgs()
    a.struct_size = ctypes.sizeof(_lib.LinearExArgs)
    a.x_dtype, a.y_dtype = _dtype_code(x, "x"), _dtype_code(y, "y")
    a.bits, a.group_size, a.M, a.N, a.K = bits, int(group_size), m, n, k
    a.x = _ptr(x)
    if layernorm is not None:
        lw, lb, eps = layernorm
        lw, lb = _f32c(lw), _f32c(lb)
        keep += [lw, lb]
        a.producer, a.ln_weight, a.ln_bias, a.ln_eps = _lib.ARCQ_PRODUCER_LAYERNORM, _ptr(lw), _ptr(lb), float(eps)
    if x_is_xhat:
        _check(layernorm is None and x.dtype == torch.float16, "x_is_xhat: x must be float16 and takes no LayerNorm")
        a.producer = _lib.ARCQ_PRODUCER_XHAT
    if next_quant is not None:
        nt, nc = _f32c(next_quant[0]), _f32c(next_quant[1])
        keep += [nt, nc]
        a.next_a_thresholds, a.next_a_codebook = _ptr(nt), _ptr(nc)
    a.activation = _lib.ARCQ_ACT_GELU if gelu else _lib.ARCQ_ACT_NONE
    (a.a_thresholds, a.a_codebook, a.packed_w, a.w_codebook, a.w_center, a.w_scale, a.w_code_sum,
     a.bias) = [_ptr(t) or None for t in keep[:8]]
    if residual is not None:
        _check(residual.is_cuda and residual.dtype == out_dtype and residual.is_contiguous()
               and tuple(residual.shape) == (m, n), "residual must be a contiguous [M, N] tensor of the output dtype")
        a.residual = _ptr(residual)
    _check_w_ws(w_hat_ws, n, k)
    a.x_hat_ws, a.w_hat_ws, a.y = _ptr(x_hat_ws), _ptr(w_hat_ws) or None, _ptr(y)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().arcq_linear_otf_ex(ctypes.byref(a), _stream()))
    return y


# ---------------------------------------------------------------------------------------------
# the layer with FP8 operands -- no counterpart in the reference; a faster, less exact stage 3
# ---------------------------------------------------------------------------------------------
FP8_MAX = 448.0          # largest finite OCP E4M3 value


def quantize_activation_fp8(x: torch.Tensor, thresholds: torch.Tensor, codebook: torch.Tensor, bits: int,
                            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Stage 1 with the reconstruction rounded to FP8 (``torch.float8_e4m3fn``, row-major ``[M, K]``) instead of fp16;
    group size 64.  Codes, ``mu`` and ``s`` are those of ``quantize_activation``."""
    _check(x.is_cuda and x.dim() == 2, "x must be a CUDA tensor of shape [M, K]")
    _check_bits(bits)
    _check_codebooks(bits, None, thresholds, codebook)
    x = x.contiguous()
    m, k = x.shape
    if out is None:
        out = torch.empty((m, k), dtype=torch.float8_e4m3fn, device=x.device)
    else:
        _check(out.dtype == torch.float8_e4m3fn and out.is_contiguous() and out.numel() >= m * k,
               "out must be a contiguous float8_e4m3fn buffer of at least M*K elements")
    thresholds, codebook = _f32c(thresholds), _f32c(codebook)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().arcq_act_quant_fp8(_ptr(x), _dtype_code(x, "x"), _ptr(thresholds), _ptr(codebook), _ptr(out),
                                                  m, k, bits, 1.0e-6, _stream()))
    return out


def fp8_weight_multiplier(w_codebook: torch.Tensor, w_center: torch.Tensor, w_scale: torch.Tensor,
                          w_code_sum: torch.Tensor) -> float:
    """Power of two that moves a layer's reconstructed weights into FP8's normal range: the largest one that keeps a
    bound on ``|w_hat|`` (``|center| + |scale| (max |cb| + |code_sum| / 64)`` over all groups) at or below half the
    largest FP8 value.  Reads the metadata back to the host: compute it once per layer."""
    w_codebook, w_center, w_scale, w_code_sum = (t.detach().float() for t in (w_codebook, w_center, w_scale, w_code_sum))
    cb = float(w_codebook.abs().max())
    bound = float((w_center.abs() + w_scale.abs() * (cb + w_code_sum.abs() / 64.0)).max())
    if not bound > 0.0:
        return 1.0
    return float(2.0 ** math.floor(math.log2(FP8_MAX / 2.0 / bound)))


def unpack_weight_fp8(packed: torch.Tensor, codebook: torch.Tensor, center: torch.Tensor, scale: torch.Tensor,
                      code_sum: torch.Tensor, bits: int, w_mult: float, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Stage 2 with the weights rounded to FP8: ``fp8(w_mult * w_hat)``, row-major ``[N, K]``; group size 64."""
    _check(packed.is_cuda and packed.dtype == torch.uint8, "packed must be a CUDA uint8 tensor")
    _check_bits(bits)
    n = packed.shape[0]
    k = center.shape[1] * 64
    _check(packed.shape[1] == (k * bits + 7) // 8, "packed row length does not match in_features*bits/8")
    _check_weights(n, k, 64, center, scale, code_sum, None)
    _check_codebooks(bits, codebook)
    if out is None:
        out = torch.empty((n, k), dtype=torch.float8_e4m3fn, device=packed.device)
    else:
        _check(out.dtype == torch.float8_e4m3fn and out.is_contiguous() and out.numel() >= n * k,
               "out must be a contiguous float8_e4m3fn buffer of at least N*K elements")
    packed = packed.contiguous()
    codebook, center, scale, code_sum = _f32c(codebook), _f32c(center), _f32c(scale), _f32c(code_sum)
    with torch.cuda.device(packed.device):
        _lib.check(_lib.load().arcq_weight_dequant_fp8(_ptr(packed), _ptr(codebook), _ptr(center), _ptr(scale),
                                                       _ptr(code_sum), _ptr(out), n, k, bits, 64, float(w_mult), _stream()))
    return out


def fp8_padded_k(k: int) -> int:
    """Row length of the FP8 GEMM's operands: ``k`` rounded up to a multiple of 128 (the padding is zero)."""
    return (int(k) + 127) // 128 * 128


def linear_otf_fp8(x: torch.Tensor, a_thresholds: torch.Tensor, a_codebook: torch.Tensor, packed_w: torch.Tensor,
                   w_codebook: torch.Tensor, w_center: torch.Tensor, w_scale: torch.Tensor, w_code_sum: torch.Tensor,
                   bias: Optional[torch.Tensor], bits: int, out_dtype: torch.dtype = torch.float16,
                   w_mult: Optional[float] = None, x8_ws: Optional[torch.Tensor] = None,
                   w8_ws: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The packed on-the-fly layer with FP8 operands (``arcq_linear_otf_fp8``, two launches): stage 1 and stage 2 as in
    ``linear_otf`` but rounded to FP8 (the weights first multiplied by ``w_mult``), then the library's own FP8 MFMA GEMM
    with fp32 accumulation, ``y = x8 w8^T / w_mult + bias``.  Faster where the layer is bound by the matrix units (the
    large models), NOT bit-compatible with the reference: each operand carries a rounding error of up to 2^-4 relative
    (fp16: 2^-11).  Group size 64.  ``x8_ws`` / ``w8_ws``: scratch of at least ``M * Kp`` / ``N * Kp`` bytes
    (``Kp = fp8_padded_k(K)``), any 1-byte dtype."""
    _check(x.is_cuda and x.dim() == 2, "x must be a CUDA tensor of shape [M, K]")
    _check_bits(bits)
    x = x.contiguous()
    m, k = x.shape
    n = packed_w.shape[0]
    _check(k % 64 == 0 and k > 0, "in_features must be a positive multiple of the group size 64")
    _check(packed_w.shape[1] == (k * bits + 7) // 8, "packed_w row length does not match K*bits/8")
    _check_weights(n, k, 64, w_center, w_scale, w_code_sum, bias)
    _check_codebooks(bits, w_codebook, a_thresholds, a_codebook)
    if w_mult is None:
        w_mult = fp8_weight_multiplier(w_codebook, w_center, w_scale, w_code_sum)
    kp = fp8_padded_k(k)
    if x8_ws is None:
        x8_ws = torch.empty(max(m * kp, 1), dtype=torch.uint8, device=x.device)
    if w8_ws is None:
        w8_ws = torch.empty(max(n * kp, 1), dtype=torch.uint8, device=x.device)
    for t, need, name in ((x8_ws, m * kp, "x8_ws"), (w8_ws, n * kp, "w8_ws")):
        _check(t.is_cuda and t.is_contiguous() and t.element_size() == 1 and t.numel() >= need,
               f"{name} must be a contiguous 1-byte CUDA buffer of at least {need} elements")
    y = torch.empty((m, n), dtype=out_dtype, device=x.device)
    a = [_f32c(a_thresholds), _f32c(a_codebook)]
    w = [packed_w.contiguous(), _f32c(w_codebook), _f32c(w_center), _f32c(w_scale), _f32c(w_code_sum)]
    b = None if bias is None or bias.numel() == 0 else _f32c(bias)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().arcq_linear_otf_fp8(
            _ptr(x), _dtype_code(x, "x"), *[_ptr(t) for t in a], *[_ptr(t) for t in w], _ptr(b), float(w_mult),
            _ptr(x8_ws), _ptr(w8_ws), _ptr(y), _dtype_code(y, "y"), m, n, k, bits, _stream()))
    return y


def linear_otf_fp8_library_gemm(x: torch.Tensor, a_thresholds: torch.Tensor, a_codebook: torch.Tensor,
                                packed_w: torch.Tensor, w_codebook: torch.Tensor, w_center: torch.Tensor,
                                w_scale: torch.Tensor, w_code_sum: torch.Tensor, bias: Optional[torch.Tensor], bits: int,
                                out_dtype: torch.dtype = torch.float16, w_mult: Optional[float] = None,
                                x8_ws: Optional[torch.Tensor] = None, w8_ws: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The same layer with the product left to the vendor library's FP8 GEMM (``torch._scaled_mm``) on row-major
    operands, three launches: kept as a timing and cross-check reference for ``linear_otf_fp8``, not used by the
    modules."""
    _check(x.is_cuda and x.dim() == 2, "x must be a CUDA tensor of shape [M, K]")
    m, k = x.shape
    n = packed_w.shape[0]
    _check(k % 16 == 0 and n % 16 == 0, "the library's FP8 GEMM needs K and N to be multiples of 16")
    if w_mult is None:
        w_mult = fp8_weight_multiplier(w_codebook, w_center, w_scale, w_code_sum)
    x8 = quantize_activation_fp8(x, a_thresholds, a_codebook, bits, out=x8_ws)
    w8 = unpack_weight_fp8(packed_w, w_codebook, w_center, w_scale, w_code_sum, bits, w_mult, out=w8_ws)
    x8 = x8.view(-1)[:m * k].view(m, k)
    w8 = w8.view(-1)[:n * k].view(n, k)
    one = torch.ones((), dtype=torch.float32, device=x.device)
    inv = torch.full((), 1.0 / float(w_mult), dtype=torch.float32, device=x.device)
    has_bias = bias is not None and bias.numel() > 0
    if has_bias and out_dtype == torch.float16:      # (the library adds a bias of the output's type; fp16 only)
        return torch._scaled_mm(x8, w8.t(), scale_a=one, scale_b=inv, bias=bias.to(torch.float16), out_dtype=out_dtype)
    y = torch._scaled_mm(x8, w8.t(), scale_a=one, scale_b=inv, out_dtype=out_dtype)
    return y + bias.to(out_dtype) if has_bias else y


def linear_fused_blocked(x_hat_blocked: torch.Tensor, m: int, k: int, packed_w: torch.Tensor, w_codebook: torch.Tensor,
                         w_center: torch.Tensor, w_scale: torch.Tensor, w_code_sum: torch.Tensor,
                         bias: Optional[torch.Tensor], bits: int, out_dtype: torch.dtype = torch.float16,
                         w_hat_ws: Optional[torch.Tensor] = None, w_hat_ready: bool = False) -> torch.Tensor:
    """``linear_fused`` on ``x_hat`` ``[m, k]`` held in the 32-row block layout (``quantize_activation_blocked``).
    ``w_hat_ready``: ``w_hat_ws`` already holds the reconstructed fp16 weights and is used as is."""
    _check(x_hat_blocked.is_cuda and x_hat_blocked.dtype == torch.float16 and x_hat_blocked.is_contiguous()
           and x_hat_blocked.numel() >= m * k, "x_hat_blocked must be a contiguous float16 CUDA buffer of M*K elements")
    _check(packed_w.is_cuda and packed_w.dtype == torch.uint8 and packed_w.dim() == 2, "packed_w must be uint8 [N, K*bits/8]")
    _check_bits(bits)
    n = packed_w.shape[0]
    _check(packed_w.shape[1] == (k * bits + 7) // 8, "packed_w row length does not match K*bits/8")
    _check_weights(n, k, 64, w_center, w_scale, w_code_sum, bias)
    _check_codebooks(bits, w_codebook)
    y = torch.empty((m, n), dtype=out_dtype, device=x_hat_blocked.device)
    b = None if bias is None or bias.numel() == 0 else _f32c(bias)
    w = [packed_w.contiguous(), _f32c(w_codebook), _f32c(w_center), _f32c(w_scale), _f32c(w_code_sum)]
    _check_w_ws(w_hat_ws, n, k)
    with torch.cuda.device(x_hat_blocked.device):
        _lib.check(_lib.load().arcq_linear_fused_blocked(
            _ptr(x_hat_blocked), *[_ptr(t) for t in w], _ptr(b), _ptr(w_hat_ws), int(bool(w_hat_ready)), _ptr(y),
            _dtype_code(y, "y"), m, n, k, bits, 64, _stream()))
    return y


# ---------------------------------------------------------------------------------------------
# index-space linears -- EXT/arcq_linear_kernel.cu:206-353
# ---------------------------------------------------------------------------------------------
def _check_index(rows: int, out_features: int, in_features: int, group_size: int, x_center, x_scale, x_code_sum, w_center,
                 w_scale, w_code_sum, product_table, bias) -> None:
    _check_weights(out_features, in_features, group_size, w_center, w_scale, w_code_sum, bias)
    need = rows * (in_features // int(group_size))
    _check(all(t.is_cuda and t.numel() >= need for t in (x_center, x_scale, x_code_sum)),
           "x_center, x_scale and x_code_sum must be CUDA tensors [rows, groups]")
    _check(product_table.is_cuda, "product_table must be CUDA tensor")
    _check(product_table.dim() == 2 and product_table.shape[0] == product_table.shape[1], "product_table must be square")


def arcq_linear_forward(packed_x: torch.Tensor, x_center: torch.Tensor, x_scale: torch.Tensor,
                        x_code_sum: torch.Tensor, packed_w: torch.Tensor, w_center: torch.Tensor,
                        w_scale: torch.Tensor, w_code_sum: torch.Tensor, product_table: torch.Tensor,
                        bias: Optional[torch.Tensor], bits: int, group_size: int, in_features: int,
                        out_features: int) -> torch.Tensor:
    """fp64-accumulated product-table linear on packed codes (EXT/arcq_linear_kernel.cu:206-278)."""
    _check(packed_x.is_cuda, "packed_x must be CUDA tensor")
    _check(packed_w.is_cuda, "packed_w must be CUDA tensor")
    _check(packed_x.dtype == torch.uint8, "packed_x must be uint8")
    _check(packed_w.dtype == torch.uint8, "packed_w must be uint8")
    _check_bits(bits)
    _check(int(in_features) % int(group_size) == 0, "in_features must be divisible by group_size")
    _check(product_table.dtype == torch.float32, "product_table must be float32")
    pc = (int(in_features) * bits + 7) // 8
    _check(packed_x.dim() == 2 and packed_x.shape[1] == pc, "packed_x row length does not match in_features*bits/8")
    _check(packed_w.dim() == 2 and packed_w.shape == (int(out_features), pc),
           "packed_w shape does not match [out_features, in_features*bits/8]")
    _check_index(packed_x.shape[0], int(out_features), int(in_features), group_size, x_center, x_scale, x_code_sum, w_center, w_scale,
                 w_code_sum, product_table, bias)
    rows = packed_x.shape[0]
    levels = product_table.shape[0]
    y = torch.empty((rows, int(out_features)), dtype=torch.float32, device=packed_x.device)
    b = None
    if bias is not None and bias.numel() > 0:
        _check(bias.is_cuda, "bias must be CUDA tensor")
        b = _f32c(bias)
    tensors = [packed_x.contiguous(), _f32c(x_center), _f32c(x_scale), _f32c(x_code_sum), packed_w.contiguous(),
               _f32c(w_center), _f32c(w_scale), _f32c(w_code_sum), _f32c(product_table)]
    with torch.cuda.device(packed_x.device):
        _lib.check(_lib.load().arcq_linear_forward_packed(
            *[_ptr(t) for t in tensors], _ptr(b), _ptr(y), rows, int(out_features), int(in_features), bits,
            int(group_size), levels, _stream()))
    return y


def arcq_linear_forward_u8(x_codes: torch.Tensor, x_center: torch.Tensor, x_scale: torch.Tensor,
                           x_code_sum: torch.Tensor, w_codes: torch.Tensor, w_center: torch.Tensor,
                           w_scale: torch.Tensor, w_code_sum: torch.Tensor, product_table: torch.Tensor,
                           bias: Optional[torch.Tensor], group_size: int) -> torch.Tensor:
    """fp32 product-table linear on byte codes, 32-lane summation order (EXT/arcq_linear_kernel.cu:280-353)."""
    _check(x_codes.is_cuda, "x_codes must be CUDA tensor")
    _check(w_codes.is_cuda, "w_codes must be CUDA tensor")
    _check(x_codes.dtype == torch.uint8, "x_codes must be uint8")
    _check(w_codes.dtype == torch.uint8, "w_codes must be uint8")
    _check(x_codes.dim() == 2, "x_codes must have shape [rows, in_features]")
    _check(w_codes.dim() == 2, "w_codes must have shape [out_features, in_features]")
    _check(x_codes.shape[1] == w_codes.shape[1], "x_codes and w_codes in_features must match")
    _check(x_codes.shape[1] % int(group_size) == 0, "in_features must be divisible by group_size")
    _check(product_table.dtype == torch.float32, "product_table must be float32")
    rows, in_features = x_codes.shape
    out_features = w_codes.shape[0]
    _check_index(rows, out_features, in_features, group_size, x_center, x_scale, x_code_sum, w_center, w_scale, w_code_sum,
                 product_table, bias)
    levels = product_table.shape[0]
    y = torch.empty((rows, out_features), dtype=torch.float32, device=x_codes.device)
    b = None
    if bias is not None and bias.numel() > 0:
        _check(bias.is_cuda, "bias must be CUDA tensor")
        b = _f32c(bias)
    tensors = [x_codes.contiguous(), _f32c(x_center), _f32c(x_scale), _f32c(x_code_sum), w_codes.contiguous(),
               _f32c(w_center), _f32c(w_scale), _f32c(w_code_sum), _f32c(product_table)]
    with torch.cuda.device(x_codes.device):
        _lib.check(_lib.load().arcq_linear_forward_u8(
            *[_ptr(t) for t in tensors], _ptr(b), _ptr(y), rows, out_features, in_features, int(group_size), levels,
            _stream()))
    return y


# ---------------------------------------------------------------------------------------------
# attention over keys and values that are kept -- no counterpart in the reference: norm and rotation
# of the heads, the pages of a cache, attention of new tokens over them.  Inference only.
# ---------------------------------------------------------------------------------------------
_NORMS = {"none": _lib.ARCQ_NORM_NONE, "rms": _lib.ARCQ_NORM_RMS, "layer": _lib.ARCQ_NORM_LAYER}
_KV_TYPES = {torch.float16: _lib.ARCQ_F16, torch.bfloat16: _lib.ARCQ_BF16}
_PAGE_TYPES = {**_KV_TYPES, torch.float8_e4m3fn: _lib.ARCQ_FP8}


class KVPages(NamedTuple):
    """The pages of a key/value cache (``kv_cache_pages`` makes them; any tuple of the same four will do).  A page holds
    ``page_size`` tokens of every key head in 16-byte pieces of ``w`` values (8 of fp16 / bf16, 16 of FP8): keys
    ``[pages, heads, head_dim / w, page_size, w]``, values ``[pages, heads, page_size / w, head_dim, w]``.  FP8 pages
    (``torch.float8_e4m3fn``) have an exponent for each token and head, int8 ``[pages, heads, page_size]``: a value is
    ``2 ** exponent`` times the FP8 value.  Slot ``p * page_size + j`` is place ``j`` of page ``p``."""
    k: torch.Tensor
    v: torch.Tensor
    k_exponents: Optional[torch.Tensor] = None
    v_exponents: Optional[torch.Tensor] = None


def kv_cache_pages(num_pages: int, heads: int, head_dim: int, page_size: int = 64, dtype: torch.dtype = torch.float16,
                   device="cuda") -> KVPages:
    """Empty pages (their memory is not cleared: attention and ``kv_cache_read`` are for slots that have been written).  ``dtype``:
    ``torch.float16``, ``torch.bfloat16`` or ``torch.float8_e4m3fn``; ``page_size`` a power of two, 16 to 2^20 (from 64 on attention reads
    them fastest), ``head_dim`` a multiple of 16, at most 256.  FP8 pages are for rows of one 16-bit type, the one they are written
    from: a value written from bfloat16 may lie outside of float16's range."""
    _check(dtype in _PAGE_TYPES, "pages hold float16, bfloat16 or float8_e4m3fn")
    _check(num_pages >= 0 and heads >= 1, "pages need at least one head")
    _check(16 <= page_size <= 1 << 20 and page_size & (page_size - 1) == 0, f"page_size must be a power of two, 16 to 2^20 (got {page_size})")
    _check(head_dim % 16 == 0 and 16 <= head_dim <= 256, f"head_dim must be a multiple of 16, at most 256 (got {head_dim})")
    fp8 = dtype == torch.float8_e4m3fn
    w = 16 if fp8 else 8
    k = torch.empty((num_pages, heads, head_dim // w, page_size, w), dtype=dtype, device=device)
    v = torch.empty((num_pages, heads, page_size // w, head_dim, w), dtype=dtype, device=device)
    exps = [torch.empty((num_pages, heads, page_size), dtype=torch.int8, device=device) for _ in range(2)] if fp8 else [None] * 2
    return KVPages(k, v, *exps)


def _no_grad(name: str, *tensors: Optional[torch.Tensor]) -> None:
    given = [t for t in tensors if t is not None]
    _check(not (torch.is_grad_enabled() and any(t.requires_grad for t in given)),
           f"{name} has no backward pass: call it under torch.no_grad() or on tensors without gradient")
    # (no_grad does not switch forward mode off)
    _check(all(forward_ad.unpack_dual(t).tangent is None for t in given),
           f"{name} has no backward pass and no forward-mode derivative: call it on tensors without tangents")


def _same_device(first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    _check(first.is_cuda, "expected CUDA tensors")
    _check(all(t is None or t.device == first.device for t in others), "all tensors must be on one device")


def _pages_args(pages) -> "tuple[_lib.KvPages, list]":
    """The pages as the library takes them, and the tensors that hold them."""
    pages = KVPages(*pages)
    k, v = pages.k, pages.v
    _check(k.dtype in _PAGE_TYPES and v.dtype == k.dtype, "pages must be float16, bfloat16 or float8_e4m3fn, keys and values alike")
    fp8 = k.dtype == torch.float8_e4m3fn
    w = 16 if fp8 else 8
    _check(k.dim() == 5 and k.shape[-1] == w, f"the keys' pages must be [pages, heads, head_dim / {w}, page_size, {w}]")
    n, h, pieces, page, _ = k.shape
    _check(page >= w and tuple(v.shape) == (n, h, page // w, pieces * w, w),
           f"the values' pages must be [pages, heads, page_size / {w}, head_dim, {w}] of the keys' sizes")
    _check(k.is_contiguous() and v.is_contiguous(), "pages must be contiguous")
    exps = [pages.k_exponents, pages.v_exponents]
    _check(all((e is not None) == fp8 for e in exps), "FP8 pages need exponents, 16-bit pages have none")
    for e in exps:
        _check(e is None or (e.dtype == torch.int8 and tuple(e.shape) == (n, h, page) and e.is_contiguous()),
               "exponents must be contiguous int8 [pages, heads, page_size]")
    _same_device(k, v, *exps)
    _no_grad("a cache", k, v)
    a = _lib.KvPages(_ptr(k), _ptr(v), _ptr(exps[0]), _ptr(exps[1]), n, h, pieces * w, page, _PAGE_TYPES[k.dtype])
    return a, [k, v, *exps]


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """``[rows, heads, dim]`` of 16 bits whose rows lie whole on 16-byte boundaries: ``t`` itself or a copy."""
    # (a dimension of one entry has any stride)
    if t.stride(2) == 1 and all(t.shape[i] <= 1 or t.stride(i) % 8 == 0 for i in (0, 1)) and t.data_ptr() % 16 == 0:
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def rotary_frequencies(pairs: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original: int = 0, fast: float = 32.0, slow: float = 1.0, device=None):
    """Radians for each position of ``pairs`` pairs, float64 ``[pairs]``, and the magnitude that goes with them, for
    ``qk_norm_rotary``: ``base ** (-i / pairs)``.  ``scaling`` for contexts ``factor`` times as long:
    ``"linear"`` divides every frequency by ``factor``; ``"base"`` raises the base so that the slowest pair does;
    ``"bands"`` divides those that turn less than ``slow`` times in the ``original`` length, leaves those that turn over
    ``fast`` times, mixes the ones between, and has magnitude ``1 + 0.1 ln(factor)``."""
    _check(pairs >= 0 and base > 0 and factor > 0, "rotary_frequencies: pairs, base and factor must be positive")
    _check(scaling in (None, "linear", "base", "bands"), f"rotary_frequencies: unknown scaling {scaling!r}")
    if scaling == "base" and pairs > 1:
        base = base * factor ** (pairs / (pairs - 1))
    f = [base ** (-i / pairs) for i in range(pairs)]
    magnitude = 1.0
    if scaling == "linear":
        f = [x / factor for x in f]
    elif scaling == "bands":
        _check(original > 0 and fast > slow, "rotary_frequencies: bands need the original length, and fast > slow")
        keep = [min(1.0, max(0.0, (original * x / (2 * math.pi) - slow) / (fast - slow))) for x in f]
        f = [x * (y + (1.0 - y) / factor) for x, y in zip(f, keep)]
        magnitude = 1.0 + 0.1 * math.log(factor)
    return torch.tensor(f, dtype=torch.float64, device=device), magnitude


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, norm: str = "none",
                   q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                   q_bias: Optional[torch.Tensor] = None, k_bias: Optional[torch.Tensor] = None, eps: float = 1.0e-6,
                   interleaved: bool = False, magnitude: float = 1.0, sections: Optional[Sequence[int]] = None, out=None):
    """Norm of every query and key head and its rotation by the token's position, in one launch (``arcq_qk_norm_rotary``).

    ``q`` ``[tokens, q_heads, head_dim]``, ``k`` ``[tokens, k_heads, head_dim]``, fp16, bf16 or fp32, of any strides (the heads
    as they lie in the qkv layer's output); ``head_dim`` even, at most 256.  ``norm``: ``"none"``, ``"rms"`` or ``"layer"``, with
    weights and biases ``[head_dim]`` or None.  ``inv_freq`` float64 ``[pairs]``: radians for each position; the first
    ``2 * pairs`` values of a head turn, pair ``i`` being values ``i`` and ``i + pairs``, or ``2 i`` and ``2 i + 1``
    (``interleaved``), and come out ``magnitude`` times as long.  ``positions`` int32 or int64 ``[tokens]``, or ``[axes, tokens]`` with
    ``sections``, the number of pairs that each axis turns.  fp32 arithmetic, angles in 64 bits, one rounding.  Returns new tensors, or
    ``out = (q_out, k_out)``, which may be ``q`` and ``k`` themselves."""
    if out is None:
        y = _lib.host().qk_norm_rotary(q, k, positions, inv_freq, _NORMS.get(norm), q_weight, k_weight, q_bias, k_bias, eps,
                                       interleaved, magnitude, sections)
        if y is not None:
            return y
    _check(norm in _NORMS, f"norm must be one of {', '.join(_NORMS)} (got {norm!r})")
    _check(q.dim() == 3 and k.dim() == 3, "q and k must have shape [tokens, heads, head_dim]")
    t, hq, d = q.shape
    hk = k.shape[1]
    _check(k.shape[0] == t and k.shape[2] == d, "q and k must have the same tokens and head_dim")
    types = {torch.float32: ARCQ_F32, **_KV_TYPES}
    _check(q.dtype in types and k.dtype == q.dtype, "q and k must both be float16, bfloat16 or float32")
    _check(positions.dtype in (torch.int32, torch.int64), "positions must be int32 or int64")
    _check(inv_freq.dtype == torch.float64 and inv_freq.dim() == 1, "inv_freq must be float64 [pairs]")
    _check(positions.dim() in (1, 2) and positions.shape[-1] == t, "positions must be [tokens] or [axes, tokens]")
    _same_device(q, k, positions, inv_freq, q_weight, k_weight, q_bias, k_bias, *(out or ()))
    _no_grad("qk_norm_rotary", q, k, inv_freq, q_weight, k_weight, q_bias, k_bias, *(out or ()))
    pairs = inv_freq.shape[0]
    axes = positions.shape[0] if positions.dim() == 2 else 1
    _check(1 <= axes <= 4, "one to four axes of positions")
    sections = [pairs] if sections is None and axes == 1 else sections
    _check(sections is not None and len(sections) == axes and sum(sections) == pairs and min(sections) >= 0,
           "sections must give the pairs of each axis of positions, all of inv_freq's in all")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight), ("q_bias", q_bias), ("k_bias", k_bias)):
        _check(w is None or w.numel() == d, f"{name} must have head_dim entries")
    # (a head's values have to lie side by side)
    q, k = (x if x.stride(2) == 1 else x.contiguous() for x in (q, k))
    if out is None:
        out = (torch.empty((t, hq, d), dtype=q.dtype, device=q.device), torch.empty((t, hk, d), dtype=q.dtype, device=q.device))
    for o, x in zip(out, (q, k)):
        _check(o.shape == x.shape and o.dtype == x.dtype and o.stride(2) == 1, "out must be two tensors like q and k, heads contiguous")
    positions = positions if positions.stride(-1) == 1 else positions.contiguous()
    inv_freq = inv_freq.contiguous()
    w = [None if x is None else _f32c(x) for x in (q_weight, q_bias, k_weight, k_bias)]
    a = _lib.QkNormRotaryArgs()
    a.dtype, a.norm, a.interleaved, a.axes = types[q.dtype], _NORMS[norm], int(bool(interleaved)), axes
    a.positions_i64 = int(positions.dtype == torch.int64)
    a.sections[:axes] = [int(x) for x in sections]
    a.eps, a.magnitude = float(eps), float(magnitude)
    a.tokens, a.q_heads, a.k_heads, a.head_dim, a.pairs = t, hq, hk, d, pairs
    a.q, a.k, a.q_out, a.k_out = (_ptr(x) for x in (q, k, *out))
    (a.q_token_stride, a.q_head_stride, a.k_token_stride, a.k_head_stride, a.q_out_token_stride, a.q_out_head_stride,
     a.k_out_token_stride, a.k_out_head_stride) = (x.stride(i) for x in (q, k, *out) for i in (0, 1))
    a.positions, a.axis_stride, a.inv_freq = _ptr(positions), positions.stride(0) if axes > 1 else 0, _ptr(inv_freq)
    a.q_weight, a.q_bias, a.k_weight, a.k_bias = (_ptr(x) or None for x in w)
    with torch.cuda.device(q.device):
        _lib.check(_lib.load().arcq_qk_norm_rotary(ctypes.byref(a), _stream()))
    return tuple(out)


def _kv_args(pages, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> "tuple[_lib.KvCacheArgs, list]":
    p, keep = _pages_args(pages)
    _check(k.dtype in _KV_TYPES and v.dtype == k.dtype, "k and v must both be float16 or bfloat16")
    _check(p.dtype in (_lib.ARCQ_FP8, _KV_TYPES[k.dtype]), "16-bit pages take and give rows of their own dtype")
    _check(slots.dtype in (torch.int32, torch.int64) and slots.dim() == 1, "slots must be int64 [rows]")
    _check(k.dim() == 3 and v.shape == k.shape and tuple(k.shape) == (slots.shape[0], p.heads, p.head_dim),
           "k and v must be [rows, heads, head_dim] of the pages, a row for each slot")
    _same_device(keep[0], k, v, slots)
    slots = slots.to(torch.int64).contiguous()
    a = _lib.KvCacheArgs()
    a.pages, a.rows, a.dtype = p, k.shape[0], _KV_TYPES[k.dtype]
    a.k, a.v, a.slots = _ptr(k), _ptr(v), _ptr(slots)
    a.k_row_stride, a.k_head_stride, a.v_row_stride, a.v_head_stride = k.stride(0), k.stride(1), v.stride(0), v.stride(1)
    return a, [k, v, slots, *keep]


def kv_cache_write(pages, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Keys and values ``[rows, heads, head_dim]`` (fp16 or bf16, any strides) into the slots ``[rows]`` of a cache's pages
    (``arcq_kv_cache_write``); a row whose slot is negative, or past the last page, is left out.  Slots have to differ: of rows
    with one slot, which one's values stay, and whether whole, is not said.  FP8 pages: each row and head with the smallest
    power of two that brings its largest magnitude to at most 448 (fp16: 2^-14 .. 2^7, bf16: 2^-110 .. 2^119, beyond
    which values saturate), rounded to nearest even; infinities and NaN become NaN."""
    if _lib.host().kv_cache_write(pages, k, v, slots) is not None:
        return
    _no_grad("kv_cache_write", k, v)
    if k.dim() == 3 and v.dim() == 3:
        k, v = _rows16(k), _rows16(v)
    a, keep = _kv_args(pages, k, v, slots)
    with torch.cuda.device(keep[0].device):
        _lib.check(_lib.load().arcq_kv_cache_write(ctypes.byref(a), _stream()))


def kv_cache_read(pages, slots: torch.Tensor, dtype: Optional[torch.dtype] = None):
    """The keys and values of the slots ``[rows]``, two tensors ``[rows, heads, head_dim]`` (``arcq_kv_cache_read``): what
    ``kv_cache_write`` put there, FP8 values widened and scaled, of ``dtype`` (by default the pages', fp16 for FP8 pages).  A slot that
    is negative, or past the last page, gives zeros."""
    out = _lib.host().kv_cache_read(pages, slots, dtype)
    if out is not None:
        return out
    p, keep = _pages_args(pages)
    dtype = dtype or (torch.float16 if p.dtype == _lib.ARCQ_FP8 else keep[0].dtype)
    k, v = (torch.empty((slots.numel(), p.heads, p.head_dim), dtype=dtype, device=keep[0].device) for _ in range(2))
    a, keep = _kv_args(pages, k, v, slots)
    with torch.cuda.device(k.device):
        _lib.check(_lib.load().arcq_kv_cache_read(ctypes.byref(a), _stream()))
    return k, v


def attention_paged_fwd(q: torch.Tensor, pages, page_table: torch.Tensor, q_offsets: torch.Tensor, kv_lengths: torch.Tensor,
                        causal: bool = True, window: int = 0, scale: Optional[float] = None,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Softmax attention of new tokens over the pages of a cache (``arcq_attention_paged_fwd``).

    ``q`` ``[tokens, q_heads, head_dim]`` fp16 or bf16 (any strides), the new tokens of all sequences one behind the other: those of
    sequence ``b`` are rows ``q_offsets[b] .. q_offsets[b + 1] - 1``, one or many, and the last of its ``kv_lengths[b]`` keys, which
    have been written to the pages ``page_table[b]`` (int32 ``[sequences, width]``, in order).  ``q_heads`` a multiple of the pages'
    heads; ``head_dim`` 32, 64, 96, 128 or 256.  ``causal``: a token sees the keys up to its own; ``window > 0``: the last ``window``
    of them.  Without ``causal`` every token sees all keys (cross attention to an encoder's states).  A token that sees no key gets
    zeros.  ``scale`` defaults to ``1 / sqrt(head_dim)``.

    Returns ``[tokens, q_heads, head_dim]`` like ``q``, or ``out``; rows behind the last sequence are not written.  Lengths
    past the table are cut to it; a page that does not exist makes the tokens that see it NaN.  Nothing is read back to the
    host, so the call can be captured."""
    if out is None:
        y = _lib.host().attention_paged(q, pages, page_table, q_offsets, kv_lengths, causal, window, scale)
        if y is not None:
            return y
    p, keep = _pages_args(pages)
    _check(q.dim() == 3 and q.shape[2] == p.head_dim, "q must be [tokens, q_heads, head_dim] of the pages' head_dim")
    _check(q.dtype in _KV_TYPES, "q must be float16 or bfloat16")
    _check(p.dtype in (_lib.ARCQ_FP8, _KV_TYPES[q.dtype]), "16-bit pages take queries of their own dtype")
    _check(page_table.dim() == 2 and page_table.dtype == torch.int32, "page_table must be int32 [sequences, width]")
    b = page_table.shape[0]
    _check(all(x.dtype == torch.int32 and x.dim() == 1 for x in (q_offsets, kv_lengths)) and q_offsets.shape[0] == b + 1
           and kv_lengths.shape[0] == b, "q_offsets must be int32 [sequences + 1] and kv_lengths int32 [sequences]")
    _same_device(q, keep[0], page_table, q_offsets, kv_lengths, out)
    _no_grad("attention_paged_fwd", q, out)
    q = _rows16(q)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        _check(out.shape == q.shape and out.dtype == q.dtype, "out must be a tensor like q")
        _check(_rows16(out) is out, "out's heads must lie whole on 16-byte boundaries")
    page_table = page_table if page_table.stride(1) == 1 or page_table.shape[1] <= 1 else page_table.contiguous()
    q_offsets, kv_lengths = q_offsets.contiguous(), kv_lengths.contiguous()
    a = _lib.AttentionPagedArgs()
    a.pages, a.q, a.out, a.dtype = p, _ptr(q), _ptr(out), _KV_TYPES[q.dtype]
    a.page_table, a.q_offsets, a.kv_lengths = _ptr(page_table), _ptr(q_offsets), _ptr(kv_lengths)
    a.tokens, a.q_heads, a.sequences, a.table_width = q.shape[0], q.shape[1], b, page_table.shape[1]
    a.table_stride, a.window, a.causal = page_table.stride(0), int(window), int(bool(causal))
    a.q_token_stride, a.q_head_stride, a.out_token_stride, a.out_head_stride = q.stride(0), q.stride(1), out.stride(0), out.stride(1)
    a.scale = p.head_dim ** -0.5 if scale is None else float(scale)
    with torch.cuda.device(q.device):
        need = _lib.load().arcq_attention_paged_workspace(ctypes.byref(a))
        _lib.check(min(need, 0))
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        a.workspace = _ptr(ws) or None
        _lib.check(_lib.load().arcq_attention_paged_fwd(ctypes.byref(a), _stream()))
    return out
