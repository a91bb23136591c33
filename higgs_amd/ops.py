"""Host-side mirror of the mlx-rs calls higgs-models makes on this path, over
the C ABI of libhiggs_hip.so. torch supplies device memory and the stream only.

Each function keeps the reference call's name and argument meaning:

    rms_norm(x, weight, eps)                 mlx_rs::fast::rms_norm / nn::RmsNorm
    rope(x, dims, traditional, base, scale, offset, freqs)
                                             mlx_rs::fast::rope (utils.rs:16-26)
    qk_norm_rope(...)                        q_norm/k_norm + transpose + apply_rope
                                             (transformer.rs:264-287)
    swiglu(gate, x)                          qwen3_next.rs:275-277
    silu_mul(gate, up)                       nn::silu(gate) * up (transformer.rs:349-353)
    gelu_approximate_mul(gate, up)           nn::gelu_approximate(gate) * up (gemma2.rs:422-427)
    gated_rms_norm(x, z, weight, eps)        swiglu(z, norm(x)) (qwen3_next.rs:1204-1205)
    add_rms_norm(x, r, weight, eps)          h = x.add(r); norm(h) (transformer.rs:413-415)
    QuantizedEmbedding(...).forward(ids)     nn::QuantizedEmbedding / QEmbedding::forward
    gather_qmm(x, w, scales, biases, rhs_indices)   qwen3_next.rs:294-363, 844-904
    gated_delta(q, k, v, a_log, a, dt_bias, b, state)
                                             qwen3_next.rs:376-451, 1152-1201
    QuantizedEmbedding(...).forward_rms_norm(ids, w, eps)
                                             embed_tokens + the first input_layernorm
                                             (transformer.rs:494, 407)
    kv_append(k, v, k_pages, v_pages, ...)   KeyValueCache::update (cache.rs:4-29, 130-312)
    kv_copy_pages(k_pages, v_pages, src, dst)   the copy of a cache (prompt_cache.rs:22-307)
    paged_attention(q, k_pages, v_pages, ...)   fast::scaled_dot_product_attention and its
                                             masks (utils.rs:28-125; gemma2.rs:219-379)
    shared_prefix_attention(q, ..., prefix_table, prefix_len)
                                             the same of a batch that begins with one prompt
                                             (prompt_cache.rs:22-307)
    kv_extend(tables, lens, ...), kv_release(...)   cache growth, lengths and offsets of a batch
                                             (cache.rs:130-312; transformer.rs:747-802)
    moe_route(logits, top_k)                 router softmax + argpartition + weights
                                             (qwen3_next.rs:949-985; qwen3_moe.rs:293-322)
    moe_combine(y, weights, shared=...)      the experts' weighted sum (qwen3_next.rs:970-985)
    OpSequence                               a decode step's per-layer ops in one launch
                                             (the layer loop, qwen3_next.rs:1508-1547)

Errors surface as HgkError (the reference returns Err(Exception::custom(..))).
Every op enqueues on torch's current CUDA/HIP stream and never synchronises.
"""
from __future__ import annotations

import ctypes as C
import math
import operator
import struct
from typing import NamedTuple, Optional, Sequence

import torch

from ._lib import (ACT_GELU_TANH, ACT_SILU, BF16, F16, F32, I32, OP_ADD_RMS_NORM, OP_GATED_RMS_NORM,
                   OP_GLU, OP_QK_NORM_ROPE, OP_RMS_NORM, SCORE_SIGMOID, SCORE_SOFTMAX, U32, HgkError, HgkOp,
                   check, f32_array, i64_array, lib)

_DT = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16, torch.int32: I32}
if hasattr(torch, "uint32"):
    _DT[torch.uint32] = U32
_TORCH = {F32: torch.float32, BF16: torch.bfloat16, F16: torch.float16}


def dtype_code(t: torch.dtype) -> int:
    try:
        return _DT[t]
    except KeyError:
        raise HgkError(1, f"unsupported dtype {t}") from None


def _promote(a: int, b: int) -> int:
    return a if a == b else F32


# A small op's call costs more on the host than on the device (the norm of 512
# rows: 11.1 us a call, about 1 us of it the kernel), so what every call does is
# kept short: pointers and streams go to ctypes as plain ints (it converts them
# by the prototype), the stream handle comes without a Stream object around it,
# and contiguous tensors are measured without making a view.
def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream(device: torch.device):
    if device.type != "cuda" or device.index is None:
        return torch.cuda.current_stream(device).cuda_stream  # raises for other devices
    return torch._C._cuda_getCurrentRawStream(device.index)


def _rows2d(x: torch.Tensor):
    """View x as [rows, n] with unit stride on n; returns (rows, n, row_stride)."""
    if x.dim() == 0:
        raise HgkError(1, "expected at least 1 dimension")
    n = x.shape[-1]
    if n > 1 and x.stride(-1) != 1:
        raise HgkError(1, "last axis must be unit-stride")
    if x.dim() == 1:
        return 1, n, n
    if n > 0 and x.is_contiguous():
        return x.numel() // n, n, n
    try:
        x2 = x.view(-1, n)
    except RuntimeError:
        raise HgkError(1, "leading axes must collapse to a single row stride") from None
    return x2.shape[0], n, x2.stride(0)


# ---------------------------------------------------------------- RMSNorm
def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float, *,
             plus_one: bool = False, out_dtype: Optional[torch.dtype] = None,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """fast::rms_norm(x, weight, eps) over the last axis. ``plus_one`` applies
    Gemma's (1 + weight) in f32 (the reference bakes it into the weight at load
    time, gemma2.rs:799-826). The default output dtype is MLX's promotion of x
    and the effective weight."""
    xd = dtype_code(x.dtype)
    wd = dtype_code(weight.dtype) if weight is not None else xd
    w_eff = (F32 if plus_one else wd) if weight is not None else xd
    od = dtype_code(out_dtype) if out_dtype is not None else _promote(xd, w_eff)
    rows, n, xs = _rows2d(x)
    if weight is not None and (weight.dim() != 1 or weight.shape[0] != n):
        raise HgkError(1, f"weight shape {tuple(weight.shape)} does not match ({n},)")
    if out is None:
        out = torch.empty(x.shape, dtype=_TORCH[od], device=x.device)
    _, _, ys = _rows2d(out)
    check(lib().hgk_rms_norm(_ptr(x), xd, xs, _ptr(weight), wd, int(plus_one), eps,
                             _ptr(out), od, ys, rows, n, _stream(x.device)))
    return out


def add_rms_norm(x: torch.Tensor, r: torch.Tensor, weight: Optional[torch.Tensor], eps: float,
                 *, plus_one: bool = False, out_dtype: Optional[torch.dtype] = None,
                 h_out: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                 write_h: bool = True):
    """The block boundary `h = x.add(residual); norm.forward(&h)`
    (transformer.rs:413-415; qwen3_next.rs:1539-1540) in one pass: returns
    (h, y). Pass ``h_out=x`` to update the residual stream in place;
    ``write_h=False`` skips h (returns None for it)."""
    xd = dtype_code(x.dtype)
    if r.dtype != x.dtype or r.shape != x.shape:
        raise HgkError(1, "x and r must match in shape and dtype")
    wd = dtype_code(weight.dtype) if weight is not None else xd
    w_eff = (F32 if plus_one else wd) if weight is not None else xd
    od = dtype_code(out_dtype) if out_dtype is not None else _promote(xd, w_eff)
    rows, n, xs = _rows2d(x)
    _, _, rs = _rows2d(r)
    if weight is not None and (weight.dim() != 1 or weight.shape[0] != n):
        raise HgkError(1, f"weight shape {tuple(weight.shape)} does not match ({n},)")
    if write_h and h_out is None:
        h_out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    hs = _rows2d(h_out)[2] if h_out is not None else 0
    if out is None:
        out = torch.empty(x.shape, dtype=_TORCH[od], device=x.device)
    _, _, ys = _rows2d(out)
    check(lib().hgk_add_rms_norm(xd, _ptr(x), xs, _ptr(r), rs, _ptr(weight), wd, int(plus_one),
                                 eps, _ptr(h_out), hs, _ptr(out), od, ys, rows, n,
                                 _stream(x.device)))
    return h_out, out


def _z_layout(z: torch.Tensor, rows: int, n: int):
    """(row_stride, group_rows, group_stride) addressing z's rows in place."""
    try:
        zr, zn, zs = _rows2d(z)
        if (zr, zn) == (rows, n):
            return zs, 0, 0
    except HgkError:
        pass
    if z.dim() >= 3 and z.shape[-1] == n and z.stride(-1) == 1:
        try:
            z3 = z.view(-1, z.shape[-2], n)
        except RuntimeError:
            raise HgkError(1, "z layout is not expressible as (groups, rows, n)") from None
        if z3.shape[0] * z3.shape[1] == rows:
            return z3.stride(1), z3.shape[1], z3.stride(0)
    raise HgkError(1, f"z shape {tuple(z.shape)} does not match {rows} rows of {n}")


def gated_rms_norm(x: torch.Tensor, z: torch.Tensor, weight: torch.Tensor, eps: float, *,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """swiglu(z, rms_norm(x, weight, eps)) = z * sigmoid(z) * norm(x).

    z may be a strided view such as the z slice of Qwen3-Next's in_proj_qkvz
    output viewed as [..., v_per_k, head_v_dim]; it is read in place."""
    xd = dtype_code(x.dtype)
    wd = dtype_code(weight.dtype)
    od = _promote(xd, _promote(xd, wd))
    rows, n, xs = _rows2d(x)
    if z.dtype != x.dtype:
        raise HgkError(1, "z must have x's dtype")
    zs, zg, zgs = _z_layout(z, rows, n)
    if out is None:
        out = torch.empty(x.shape, dtype=_TORCH[od], device=x.device)
    _, _, os_ = _rows2d(out)
    check(lib().hgk_gated_rms_norm(xd, _ptr(x), xs, _ptr(z), zs, zg, zgs, _ptr(weight), wd,
                                   eps, _ptr(out), od, os_, rows, n, _stream(x.device)))
    return out


# ---------------------------------------------------------------- RoPE
def rope_inv_freq(base: float, dims: int, freqs: Optional[Sequence[float]] = None):
    inv = (C.c_float * (dims // 2))()
    fr = None if freqs is None else f32_array(list(freqs))
    check(lib().hgk_rope_inv_freq(base, dims, fr, inv))
    return list(inv)


def llama3_rope_freqs(base: float, dims: int, factor: float, low_freq_factor: float,
                      high_freq_factor: float, original_max_position: float):
    """mlx-lm Llama3RoPE frequency table (pass as ``freqs`` to rope)."""
    f = (C.c_float * (dims // 2))()
    check(lib().hgk_llama3_rope_freqs(base, dims, factor, low_freq_factor, high_freq_factor,
                                      original_max_position, f))
    return list(f)


def _freqs_arg(freqs):
    if freqs is None:
        return None
    if isinstance(freqs, torch.Tensor):
        freqs = freqs.detach().to("cpu", torch.float32).tolist()
    return f32_array(list(freqs))


def _offsets_arg(offsets, batch, device):
    if offsets is None:
        return None, None
    if not isinstance(offsets, torch.Tensor):
        offsets = torch.tensor(list(offsets), dtype=torch.int32, device=device)
    if offsets.dtype != torch.int32 or offsets.device != device or offsets.numel() != batch:
        raise HgkError(1, f"offsets must be int32[{batch}] on {device}")
    offsets = offsets.contiguous()
    return offsets, _ptr(offsets)


def rope(x: torch.Tensor, dims: int, traditional: bool = False, base: Optional[float] = 10000.0,
         scale: float = 1.0, offset: int = 0, freqs=None, *, offsets=None,
         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """fast::rope(x, dims, traditional, base, scale, offset, freqs).

    x is [..., L, D] with positions along axis -2, as MLX's rope; leading axes
    are flattened to [N, ...]. For 4-D x [B, H, L, D] (the reference's
    post-transpose layout), ``offsets`` (int32[B]) gives each sequence its own
    offset, replacing forward_batched's per-request loop."""
    if (freqs is None) == (base is None):
        raise HgkError(1, "exactly one of base and freqs must be given")
    if x.dim() < 3:
        raise HgkError(1, "rope expects at least 3 dimensions")
    D, L = x.shape[-1], x.shape[-2]
    if x.dim() == 3:
        B, H = x.shape[0], 1
        xs = (x.stride(0), x.stride(1), 0)
    else:
        xv = x.reshape(-1, x.shape[-3], L, D) if x.dim() > 4 else x
        B, H = xv.shape[0], xv.shape[1]
        xs = (xv.stride(0), xv.stride(2), xv.stride(1))
        x = xv
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out.dim() == 3:
        ys = (out.stride(0), out.stride(1), 0)
    else:
        ys = (out.stride(0), out.stride(2), out.stride(1))
    offs, offs_p = _offsets_arg(offsets, B, x.device)
    check(lib().hgk_rope(dtype_code(x.dtype), _ptr(x), i64_array(xs), _ptr(out), i64_array(ys),
                         B, L, H, D, dims, int(traditional), float(base or 0.0), scale,
                         _freqs_arg(freqs), offset, offs_p, _stream(x.device)))
    return out


def qk_norm_rope(q: torch.Tensor, k: Optional[torch.Tensor], q_norm_w: Optional[torch.Tensor],
                 k_norm_w: Optional[torch.Tensor], eps: float, dims: int, base: float = 10000.0,
                 scale: float = 1.0, offset: int = 0, freqs=None, *, offsets=None,
                 q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None):
    """Per-head RMSNorm + RoPE for q [B, L, Hq, D] and k [B, L, Hk, D] (the
    projection layout, any strides with unit D stride). Outputs default to the
    reference's post-transpose [B, H, L, D] contiguous layout."""
    B, L, Hq, D = q.shape
    wd = dtype_code(q_norm_w.dtype if q_norm_w is not None else
                    (k_norm_w.dtype if k_norm_w is not None else q.dtype))
    if q_out is None:
        q_out = torch.empty((B, Hq, L, D), dtype=q.dtype, device=q.device)
    qos = (q_out.stride(0), q_out.stride(2), q_out.stride(1))
    Hk = 0
    ks = kos = (0, 0, 0)
    if k is not None:
        Hk = k.shape[2]
        if k_out is None:
            k_out = torch.empty((B, Hk, L, D), dtype=k.dtype, device=k.device)
        ks = (k.stride(0), k.stride(1), k.stride(2))
        kos = (k_out.stride(0), k_out.stride(2), k_out.stride(1))
    offs, offs_p = _offsets_arg(offsets, B, q.device)
    qs = (q.stride(0), q.stride(1), q.stride(2))
    check(lib().hgk_qk_norm_rope(
        dtype_code(q.dtype), _ptr(q), i64_array(qs), _ptr(q_out), i64_array(qos), Hq,
        _ptr(q_norm_w), _ptr(k), i64_array(ks), _ptr(k_out), i64_array(kos), Hk,
        _ptr(k_norm_w), wd, eps, B, L, D, dims, float(base or 0.0), scale,
        _freqs_arg(freqs), offset, offs_p, _stream(q.device)))
    return q_out, k_out


# ---------------------------------------------------------------- GLU
def _glu(act: int, gate: torch.Tensor, up: torch.Tensor, out_dtype, out):
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise HgkError(1, "gate and up must match in shape and dtype")
    xd = dtype_code(gate.dtype)
    od = dtype_code(out_dtype) if out_dtype is not None else xd
    rows, n, gs = _rows2d(gate)
    _, _, us = _rows2d(up)
    if out is None:
        out = torch.empty(gate.shape, dtype=_TORCH[od], device=gate.device)
    _, _, os_ = _rows2d(out)
    check(lib().hgk_glu(act, xd, _ptr(gate), gs, _ptr(up), us, _ptr(out), od, os_, rows, n,
                        _stream(gate.device)))
    return out


def silu_mul(gate, up, *, out_dtype=None, out=None):
    """nn::silu(gate) * up (transformer.rs:349-353)."""
    return _glu(ACT_SILU, gate, up, out_dtype, out)


def swiglu(gate, x, *, out=None):
    """swiglu(gate, x) = gate * sigmoid(gate) * x (qwen3_next.rs:275-277)."""
    return _glu(ACT_SILU, gate, x, None, out)


def gelu_approximate_mul(gate, up, *, out_dtype=None, out=None):
    """nn::gelu_approximate(gate) * up (gemma2.rs:422-427)."""
    return _glu(ACT_GELU_TANH, gate, up, out_dtype, out)


def fused_gate_up_swiglu(gate_up: torch.Tensor, *, out=None):
    """phi3-style fused projection [.., 2I]: silu(first half) * second half
    (phi3.rs:261-265), read in place through row strides."""
    I2 = gate_up.shape[-1]
    return _glu(ACT_SILU, gate_up[..., : I2 // 2], gate_up[..., I2 // 2:], None, out)


# ---------------------------------------------------------------- gather_qmm
def gather_qmm(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor,
               rhs_indices: torch.Tensor, transpose: bool = True, group_size: int = 64,
               bits: int = 4, *, x_row_div: int = 1, lhs_indices: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gather_qmm(x, w, scales, biases, rhs_indices, transpose, group_size, bits)
    as SwitchMlpWeights::forward_gather uses it (qwen3_next.rs:844-904): one
    row of x per (token, expert) pair. x is [R, K]; w [E, N, K*bits/32] packed
    32-bit words; rhs_indices [P] expert per pair; pair p reads x row
    lhs_indices[p], or p // x_row_div (x_row_div = top_k broadcasts a token
    over its experts). Returns y [P, N] in x's dtype."""
    if not transpose:
        raise HgkError(2, "gather_qmm: only transpose=True (weights stored [N, K]) is implemented")
    if x.dim() != 2 or x.stride(-1) != 1:
        raise HgkError(1, "x must be [rows, K] with a unit-stride last axis")
    if w.dim() != 3 or scales.dim() != 3 or scales.shape != biases.shape:
        raise HgkError(1, "w must be [E, N, K/8]; scales and biases [E, N, K/group]")
    if scales.dtype != biases.dtype:
        raise HgkError(1, "scales and biases must share a dtype")
    E, N = w.shape[0], w.shape[1]
    K = x.shape[1]
    P = rhs_indices.numel()
    idx = rhs_indices.reshape(-1).contiguous()
    lhs = None if lhs_indices is None else lhs_indices.reshape(-1).contiguous()
    if out is None:
        out = torch.empty((P, N), dtype=x.dtype, device=x.device)
    check(lib().hgk_gather_qmm(dtype_code(x.dtype), _ptr(x), x.shape[0], x.stride(0), x_row_div,
                               _ptr(lhs), _ptr(w.contiguous()), _ptr(scales.contiguous()),
                               _ptr(biases.contiguous()), dtype_code(scales.dtype), E, N, K,
                               group_size, bits, _ptr(idx), dtype_code(idx.dtype), P, _ptr(out),
                               out.stride(0), _stream(x.device)))
    return out


def gather_qmm_swiglu(x: torch.Tensor, w_gate: torch.Tensor, scales_gate: torch.Tensor,
                      biases_gate: torch.Tensor, w_up: torch.Tensor, scales_up: torch.Tensor,
                      biases_up: torch.Tensor, rhs_indices: torch.Tensor, group_size: int = 64,
                      bits: int = 4, *, x_row_div: int = 1,
                      lhs_indices: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """swiglu(gather_qmm(x, gate...), gather_qmm(x, up...)) -- the gate/up half of
    SwitchMlpWeights::forward_gather (qwen3_next.rs:862-886) -- in one launch
    where a fused kernel applies (the per-pair decode kernel, or the grouped
    matrix-core kernel's fused form at 16 or more pairs per expert), else as
    the three calls. Returns [P, N] in x's dtype."""
    E, N = w_gate.shape[0], w_gate.shape[1]
    K = x.shape[1]
    idx = rhs_indices.reshape(-1).contiguous()
    P = idx.numel()
    lhs = None if lhs_indices is None else lhs_indices.reshape(-1).contiguous()
    if out is None:
        out = torch.empty((P, N), dtype=x.dtype, device=x.device)
    if w_up.shape != w_gate.shape or scales_up.shape != scales_gate.shape:
        raise HgkError(1, "gate and up weights must have the same shapes")
    for name, t in (("biases_gate", biases_gate), ("scales_up", scales_up), ("biases_up", biases_up)):
        # one scales dtype reaches the kernel for both projections
        if t.dtype != scales_gate.dtype:
            raise HgkError(1, f"{name} dtype {t.dtype} differs from scales_gate's {scales_gate.dtype}")
    st = lib().hgk_gather_qmm_swiglu(
        dtype_code(x.dtype), _ptr(x), x.shape[0], x.stride(0), x_row_div, _ptr(lhs),
        _ptr(w_gate.contiguous()), _ptr(scales_gate.contiguous()), _ptr(biases_gate.contiguous()),
        _ptr(w_up.contiguous()), _ptr(scales_up.contiguous()), _ptr(biases_up.contiguous()),
        dtype_code(scales_gate.dtype), E, N, K, group_size, bits, _ptr(idx),
        dtype_code(idx.dtype), P, _ptr(out), out.stride(0), _stream(x.device))
    if st == 2:  # not the fused kernel's regime: the reference's three calls
        g = gather_qmm(x, w_gate, scales_gate, biases_gate, idx, True, group_size, bits,
                       x_row_div=x_row_div, lhs_indices=lhs)
        u = gather_qmm(x, w_up, scales_up, biases_up, idx, True, group_size, bits,
                       x_row_div=x_row_div, lhs_indices=lhs)
        return swiglu(g, u, out=out)
    check(st)
    return out


def quantized_matmul(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor,
                     biases: torch.Tensor, transpose: bool = True, group_size: int = 64,
                     bits: int = 4, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """quantized_matmul(x, w, scales, biases, transpose, group_size, bits) as
    QLinear::forward calls it (qwen3_next.rs:174-221): x [..., K], w [N,
    K*bits/32] packed 32-bit words, scales/biases [N, K/group_size]. Returns
    y [..., N] in x's dtype. bf16 with group 64 runs on the matrix cores from 16
    rows on, and from 2 rows where K is 512, 1024, 2048 or 4096; fewer rows, f16
    and other groups run on the GEMV kernels."""
    if not transpose:
        raise HgkError(2, "quantized_matmul: only transpose=True (weights stored [N, K]) is implemented")
    if w.dim() != 2 or scales.dim() != 2 or scales.shape != biases.shape:
        raise HgkError(1, "w must be [N, K/8]; scales and biases [N, K/group]")
    if scales.dtype != biases.dtype:
        raise HgkError(1, "scales and biases must share a dtype")
    K = x.shape[-1]
    N = w.shape[0]
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    M = x2.shape[0]
    if out is None:
        out = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=x.device)
    o2 = out if out.dim() == 2 and out.shape[1] == N else out.view(-1, N)
    check(lib().hgk_quantized_matmul(dtype_code(x.dtype), _ptr(x2), M, x2.stride(0) if M else K,
                                     _ptr(w.contiguous()), _ptr(scales.contiguous()),
                                     _ptr(biases.contiguous()), dtype_code(scales.dtype), N, K,
                                     group_size, bits, _ptr(o2), o2.stride(0) if M else N,
                                     _stream(x.device)))
    return out


# ---------------------------------------------------------------- GatedDeltaNet
def gdn_qk_norm_weights(head_k_dim: int, dtype: torch.dtype, device):
    """GatedDeltaNet's constant q/k norm weights (qwen3_next.rs:1075-1094, cast to the input dtype at 1165-1169):
    s = 1/sqrt(Dk) in f32; q's weight is s*s, k's is s, cast to `dtype`."""
    s = torch.tensor(1.0, dtype=torch.float32) / torch.sqrt(torch.tensor(float(head_k_dim)))
    wq = torch.full((head_k_dim,), float(s * s), dtype=torch.float32).to(dtype)
    wk = torch.full((head_k_dim,), float(s), dtype=torch.float32).to(dtype)
    return wq.to(device), wk.to(device)


def gated_delta(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, a_log: torch.Tensor,
                a: torch.Tensor, dt_bias: torch.Tensor, b: torch.Tensor,
                state: Optional[torch.Tensor] = None, *, q_norm_w: Optional[torch.Tensor] = None,
                k_norm_w: Optional[torch.Tensor] = None, eps: float = 1e-6,
                state_out: Optional[torch.Tensor] = None):
    """The gated-delta recurrence (gated_delta_kernel_ffi, qwen3_next.rs:376-451)
    with the optional constant-weight q/k RMSNorm fused in: q, k [B, T, Hk, Dk],
    v [B, T, Hv, Dv], a, b [B, T, Hv], a_log, dt_bias [Hv], state [B, Hv, Dv, Dk]
    or None (zeros). Returns (y [B, T, Hv, Dv], new_state)."""
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2], v.shape[3]
    for t in (q, k, v, a, b):
        if not t.is_contiguous() or t.dtype != q.dtype:
            raise HgkError(1, "q, k, v, a, b must be contiguous and share a dtype")
    if a_log.dtype != dt_bias.dtype:
        raise HgkError(1, "a_log and dt_bias must share a dtype")
    y = torch.empty((B, T, Hv, Dv), dtype=q.dtype, device=q.device)
    if state_out is None:
        state_out = torch.empty((B, Hv, Dv, Dk), dtype=q.dtype, device=q.device)
    check(lib().hgk_gated_delta(dtype_code(q.dtype), _ptr(q), _ptr(k), _ptr(v),
                                _ptr(a_log.contiguous()), _ptr(a), _ptr(dt_bias.contiguous()),
                                _ptr(b), dtype_code(a_log.dtype),
                                None if state is None else _ptr(state.contiguous()),
                                _ptr(q_norm_w), _ptr(k_norm_w), eps, B, T, Hk, Dk, Hv, Dv,
                                _ptr(y), _ptr(state_out), _stream(q.device)))
    return y, state_out


def gated_delta_gated_norm(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                           a_log: torch.Tensor, a: torch.Tensor, dt_bias: torch.Tensor,
                           b: torch.Tensor, state: Optional[torch.Tensor], z: torch.Tensor,
                           norm_weight: torch.Tensor, norm_eps: float, *,
                           q_norm_w: Optional[torch.Tensor] = None,
                           k_norm_w: Optional[torch.Tensor] = None, eps: float = 1e-6,
                           state_out: Optional[torch.Tensor] = None,
                           out: Optional[torch.Tensor] = None):
    """One decode token of GatedDeltaNet from the recurrence through its gated
    output norm (qwen3_next.rs:1185-1205): swiglu(z, norm(gated_delta(...).y))
    in one launch where it applies, else as the two calls. q, k [B, 1, Hk, Dk],
    v [B, 1, Hv, Dv], a, b [B, 1, Hv]; z [B, 1, Hv, Dv] (may be a strided view
    of in_proj_qkvz). Returns (out [B, 1, Hv, Dv], new_state)."""
    B, T, Hk, Dk = q.shape
    Hv, Dv = v.shape[2], v.shape[3]
    if T != 1:
        raise HgkError(1, "gated_delta_gated_norm is the one-token (decode) form")
    for t in (q, k, v, a, b):
        if not t.is_contiguous() or t.dtype != q.dtype:
            raise HgkError(1, "q, k, v, a, b must be contiguous and share a dtype")
    if a_log.dtype != dt_bias.dtype:
        raise HgkError(1, "a_log and dt_bias must share a dtype")
    if state_out is None:
        state_out = torch.empty((B, Hv, Dv, Dk), dtype=q.dtype, device=q.device)
    if out is None:
        out = torch.empty((B, T, Hv, Dv), dtype=q.dtype, device=q.device)
    zs, zg, zgs = _z_layout(z, B * Hv, Dv)
    st = lib().hgk_gated_delta_gated_norm(
        dtype_code(q.dtype), _ptr(q), _ptr(k), _ptr(v), _ptr(a_log.contiguous()), _ptr(a),
        _ptr(dt_bias.contiguous()), _ptr(b), dtype_code(a_log.dtype),
        None if state is None else _ptr(state.contiguous()), _ptr(q_norm_w), _ptr(k_norm_w), eps,
        B, Hk, Dk, Hv, Dv, _ptr(state_out), None, _ptr(z), zs, zg, zgs, _ptr(norm_weight),
        dtype_code(norm_weight.dtype), norm_eps, _ptr(out), _stream(q.device))
    if st == 2:  # outside the fused form: the reference's two calls
        y, state_out = gated_delta(q, k, v, a_log, a, dt_bias, b, state, q_norm_w=q_norm_w,
                                   k_norm_w=k_norm_w, eps=eps, state_out=state_out)
        gated_rms_norm(y, z, norm_weight, norm_eps, out=out)
        return out, state_out
    check(st)
    return out, state_out


# ---------------------------------------------------------------- paged cache
# hgk_kv_pages and hgk_kv_batch as one pack call each (native alignment is the
# C layout): shorter on the host than filling ctypes structures field by field
_KV_PAGES = struct.Struct("@iiqqqP3qP3q")
_KV_BATCH = struct.Struct("@qqPqqPP")


def _pool(k_pages: torch.Tensor, v_pages: torch.Tensor, what: str):
    """The packed hgk_kv_pages of pools [n_pages, page_size, Hk, D]."""
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
        raise HgkError(1, f"{what}: pages must be [n_pages, page_size, kv_heads, head_dim], "
                          "keys and values alike")
    if k_pages.dtype != v_pages.dtype or k_pages.device != v_pages.device:
        raise HgkError(1, f"{what}: key and value pages must share dtype and device")
    n, ps, hk, d = k_pages.shape
    ks, vs = k_pages.stride(), v_pages.stride()
    if ks[3] != 1 or vs[3] != 1:
        raise HgkError(1, f"{what}: last axis must be unit-stride")
    return _KV_PAGES.pack(dtype_code(k_pages.dtype), ps, n, hk, d, k_pages.data_ptr(), *ks[:3],
                          v_pages.data_ptr(), *vs[:3])


def _kv_batch(tokens: int, block_table: torch.Tensor, kv_lens: torch.Tensor, q_starts, device,
              what: str):
    """The packed hgk_kv_batch."""
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.stride(1) != 1 \
            and block_table.shape[1] > 1:
        raise HgkError(1, f"{what}: block_table must be int32 [batch, pages] with a unit-stride last axis")
    batch = block_table.shape[0]
    if kv_lens.dtype != torch.int32 or kv_lens.shape != (batch,) or not kv_lens.is_contiguous():
        raise HgkError(1, f"{what}: kv_lens must be contiguous int32[{batch}]")
    if block_table.device != device or kv_lens.device != device:
        raise HgkError(1, f"{what}: operands on different devices")
    if q_starts is not None and (q_starts.dtype != torch.int32 or q_starts.shape != (batch + 1,)
                                 or not q_starts.is_contiguous() or q_starts.device != device):
        raise HgkError(1, f"{what}: q_starts must be contiguous int32[{batch + 1}] on {device}")
    return _KV_BATCH.pack(batch, tokens, block_table.data_ptr(), block_table.stride(0),
                          block_table.shape[1], kv_lens.data_ptr(),
                          0 if q_starts is None else q_starts.data_ptr())


def _token_rows(t: torch.Tensor, pages: torch.Tensor, what: str, name: str):
    """(token, head) strides of a [tokens, heads, D] operand, packed."""
    if t.dim() != 3 or t.shape[2] != pages.shape[3]:
        raise HgkError(1, f"{what}: {name} must be [tokens, heads, {pages.shape[3]}]")
    if t.dtype != pages.dtype or t.device != pages.device:
        raise HgkError(1, f"{what}: {name} must share the pages' dtype and device")
    st = t.stride()
    if st[2] != 1:
        raise HgkError(1, f"{what}: {name}: last axis must be unit-stride")
    return _TWO.pack(st[0], st[1])


_TWO = struct.Struct("@qq")


def _kv_call(device: torch.device, fn, *args):
    """fn(*args, stream) with the device current, as a launch needs: a stream
    takes launches of its own device only."""
    if device.type != "cuda":
        raise HgkError(1, f"operands must be on the GPU, not on {device}")
    if device.index == torch._C._cuda_getDevice():
        check(fn(*args, torch._C._cuda_getCurrentRawStream(device.index)))
    else:
        with torch.cuda.device(device):
            check(fn(*args, torch._C._cuda_getCurrentRawStream(device.index)))


def kv_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
              block_table: Optional[torch.Tensor] = None, kv_lens: Optional[torch.Tensor] = None, *,
              q_starts: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None) -> None:
    """Writes new tokens' keys and values, k and v [T, Hk, D] (any token and
    head strides), into their sequences' pages [n_pages, page_size, Hk, D].

    block_table int32 [B, P] names each sequence's pages in order; kv_lens
    int32 [B] counts its tokens with the new ones, which are its last. Sequence
    b owns rows q_starts[b] .. q_starts[b+1]-1 of k and v (int32 [B+1]);
    without q_starts, row b is its one new token. Rows of no sequence,
    positions beyond the table and pages outside the pool are skipped. The key
    pages may not lie on the value pages, unless k is v and they are the same.

    With ``slots`` (int64 [T], as kv_extend gives them) row t goes to place
    slots[t] % page_size of page slots[t] // page_size instead, and a slot below
    zero or past the pool is skipped; no table, lengths or starts are given then."""
    what = "kv_append"
    pool = _pool(k_pages, v_pages, what)
    ks, vs = _token_rows(k, k_pages, what, "k"), _token_rows(v, k_pages, what, "v")
    if k.shape != v.shape or k.shape[1] != k_pages.shape[2]:
        raise HgkError(1, f"{what}: k and v must be [tokens, {k_pages.shape[2]}, {k_pages.shape[3]}]")
    dev = k_pages.device
    if slots is not None:
        if block_table is not None or kv_lens is not None or q_starts is not None:
            raise HgkError(1, f"{what}: slots stand in place of block_table, kv_lens and q_starts")
        if slots.dtype != torch.int64 or slots.shape != (k.shape[0],) or not slots.is_contiguous() \
                or slots.device != dev:
            raise HgkError(1, f"{what}: slots must be contiguous int64[{k.shape[0]}] on {dev}")
        _kv_call(dev, lib().hgk_kv_append_slots, pool, slots.data_ptr(), k.shape[0], k.data_ptr(), ks,
                 v.data_ptr(), vs)
        return
    if block_table is None or kv_lens is None:
        raise HgkError(1, f"{what}: block_table and kv_lens, or slots, must be given")
    batch = _kv_batch(k.shape[0], block_table, kv_lens, q_starts, dev, what)
    _kv_call(dev, lib().hgk_kv_append, pool, batch, k.data_ptr(), ks, v.data_ptr(), vs)


def kv_copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, src: Sequence[int],
                  dst: Sequence[int]) -> None:
    """Copies page src[i] to page dst[i], keys and values, for lists of page
    indices held on the host. Pages are [n_pages, page_size, Hk, D], or
    [layers, n_pages, ...] to copy them in every layer. A destination may
    neither be named twice nor be a source."""
    what = "kv_copy_pages"
    layers, strides = 1, None
    if k_pages.dim() == 5 and k_pages.shape == v_pages.shape:
        layers = k_pages.shape[0]
        strides = _TWO.pack(k_pages.stride(0), v_pages.stride(0))
        if layers == 0:
            return
        k_pages, v_pages = k_pages[0], v_pages[0]
    pool = _pool(k_pages, v_pages, what)
    if len(src) != len(dst):
        raise HgkError(1, f"{what}: {len(src)} sources for {len(dst)} destinations")
    n = len(src)
    try:
        pairs = [operator.index(i) for i in (*src, *dst)]
    except TypeError:
        raise HgkError(1, f"{what}: src and dst must be sequences of page indices") from None
    if n and not -2 ** 31 <= min(pairs) <= max(pairs) < 2 ** 31:  # ctypes would keep the low 32 bits
        raise HgkError(1, f"{what}: a page index outside the pages")
    s, d = (C.c_int32 * n)(*pairs[:n]), (C.c_int32 * n)(*pairs[n:])
    dev = k_pages.device
    _kv_call(dev, lib().hgk_kv_copy_pages, pool, layers, strides, C.addressof(s), C.addressof(d), n)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    block_table: torch.Tensor, kv_lens: torch.Tensor, *,
                    scale: Optional[float] = None, window: int = 0, sinks: int = 0,
                    softcap: float = 0.0, q_starts: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of new tokens over their sequences' pages, which hold
    the new tokens too (kv_append first). q [T, Hq, D] with any token and head
    strides; pages, block_table, kv_lens and q_starts as in kv_append: prompts
    of any lengths over any cached prefix, or, without q_starts, one token per
    sequence. Query head h reads kv head h // (Hq // Hk).

    ``scale`` is 1/sqrt(D) unless given. ``window`` > 0 keeps the last
    ``window`` keys visible, and of the keys before them the first ``sinks``.
    ``softcap`` > 0 replaces a score s by softcap * tanh(s / softcap). A query
    that sees no key gives zeros. Rows of no sequence are not written (without
    ``out`` they hold whatever the new tensor held). ``out`` must not share
    memory with the other operands. Returns [T, Hq, D]."""
    what = "paged_attention"
    pool = _pool(k_pages, v_pages, what)
    qs = _token_rows(q, k_pages, what, "q")
    T, hq, d = q.shape
    if out is None:
        out = torch.empty((T, hq, d), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape:
        raise HgkError(1, f"{what}: out shape {tuple(out.shape)} is not q's")
    if not (0 <= window < 2 ** 63 and 0 <= sinks < 2 ** 63):
        raise HgkError(1, f"{what}: window={window}, sinks={sinks}")
    os_ = _token_rows(out, k_pages, what, "out")
    dev = k_pages.device
    batch = _kv_batch(T, block_table, kv_lens, q_starts, dev, what)
    L = lib()
    need = L.hgk_paged_attention_workspace(pool, batch, hq, window, sinks)
    if need < 0:  # the call refuses the same sizes, with their status
        check(L.hgk_paged_attention(pool, batch, None, None, hq, 1.0, 0.0, window, sinks, None, None, None, 0, None))
    # a workspace of the call's own, from the current stream's pool of memory
    ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
    _kv_call(dev, L.hgk_paged_attention, pool, batch, q.data_ptr(), qs, hq,
             1.0 / math.sqrt(d) if scale is None else scale, softcap, window, sinks,
             out.data_ptr(), os_, None if ws is None else ws.data_ptr(), need)
    return out


def shared_prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                            block_table: torch.Tensor, kv_lens: torch.Tensor, prefix_table: torch.Tensor,
                            prefix_len: int, *, scale: Optional[float] = None, window: int = 0, sinks: int = 0,
                            softcap: float = 0.0, q_starts: Optional[torch.Tensor] = None,
                            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """paged_attention of sequences that all begin with the same ``prefix_len``
    tokens (a host number), whose keys and values are on the pages
    ``prefix_table`` (int32 [P]): they are read and multiplied once for the
    whole batch. kv_lens, positions, ``window`` and ``sinks`` count from a
    sequence's first token, prefix included, so the result is paged_attention's;
    block_table's entries are read from position prefix_len on (one that holds
    tokens on both sides of it is the sequence's own). A sequence shorter than
    the prefix sees its beginning. Everything else as paged_attention."""
    what = "shared_prefix_attention"
    pool = _pool(k_pages, v_pages, what)
    qs = _token_rows(q, k_pages, what, "q")
    T, hq, d = q.shape
    if out is None:
        out = torch.empty((T, hq, d), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape:
        raise HgkError(1, f"{what}: out shape {tuple(out.shape)} is not q's")
    if not (0 <= window < 2 ** 63 and 0 <= sinks < 2 ** 63):
        raise HgkError(1, f"{what}: window={window}, sinks={sinks}")
    prefix_len = operator.index(prefix_len)
    if not 0 <= prefix_len < 2 ** 63:
        raise HgkError(1, f"{what}: prefix_len={prefix_len}")
    os_ = _token_rows(out, k_pages, what, "out")
    dev = k_pages.device
    if prefix_table.dtype != torch.int32 or prefix_table.dim() != 1 or not prefix_table.is_contiguous() \
            or prefix_table.device != dev:
        raise HgkError(1, f"{what}: prefix_table must be contiguous int32 [pages] on {dev}")
    batch = _kv_batch(T, block_table, kv_lens, q_starts, dev, what)
    L, pw = lib(), prefix_table.shape[0]
    need = L.hgk_shared_prefix_attention_workspace(pool, batch, pw, prefix_len, hq, window, sinks)
    if need < 0:  # the call refuses the same sizes, with their status
        check(L.hgk_shared_prefix_attention(pool, batch, None, pw, prefix_len, None, None, hq, 1.0, 0.0, window,
                                            sinks, None, None, None, 0, None))
    ws = torch.empty((need,), dtype=torch.uint8, device=dev) if need else None
    _kv_call(dev, L.hgk_shared_prefix_attention, pool, batch, prefix_table.data_ptr(), pw, prefix_len, q.data_ptr(),
             qs, hq, 1.0 / math.sqrt(d) if scale is None else scale, softcap, window, sinks, out.data_ptr(), os_,
             None if ws is None else ws.data_ptr(), need)
    return out


# ---------------------------------------------------------------- pages on the GPU
_KV_TABLES = struct.Struct("@iqPqqPPqP")


class KVStep(NamedTuple):
    """What kv_extend gives: a call's table, lengths, starts, places and
    positions, and the state after it."""
    block_table: torch.Tensor
    kv_lens: torch.Tensor
    q_starts: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    lens: torch.Tensor
    n_free: torch.Tensor
    status: torch.Tensor


class KVState(NamedTuple):
    """The state after kv_release."""
    lens: torch.Tensor
    n_free: torch.Tensor
    status: torch.Tensor


def _ints(t: torch.Tensor, n: int, dev, what: str, name: str) -> int:
    """The address of a contiguous int32 [n] (n < 0: of any length) on dev."""
    if t.dtype != torch.int32 or t.dim() != 1 or t.device != dev:
        raise HgkError(1, f"{what}: {name} must be int32 [{'n' if n < 0 else n}] on {dev}")
    m = t.shape[0]
    if (m != n and n >= 0) or (m > 1 and t.stride(0) != 1):
        raise HgkError(1, f"{what}: {name} must be contiguous int32[{'n' if n < 0 else n}]")
    return t.data_ptr()


def _kv_tables(tables, lens, free_pages, n_free, page_size, what):
    """The packed hgk_kv_tables, the rows and the pages of a row."""
    if tables.dim() != 2 or tables.dtype != torch.int32:
        raise HgkError(1, f"{what}: tables must be int32 [sequences, pages]")
    dev, (rows, width), (stride, unit) = tables.device, tables.shape, tables.stride()
    if unit != 1 and width > 1:
        raise HgkError(1, f"{what}: tables: last axis must be unit-stride")
    if not 1 <= page_size <= 65536:
        raise HgkError(1, f"{what}: page_size={page_size} must be a power of two in 1..65536")
    return _KV_TABLES.pack(page_size, rows, tables.data_ptr(), stride, width, _ints(lens, rows, dev, what, "lens"),
                           _ints(free_pages, -1, dev, what, "free_pages"), free_pages.shape[0],
                           _ints(n_free, 1, dev, what, "n_free")), rows, width


def kv_extend(tables: torch.Tensor, lens: torch.Tensor, free_pages: torch.Tensor, n_free: torch.Tensor,
              counts: torch.Tensor, page_size: int, tokens: int, *, seqs: Optional[torch.Tensor] = None,
              inplace: bool = False) -> KVStep:
    """Gives sequences room for their new tokens without the host: pages come
    off a stack on the GPU, and the table, lengths, starts, places and positions
    of a call over the new tokens are worked out there.

    tables int32 [S, W] (pages of every resident sequence in order; written in
    place), lens int32 [S] (their tokens), free_pages int32 [N] (a stack: its
    first n_free[0] entries are free), n_free int32 [1]. ``counts`` int32 [B]
    new tokens of the sequences in rows ``seqs`` (int32 [B], any order; without
    it of every row); the last page of one that has room for more is its own.
    ``tokens`` rows is what the packed array of new tokens has; those behind the
    last sequence's belong to none.

    Returns KVStep: block_table [B, W] (the tables themselves without seqs; else
    a copy of the batch's rows, -1 behind their last page), kv_lens [B],
    q_starts [B+1], slots int64 [tokens] (page * page_size + place, -1: none),
    positions [tokens], and the state after: lens [S], n_free [1] (new tensors,
    or with ``inplace`` the ones given). A call that cannot be done whole changes
    nothing and gives a step without new tokens; status [1] tells why (a sum of
    TABLES_PAGES 1, TABLES_WIDTH 2, TABLES_SEQUENCE 4, TABLES_TOKENS 8)."""
    what = "kv_extend"
    state, rows, width = _kv_tables(tables, lens, free_pages, n_free, page_size, what)
    dev = tables.device
    batch = rows if seqs is None else seqs.shape[0] if seqs.dim() == 1 else -1
    c = _ints(counts, batch, dev, what, "counts")
    s = 0 if seqs is None else _ints(seqs, batch, dev, what, "seqs")
    tokens = operator.index(tokens)
    if not 0 <= tokens <= 2 ** 30:
        raise HgkError(1, f"{what}: tokens={tokens}")
    # one array for the small results, the call's workspace of batch + 1 at its end
    small = 3 * batch + tokens + 3
    if inplace:
        ints = torch.empty((small,), dtype=torch.int32, device=dev)
        kv_lens, starts, positions, status, ws = ints.split_with_sizes([batch, batch + 1, tokens, 1, batch + 1])
        lens_out, n_out = lens, n_free
    else:
        ints = torch.empty((small + rows + 1,), dtype=torch.int32, device=dev)
        kv_lens, starts, positions, status, lens_out, n_out, ws = ints.split_with_sizes(
            [batch, batch + 1, tokens, 1, rows, 1, batch + 1])
    slots = torch.empty((tokens,), dtype=torch.int64, device=dev)
    table = tables if seqs is None else torch.empty((batch, width), dtype=torch.int32, device=dev)
    _kv_call(dev, lib().hgk_kv_extend, state, s, c, batch, tokens, lens_out.data_ptr(), n_out.data_ptr(),
             kv_lens.data_ptr(), starts.data_ptr(), slots.data_ptr(), positions.data_ptr(),
             0 if seqs is None else table.data_ptr(), width, status.data_ptr(), ws.data_ptr())
    return KVStep(table, kv_lens, starts, slots, positions, lens_out, n_out, status)


def kv_release(tables: torch.Tensor, lens: torch.Tensor, free_pages: torch.Tensor, n_free: torch.Tensor,
               page_size: int, *, seqs: Optional[torch.Tensor] = None, keep: Optional[torch.Tensor] = None,
               owned_from: Optional[torch.Tensor] = None, inplace: bool = False) -> KVState:
    """Cuts sequences down to their first ``keep`` tokens (int32 [B]; without it
    to none: they end) and puts the pages that they no longer need on the stack
    of free ones. tables, lens, free_pages, n_free, seqs and ``inplace`` as
    kv_extend; the first ``owned_from`` (int32 [S]) pages of a row are not its
    own and stay. Returns KVState: lens [S], n_free [1], status [1] (as
    kv_extend; nothing is changed where it is not zero)."""
    what = "kv_release"
    state, rows, _ = _kv_tables(tables, lens, free_pages, n_free, page_size, what)
    dev = tables.device
    batch = rows if seqs is None else seqs.shape[0] if seqs.dim() == 1 else -1
    s = 0 if seqs is None else _ints(seqs, batch, dev, what, "seqs")
    k = 0 if keep is None else _ints(keep, batch, dev, what, "keep")
    o = 0 if owned_from is None else _ints(owned_from, rows, dev, what, "owned_from")
    if inplace:
        status, ws = torch.empty((batch + 2,), dtype=torch.int32, device=dev).split_with_sizes([1, batch + 1])
        lens_out, n_out = lens, n_free
    else:
        status, lens_out, n_out, ws = torch.empty((batch + rows + 3,), dtype=torch.int32, device=dev).split_with_sizes(
            [1, rows, 1, batch + 1])
    _kv_call(dev, lib().hgk_kv_release, state, s, k, o, batch, lens_out.data_ptr(), n_out.data_ptr(),
             status.data_ptr(), ws.data_ptr())
    return KVState(lens_out, n_out, status)


# ---------------------------------------------------------------- routed experts
_SCORES = {"softmax": SCORE_SOFTMAX, "sigmoid": SCORE_SIGMOID}


def moe_route(logits: torch.Tensor, top_k: int, *, scores: str = "softmax", bias: Optional[torch.Tensor] = None,
              groups: int = 1, top_groups: int = 1, group_top: int = 1, renormalize: bool = False,
              scale: float = 1.0):
    """The experts of every token and their weights, from logits [..., E] (bf16,
    f16 or f32). With s = softmax or sigmoid (``scores``) of a token's logits the
    top_k greatest s + bias (f32 [E]) are chosen, greatest first, equal ones by
    the lower index; with ``top_groups`` < ``groups`` only from the best of E /
    groups experts in a row, a group counting for its greatest s + bias or the
    sum of its two greatest (``group_top`` 1 or 2). Returns (weights f32 [..., top_k],
    experts int32 [..., top_k]): weights are scale * s, divided by the token's sum
    of them first with ``renormalize``. A NaN logit counts as -inf; a token without
    any logit above -inf has weights of 0 (softmax). E up to 1024, top_k up to 64,
    up to 64 groups, of at most 16 experts in each of a group's share of 64 lanes."""
    what = "moe_route"
    if logits.dim() < 1:
        raise HgkError(1, f"{what}: logits must have at least 1 dimension")
    if scores not in _SCORES:
        raise HgkError(1, f"{what}: scores={scores!r} (softmax or sigmoid)")
    dev = logits.device
    rows, n, stride = _rows2d(logits)
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,) or not bias.is_contiguous()
                             or bias.device != dev):
        raise HgkError(1, f"{what}: bias must be contiguous float32[{n}] on {dev}")
    top_k = operator.index(top_k)
    if not 1 <= top_k <= n:
        raise HgkError(1, f"{what}: top_k={top_k} of {n} experts")
    shape = (*logits.shape[:-1], top_k)
    weights = torch.empty(shape, dtype=torch.float32, device=dev)
    experts = torch.empty(shape, dtype=torch.int32, device=dev)
    _kv_call(dev, lib().hgk_moe_route, dtype_code(logits.dtype), logits.data_ptr(), stride, _ptr(bias),
             _SCORES[scores], rows, n, top_k, groups, top_groups, group_top, int(renormalize), scale,
             weights.data_ptr(), experts.data_ptr())
    return weights, experts


def moe_combine(y: torch.Tensor, weights: torch.Tensor, *, shared: Optional[torch.Tensor] = None,
                shared_gate: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t] = sum_i weights[t, i] * y[t * top_k + i] + sigmoid(shared_gate[t]) *
    shared[t]: the experts' outputs y [T * top_k, H] (gather_qmm's, or [..., top_k,
    H]) under moe_route's weights f32 [..., top_k], and the shared expert's
    [..., H] with its gate's logits [...] or [..., 1], if given. A pair of weight
    zero is left out, whatever its row of y holds. Sums are f32, rounded once.
    Returns [..., H] of y's dtype; ``out`` may be ``shared``."""
    what = "moe_combine"
    if weights.dim() < 1 or weights.dtype != torch.float32:
        raise HgkError(1, f"{what}: weights must be float32 [..., top_k]")
    dev = y.device
    rows, n, ys = _rows2d(y)
    tokens, top_k, ws = _rows2d(weights)
    if rows != tokens * top_k:
        raise HgkError(1, f"{what}: {rows} rows of y for {tokens} tokens of {top_k} experts")
    shape = (*weights.shape[:-1], n)
    ss = gs = gd = 0
    if shared is not None:
        if shared.dtype != y.dtype or shared.shape != shape:
            raise HgkError(1, f"{what}: shared must be {y.dtype} {list(shape)}")
        ss = _rows2d(shared)[2]
    if shared_gate is not None:
        lead = shape[:-1]
        if shared_gate.shape != (*lead, 1):
            if shared_gate.shape != lead:
                raise HgkError(1, f"{what}: shared_gate must be {list(lead)} or {[*lead, 1]}")
            shared_gate = shared_gate.unsqueeze(-1)
        gd, gs = dtype_code(shared_gate.dtype), _rows2d(shared_gate)[2]
    if weights.device != dev or (shared is not None and shared.device != dev) \
            or (shared_gate is not None and shared_gate.device != dev) or (out is not None and out.device != dev):
        raise HgkError(1, f"{what}: operands on different devices")
    if out is None:
        out, os_ = torch.empty(shape, dtype=y.dtype, device=dev), n
    elif out.shape != shape or out.dtype != y.dtype:
        raise HgkError(1, f"{what}: out must be {y.dtype} {list(shape)}")
    else:
        os_ = _rows2d(out)[2]
    _kv_call(dev, lib().hgk_moe_combine, dtype_code(y.dtype), y.data_ptr(), ys, weights.data_ptr(), ws, top_k,
             _ptr(shared), ss, _ptr(shared_gate), gd, gs, out.data_ptr(), os_, tokens, n)
    return out


# ---------------------------------------------------------------- embedding
class QuantizedEmbedding:
    """nn::QuantizedEmbedding: 4-bit affine table (weight u32 [V, H/8], scales
    and biases [V, H/group] in bf16/f16). forward(ids) gathers and
    dequantizes only the requested rows; out_scale applies Gemma's
    bf16(sqrt(H)) embedding scale in the same pass (gemma2.rs:587-600)."""

    def __init__(self, weight: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor,
                 group_size: int = 64, bits: int = 4):
        if weight.dtype not in (torch.int32, getattr(torch, "uint32", torch.int32)):
            raise HgkError(1, "weight must hold packed 32-bit words")
        self.weight, self.scales, self.biases = weight, scales, biases
        self.group_size, self.bits = group_size, bits
        self.vocab = weight.shape[0]
        self.hidden = weight.shape[1] * 32 // bits

    def forward(self, ids: torch.Tensor, *, out_scale: float = 0.0,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
        idd = dtype_code(ids.dtype)
        sd = dtype_code(self.scales.dtype)
        flat = ids.reshape(-1).contiguous()
        if out is None:
            out = torch.empty((flat.numel(), self.hidden), dtype=_TORCH[sd], device=ids.device)
        check(lib().hgk_quantized_embedding(
            _ptr(flat), idd, flat.numel(), _ptr(self.weight), _ptr(self.scales),
            _ptr(self.biases), sd, self.vocab, self.hidden, self.group_size, self.bits,
            out_scale, _ptr(out), out.stride(0), _stream(ids.device)))
        return out.reshape(*ids.shape, self.hidden)

    __call__ = forward

    def forward_rms_norm(self, ids: torch.Tensor, weight: torch.Tensor, eps: float, *,
                         plus_one: bool = False, out_scale: float = 0.0,
                         out_dtype: Optional[torch.dtype] = None, write_h: bool = True):
        """forward(ids) followed by the first block's input RMSNorm, in one
        pass: returns (h, y), both [*ids.shape, hidden]; h is None when
        ``write_h`` is False."""
        idd = dtype_code(ids.dtype)
        sd = dtype_code(self.scales.dtype)
        wd = dtype_code(weight.dtype)
        w_eff = F32 if plus_one else wd
        od = dtype_code(out_dtype) if out_dtype is not None else _promote(sd, w_eff)
        flat = ids.reshape(-1).contiguous()
        T = flat.numel()
        h = (torch.empty((T, self.hidden), dtype=_TORCH[sd], device=ids.device)
             if write_h else None)
        y = torch.empty((T, self.hidden), dtype=_TORCH[od], device=ids.device)
        check(lib().hgk_quantized_embedding_rms_norm(
            _ptr(flat), idd, T, _ptr(self.weight), _ptr(self.scales), _ptr(self.biases), sd,
            self.vocab, self.hidden, self.group_size, self.bits, out_scale, _ptr(h),
            self.hidden, _ptr(weight), wd, int(plus_one), eps, _ptr(y), od, self.hidden,
            _stream(ids.device)))
        shape = (*ids.shape, self.hidden)
        return (None if h is None else h.reshape(shape)), y.reshape(shape)


def gemma_embed_scale(hidden: int) -> float:
    """sqrt(hidden) as the reference computes it (f32), before the cast to the
    activation dtype that the kernel applies."""
    return float(math.sqrt(float(hidden)))


# ---------------------------------------------------------------- op sequence
def _tok_rows(t: torch.Tensor, what: str):
    """(rows, n, token stride, row stride) of a [T, n] or [T, rows, n] view
    with a unit-stride last axis."""
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise HgkError(1, f"{what}: the last axis must have unit stride")
    if t.dim() == 2:
        return 1, t.shape[1], t.stride(0), t.shape[1]
    if t.dim() == 3:
        return t.shape[1], t.shape[2], t.stride(0), t.stride(1)
    raise HgkError(1, f"{what}: expected [tokens, n] or [tokens, rows, n]")


class OpSequence:
    """A decode step's per-layer ops -- input_layernorm (residual add +
    RMSNorm), the gated RMSNorm or q/k RMSNorm + RoPE, post_attention_layernorm,
    the experts' SwiGLU, layer after layer as the loop of qwen3_next.rs:1508-1547
    calls them -- recorded once, uploaded once, then run over a batch of tokens
    in one launch (hgk_op_list_upload / hgk_op_list_run). Every operand is a
    view whose first axis is the token; the recorded addresses are used at
    every run, so the tensors must stay alive and in place (this object keeps
    references to them). Results are the same bits as the separate calls."""

    def __init__(self, dtype: torch.dtype, device):
        if dtype not in (torch.bfloat16, torch.float16):
            raise HgkError(2, "OpSequence: bf16 or f16 only")
        self.dtype, self.device = dtype, torch.device(device)
        self._ops, self._keep, self._list, self._uploaded = [], [], None, 0

    def _check(self, *ts):
        for t in ts:
            if t is not None and t.dtype != self.dtype:
                raise HgkError(1, f"OpSequence: operand dtype {t.dtype}, list dtype {self.dtype}")
        self._keep.extend(t for t in ts if t is not None)

    def __len__(self):
        return len(self._ops)

    def rms_norm(self, x, weight, eps, y):
        """y = rms_norm(x, weight, eps) (weight may be None)."""
        self._check(x, weight, y)
        rows, n, xt, xr = _tok_rows(x, "x")
        _, _, yt, yr = _tok_rows(y, "y")
        self._ops.append(HgkOp(kind=OP_RMS_NORM, rows=rows, n=n, eps=eps, x=x.data_ptr(), x_tok=xt,
                               x_row=xr, w=None if weight is None else weight.data_ptr(),
                               y=y.data_ptr(), y_tok=yt, y_row=yr))
        return self

    def add_rms_norm(self, x, r, weight, eps, y, h=None):
        """h = x + r (written when h is given); y = rms_norm(h, weight, eps)."""
        self._check(x, r, weight, y, h)
        rows, n, xt, xr = _tok_rows(x, "x")
        _, _, rt, rr = _tok_rows(r, "r")
        _, _, yt, yr = _tok_rows(y, "y")
        ht, hr = (0, 0) if h is None else _tok_rows(h, "h")[2:]
        self._ops.append(HgkOp(kind=OP_ADD_RMS_NORM, rows=rows, n=n, eps=eps, x=x.data_ptr(),
                               x_tok=xt, x_row=xr, r=r.data_ptr(), r_tok=rt, r_row=rr,
                               w=None if weight is None else weight.data_ptr(), y=y.data_ptr(),
                               y_tok=yt, y_row=yr, h=None if h is None else h.data_ptr(),
                               h_tok=ht, h_row=hr))
        return self

    def gated_rms_norm(self, x, z, weight, eps, y):
        """y = swiglu(z, rms_norm(x, weight, eps)). x, y: [T, rows, n]; z:
        [T, rows, n] or [T, groups, rows_per_group, n] (e.g. the z slice of
        in_proj_qkvz, read in place)."""
        self._check(x, z, weight, y)
        rows, n, xt, xr = _tok_rows(x, "x")
        _, _, yt, yr = _tok_rows(y, "y")
        if z.dim() == 4:
            if z.shape[1] * z.shape[2] != rows or z.shape[3] != n or z.stride(3) != 1:
                raise HgkError(1, "z must be [T, groups, rows_per_group, n] covering x's rows")
            zt, zr, zg, zgs = z.stride(0), z.stride(2), z.shape[2], z.stride(1)
        else:
            _, _, zt, zr = _tok_rows(z, "z")
            zg, zgs = 0, 0
        self._ops.append(HgkOp(kind=OP_GATED_RMS_NORM, rows=rows, n=n, eps=eps, x=x.data_ptr(),
                               x_tok=xt, x_row=xr, r=z.data_ptr(), r_tok=zt, r_row=zr,
                               z_group_rows=zg, z_group_stride=zgs, w=weight.data_ptr(),
                               y=y.data_ptr(), y_tok=yt, y_row=yr))
        return self

    def qk_norm_rope(self, q, k, q_weight, k_weight, eps, dims, base, q_out, k_out, *,
                     scale=1.0, offset=0, offsets=None, freqs=None):
        """q/k RMSNorm (weights may be None) and RoPE of one new token per
        sequence at position offsets[t] (or offset) times scale: q [T, Hq, D]
        (a head may sit in a wider block, as Qwen3-Next's q), k [T, Hk, D];
        outputs q_out [T, Hq, D], k_out [T, Hk, D] (any token/head strides)."""
        self._check(q, k, q_weight, k_weight, q_out, k_out)
        hq, D, qt, qr = _tok_rows(q, "q")
        hk, _, kt, kr = _tok_rows(k, "k")
        _, _, yt, yr = _tok_rows(q_out, "q_out")
        _, _, ht, hr = _tok_rows(k_out, "k_out")
        if offsets is not None:
            if offsets.dtype != torch.int32 or offsets.device != q.device:
                raise HgkError(1, "offsets must be int32 on q's device")
            self._keep.append(offsets)
        fr = _freqs_arg(freqs)
        if fr is not None:
            self._keep.append(fr)
        self._ops.append(HgkOp(kind=OP_QK_NORM_ROPE, rows=hq, n=D, eps=eps, x=q.data_ptr(),
                               x_tok=qt, x_row=qr, r=k.data_ptr(), r_tok=kt, r_row=kr,
                               w=None if q_weight is None else q_weight.data_ptr(),
                               w2=None if k_weight is None else k_weight.data_ptr(),
                               y=q_out.data_ptr(), y_tok=yt, y_row=yr, h=k_out.data_ptr(),
                               h_tok=ht, h_row=hr, k_heads=hk, dims=dims,
                               base=0.0 if base is None else base, freqs=fr, scale=scale,
                               offsets=None if offsets is None else offsets.data_ptr(),
                               offset=offset))
        return self

    def glu(self, act, gate, up, y):
        """y = act(gate) * up (ACT_SILU: swiglu; ACT_GELU_TANH: GeGLU)."""
        self._check(gate, up, y)
        rows, n, gt, gr = _tok_rows(gate, "gate")
        _, _, ut, ur = _tok_rows(up, "up")
        _, _, yt, yr = _tok_rows(y, "y")
        self._ops.append(HgkOp(kind=OP_GLU, rows=rows, n=n, act=act, x=gate.data_ptr(), x_tok=gt,
                               x_row=gr, r=up.data_ptr(), r_tok=ut, r_row=ur, y=y.data_ptr(),
                               y_tok=yt, y_row=yr))
        return self

    def upload(self):
        """Writes the recorded ops into a device list (done by run() when
        ops were added since the last upload)."""
        n = len(self._ops)
        if n == 0:
            raise HgkError(1, "OpSequence: no ops")
        nbytes = lib().hgk_op_list_bytes(n)
        if nbytes < 0:
            raise HgkError(1, f"OpSequence: {n} ops is too many")
        self._list = torch.empty(((nbytes + 15) // 16 * 16,), dtype=torch.uint8, device=self.device)
        arr = (HgkOp * n)(*self._ops)
        check(lib().hgk_op_list_upload(dtype_code(self.dtype), arr, n, _ptr(self._list),
                                       self._list.numel(), _stream(self.device)))
        self._uploaded = n
        return self

    def run(self, tokens: int):
        """Every op over tokens 0..tokens-1, in one launch on the current stream."""
        if self._uploaded != len(self._ops):
            self.upload()
        check(lib().hgk_op_list_run(dtype_code(self.dtype), _ptr(self._list), self._uploaded,
                                    tokens, _stream(self.device)))
