"""The reference operator interface (FO/src/ops.rs) over the gfx950 C ABI.

Each function keeps the argument order and in-place semantics of the reference's
`#[device] fn` (the `device` handle becomes torch device memory on the current HIP
stream). Tensors are torch tensors on a ROCm device:

  bf16 tensors    torch.bfloat16 (or int16/uint16 bit views)
  E4M3 / E2M1 / E8M0 codes    torch.uint8 (E4M3 may also be torch.float8_e4m3fn)
  per-channel scales    torch.float32 (ops.rs uses bf16: pass torch.bfloat16 and the
                        exact bf16 entry point is used)

Errors from the library raise MoaError; nothing falls back to a CPU path. In checked mode
(set_checked(True), or MOA_CHECK_DEVICE_ERRORS=1 in the environment) every operator call is
followed by device_errors(), which synchronises, and any device-side error bit raises MoaError
(MOA_ERROR_DEVICE_STATE); off by default, since the check synchronises the stream.
"""
from __future__ import annotations

import ctypes as C
import os
import struct

import torch

from . import _lib

_checked = os.environ.get("MOA_CHECK_DEVICE_ERRORS", "") not in ("", "0")


def set_checked(on: bool) -> None:
    """Checked mode on or off (see the module docstring)."""
    global _checked
    _checked = bool(on)


def _call(name: str, *args) -> None:
    """One operator entry point; in checked mode, then the device's error bits."""
    _lib.call(name, *args)
    if _checked:
        bits = device_errors()
        if bits:
            raise _lib.MoaError(-5, f"{name}: device error bits {bits:#x} (1 rope offset, 2 kv offset, "
                                    f"4 expired wait: the device state is now tripped, see clear_device_state; "
                                    f"8 paged-cache argument)")

H, L, NS, GS, DS, QS, PS, TS, E, W = 3840, 15360, 8, 2, 256, 4096, 2048, 1024, 32768, 262144


def _ptr(t: torch.Tensor | None, name: str, dtypes, numel: int | None = None):
    """The tensor's device address after the checks (an int: the signatures declare void*, so
    ctypes converts it). The cheapest torch attributes are used: every operator call runs this for
    each of its tensors, and `t.device` alone costs about 0.4 us per tensor."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must live on a ROCm device, got {t.device}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: dtype {t.dtype} not in {dtypes}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name}: expected {numel} elements, got {t.numel()}")
    return t.data_ptr()


_BF16 = (torch.bfloat16, torch.int16, torch.uint16)
_U8 = (torch.uint8, torch.float8_e4m3fn)
_F32 = (torch.float32,)
_I32 = (torch.int32,)
_I64 = (torch.int64,)


def _stream(t: torch.Tensor) -> int:
    """The current HIP stream of the current device (its handle as an int). The library serves a
    call from the scratch of the current device, so the call's tensors must live there: a tensor
    of another device is refused here rather than run against the wrong device's scratch. The handle
    is asked for as a number: torch.cuda.current_stream builds a Stream object around it, 1.14 us of
    host time per call against 0.08, and the small calls are bound by the host."""
    dev = t.get_device()
    cur = torch.cuda.current_device()
    if dev != cur:
        raise ValueError(f"the call's tensors live on cuda:{dev} but the current device is cuda:{cur}; "
                         f"call it under torch.cuda.device({dev})")
    return torch._C._cuda_getCurrentRawStream(dev)


def _rows(x: torch.Tensor, width: int, name: str) -> int:
    if x.numel() % width:
        raise ValueError(f"{name}: {x.numel()} elements is not a multiple of {width}")
    return x.numel() // width


def _scales(*ts):
    kinds = {t.dtype for t in ts}
    if kinds == {torch.float32}:
        return _F32, False
    if kinds <= set(_BF16):
        return _BF16, True
    raise TypeError(f"per-channel scales must all be float32 or all bfloat16, got {kinds}")


def sliding_project_qkv(x, q_weight, k_weight, v_weight, q_weight_scale, k_weight_scale, v_weight_scale,
                        input_rms_weight, q_rms_weight, k_rms_weight, kv_offset, rope_offset, cos, sin,
                        k_cache, v_cache, q_out) -> None:
    """ops::sliding_project_qkv (FO/src/ops.rs:37-76). Writes q_out and the K/V cache slot(s)."""
    M = _rows(x, H, "x")
    sd, bf = _scales(q_weight_scale, k_weight_scale, v_weight_scale)
    args = [
        _ptr(x, "x", _BF16), _ptr(q_weight, "q_weight", _U8, QS * H), _ptr(k_weight, "k_weight", _U8, PS * H),
        _ptr(v_weight, "v_weight", _U8, PS * H), _ptr(q_weight_scale, "q_weight_scale", sd, QS),
        _ptr(k_weight_scale, "k_weight_scale", sd, PS), _ptr(v_weight_scale, "v_weight_scale", sd, PS),
        _ptr(input_rms_weight, "input_rms_weight", _BF16, H), _ptr(q_rms_weight, "q_rms_weight", _BF16, DS),
        _ptr(k_rms_weight, "k_rms_weight", _BF16, DS), _ptr(kv_offset, "kv_offset", _I32, 1),
        _ptr(rope_offset, "rope_offset", _I32, 1), _ptr(cos, "cos", _BF16, E * DS), _ptr(sin, "sin", _BF16, E * DS),
        _ptr(k_cache, "k_cache", _BF16, TS * NS * DS), _ptr(v_cache, "v_cache", _BF16, TS * NS * DS),
        _ptr(q_out, "q_out", _BF16, M * QS),
    ]
    name = "moa_sliding_project_qkv_bf16_scales" if bf else "moa_sliding_project_qkv"
    _call(name, *args, M, _stream(x))


def sliding_attention(q, k, v, mask, out) -> None:
    """ops::sliding_attention (FO/src/ops.rs:118-128): out = softmax over the slots with mask != 0 of
    q . k_t (scale 1.0), times v. q / out [M, 8, 2, 256] bf16, k / v [1024, 8, 256] bf16 (the ring
    caches), mask [M, 1024] f32."""
    M = _rows(q, QS, "q")
    args = [
        _ptr(q, "q", _BF16), _ptr(k, "k", _BF16, TS * NS * DS), _ptr(v, "v", _BF16, TS * NS * DS),
        _ptr(mask, "mask", _F32, M * TS), _ptr(out, "out", _BF16, M * QS),
    ]
    _call("moa_sliding_attention", *args, M, _stream(q))


GF, DF, QF, PF, TF = 16, 512, 8192, 512, 512  # full-attention layers (FO/src/axes.rs)


def full_project_qkv(x, q_weight, k_weight, q_weight_scale, k_weight_scale, input_rms_weight, q_rms_weight,
                     k_rms_weight, kv_offset, rope_offset, cos, sin, k_cache, v_cache, q_out) -> None:
    """ops::full_project_qkv (FO/src/ops.rs:78-116). k_cache / v_cache are the position's page
    [512, 512]; V is the unweighted norm of the raw K projection. bf16 per-row weight scales."""
    M = _rows(x, H, "x")
    args = [
        _ptr(x, "x", _BF16), _ptr(q_weight, "q_weight", _U8, QF * H), _ptr(k_weight, "k_weight", _U8, PF * H),
        _ptr(q_weight_scale, "q_weight_scale", _BF16, QF), _ptr(k_weight_scale, "k_weight_scale", _BF16, PF),
        _ptr(input_rms_weight, "input_rms_weight", _BF16, H), _ptr(q_rms_weight, "q_rms_weight", _BF16, DF),
        _ptr(k_rms_weight, "k_rms_weight", _BF16, DF), _ptr(kv_offset, "kv_offset", _I32, 1),
        _ptr(rope_offset, "rope_offset", _I32, 1), _ptr(cos, "cos", _BF16, E * DF), _ptr(sin, "sin", _BF16, E * DF),
        _ptr(k_cache, "k_cache", _BF16, TF * DF), _ptr(v_cache, "v_cache", _BF16, TF * DF),
        _ptr(q_out, "q_out", _BF16, M * QF),
    ]
    _call("moa_full_project_qkv", *args, M, _stream(x))


def _full_page(name, q, k, v, mask, running_max, running_sum, out):
    M = _rows(q, QF, "q")
    args = [
        _ptr(q, "q", _BF16), _ptr(k, "k", _BF16, TF * DF), _ptr(v, "v", _BF16, TF * DF),
        _ptr(mask, "mask", _F32, M * TF), _ptr(running_max, "running_max", _F32, M * GF),
        _ptr(running_sum, "running_sum", _F32, M * GF), _ptr(out, "out", _BF16, M * QF),
    ]
    _call(name, *args, M, _stream(q))


def full_attention_first_page(q, k, v, mask, running_max, running_sum, out) -> None:
    """ops::full_attention_first_page (FO/src/ops.rs:148-160): starts the running softmax state
    (max, sum [M, 16] f32; out [M, 16, 512] bf16, un-normalised) from one 512-slot page."""
    _full_page("moa_full_attention_first_page", q, k, v, mask, running_max, running_sum, out)


def full_attention_page(q, k, v, mask, running_max, running_sum, out) -> None:
    """ops::full_attention_page (FO/src/ops.rs:162-174): folds one more page into the state."""
    _full_page("moa_full_attention_page", q, k, v, mask, running_max, running_sum, out)


def full_attention(q, k_pages, v_pages, masks, running_max, running_sum, out) -> None:
    """The state full_attention_first_page + full_attention_page over pages 1 .. P-1 leave, in two
    launches: k_pages / v_pages [P, 512, 512] bf16 (contiguous), masks [P, M, 512] f32."""
    M = _rows(q, QF, "q")
    P = _rows(k_pages, TF * DF, "k_pages")
    args = [
        _ptr(q, "q", _BF16), _ptr(k_pages, "k_pages", _BF16), _ptr(v_pages, "v_pages", _BF16, P * TF * DF),
        _ptr(masks, "masks", _F32, P * M * TF),
    ]
    tail = [_ptr(running_max, "running_max", _F32, M * GF), _ptr(running_sum, "running_sum", _F32, M * GF),
            _ptr(out, "out", _BF16, M * QF)]
    _call("moa_full_attention", *args, P, *tail, M, _stream(q))


def full_attention_output(x, running_sum, post_attn_rms_weight, o_weight, o_weight_scale, residual) -> None:
    """ops::full_attention_output (FO/src/ops.rs:176-199): x / running_sum, the O projection
    (K = 8192, bf16 per-row scales), post-norm and residual add, in place."""
    M = _rows(x, QF, "x")
    args = [
        _ptr(x, "x", _BF16), _ptr(running_sum, "running_sum", _F32, M * GF),
        _ptr(post_attn_rms_weight, "post_attn_rms_weight", _BF16, H), _ptr(o_weight, "o_weight", _U8, H * QF),
        _ptr(o_weight_scale, "o_weight_scale", _BF16, H), _ptr(residual, "residual", _BF16, M * H),
    ]
    _call("moa_full_attention_output", *args, M, _stream(x))


def final_norm_and_logits(input, rms_weight, lm_head_weight, out) -> None:
    """ops::final_norm_and_logits (FO/src/ops.rs:241-298): out = softcap30(bf16(RMSNorm(input) .
    lm_head_weight^T)). input [M, 3840] bf16, lm_head_weight [262144, 3840] bf16, out [M, 262144] bf16."""
    M = _rows(input, H, "input")
    args = [
        _ptr(input, "input", _BF16), _ptr(rms_weight, "rms_weight", _BF16, H),
        _ptr(lm_head_weight, "lm_head_weight", _BF16, W * H), _ptr(out, "out", _BF16, M * W),
    ]
    _call("moa_final_norm_and_logits", *args, M, _stream(input))


def sliding_attention_output(x, post_attn_rms_weight, o_weight, o_weight_scale, residual) -> None:
    """ops::sliding_attention_output (FO/src/ops.rs:130-146). Updates residual in place."""
    M = _rows(x, QS, "x")
    sd, bf = _scales(o_weight_scale)
    args = [
        _ptr(x, "x", _BF16), _ptr(post_attn_rms_weight, "post_attn_rms_weight", _BF16, H),
        _ptr(o_weight, "o_weight", _U8, H * QS), _ptr(o_weight_scale, "o_weight_scale", sd, H),
        _ptr(residual, "residual", _BF16, M * H),
    ]
    name = "moa_sliding_attention_output_bf16_scales" if bf else "moa_sliding_attention_output"
    _call(name, *args, M, _stream(x))


def decoder_feedforward(residual, pre_ff_rms_weight, up_weight_packed, gate_weight_packed, down_weight_packed,
                        up_weight_scale, gate_weight_scale, down_weight_scale, up_global_scale, gate_global_scale,
                        down_global_scale, post_ff_rms_weight, layer_scalar) -> None:
    """ops::decoder_feedforward (FO/src/ops.rs:201-239), NVFP4 weights. Updates residual in place."""
    M = _rows(residual, H, "residual")
    args = [
        _ptr(residual, "residual", _BF16), _ptr(pre_ff_rms_weight, "pre_ff_rms_weight", _BF16, H),
        _ptr(up_weight_packed, "up_weight_packed", _U8, L * H // 2),
        _ptr(gate_weight_packed, "gate_weight_packed", _U8, L * H // 2),
        _ptr(down_weight_packed, "down_weight_packed", _U8, H * L // 2),
        _ptr(up_weight_scale, "up_weight_scale", _U8, L * H // 16),
        _ptr(gate_weight_scale, "gate_weight_scale", _U8, L * H // 16),
        _ptr(down_weight_scale, "down_weight_scale", _U8, H * L // 16),
        _ptr(up_global_scale, "up_global_scale", _F32, 1), _ptr(gate_global_scale, "gate_global_scale", _F32, 1),
        _ptr(down_global_scale, "down_global_scale", _F32, 1),
        _ptr(post_ff_rms_weight, "post_ff_rms_weight", _BF16, H), _ptr(layer_scalar, "layer_scalar", _BF16, 8),
    ]
    _call("moa_decoder_feedforward", *args, M, _stream(residual))


def decoder_feedforward_fp8(residual, pre_ff_rms_weight, up_weight, gate_weight, down_weight, up_weight_scale,
                            gate_weight_scale, down_weight_scale, post_ff_rms_weight=None, layer_scalar=None) -> None:
    """GeGLU FFN with FP8 E4M3 weights and f32 per-channel scales."""
    M = _rows(residual, H, "residual")
    args = [
        _ptr(residual, "residual", _BF16), _ptr(pre_ff_rms_weight, "pre_ff_rms_weight", _BF16, H),
        _ptr(up_weight, "up_weight", _U8, L * H), _ptr(gate_weight, "gate_weight", _U8, L * H),
        _ptr(down_weight, "down_weight", _U8, H * L), _ptr(up_weight_scale, "up_weight_scale", _F32, L),
        _ptr(gate_weight_scale, "gate_weight_scale", _F32, L), _ptr(down_weight_scale, "down_weight_scale", _F32, H),
        _ptr(post_ff_rms_weight, "post_ff_rms_weight", _BF16, H), _ptr(layer_scalar, "layer_scalar", _BF16, 8),
    ]
    _call("moa_decoder_feedforward_fp8", *args, M, _stream(residual))


def decoder_feedforward_mxfp4(residual, pre_ff_rms_weight, up_weight_packed, gate_weight_packed, down_weight_packed,
                              up_weight_scale, gate_weight_scale, down_weight_scale, post_ff_rms_weight=None,
                              layer_scalar=None) -> None:
    """GeGLU FFN with MXFP4 weights (E2M1 + E8M0 per 32)."""
    M = _rows(residual, H, "residual")
    args = [
        _ptr(residual, "residual", _BF16), _ptr(pre_ff_rms_weight, "pre_ff_rms_weight", _BF16, H),
        _ptr(up_weight_packed, "up_weight_packed", _U8, L * H // 2),
        _ptr(gate_weight_packed, "gate_weight_packed", _U8, L * H // 2),
        _ptr(down_weight_packed, "down_weight_packed", _U8, H * L // 2),
        _ptr(up_weight_scale, "up_weight_scale", _U8, L * H // 32),
        _ptr(gate_weight_scale, "gate_weight_scale", _U8, L * H // 32),
        _ptr(down_weight_scale, "down_weight_scale", _U8, H * L // 32),
        _ptr(post_ff_rms_weight, "post_ff_rms_weight", _BF16, H), _ptr(layer_scalar, "layer_scalar", _BF16, 8),
    ]
    _call("moa_decoder_feedforward_mxfp4", *args, M, _stream(residual))


def _o_args(x, post_attn_rms_weight, o_weight, o_weight_scale, residual, scale_dtypes):
    M = _rows(x, QS, "x")
    return M, [
        _ptr(x, "x", _BF16), _ptr(post_attn_rms_weight, "post_attn_rms_weight", _BF16, H),
        _ptr(o_weight, "o_weight", _U8, H * QS), _ptr(o_weight_scale, "o_weight_scale", scale_dtypes, H),
        _ptr(residual, "residual", _BF16, M * H),
    ]


def sliding_attention_output_feedforward(x, post_attn_rms_weight, o_weight, o_weight_scale, residual,
                                         pre_ff_rms_weight, up_weight_packed, gate_weight_packed, down_weight_packed,
                                         up_weight_scale, gate_weight_scale, down_weight_scale, up_global_scale,
                                         gate_global_scale, down_global_scale, post_ff_rms_weight,
                                         layer_scalar) -> None:
    """The tail of the reference's sliding-layer step (FO/src/host/runtime.rs:440-459, 543-571):
    sliding_attention_output (bf16 O scales, as ops.rs:136) then decoder_feedforward (NVFP4) on the
    same residual, in place. One launch per token row; the same bits as the two calls in turn."""
    M, args = _o_args(x, post_attn_rms_weight, o_weight, o_weight_scale, residual, _BF16)
    args += [
        _ptr(pre_ff_rms_weight, "pre_ff_rms_weight", _BF16, H),
        _ptr(up_weight_packed, "up_weight_packed", _U8, L * H // 2),
        _ptr(gate_weight_packed, "gate_weight_packed", _U8, L * H // 2),
        _ptr(down_weight_packed, "down_weight_packed", _U8, H * L // 2),
        _ptr(up_weight_scale, "up_weight_scale", _U8, L * H // 16),
        _ptr(gate_weight_scale, "gate_weight_scale", _U8, L * H // 16),
        _ptr(down_weight_scale, "down_weight_scale", _U8, H * L // 16),
        _ptr(up_global_scale, "up_global_scale", _F32, 1), _ptr(gate_global_scale, "gate_global_scale", _F32, 1),
        _ptr(down_global_scale, "down_global_scale", _F32, 1),
        _ptr(post_ff_rms_weight, "post_ff_rms_weight", _BF16, H), _ptr(layer_scalar, "layer_scalar", _BF16, 8),
    ]
    _call("moa_sliding_attention_output_feedforward", *args, M, _stream(x))


def sliding_attention_output_feedforward_fp8(x, post_attn_rms_weight, o_weight, o_weight_scale, residual,
                                             pre_ff_rms_weight, up_weight, gate_weight, down_weight, up_weight_scale,
                                             gate_weight_scale, down_weight_scale, post_ff_rms_weight=None,
                                             layer_scalar=None) -> None:
    """sliding_attention_output (f32 O scales) then decoder_feedforward_fp8 on the same residual
    (BASELINE configs 1 then 0), in place: one launch per token row, the same bits as the two calls."""
    M, args = _o_args(x, post_attn_rms_weight, o_weight, o_weight_scale, residual, _F32)
    args += [
        _ptr(pre_ff_rms_weight, "pre_ff_rms_weight", _BF16, H),
        _ptr(up_weight, "up_weight", _U8, L * H), _ptr(gate_weight, "gate_weight", _U8, L * H),
        _ptr(down_weight, "down_weight", _U8, H * L), _ptr(up_weight_scale, "up_weight_scale", _F32, L),
        _ptr(gate_weight_scale, "gate_weight_scale", _F32, L), _ptr(down_weight_scale, "down_weight_scale", _F32, H),
        _ptr(post_ff_rms_weight, "post_ff_rms_weight", _BF16, H), _ptr(layer_scalar, "layer_scalar", _BF16, 8),
    ]
    _call("moa_sliding_attention_output_feedforward_fp8", *args, M, _stream(x))


def sliding_attention_output_feedforward_mxfp4(x, post_attn_rms_weight, o_weight, o_weight_scale, residual,
                                               pre_ff_rms_weight, up_weight_packed, gate_weight_packed,
                                               down_weight_packed, up_weight_scale, gate_weight_scale,
                                               down_weight_scale, post_ff_rms_weight=None,
                                               layer_scalar=None) -> None:
    """sliding_attention_output (f32 O scales) then decoder_feedforward_mxfp4 on the same residual."""
    M, args = _o_args(x, post_attn_rms_weight, o_weight, o_weight_scale, residual, _F32)
    args += [
        _ptr(pre_ff_rms_weight, "pre_ff_rms_weight", _BF16, H),
        _ptr(up_weight_packed, "up_weight_packed", _U8, L * H // 2),
        _ptr(gate_weight_packed, "gate_weight_packed", _U8, L * H // 2),
        _ptr(down_weight_packed, "down_weight_packed", _U8, H * L // 2),
        _ptr(up_weight_scale, "up_weight_scale", _U8, L * H // 32),
        _ptr(gate_weight_scale, "gate_weight_scale", _U8, L * H // 32),
        _ptr(down_weight_scale, "down_weight_scale", _U8, H * L // 32),
        _ptr(post_ff_rms_weight, "post_ff_rms_weight", _BF16, H), _ptr(layer_scalar, "layer_scalar", _BF16, 8),
    ]
    _call("moa_sliding_attention_output_feedforward_mxfp4", *args, M, _stream(x))


# ---- the paged KV cache (include/moa_paged.h; no counterpart in the reference, which serves one sequence)

_PAGED_STRUCT = struct.Struct("=7Q9q8i")  # moa_paged_cache


class PagedCache:
    """Many sequences' K and V over one pool of pages, as the paged_* operators take it. The tensors stay the
    caller's; this handle checks them once and holds them.

      k_pages, v_pages    bf16, or E4M3 codes (float8_e4m3fn / uint8) [layers, pages, slots, kv_heads, head_dim], or
                          without the layers; head_dim 64, 128, 256 or 512, dense; other strides multiples of 16 bytes
      page_table          int32 [sequences, columns], dense rows: position t of sequence s lies in page
                          page_table[s, t // slots] at slot t % slots
      seq_lens            int32 [sequences]: positions of each sequence (0: a free one)
      ref_counts          int32 [pages]: the table entries in use that name the page (0: a free page)
      k_scale, v_scale    with E4M3 pages: f32 [layers, kv_heads] (or [kv_heads]), a value is code * scale

    A new cache has seq_lens and ref_counts zero. Calls that find a bad value in the state or in an index tensor
    leave it out and raise bit 8 of device_errors() (each operator says what is left out)."""

    def __init__(self, k_pages, v_pages, page_table, seq_lens, ref_counts, k_scale=None, v_scale=None):
        for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages"), (page_table, "page_table"), (seq_lens, "seq_lens"),
                        (ref_counts, "ref_counts")):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
        k_pages, v_pages = (t.detach()[None] if t.dim() == 4 else t.detach() for t in (k_pages, v_pages))
        if k_pages.dim() != 5 or k_pages.shape != v_pages.shape:
            raise ValueError(f"k_pages and v_pages must both be [layers, pages, slots, kv_heads, head_dim], got "
                             f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
        if 0 in k_pages.shape:
            raise ValueError(f"k_pages and v_pages must not be empty, got {tuple(k_pages.shape)}")
        e4m3 = k_pages.dtype in _U8
        if k_pages.dtype not in _BF16 + _U8 or (v_pages.dtype in _U8) != e4m3 or v_pages.dtype not in _BF16 + _U8:
            raise TypeError(f"k_pages and v_pages must both be bf16 or both be E4M3, got {k_pages.dtype} and {v_pages.dtype}")
        for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
            if not t.is_cuda:
                raise ValueError(f"{name} must live on a ROCm device, got {t.device}")
            if t.stride(4) != 1:
                raise ValueError(f"{name}: head_dim must be dense")
        layers, pages, slots, heads, dim = k_pages.shape
        if page_table.dim() != 2 or page_table.dtype != torch.int32 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
            raise ValueError("page_table must be int32 [sequences, columns] with dense rows")
        if not page_table.is_cuda:
            raise ValueError(f"page_table must live on a ROCm device, got {page_table.device}")
        seqs, columns = page_table.shape
        table_stride = page_table.stride(0) if seqs > 1 else columns
        self._keep = [k_pages, v_pages, page_table.detach(), seq_lens.detach(), ref_counts.detach()]
        ptrs = [k_pages.data_ptr(), v_pages.data_ptr()]
        for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if e4m3 and t is None:
                raise ValueError(f"E4M3 pages need {name}")
            if not e4m3 and t is not None:
                raise ValueError(f"bf16 pages have no scales: {name} must be None")
            ptrs.append(_ptr(t, name, _F32, layers * heads) or 0)
            self._keep.append(t if t is None else t.detach())
        ptrs += [page_table.data_ptr(), _ptr(seq_lens, "seq_lens", _I32, seqs), _ptr(ref_counts, "ref_counts", _I32, pages)]
        device = k_pages.get_device()
        if any(t is not None and t.get_device() != device for t in self._keep):
            raise ValueError("the cache's tensors must live on one device")
        self.layers, self.pages, self.slots, self.kv_heads, self.head_dim = layers, pages, slots, heads, dim
        self.sequences, self.columns, self.device_index = seqs, columns, device
        self._struct = _PAGED_STRUCT.pack(*ptrs, *k_pages.stride()[:4], *v_pages.stride()[:4], table_stride, layers, pages,
                                          slots, heads, dim, int(e4m3), seqs, columns)


def _index(t, name, cache, numel):
    """The address of an int32 index tensor of a call on `cache` (numel: None for any number)."""
    if not isinstance(cache, PagedCache):
        raise TypeError("cache must be a PagedCache")
    p = _ptr(t, name, _I32, numel if numel is None else getattr(cache, numel[0]) + numel[1])
    if p is None:
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.get_device() != cache.device_index:
        raise ValueError(f"{name} lives on cuda:{t.get_device()}, the cache on cuda:{cache.device_index}")
    return p


def _cache_stream(cache) -> int:
    """The current stream of the cache's device, which must be the current one (as _stream)."""
    cur = torch.cuda.current_device()
    if cache.device_index != cur:
        raise ValueError(f"the cache lives on cuda:{cache.device_index} but the current device is cuda:{cur}; "
                         f"call it under torch.cuda.device({cache.device_index})")
    return torch._C._cuda_getCurrentRawStream(cur)


def _row_tensor(t, name, cache, heads):
    """Address, row stride and rows of a bf16 [rows, heads, head_dim] tensor whose rows may lie apart. (Tuples are unpacked
    and compared whole: every call runs this for each of its tensors.)"""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.get_device() != cache.device_index:
        raise ValueError(f"{name} must live on cuda:{cache.device_index} as the cache does, got {t.device}")
    if t.dtype not in _BF16:
        raise TypeError(f"{name}: dtype {t.dtype} not in {_BF16}")
    shape = t.shape
    if len(shape) != 3 or shape[2] != cache.head_dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name} must be [rows, {heads or 'heads'}, {cache.head_dim}], got {tuple(shape)}")
    rows, h, d = shape
    row, head, one = t.stride()
    if one != 1 or (head != d and h > 1):
        raise ValueError(f"{name}: heads and head_dim must be dense")
    return t.data_ptr(), (row if rows > 1 else h * d), rows


def paged_cache_reserve(cache, new_tokens) -> None:
    """Grows every sequence s by new_tokens[s] positions (int32 [sequences]): the lowest free pages, in the order of the
    sequences. All or nothing: where it cannot be served whole the state stays and bit 8 is raised."""
    p = _index(new_tokens, "new_tokens", cache, ("sequences", 0))
    _call("moa_paged_cache_reserve", cache._struct, p, _cache_stream(cache))


def paged_cache_append(cache, k, v, row_starts, layer=0) -> None:
    """Writes one layer's K and V rows of a step's new tokens: k, v bf16 [rows, kv_heads, head_dim] (rows may lie apart).
    Rows row_starts[s] .. row_starts[s + 1] - 1 (int32 [sequences + 1]) are the last positions of sequence s, so reserve
    first. E4M3 pages take the nearest code of x / scale, at most +-448. A row whose position or page is out of range, or
    whose sequence's starts descend, is not written (bit 8)."""
    p = _index(row_starts, "row_starts", cache, ("sequences", 1))
    kp, kr, rows = _row_tensor(k, "k", cache, cache.kv_heads)
    vp, vr, vrows = _row_tensor(v, "v", cache, cache.kv_heads)
    if vrows != rows:
        raise ValueError(f"v: expected {rows} rows, got {vrows}")
    _call("moa_paged_cache_append", cache._struct, kp, kr, vp, vr, p, rows, layer, _cache_stream(cache))


def paged_cache_fork(cache, parents, children) -> None:
    """Makes the empty sequences children[i] copies of parents[i] (int32 [count]): full pages are shared, the partly
    filled last page of every layer is copied to the lowest free page. All or nothing (bit 8): see moa_paged.h."""
    p, c = _index(parents, "parents", cache, None), _index(children, "children", cache, None)
    n = children.numel()
    if parents.numel() != n:
        raise ValueError(f"parents: expected {n} elements, got {parents.numel()}")
    _call("moa_paged_cache_fork", cache._struct, p, c, n, _cache_stream(cache))


def paged_cache_free(cache, sequences) -> None:
    """Ends the listed sequences (int32 [count]): their length becomes 0 and their pages lose a reference. Empty and
    repeated ones change nothing; an index or a length out of range is left out (bit 8)."""
    p = _index(sequences, "sequences", cache, None)
    _call("moa_paged_cache_free", cache._struct, p, sequences.numel(), _cache_stream(cache))


def paged_cache_compact(cache) -> None:
    """Moves the n live pages to pages 0 .. n - 1 in every layer, page table and reference counts with them: those at n
    and beyond go, in order, to the free pages below n. A length out of range leaves all as it was, a table entry outside the
    pool stays (bit 8)."""
    if not isinstance(cache, PagedCache):
        raise TypeError("cache must be a PagedCache")
    _call("moa_paged_cache_compact", cache._struct, _cache_stream(cache))


def paged_attention(q, cache, row_starts, out, layer=0, window=0, scale=1.0, max_rows=None) -> None:
    """Attention of a batch's new rows over one layer of a paged cache, their own positions included (append first).
    q, out bf16 [rows, q_heads, head_dim] (rows may lie apart; out may be q). Rows row_starts[s] .. row_starts[s + 1] - 1
    (int32 [sequences + 1]) are the last tokens of sequence s: row i of n stands at position seq_lens[s] - n + i and sees
    the positions up to its own, the last `window` of them if window > 0. A row that sees nothing gives zeros, rows of no
    sequence are left as they were. max_rows: the most rows a sequence has in this call (default: all rows; the
    right number makes the call faster). A sequence with a bad length, bad row starts or more rows than max_rows is left
    out, and so is at least every row that sees a page outside the pool (bit 8)."""
    p = _index(row_starts, "row_starts", cache, ("sequences", 1))
    qp, qr, rows = _row_tensor(q, "q", cache, None)
    op, orow, orows = _row_tensor(out, "out", cache, q.shape[1])
    if orows != rows:
        raise ValueError(f"out: expected {rows} rows, got {orows}")
    _call("moa_paged_attention", qp, qr, cache._struct, p, op, orow, rows, q.shape[1], layer, window, scale,
          rows if max_rows is None else max_rows, _cache_stream(cache))


def _masks(t, rows, device_index):
    """Address and words of the nodes' masks: int64 [rows, words], dense."""
    p = _ptr(t, "masks", _I64)
    if p is None:
        raise TypeError("masks must be a torch.Tensor")
    if t.dim() != 2 or t.shape[0] != rows:
        raise ValueError(f"masks must be [{rows}, words], got {tuple(t.shape)}")
    if t.get_device() != device_index:
        raise ValueError(f"masks lives on cuda:{t.get_device()}, the call's other tensors on cuda:{device_index}")
    return p, t.shape[1]


def paged_tree_attention(q, cache, row_starts, masks, out, layer=0, window=0, scale=1.0, max_rows=None) -> None:
    """Attention of drafted trees, appended as their sequences' last positions: row i of a sequence's n is node i, at position
    seq_lens[s] - n + i, and sees the positions before the tree and the nodes of its mask (int64 [rows, words], 1 to 4 words; bit
    j % 64 of word j // 64: node j, itself among them). A window (0, or at least max_rows) counts from a node's depth, the number of
    nodes that it sees. A row without bits gives zeros. Otherwise as paged_attention; max_rows, the most rows a sequence has, is at most
    64 * words and the rows of the call, the default where it is not said (so a smaller window asks for a max_rows of its own)."""
    p = _index(row_starts, "row_starts", cache, ("sequences", 1))
    qp, qr, rows = _row_tensor(q, "q", cache, None)
    op, orow, orows = _row_tensor(out, "out", cache, q.shape[1])
    if orows != rows:
        raise ValueError(f"out: expected {rows} rows, got {orows}")
    mp, words = _masks(masks, rows, cache.device_index)
    _call("moa_paged_tree_attention", qp, qr, cache._struct, p, mp, words, op, orow, rows, q.shape[1], layer, window, scale,
          min(rows, 64 * max(words, 1)) if max_rows is None else max_rows, _cache_stream(cache))


def paged_tree_commit(cache, row_starts, masks, leaves) -> None:
    """Ends a speculative step: the nodes that node leaves[s] (int32 [sequences], -1: none is kept) of a sequence sees become its
    positions behind those before the tree, in order and in every layer; the sequence ends there, and pages that it no longer
    reaches are free. row_starts and masks as in paged_tree_attention; a sequence without rows is left alone. A sequence whose rows,
    length or leaf are out of range, or with a node in a page that is outside the pool or not its alone, stays as it was (bit 8)."""
    p = _index(row_starts, "row_starts", cache, ("sequences", 1))
    leaf = _index(leaves, "leaves", cache, ("sequences", 0))
    rows = masks.shape[0] if isinstance(masks, torch.Tensor) and masks.dim() == 2 else -1
    mp, words = _masks(masks, rows, cache.device_index)
    _call("moa_paged_tree_commit", cache._struct, p, mp, words, leaf, rows, _cache_stream(cache))


def paged_cache_reorder(cache, parents, beams) -> None:
    """Sequences 0 .. len(parents) - 1 are groups of `beams`; every sequence s of them becomes what parents[s] (int32, a sequence of its
    group) was: full pages are shared, a partly filled last page stays with one of its children and its slots in use are copied
    for the others, first into the last pages of sequences that are nobody's parent, then into the lowest free pages. All or
    nothing (bit 8): see moa_paged.h."""
    p = _index(parents, "parents", cache, None)
    _call("moa_paged_cache_reorder", cache._struct, p, parents.numel(), beams, _cache_stream(cache))


def _logits(t):
    """Address, row stride, rows and columns of bf16 logits [rows, vocab] whose rows may lie apart."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("logits must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"logits must live on a ROCm device, got {t.device}")
    if t.dtype not in _BF16:
        raise TypeError(f"logits: dtype {t.dtype} not in {_BF16}")
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError("logits must be [rows, vocab] with dense rows")
    rows, vocab = t.shape
    return t.data_ptr(), (t.stride(0) if rows > 1 else vocab), rows, vocab


def _beside(t, name, logits, dtypes, numel):
    p = _ptr(t, name, dtypes, numel)
    if p is None:
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.get_device() != logits.get_device():
        raise ValueError(f"{name} lives on cuda:{t.get_device()}, the logits on cuda:{logits.get_device()}")
    return p


def tree_verify(logits, tokens, row_starts, masks, best, leaves, next_tokens) -> None:
    """Greedy verification of drafted trees (row_starts [sequences + 1] and masks as in paged_tree_attention): best[row] is the token of
    the row's largest logit (bf16 [rows, vocab], rows may lie apart), ties to the lowest. From node 0 of a sequence the walk goes to
    the lowest child whose token (int32 [rows]) is its best, as long as there is one: leaves[s] is the node where it ends,
    next_tokens[s] that node's best; -1 both for a sequence without rows or whose first row is no node."""
    lp, stride, rows, vocab = _logits(logits)
    n = leaves.numel() if isinstance(leaves, torch.Tensor) else None
    mp, words = _masks(masks, rows, logits.get_device())
    args = [_beside(tokens, "tokens", logits, _I32, rows), _beside(row_starts, "row_starts", logits, _I32, None if n is None else n + 1), mp, words,
            _beside(best, "best", logits, _I32, rows), _beside(leaves, "leaves", logits, _I32, None),
            _beside(next_tokens, "next_tokens", logits, _I32, n)]
    _call("moa_tree_verify", lp, stride, *args, rows, vocab, n, _stream(logits))


def beam_select(logits, scores, finished, out_scores, out_finished, parents, tokens, beams, eos=-1) -> None:
    """A beam search's step over groups of `beams` rows (bf16 logits [rows, vocab], rows may lie apart): the `beams` best of a group's
    candidates, in descending order, ties to the lowest row and token. A candidate is scores[row] + log softmax(logits[row])[token]; a
    finished row has the one candidate eos at its score. parents: the rows that the best come from, as paged_cache_reorder takes them.
    out_scores may be scores (f32 [rows]), out_finished may be finished (int32 [rows]). See moa_search.h for rows without candidates."""
    lp, stride, rows, vocab = _logits(logits)
    if not isinstance(beams, int) or beams < 1 or rows % beams:
        raise ValueError(f"the rows must be groups of beams, got {rows} rows and {beams} beams")
    args = [_beside(scores, "scores", logits, _F32, rows), _beside(finished, "finished", logits, _I32, rows),
            _beside(out_scores, "out_scores", logits, _F32, rows), _beside(out_finished, "out_finished", logits, _I32, rows),
            _beside(parents, "parents", logits, _I32, rows), _beside(tokens, "tokens", logits, _I32, rows)]
    _call("moa_beam_select", lp, stride, *args, rows // beams, beams, vocab, eos, _stream(logits))


def fp8_scaled_projection(x, w, scale, out) -> None:
    """scaled_projection (FO/scripts/generate_references.py:265-274): out = bf16((x . W^T) * scale)."""
    N, K = w.shape
    M = _rows(x, K, "x")
    args = [_ptr(x, "x", _BF16), _ptr(w, "w", _U8, N * K), _ptr(scale, "scale", _F32, N),
            _ptr(out, "out", _BF16, M * N)]
    _call("moa_fp8_scaled_projection", *args, M, N, K, _stream(x))


def device_errors(device: torch.device | None = None) -> int:
    """Synchronise the current stream of `device` (default: the current device); return and clear
    that device's kernel-raised error bits."""
    bits = C.c_uint32(0)
    with torch.cuda.device(device):  # the library reads the bits of the current device
        s = torch.cuda.current_stream().cuda_stream
        _lib.call("moa_device_errors", C.c_void_p(s), C.byref(bits))
    return int(bits.value)


def clear_device_state(device: int = 0) -> None:
    """moa_clear_device_state: acknowledge a tripped device (an expired wait's outputs restored)."""
    _lib.call("moa_clear_device_state", device)


def format_selftest(device="cuda") -> torch.Tensor:
    out = torch.zeros(721924, dtype=torch.int32, device=device)  # layout: moa_decode.hip format_selftest_kernel
    _lib.call("moa_format_selftest", C.c_void_p(out.data_ptr()), _stream(out))
    return out


def init(device: int = 0) -> None:
    _lib.call("moa_init", device)
