"""SwiGLU of the experts' rows as operators of their own, forward (to BF16, or straight to FP8 with FP32 scales) and backward, for callers
that run the grouped GEMMs themselves; the Mega-MoE layers fuse the forward form into their gate/up GEMM."""
import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from .block_scaled import check_same_device
from .permute import _check_out, _check_rows, _stride
from .runtime import get_mk_alignment_for_contiguous_layout
from .utils.math import ceil_div


def _check_call(gate_up, grouped_layout, activation_clamp):
    _check_rows(gate_up, None, None, (torch.bfloat16,), 'gate_up')
    if gate_up.size(1) % 2 != 0:
        raise RuntimeError('gate_up must hold [gate | up] rows of even width')
    if grouped_layout is not None and not (grouped_layout.is_cuda and grouped_layout.dtype == torch.int32 and grouped_layout.dim() == 1 and
                                           grouped_layout.is_contiguous() and grouped_layout.numel() > 0):
        raise RuntimeError('grouped_layout must be a contiguous CUDA int32 tensor, one end row per group')
    if activation_clamp is not None and not ctypes.c_float(activation_clamp).value > 0:  # in FP32, where zero stands for no clamp
        raise RuntimeError('activation_clamp must be positive (None: no clamp)')
    layout = (grouped_layout.data_ptr(), grouped_layout.numel(), get_mk_alignment_for_contiguous_layout()) if grouped_layout is not None else (None, 0, 0)
    return gate_up.size(0), gate_up.size(1) // 2, layout + (float(activation_clamp) if activation_clamp is not None else 0.0,)


def swiglu(gate_up: torch.Tensor, grouped_layout: Optional[torch.Tensor] = None, activation_clamp: Optional[float] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``silu(gate) * up`` of bfloat16 rows ``[gate | up]`` ([rows, 2 * inter]) as bfloat16 [rows, inter]; with ``activation_clamp`` c the gate
    is min(gate, c) and up is clamped to [-c, c]. FP32 arithmetic, one rounding. With ``grouped_layout`` (the psum layout of the
    grouped GEMMs) only rows below the last group's aligned end are computed, the rest of the result is left as it is."""
    rows, inter, call = _check_call(gate_up, grouped_layout, activation_clamp)
    if out is None:
        with _lib.on_device(gate_up.device):
            out = torch.empty((rows, inter), dtype=torch.bfloat16, device=gate_up.device)
    else:
        _check_rows(out, rows, inter, (torch.bfloat16,), 'out')
        _check_out(out, (gate_up, grouped_layout))
    check_same_device(gate_up, out, grouped_layout)
    with _lib.on_device(gate_up.device):
        _lib.check(_lib.lib().dgb200_swiglu(gate_up.data_ptr(), _stride(gate_up), out.data_ptr(), _stride(out), rows, inter, *call,
                                            _lib.current_stream_ptr()))
    return out


def swiglu_backward(d_act: torch.Tensor, gate_up: torch.Tensor, grouped_layout: Optional[torch.Tensor] = None,
                    activation_clamp: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of ``swiglu`` with respect to ``gate_up``: bfloat16 ``[d_gate | d_up]``, zero where a clamp holds; rows as there."""
    rows, inter, call = _check_call(gate_up, grouped_layout, activation_clamp)
    _check_rows(d_act, rows, inter, (torch.bfloat16,), 'd_act')
    if out is None:
        with _lib.on_device(gate_up.device):
            out = torch.empty((rows, 2 * inter), dtype=torch.bfloat16, device=gate_up.device)
    else:
        _check_rows(out, rows, 2 * inter, (torch.bfloat16,), 'out')
        _check_out(out, (gate_up, d_act, grouped_layout))
    check_same_device(gate_up, d_act, out, grouped_layout)
    with _lib.on_device(gate_up.device):
        _lib.check(_lib.lib().dgb200_swiglu_backward(d_act.data_ptr(), _stride(d_act), gate_up.data_ptr(), _stride(gate_up), out.data_ptr(),
                                                     _stride(out), rows, inter, *call, _lib.current_stream_ptr()))
    return out


def swiglu_per_token_cast_to_fp8(gate_up: torch.Tensor, grouped_layout: Optional[torch.Tensor] = None, activation_clamp: Optional[float] = None,
                                 out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``swiglu`` and the quantiser after it in one pass: (float8_e4m3fn [rows, inter], float32 scales [rows, ceil(inter / 128)]) from the
    FP32 products, sf = max(amax, 1e-4) / 448 of each 128 columns. ``inter`` must be a multiple of 8."""
    rows, inter, call = _check_call(gate_up, grouped_layout, activation_clamp)
    if inter % 8 != 0:
        raise RuntimeError(f'inter ({inter}) must be a multiple of 8')
    if out is None:
        with _lib.on_device(gate_up.device):
            q = torch.empty((rows, inter), dtype=torch.float8_e4m3fn, device=gate_up.device)
            sf = torch.empty((rows, ceil_div(inter, 128)), dtype=torch.float32, device=gate_up.device)
    else:
        if not isinstance(out, tuple) or len(out) != 2:
            raise RuntimeError('out must be a pair (rows, scales)')
        q, sf = out
        _check_rows(q, rows, inter, (torch.float8_e4m3fn,), 'out')
        _check_rows(sf, rows, ceil_div(inter, 128), (torch.float32,), 'the scales of out')
        _check_out(q, (gate_up, grouped_layout))
        _check_out(sf, (gate_up, grouped_layout, q), 'the scales of out')
    check_same_device(gate_up, q, sf, grouped_layout)
    with _lib.on_device(gate_up.device):
        _lib.check(_lib.lib().dgb200_swiglu_per_token_cast_to_fp8(gate_up.data_ptr(), _stride(gate_up), q.data_ptr(), _stride(q), sf.data_ptr(),
                                                                  _stride(sf), rows, inter, *call, _lib.current_stream_ptr()))
    return q, sf
