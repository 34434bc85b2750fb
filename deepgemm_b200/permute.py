"""Tokens sorted by expert and back, with the gradients of both, for callers that run the grouped GEMMs themselves (a training step,
or a layer of their own). The Mega-MoE layers do this inside their calls; the reference has no such operators.

    plan = moe_dispatch_plan(topk_idx, num_experts)
    rows = moe_permute(x, plan)                                   # forward
    m_grouped_..._contiguous((rows, ...), ..., grouped_layout=plan.expert_end, use_psum_layout=True)
    y = moe_unpermute(rows_out, plan, topk_weights)
    d_rows_out, d_weights = moe_unpermute_backward(dy, rows_out, plan, topk_weights)
    dx = moe_permute_backward(d_rows, plan)

Every function allocates its result on the current stream or writes into ``out``; nothing synchronises, nothing is kept
between calls, and all of them can be captured into a CUDA graph."""
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib
from .block_scaled import check_same_device, span
from .runtime import get_mk_alignment_for_contiguous_layout

_MAX_TOPK, _MAX_EXPERTS = 32, 1024


def _capacity(entries: int, experts: int, alignment: int) -> int:
    step = max(alignment, 8)
    return -(-(entries + min(experts, entries) * (alignment - 1)) // step) * step


class MoeDispatchPlan(NamedTuple):
    """Where every (token, k) entry goes. ``expert_end`` is the psum layout of the grouped GEMMs of the same alignment."""
    dest_row: torch.Tensor      # int32 [tokens, topk], -1 = masked entry
    expert_start: torch.Tensor  # int32 [experts], multiples of `alignment`
    expert_end: torch.Tensor    # int32 [experts]
    alignment: int

    @property
    def num_experts(self) -> int:
        return self.expert_end.numel()

    @property
    def capacity(self) -> int:
        """Rows that hold the sorted tokens however they are routed (known without reading the plan back), rounded up to a multiple
        of 8 or of the alignment, whichever is larger."""
        return _capacity(self.dest_row.numel(), self.num_experts, self.alignment)


def _check_plan(plan: MoeDispatchPlan):
    """Returns (tokens, topk, experts, capacity)."""
    dest, start, end, alignment = plan
    if not (dest.is_cuda and dest.dtype == torch.int32 and dest.dim() == 2 and dest.is_contiguous()):
        raise RuntimeError('plan.dest_row must be a contiguous CUDA int32 [tokens, topk] tensor')
    if not (end.is_cuda and end.dtype == torch.int32 and end.dim() == 1 and end.is_contiguous()):
        raise RuntimeError('plan.expert_end must be a contiguous CUDA int32 [experts] tensor')
    tokens, topk = dest.shape
    if not 1 <= topk <= _MAX_TOPK:
        raise RuntimeError(f'num_topk must be in [1, {_MAX_TOPK}]')
    experts = end.numel()
    if not 1 <= experts <= _MAX_EXPERTS or start.shape != end.shape:
        raise RuntimeError(f'the plan must hold 1 to {_MAX_EXPERTS} experts')
    if not 1 <= alignment < 2 ** 31:
        raise RuntimeError('the alignment must be positive')
    if tokens >= 2 ** 31:
        raise RuntimeError('the plan is too large')
    return tokens, topk, experts, _capacity(tokens * topk, experts, alignment)


def _check_rows(t: torch.Tensor, rows: Optional[int], width: Optional[int], dtypes, name: str):
    if not (t.is_cuda and t.dim() == 2 and t.dtype in dtypes):
        raise RuntimeError(f'{name} must be a 2-D CUDA tensor, one of {", ".join(map(str, dtypes))}')
    height, columns = t.shape
    row_stride, inner = t.stride()
    if inner != 1 and columns != 1:
        raise RuntimeError(f'{name} must have unit inner stride')
    if (rows is not None and height != rows) or (width is not None and columns != width) or columns == 0:
        raise RuntimeError(f'{name} has shape {(height, columns)}, expected ({rows if rows is not None else "any"}, '
                           f'{width if width is not None else "at least 1"})')
    if height >= 2 ** 31 or columns >= 2 ** 31:
        raise RuntimeError(f'{name} is too large')
    if height > 1 and row_stride < columns:
        raise RuntimeError(f'rows of {name} must not overlap')


def _stride(t: torch.Tensor) -> int:
    """Row stride in elements; a single row's is its width, whatever torch says."""
    return t.stride(0) if t.size(0) > 1 else t.size(1)


def _check_out(out: torch.Tensor, inputs, name='out'):
    start, end = span(out)
    for t in inputs:
        if t is not None:
            t_start, t_end = span(t)
            if t_start < end and start < t_end and t_start < t_end and start < end:
                raise RuntimeError(f'{name} must not overlap an input')


def moe_dispatch_plan(topk_idx: torch.Tensor, num_experts: int, alignment: Optional[int] = None) -> MoeDispatchPlan:
    """Stable sort of the (token, k) entries of ``topk_idx`` (int64 [tokens, topk]; an index outside [0, num_experts), -1 by
    convention, masks its entry) by expert. Every expert's segment starts at a multiple of ``alignment`` (default: the
    contiguous-layout alignment); empty segments take no rows."""
    if not (topk_idx.is_cuda and topk_idx.dtype == torch.int64 and topk_idx.dim() == 2 and topk_idx.is_contiguous()):
        raise RuntimeError('topk_idx must be a contiguous CUDA int64 [tokens, topk] tensor')
    alignment = get_mk_alignment_for_contiguous_layout() if alignment is None else int(alignment)
    tokens, topk = topk_idx.shape
    if tokens >= 2 ** 31:
        raise RuntimeError('topk_idx is too large')
    if not 1 <= topk <= _MAX_TOPK:
        raise RuntimeError(f'num_topk must be in [1, {_MAX_TOPK}]')
    if not 1 <= num_experts <= _MAX_EXPERTS:
        raise RuntimeError(f'num_experts must be in [1, {_MAX_EXPERTS}]')
    if not 1 <= alignment < 2 ** 31:
        raise RuntimeError('the alignment must be positive')
    lib = _lib.lib()
    workspace_bytes = lib.dgb200_moe_dispatch_plan_workspace_bytes(tokens, topk, num_experts)
    with _lib.on_device(topk_idx.device):
        dest = topk_idx.new_empty((tokens, topk), dtype=torch.int32)
        start, end = topk_idx.new_empty((2, num_experts), dtype=torch.int32).unbind(0)
        workspace = topk_idx.new_empty(workspace_bytes, dtype=torch.int8) if workspace_bytes else None
        _lib.check(lib.dgb200_moe_dispatch_plan(
            topk_idx.data_ptr(), tokens, topk, num_experts, alignment, dest.data_ptr(), start.data_ptr(), end.data_ptr(),
            workspace.data_ptr() if workspace is not None else None, _lib.current_stream_ptr()))
    return MoeDispatchPlan(dest, start, end, alignment)


def moe_permute(x: Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]], plan: MoeDispatchPlan, out=None, zero_padding: bool = True):
    """``rows[plan.dest_row[t, k]] = x[t]`` for every entry that is not masked. ``x`` is bfloat16 or float32 [tokens, hidden], or the pair
    (float8_e4m3fn [tokens, hidden], float32 scales [tokens, blocks]) of a quantiser, then so is the result. The rows between a
    segment's end and its aligned end become zero (``zero_padding``; the K-grouped GEMMs need that, the m-grouped ones do
    not); rows behind the last segment are left as they are. ``out``: a buffer (or pair) of at least ``plan.capacity`` rows."""
    tokens, topk, experts, capacity = _check_plan(plan)
    dest, end = plan.dest_row, plan.expert_end
    pair = isinstance(x, tuple)
    if (pair and len(x) != 2) or (out is not None and (isinstance(out, tuple) != pair or (pair and len(out) != 2))):
        raise RuntimeError('x and out must both be pairs (rows, scales), or both tensors')
    q, sf = x if pair else (x, None)
    _check_rows(q, tokens, None, (torch.float8_e4m3fn,) if pair else (torch.bfloat16, torch.float32), 'x')
    if pair:
        _check_rows(sf, tokens, None, (torch.float32,), 'the scales')
    with _lib.on_device(q.device):
        if out is None:
            rows = torch.empty((capacity, q.size(1)), dtype=q.dtype, device=q.device)
            rows_sf = torch.empty((capacity, sf.size(1)), dtype=torch.float32, device=q.device) if pair else None
        else:
            rows, rows_sf = out if pair else (out, None)
            _check_rows(rows, None, q.size(1), (q.dtype,), 'out')
            if rows.size(0) < capacity:
                raise RuntimeError(f'out needs at least plan.capacity ({capacity}) rows, got {rows.size(0)}')
            _check_out(rows, (q, sf, dest, end))
            if pair:
                _check_rows(rows_sf, rows.size(0), sf.size(1), (torch.float32,), 'the scales of out')
                _check_out(rows_sf, (q, sf, rows, dest, end), 'the scales of out')
        check_same_device(q, sf, rows, rows_sf, dest, end)
        size = q.element_size()
        _lib.check(_lib.lib().dgb200_moe_permute(
            q.data_ptr(), q.size(1) * size, _stride(q) * size, rows.data_ptr(), _stride(rows) * size, sf.data_ptr() if pair else None,
            sf.size(1) if pair else 0, _stride(sf) if pair else 0, rows_sf.data_ptr() if pair else None, _stride(rows_sf) if pair else 0,
            dest.data_ptr(), end.data_ptr(), tokens, topk, experts, plan.alignment, rows.size(0), int(zero_padding), _lib.current_stream_ptr()))
    return (rows, rows_sf) if pair else rows


def moe_unpermute(rows: torch.Tensor, plan: MoeDispatchPlan, topk_weights: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[t] = sum_k topk_weights[t, k] * rows[plan.dest_row[t, k]]``, summed in ascending k in FP32 and rounded once; masked
    entries add nothing. ``rows`` bfloat16 or float32 [>= plan.capacity, hidden]; ``topk_weights`` float32 [tokens, topk] or None
    (every weight one); returns [tokens, hidden] of the type of ``rows``."""
    tokens, topk, experts, capacity = _check_plan(plan)
    _check_rows(rows, None, None, (torch.bfloat16, torch.float32), 'rows')
    if rows.size(0) < capacity:
        raise RuntimeError(f'rows must hold plan.capacity ({capacity}) rows, got {rows.size(0)}')
    _check_weights(topk_weights, plan)
    with _lib.on_device(rows.device):
        if out is None:
            out = torch.empty((tokens, rows.size(1)), dtype=rows.dtype, device=rows.device)
        else:
            _check_rows(out, tokens, rows.size(1), (rows.dtype,), 'out')
            _check_out(out, (rows, topk_weights, plan.dest_row))
        check_same_device(rows, out, topk_weights, plan.dest_row)
        _lib.check(_lib.lib().dgb200_moe_unpermute(
            rows.data_ptr(), _stride(rows), topk_weights.data_ptr() if topk_weights is not None else None, plan.dest_row.data_ptr(),
            out.data_ptr(), _stride(out), tokens, topk, rows.size(1), rows.size(0), int(rows.dtype == torch.float32), _lib.current_stream_ptr()))
    return out


def moe_permute_backward(d_rows: torch.Tensor, plan: MoeDispatchPlan, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of ``moe_permute``: ``dx[t] = sum_k d_rows[plan.dest_row[t, k]]`` (FP32 sum, rounded once)."""
    return moe_unpermute(d_rows, plan, None, out)


def _check_weights(topk_weights, plan):
    if topk_weights is not None and not (topk_weights.is_cuda and topk_weights.dtype == torch.float32 and topk_weights.is_contiguous() and
                                         topk_weights.shape == plan.dest_row.shape):
        raise RuntimeError(f'topk_weights must be a contiguous CUDA float32 tensor of shape {tuple(plan.dest_row.shape)}')


def moe_unpermute_backward(dy: torch.Tensor, rows: torch.Tensor, plan: MoeDispatchPlan, topk_weights: Optional[torch.Tensor] = None,
                           out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gradients of ``moe_unpermute``: ``(d_rows, d_weights)`` with ``d_rows[plan.dest_row[t, k]] = topk_weights[t, k] * dy[t]`` (padding
    rows of the segments zero, rows behind the last segment left as they are; written into ``out`` if given) and
    ``d_weights[t, k] = <rows[plan.dest_row[t, k]], dy[t]>``, float32, zero for masked entries."""
    tokens, topk, experts, capacity = _check_plan(plan)
    _check_rows(rows, None, None, (torch.bfloat16, torch.float32), 'rows')
    if rows.size(0) < capacity:
        raise RuntimeError(f'rows must hold plan.capacity ({capacity}) rows, got {rows.size(0)}')
    _check_rows(dy, tokens, rows.size(1), (rows.dtype,), 'dy')
    _check_weights(topk_weights, plan)
    with _lib.on_device(rows.device):
        if out is None:
            out = torch.empty((rows.size(0), rows.size(1)), dtype=rows.dtype, device=rows.device)
        else:
            _check_rows(out, rows.size(0), rows.size(1), (rows.dtype,), 'out')
            _check_out(out, (rows, dy, topk_weights, plan.dest_row, plan.expert_end))
        d_weights = torch.empty((tokens, topk), dtype=torch.float32, device=rows.device)
        check_same_device(rows, dy, out, topk_weights, plan.dest_row, plan.expert_end)
        _lib.check(_lib.lib().dgb200_moe_unpermute_backward(
            dy.data_ptr(), _stride(dy), rows.data_ptr(), _stride(rows), topk_weights.data_ptr() if topk_weights is not None else None,
            plan.dest_row.data_ptr(), plan.expert_end.data_ptr(), out.data_ptr(), _stride(out), d_weights.data_ptr(), tokens, topk,
            experts, plan.alignment, rows.size(1), rows.size(0), int(rows.dtype == torch.float32), _lib.current_stream_ptr()))
    return out, d_weights
