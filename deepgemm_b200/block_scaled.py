"""FP8 GEMMs whose operands carry FP32 scales, one per 1 x 128 values of a and per 128 x 128 of b: what the entry points of
``gemm`` do with float32 scales and ``disable_ue8m0_cast=True`` (the reference's FP32-scale kernels, csrc/apis/gemm.hpp:73-124,
:166-297, exist for the previous architecture only)."""
import struct

import torch

from . import _lib
from .layout import check_sf_layout

# dgb200_fp8_block_scaled_gemm_args of include/dgb200.h: size, seven pointers, eight strides, ten ints. Packed by hand: a
# ctypes.Structure takes 6 us to fill, a third of what a small call takes on the host.
_ARGS = struct.Struct('@N7P8q10i')

LAYOUT_ROW_IDS, LAYOUT_PSUM, LAYOUT_MASKED, LAYOUT_DENSE = range(4)


def check_same_device(first, *tensors):
    """Pointers of one call go to one device."""
    index = first.get_device()
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise RuntimeError(f'all tensors of a call must be on one device, got {first.device} and {t.device}')


def span(t: torch.Tensor):
    """First byte and one past the last of a tensor's memory."""
    start = t.data_ptr()
    if t.is_contiguous():
        return start, start + t.nbytes
    if t.numel() == 0:
        return start, start
    return start, start + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory spans of two tensors meet."""
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1 and a0 < a1 and b0 < b1


def wanted(a_sf: torch.Tensor, b_sf: torch.Tensor, disable_ue8m0_cast: bool) -> bool:
    """Scales stay FP32: both are float32 and the caller does not want them cast to powers of two."""
    return bool(disable_ue8m0_cast) and a_sf.dtype == torch.float32 and b_sf.dtype == torch.float32


def _check_recipe(recipe, recipe_a, recipe_b):
    if (recipe_a is None) != (recipe_b is None):
        raise RuntimeError('recipe_a and recipe_b must be given together')
    if recipe is not None and recipe_a is not None:
        raise RuntimeError('give either recipe or the recipe_a / recipe_b pair')
    pair = (tuple(recipe_a), tuple(recipe_b)) if recipe_a is not None else None
    if (recipe is not None and tuple(recipe) != (1, 128, 128)) or (pair is not None and pair != ((1, 128), (128, 128))):
        raise RuntimeError('FP32 scales that are not cast need the recipe (1, 128, 128)')


def _check_operand(t, name, dims):
    if not (t.is_cuda and t.dtype == torch.float8_e4m3fn and t.dim() == dims):
        raise RuntimeError(f'{name} must be a {dims}-D CUDA float8_e4m3fn tensor')


def run(a, b, d, c, layout, layout_kind, recipe, recipe_a, recipe_b, alignment=128, store_padding=False, expected_m=0):
    """Checks and the call. ``a`` [M, K] (masked: [G, M, K]); ``b`` [N, K] (dense) or [G, N, K], K-major or the transposed view
    of a contiguous tensor."""
    (a_q, a_sf), (b_q, b_sf) = a, b
    _check_recipe(recipe, recipe_a, recipe_b)
    masked, dense = layout_kind == LAYOUT_MASKED, layout_kind == LAYOUT_DENSE
    _check_operand(a_q, 'a', 3 if masked else 2)
    _check_operand(b_q, 'b', 2 if dense else 3)
    if not a_q.is_contiguous():
        raise RuntimeError('a must be K-major and contiguous')
    b_mn_major = not b_q.is_contiguous()
    if b_mn_major and not b_q.transpose(-1, -2).is_contiguous():
        raise RuntimeError('b must be K-major and contiguous, or the transposed view of a contiguous tensor')
    m, k = a_q.shape[-2:]
    n, k_b = b_q.shape[-2:]
    groups = 1 if dense else b_q.size(0)
    if k != k_b:
        raise RuntimeError(f'K mismatch: a has {k}, b has {k_b}')
    if masked and a_q.size(0) != groups:
        raise RuntimeError(f'group count mismatch: a has {a_q.size(0)}, b has {groups}')
    if max(m, n, k, groups) >= 2 ** 31:
        raise RuntimeError('the operands are too large')
    if n % 8 != 0 or k % 16 != 0 or n == 0 or k == 0:
        raise RuntimeError(f'n ({n}) must be a positive multiple of 8 and k ({k}) of 16')
    if b_mn_major and n % 16 != 0:
        raise RuntimeError(f'an MN-major b needs n ({n}) to be a multiple of 16')
    check_sf_layout(a_sf, m, k, 1, 128, groups if masked else None, type_check=torch.float32)
    check_sf_layout(b_sf, n, k, 128, 128, None if dense else groups, type_check=torch.float32)
    shape = (groups, m, n) if masked else (m, n)
    kinds = (torch.bfloat16, torch.float32) if dense else (torch.bfloat16,)
    if not (d.is_cuda and tuple(d.shape) == shape and d.dtype in kinds and d.stride(-1) == 1):
        raise RuntimeError(f'd must be a CUDA tensor of shape {shape} with unit stride on N, {" or ".join(map(str, kinds))}')
    if masked and not d.is_contiguous():
        raise RuntimeError('d must be contiguous')
    row_stride = d.stride(-2) if m > 1 else n
    if row_stride < n or row_stride * d.element_size() % 16 != 0:
        raise RuntimeError('d rows must be 16-byte aligned and not overlap')
    if c is not None:
        if not (c.is_cuda and c.dtype == torch.float32 and d.dtype == torch.float32 and c.shape == d.shape):
            raise RuntimeError('c must be a CUDA float32 tensor of the shape of a float32 d')
        same = c.data_ptr() == d.data_ptr() and c.stride() == d.stride()
        if not same and (overlap(c, d) or c.stride(-1) != 1 or (m > 1 and (c.stride(-2) % 4 != 0 or c.stride(-2) < n)) or c.data_ptr() % 16 != 0):
            c = c.clone(memory_format=torch.contiguous_format)
    check_same_device(a_q, a_sf, b_q, b_sf, d, c, layout)
    if m == 0:
        return
    d0, d1 = span(d)
    for t in (a_q, a_sf, b_q, b_sf) if layout is None else (a_q, a_sf, b_q, b_sf, layout):
        t0, t1 = span(t)
        if t0 < d1 and d0 < t1:
            raise RuntimeError('d must not overlap an operand')
    args = _ARGS.pack(
        _ARGS.size, a_q.data_ptr(), a_sf.data_ptr(), b_q.data_ptr(), b_sf.data_ptr(), d.data_ptr(), c.data_ptr() if c is not None else 0,
        layout.data_ptr() if layout is not None else 0, a_sf.stride(0) if masked else 0, a_sf.stride(-2), a_sf.stride(-1),
        0 if dense else b_sf.stride(0), b_sf.stride(-2), b_sf.stride(-1), row_stride,
        (c.stride(-2) if m > 1 else n) if c is not None else 0, m, n, k, groups, layout_kind, alignment,
        int(bool(store_padding)), min(int(expected_m), m), int(b_mn_major), int(d.dtype == torch.float32))
    with _lib.on_device(d.device):
        _lib.check(_lib.lib().dgb200_fp8_block_scaled_gemm(args, _lib.current_stream_ptr()))
