"""Calls that the operators around the experts' GEMMs refuse, on the CPU: every one ends before a kernel is launched."""
import ctypes
import struct

import pytest
import torch

import deepgemm_b200 as dg
from deepgemm_b200 import _lib, block_scaled, build

P, NULL = ctypes.c_void_p(4096), None


@pytest.fixture(scope='module')
def lib():
    build.build()
    return _lib.lib()


def refused(lib, rc, fragment):
    assert rc == 1 and fragment in lib.dgb200_last_error().decode(), (rc, lib.dgb200_last_error())


FIELDS = ['size', 'a', 'sfa', 'b', 'sfb', 'd', 'c', 'layout', 'sfa_group_stride', 'sfa_row_stride', 'sfa_k_stride', 'sfb_group_stride',
          'sfb_n_stride', 'sfb_k_stride', 'd_row_stride', 'c_row_stride', 'm', 'n', 'k', 'num_groups', 'layout_kind', 'alignment', 'store_padding',
          'expected_m', 'b_mn_major', 'd_is_fp32']


@pytest.mark.parametrize('change, fragment', [
    (dict(size=160), 'another size'), (dict(layout_kind=4), 'layout kind'), (dict(m=-1), 'm must be'), (dict(n=0), 'm must be'),
    (dict(n=260), 'multiple of 8'), (dict(k=130), 'of 16'), (dict(b_mn_major=1, n=264), 'MN-major'), (dict(num_groups=2), 'one group'),
    (dict(layout_kind=1, num_groups=513), '512'), (dict(layout_kind=2, num_groups=513), '512'), (dict(layout_kind=1, alignment=6), 'alignment'),
    (dict(layout_kind=0, alignment=64), 'multiple of 128'), (dict(a=0), 'null'), (dict(sfa=0), 'null'), (dict(b=0), 'null'), (dict(sfb=0), 'null'),
    (dict(d=0), 'null'), (dict(layout_kind=1, layout=0), 'null'), (dict(a=4100), '16-byte'), (dict(b=4104), '16-byte'), (dict(sfa=4098), '4-byte'),
    (dict(sfb=4097), '4-byte'), (dict(d=4104), 'd must be 16-byte'), (dict(d_row_stride=128), 'row stride'), (dict(d_row_stride=260), 'row stride'),
    (dict(c=4096), 'c needs'), (dict(c=4096, d_is_fp32=1, layout_kind=1), 'c needs'), (dict(c=4100, d_is_fp32=1), 'c must'),
    (dict(c=4096, d_is_fp32=1, c_row_stride=100), 'c must'),
])
def test_gemm_c_abi(lib, change, fragment):
    fields = dict(size=168, a=4096, sfa=4096, b=4096, sfb=4096, d=4096, c=0, layout=4096, sfa_group_stride=0, sfa_row_stride=1, sfa_k_stride=1,
                  sfb_group_stride=0, sfb_n_stride=1, sfb_k_stride=1, d_row_stride=256, c_row_stride=256, m=64, n=256, k=256, num_groups=1,
                  layout_kind=3, alignment=128, store_padding=0, expected_m=64, b_mn_major=0, d_is_fp32=0)
    if 'n' in change and change['n'] > 256:
        fields['d_row_stride'] = 512
    fields.update(change)
    assert block_scaled._ARGS.size == 168
    refused(lib, lib.dgb200_fp8_block_scaled_gemm(struct.pack('@N7P8q10i', *(fields[f] for f in FIELDS)), NULL), fragment)
    refused(lib, lib.dgb200_fp8_block_scaled_gemm(None, NULL), 'another size')


def test_quantisers_c_abi(lib):
    token, block = lib.dgb200_per_token_cast_to_fp8_f32_scales, lib.dgb200_per_block_cast_to_fp8
    refused(lib, token(P, 100, 4, 100, 128, P, 112, P, 1, NULL), 'multiple of 16')
    refused(lib, token(NULL, 128, 4, 128, 128, P, 128, P, 1, NULL), 'null')
    refused(lib, token(P, 128, 4, 128, 64, P, 128, P, 2, NULL), 'gran_k')
    refused(lib, token(P, 132, 4, 128, 128, P, 128, P, 1, NULL), '16-byte')
    refused(lib, token(P, 64, 4, 128, 128, P, 128, P, 1, NULL), 'cover k')
    refused(lib, token(P, 128, 4, 128, 32, P, 128, P, 3, NULL), 'scale rows')
    refused(lib, block(P, 0, 256, 1, 4, 256, 0, P, 0, 256, P, 0, 1, NULL), 'scale rows')
    refused(lib, block(P, 4, 256, 2, 4, 256, 0, P, 0, 256, P, 0, 2, NULL), '16-byte')
    refused(lib, block(P, 0, 256, 65536, 4, 256, 0, P, 0, 256, P, 0, 2, NULL), 'groups')


def test_plan_and_permutation_c_abi(lib):
    plan = lib.dgb200_moe_dispatch_plan
    refused(lib, plan(P, 4, 0, 8, 16, P, P, P, NULL, NULL), 'num_topk')
    refused(lib, plan(P, 4, 33, 8, 16, P, P, P, NULL, NULL), 'num_topk')
    refused(lib, plan(P, 4, 2, 1025, 16, P, P, P, NULL, NULL), 'experts')
    refused(lib, plan(P, 4, 2, 8, 0, P, P, P, NULL, NULL), 'alignment')
    refused(lib, plan(NULL, 4, 2, 8, 16, P, P, P, NULL, NULL), 'null')
    refused(lib, plan(P, 4, 2, 8, 16, NULL, P, P, NULL, NULL), 'null')
    refused(lib, plan(P, 100000, 8, 8, 16, P, P, P, NULL, NULL), 'workspace')
    refused(lib, plan(P, 2 ** 28, 8, 8, 16, P, P, P, P, NULL), 'too many')
    assert lib.dgb200_moe_dispatch_plan_workspace_bytes(-1, 1, 1) == -1
    assert lib.dgb200_moe_dispatch_plan_workspace_bytes(100, 8, 256) == 0 < lib.dgb200_moe_dispatch_plan_workspace_bytes(100000, 8, 256)
    permute = lib.dgb200_moe_permute
    refused(lib, permute(P, 128, 64, P, 128, NULL, 0, 0, NULL, 0, P, P, 4, 2, 8, 16, 100, 1, NULL), 'row strides')
    refused(lib, permute(P, 128, 128, NULL, 128, NULL, 0, 0, NULL, 0, P, P, 4, 2, 8, 16, 100, 1, NULL), 'null')
    refused(lib, permute(P, 128, 128, P, 128, P, 1, 1, NULL, 0, P, P, 4, 2, 8, 16, 100, 1, NULL), 'scale factors')
    refused(lib, permute(P, 128, 128, P, 128, P, 2, 1, P, 2, P, P, 4, 2, 8, 16, 100, 1, NULL), 'scale rows')
    back = lib.dgb200_moe_unpermute
    refused(lib, back(P, 32, P, P, P, 64, 4, 2, 64, 100, 0, NULL), 'row strides')
    refused(lib, back(NULL, 64, P, P, P, 64, 4, 2, 64, 100, 0, NULL), 'null')
    refused(lib, back(P, 64, P, P, P, 64, 4, 40, 64, 100, 0, NULL), 'num_topk')
    refused(lib, back(ctypes.c_void_p(4098), 64, P, P, P, 64, 4, 2, 64, 100, 1, NULL), 'aligned')
    grad = lib.dgb200_moe_unpermute_backward
    refused(lib, grad(NULL, 64, P, 64, P, P, P, P, 64, P, 4, 2, 8, 16, 64, 100, 0, NULL), 'null')
    refused(lib, grad(P, 64, P, 64, P, P, NULL, P, 64, P, 4, 2, 8, 16, 64, 100, 0, NULL), 'null')
    refused(lib, grad(P, 64, P, 64, P, P, P, P, 64, NULL, 4, 2, 8, 16, 64, 100, 0, NULL), 'null')


def test_swiglu_c_abi(lib):
    refused(lib, lib.dgb200_swiglu(NULL, 128, P, 64, 4, 64, NULL, 0, 0, 0.0, NULL), 'null')
    refused(lib, lib.dgb200_swiglu(P, 64, P, 64, 4, 64, NULL, 0, 0, 0.0, NULL), 'row strides')
    refused(lib, lib.dgb200_swiglu(P, 128, P, 64, 4, 0, NULL, 0, 0, 0.0, NULL), 'inter')
    refused(lib, lib.dgb200_swiglu(P, 128, P, 64, 4, 64, P, 0, 128, 0.0, NULL), 'layout')
    refused(lib, lib.dgb200_swiglu_backward(NULL, 64, P, 128, P, 128, 4, 64, NULL, 0, 0, 0.0, NULL), 'null')
    refused(lib, lib.dgb200_swiglu_per_token_cast_to_fp8(P, 120, P, 60, P, 1, 4, 60, NULL, 0, 0, 0.0, NULL), 'multiple of 8')
    refused(lib, lib.dgb200_swiglu_per_token_cast_to_fp8(P, 512, P, 256, P, 1, 4, 256, NULL, 0, 0, 0.0, NULL), 'scale rows')


def test_python_refuses_cpu_tensors_and_wrong_types():
    q, sf, d = torch.zeros(4, 128, dtype=torch.float8_e4m3fn), torch.ones(4, 1), torch.zeros(4, 4, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match='CUDA'):
        dg.fp8_gemm_nt((q, sf), (q, sf[:1]), d, disable_ue8m0_cast=True)
    with pytest.raises(RuntimeError, match='recipe'):
        dg.fp8_gemm_nt((q, sf), (q, sf), d, recipe=(1, 1, 128), disable_ue8m0_cast=True)
    with pytest.raises(RuntimeError, match='together'):
        dg.fp8_gemm_nt((q, sf), (q, sf), d, recipe_a=(1, 128), disable_ue8m0_cast=True)
    layout = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match='grouped_layout'):
        dg.m_grouped_fp8_gemm_nt_contiguous((q, sf), (q[None], sf[None]), d, layout, disable_ue8m0_cast=True, use_psum_layout=True)
    with pytest.raises(RuntimeError, match='masked_m'):
        dg.m_grouped_fp8_gemm_nt_masked((q[None], sf[None]), (q[None], sf[None]), d[None], layout, 1, disable_ue8m0_cast=True)
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    for call in (lambda: dg.utils.per_token_cast_to_fp8(x, use_ue8m0=False), lambda: dg.utils.per_block_cast_to_fp8(x, use_ue8m0=False),
                 lambda: dg.swiglu(x), lambda: dg.swiglu_backward(x, x), lambda: dg.swiglu_per_token_cast_to_fp8(x),
                 lambda: dg.moe_dispatch_plan(torch.zeros(4, 2, dtype=torch.int64), 8)):
        with pytest.raises(RuntimeError, match='CUDA'):
            call()
    with pytest.raises(RuntimeError, match='use_ue8m0'):
        dg.utils.per_token_cast_to_fp8(x, use_ue8m0=False, use_packed_ue8m0=True)
    with pytest.raises(RuntimeError, match='128 x 128'):
        dg.utils.per_block_cast_to_fp8(x, use_ue8m0=False, gran_k=32)
    plan = dg.MoeDispatchPlan(torch.zeros(4, 2, dtype=torch.int32), layout, layout, 16)
    assert plan.capacity == 32 and plan.num_experts == 1
    for call in (lambda: dg.moe_permute(x, plan), lambda: dg.moe_unpermute(x, plan), lambda: dg.moe_permute_backward(x, plan),
                 lambda: dg.moe_unpermute_backward(x, x, plan)):
        with pytest.raises(RuntimeError, match='dest_row'):
            call()


@pytest.mark.gpu
def test_python_refusals_on_the_gpu():
    cuda = lambda *shape, dtype=torch.bfloat16: torch.zeros(*shape, dtype=torch.float32, device='cuda').to(dtype)
    q, sf = cuda(64, 256, dtype=torch.float8_e4m3fn), cuda(64, 2, dtype=torch.float32)
    b, sfb, d = cuda(128, 256, dtype=torch.float8_e4m3fn), cuda(1, 2, dtype=torch.float32), cuda(64, 128)
    gemm = lambda a=(q, sf), b=(b, sfb), d=d, **kw: dg.fp8_gemm_nt(a, b, d, disable_ue8m0_cast=True, **kw)
    for call, match in ((lambda: gemm(a=(q, sf[:, :1])), 'K extent'), (lambda: gemm(b=(b, sf)), 'MN extent'), (lambda: gemm(d=d[:, :120]), 'shape'),
                        (lambda: gemm(d=d.half()), 'd must'), (lambda: gemm(c=cuda(64, 128, dtype=torch.float32)), 'c must'),
                        (lambda: gemm(b=(b.view(torch.int8), sfb)), 'float8'), (lambda: gemm(a=(q[:, ::2], sf)), 'contiguous'),
                        (lambda: gemm(d=q.view(torch.bfloat16)), 'overlap'), (lambda: gemm(d=d[:1].expand(64, 128)), 'aligned and not overlap'),
                        (lambda: gemm(a=(cuda(64, 120, dtype=torch.float8_e4m3fn), sf[:, :1]), b=(cuda(128, 120, dtype=torch.float8_e4m3fn), sfb[:, :1])), 'of 16')):
        with pytest.raises(RuntimeError, match=match):
            call()
    idx = torch.zeros(5, 2, dtype=torch.int64, device='cuda')
    plan = dg.moe_dispatch_plan(idx, 4, alignment=8)
    x = cuda(5, 64)
    for call, match in ((lambda: dg.moe_dispatch_plan(idx.int(), 4), 'int64'), (lambda: dg.moe_dispatch_plan(idx.t(), 4), 'contiguous'),
                        (lambda: dg.moe_dispatch_plan(idx, 0), 'num_experts'), (lambda: dg.moe_permute(x[:4], plan), 'shape'),
                        (lambda: dg.moe_permute(x.half(), plan), '2-D CUDA'), (lambda: dg.moe_permute(x, plan, out=cuda(plan.capacity - 1, 64)), 'at least'),
                        (lambda: dg.moe_permute((x, x), plan), '2-D CUDA'), (lambda: dg.moe_unpermute(x, plan), 'capacity'),
                        (lambda: dg.moe_unpermute(cuda(plan.capacity, 64), plan, cuda(5, 3, dtype=torch.float32)), 'topk_weights'),
                        (lambda: dg.moe_unpermute(cuda(plan.capacity, 64), plan, cuda(5, 2)), 'topk_weights')):
        with pytest.raises(RuntimeError, match=match):
            call()
    store = cuda(plan.capacity + 5, 64)
    with pytest.raises(RuntimeError, match='overlap'):
        dg.moe_permute(store[:5], plan, out=store[:plan.capacity])
    with pytest.raises(RuntimeError, match='overlap'):
        dg.moe_unpermute_backward(x, store, plan, out=store)
    wide = cuda(6, 128)
    for call, match in ((lambda: dg.swiglu(wide[:, :127]), 'even'), (lambda: dg.swiglu(wide.float()), '2-D CUDA'),
                        (lambda: dg.swiglu(wide, out=wide[:, :64]), 'overlap'), (lambda: dg.swiglu(wide, activation_clamp=0.0), 'positive'),
                        (lambda: dg.swiglu(wide, activation_clamp=float('nan')), 'positive'),
                        (lambda: dg.swiglu(wide, grouped_layout=idx[0]), 'int32'), (lambda: dg.swiglu_backward(wide, wide), 'shape'),
                        (lambda: dg.swiglu_per_token_cast_to_fp8(wide[:, :72]), 'multiple of 8'), (lambda: dg.swiglu(wide.t()), 'unit inner')):
        with pytest.raises(RuntimeError, match=match):
            call()


LARGE = 2 ** 31 - 1  # counts of tiles, vectors and rows are 32-bit: sizes near their end are refused


def test_sizes_near_the_end_of_32_bits(lib):
    fields = dict(size=168, a=4096, sfa=4096, b=4096, sfb=4096, d=4096, c=0, layout=4096, sfa_group_stride=0, sfa_row_stride=1, sfa_k_stride=1,
                  sfb_group_stride=0, sfb_n_stride=1, sfb_k_stride=1, d_row_stride=256, c_row_stride=256, m=64, n=256, k=256, num_groups=1,
                  layout_kind=3, alignment=128, store_padding=0, expected_m=64, b_mn_major=0, d_is_fp32=0)
    for change in (dict(m=LARGE), dict(n=2 ** 31 - 16, d_row_stride=2 ** 31), dict(k=2 ** 31 - 16)):
        args = struct.pack('@N7P8q10i', *({**fields, **change}[f] for f in FIELDS))
        refused(lib, lib.dgb200_fp8_block_scaled_gemm(args, NULL), 'too large')
    refused(lib, lib.dgb200_per_token_cast_to_fp8_f32_scales(P, 16, LARGE, 16, 128, P, 16, P, 1, NULL), 'too large')
    refused(lib, lib.dgb200_moe_dispatch_plan(P, LARGE, 1, 1, 1, P, P, P, P, NULL), 'too many')
    refused(lib, lib.dgb200_moe_dispatch_plan(P, 1, 1, 1, LARGE, P, P, P, NULL, NULL), 'alignment')
    refused(lib, lib.dgb200_moe_permute(P, 128, 128, P, 128, NULL, 0, 0, NULL, 0, P, P, 0, 1, 1, LARGE, 4, 1, NULL), 'alignment')
    refused(lib, lib.dgb200_moe_unpermute(P, 2 ** 31, P, P, P, 2 ** 31, 4, 2, LARGE, 100, 0, NULL), 'hidden')
    refused(lib, lib.dgb200_swiglu(P, 2 ** 32, P, 2 ** 31, 4, LARGE, NULL, 0, 0, 0.0, NULL), 'too large')
    refused(lib, lib.dgb200_swiglu_backward(P, 64, P, 128, P, 128, LARGE, 64, NULL, 0, 0, 0.0, NULL), 'too large')


def test_python_refuses_sizes_beyond_32_bits(monkeypatch):
    # a row that repeats stands for a buffer of that many rows
    for t in (torch.zeros(1, 1).expand(2 ** 31, 1), torch.zeros(1, 1).expand(1, 2 ** 31)):
        monkeypatch.setattr(torch.Tensor, 'is_cuda', True)
        from deepgemm_b200.permute import _check_rows
        with pytest.raises(RuntimeError, match='too large|inner stride'):
            _check_rows(t, None, None, (torch.float32,), 'out')
    with pytest.raises(RuntimeError, match='too large'):
        dg.utils.per_token_cast_to_fp8(torch.zeros(1, 16, dtype=torch.bfloat16).expand(2 ** 31, 16), use_ue8m0=False)
    with pytest.raises(RuntimeError, match='too large'):
        dg.utils.per_block_cast_to_fp8(torch.zeros(1, 16, dtype=torch.bfloat16).expand(2 ** 31, 16), use_ue8m0=False)
    with pytest.raises(RuntimeError, match='too large'):
        dg.moe_dispatch_plan(torch.zeros(2 ** 31, 0, dtype=torch.int64), 8)


@pytest.mark.gpu
def test_more_python_refusals_on_the_gpu():
    plan = dg.moe_dispatch_plan(torch.zeros(5, 2, dtype=torch.int64, device='cuda'), 4, alignment=8)
    x = torch.zeros(5, 64, dtype=torch.bfloat16, device='cuda')
    rows = torch.zeros(plan.capacity, 64, dtype=torch.bfloat16, device='cuda')
    with pytest.raises(RuntimeError, match='pairs'):
        dg.moe_permute(x, plan, out=(rows, rows))
    store = torch.zeros(128 * 128 * 2 + 16, dtype=torch.uint8, device='cuda')
    d, layout = store[:128 * 128 * 2].view(torch.bfloat16).view(128, 128), store[256:260].view(torch.int32)
    a, sfa = torch.zeros(128, 128, device='cuda').to(torch.float8_e4m3fn), torch.ones(128, 1, device='cuda')
    with pytest.raises(RuntimeError, match='overlap'):
        dg.m_grouped_fp8_gemm_nt_contiguous((a, sfa), (a[None], sfa[None, :1]), d, layout, disable_ue8m0_cast=True, use_psum_layout=True)
