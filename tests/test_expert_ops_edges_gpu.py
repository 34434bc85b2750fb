"""Calls of the operators around the experts' GEMMs at the ends of their ranges, against FP64."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def dg():
    import deepgemm_b200
    yield deepgemm_b200
    from deepgemm_b200 import _lib
    assert _lib.device_status()[0] == 0


@pytest.mark.parametrize('form', [(0, -1), (128, 0), (256, 0), (256, 1)])
@pytest.mark.parametrize('nn', [False, True])
def test_padding_rows_are_zero_whatever_their_scales_hold(dg, form, nn):
    """ensure_zero_padding: rows between a group's end and its aligned end are zero where a's are; nothing has written scales for them."""
    from deepgemm_b200 import _lib
    g = torch.Generator(device='cuda').manual_seed(1)
    n, k, ends, rows = 272, 656, [5, 128, 387, 512], 700
    codes = torch.randint(1, 0x70, (rows, k), generator=g, device='cuda', dtype=torch.uint8)
    sfa = torch.rand(rows, 6, generator=g, device='cuda') + 0.5
    padding = torch.zeros(rows, dtype=torch.bool, device='cuda')
    for e in ends:
        padding[e:-(-e // 128) * 128] = True
    codes[padding] = 0
    b = torch.randint(1, 0x70, (4, k, n) if nn else (4, n, k), generator=g, device='cuda', dtype=torch.uint8).view(torch.float8_e4m3fn)
    sfb = torch.rand((4, 6, 3) if nn else (4, 3, 6), generator=g, device='cuda') + 0.5
    gemm = dg.m_grouped_fp8_gemm_nn_contiguous if nn else dg.m_grouped_fp8_gemm_nt_contiguous
    outs = []
    try:
        for knob, value in zip(('block_n', 'pair'), form):
            _lib.check(_lib.lib().dgb200_set_tuning(knob.encode(), value))
        for bad in (1.0, float('nan'), float('inf')):
            sfa[padding] = bad
            d = torch.full((rows, n), float('nan'), dtype=torch.bfloat16, device='cuda')
            gemm((codes.view(torch.float8_e4m3fn), sfa), (b, sfb), d, torch.tensor(ends, dtype=torch.int32, device='cuda'), disable_ue8m0_cast=True,
                 use_psum_layout=True)
            assert (d[padding] == 0).all() and torch.isfinite(d[:512].float()).all() and torch.isnan(d[512:].float()).all()
            outs.append(d[:512])
    finally:
        for knob, value in (('block_n', 0), ('pair', -1)):
            _lib.check(_lib.lib().dgb200_set_tuning(knob.encode(), value))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
