"""FP8 quantisers with FP32 scales: bit for bit what FP32 division and one rounding to E4M3 give."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def dg():
    import deepgemm_b200
    return deepgemm_b200


def reference(x, rows_per_block, gran_k, ue8m0=False):
    """x [G, N, K] on the CPU (whose FP32 division is IEEE's)."""
    x = x.float()
    g, n, k = x.shape
    q, nb, kb = torch.empty_like(x), -(-n // rows_per_block), -(-k // gran_k)
    sf = torch.empty(g, nb, kb)
    for r in range(nb):
        for c in range(kb):
            part = x[:, r * rows_per_block:(r + 1) * rows_per_block, c * gran_k:(c + 1) * gran_k]
            s = part.abs().amax(dim=(1, 2)).clamp(min=1e-4) / torch.tensor(448.0)
            if ue8m0:
                s = torch.exp2(torch.ceil(torch.log2(s.double()))).float()
            sf[:, r, c] = s
            q[:, r * rows_per_block:(r + 1) * rows_per_block, c * gran_k:(c + 1) * gran_k] = part / s[:, None, None]
    return q.to(torch.float8_e4m3fn), sf


def values(*shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * scale * torch.exp2(torch.randint(-12, 6, shape, generator=g).float())
    return x.bfloat16()


def same(a, b):
    return torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize('rows, k', [(1, 16), (1, 7168), (3, 144), (31, 2048), (257, 1040), (1000, 528), (40, 128)])
@pytest.mark.parametrize('gran_k', [32, 128])
@pytest.mark.parametrize('scale', [1.0, 1e-30, 1e30, 1e-7])
def test_per_token(dg, rows, k, gran_k, scale):
    x = values(rows, k, seed=1, scale=scale)
    q, sf = dg.utils.per_token_cast_to_fp8(x.cuda(), use_ue8m0=False, gran_k=gran_k)
    want_q, want_sf = reference(x[:, None], 1, gran_k)
    assert torch.equal(sf.cpu(), want_sf[:, 0]) and same(q, want_q[:, 0])


@pytest.mark.parametrize('rows, k', [(20001, 528), (9999, 1040), (20000, 16), (5003, 2032)])
@pytest.mark.parametrize('gran_k', [32, 128])
def test_per_token_many_rows_with_a_short_last_block(dg, rows, k, gran_k):
    x = values(rows, k, seed=4)
    q, sf = dg.utils.per_token_cast_to_fp8(x.cuda(), use_ue8m0=False, gran_k=gran_k)
    want_q, want_sf = reference(x[:, None], 1, gran_k)
    assert torch.equal(sf.cpu(), want_sf[:, 0]) and same(q, want_q[:, 0])


@pytest.mark.parametrize('shape', [(1, 16), (128, 128), (130, 272), (7, 1024), (513, 144), (3, 256, 128), (2, 200, 400), (5, 1, 16)])
@pytest.mark.parametrize('ue8m0', [False, True])
@pytest.mark.parametrize('scale', [1.0, 1e-30])
def test_per_block(dg, shape, ue8m0, scale):
    x = values(*shape, seed=2, scale=scale)
    q, sf = dg.utils.per_block_cast_to_fp8(x.cuda(), use_ue8m0=ue8m0)
    want_q, want_sf = reference(x if x.dim() == 3 else x[None], 128, 128, ue8m0)
    assert torch.equal(sf.cpu(), want_sf if x.dim() == 3 else want_sf[0])
    assert same(q, want_q if x.dim() == 3 else want_q[0])


def test_every_bf16_mantissa_against_division(dg):
    """All 128 mantissas of x against all of the maximum: each row holds one maximum and every value below it in two binades."""
    tops = (128 + torch.arange(128.0)) * 2.0 ** -7
    below = torch.cat([(128 + torch.arange(128.0)) * 2.0 ** e for e in (-9, -13, -16)])
    x = torch.cat([tops[:, None], below.expand(128, -1).clamp(max=0.99), torch.zeros(128, 127)], dim=1).bfloat16()
    x = torch.cat([x, -x[:, 1:], x[:, :1]], dim=1)[:, :1008]
    q, sf = dg.utils.per_token_cast_to_fp8(x.cuda(), use_ue8m0=False)
    want_q, want_sf = reference(x[:, None], 1, 128)
    assert torch.equal(sf.cpu(), want_sf[:, 0]) and same(q, want_q[:, 0])


def test_strides_and_special_values(dg):
    store = values(6, 300, 320, seed=3).cuda()
    x = store[::2, 20:230, 16:288]
    q, sf = dg.utils.per_block_cast_to_fp8(x, use_ue8m0=False)
    want_q, want_sf = reference(x.cpu(), 128, 128)
    assert torch.equal(sf.cpu(), want_sf) and same(q, want_q)
    for view in (store[0, :, 3:35], store[1].t()[:, :288], store[2, ::3, :160], store[3, :1, :64].expand(5, 64)):
        q, sf = dg.utils.per_token_cast_to_fp8(view, use_ue8m0=False)
        want_q, want_sf = reference(view.cpu()[:, None], 1, 128)
        assert torch.equal(sf.cpu(), want_sf[:, 0]) and same(q, want_q[:, 0])
    x = torch.ones(2, 256, dtype=torch.bfloat16, device='cuda')
    x[0, 3], x[1, 130] = float('inf'), float('nan')
    for q, sf in (dg.utils.per_token_cast_to_fp8(x, use_ue8m0=False), dg.utils.per_block_cast_to_fp8(x, use_ue8m0=False)):
        v = q.float()
        assert torch.isnan(v[0, 3]) and (v[0, 4:128] == 0).all() and torch.isinf(sf.flatten()[0])
        assert torch.isnan(v[1, 130]) and (v[1, 131:] == 448).all() and (v[0, 128:] == 448).all()


def test_no_rows(dg):
    q, sf = dg.utils.per_token_cast_to_fp8(torch.empty((0, 256), dtype=torch.bfloat16, device='cuda'), use_ue8m0=False)
    assert q.shape == (0, 256) and sf.shape == (0, 2)
    q, sf = dg.utils.per_block_cast_to_fp8(torch.empty((0, 128, 256), dtype=torch.bfloat16, device='cuda'), use_ue8m0=False)
    assert q.shape == (0, 128, 256) and sf.shape == (0, 1, 2)
