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


# ------------------------------------------------------------------------------------------------------- gates far below zero
# The sigmoid's relative error there is the exponential's: 2 + 1.16 |g| half steps (2^-24 each, the documented bound of the fast one is in whole
# ones) and a few roundings: (1.16 |g| + 12) * 2^-23 of the value, or of the terms of the gate's gradient. One rounding to BF16.

def far_case(inter, seed):
    """Gates from 0 to -170 in every step of BF16 that lies there, with values of `up` that keep the product among ordinary numbers."""
    g = torch.Generator(device='cuda').manual_seed(seed)
    gate = torch.cat([torch.arange(-170.0, -60.0, 0.5), torch.arange(-60.0, 0.0, 0.25)])
    gate = gate.bfloat16().unique().cuda()
    gate = gate[torch.randint(0, gate.numel(), (64, inter), generator=g, device='cuda')]
    size = torch.exp2((-gate.float() * 1.4427).clamp(max=118.0) + torch.rand(64, inter, generator=g, device='cuda') * 6 - 3)
    up = (size * torch.where(torch.rand(64, inter, generator=g, device='cuda') < 0.5, -1.0, 1.0)).bfloat16()
    dy = torch.randn(64, inter, generator=g, device='cuda').bfloat16()
    return torch.cat([gate, up], dim=1), dy


def far_reference(x, dy):
    inter = x.shape[1] // 2
    g, u, dy = x[:, :inter].double(), x[:, inter:].double(), dy.double()
    s = torch.exp(g) / (1 + torch.exp(g))
    return g * s * u, dy * u * s * (1 + g * (1 - s)), dy * g * s, dy.abs() * u.abs() * s * (1 + g.abs())


@pytest.mark.parametrize('inter', [7, 264])
@pytest.mark.parametrize('clamp', [None, 3e38])
def test_gates_far_below_zero(dg, inter, clamp):
    x, dy = far_case(inter, seed=3)
    y, d_gate, d_up, terms = far_reference(x, dy)
    error = (1.16 * x[:, :inter].double().abs() + 12) * 2.0 ** -23
    smallest = 2.0 ** -134  # half a step of BF16's subnormal numbers
    got = dg.swiglu(x, activation_clamp=clamp).double()
    assert ((got - y).abs() <= y.abs() * (2.0 ** -8 + error) + smallest).all()
    got = dg.swiglu_backward(dy, x, activation_clamp=clamp).double()
    assert ((got[:, :inter] - d_gate).abs() <= d_gate.abs() * 2.0 ** -8 + terms * error * 1.01 + smallest).all()
    assert ((got[:, inter:] - d_up).abs() <= d_up.abs() * (2.0 ** -8 + error) + smallest).all()
    if inter % 8 == 0:
        q, sf = dg.swiglu_per_token_cast_to_fp8(x, activation_clamp=clamp)
        blocks = -(-inter // 128)
        amax = torch.nn.functional.pad(y, (0, blocks * 128 - inter)).view(64, blocks, 128).abs().amax(dim=-1)
        scale = amax.clamp(min=1e-4) / 448
        assert ((sf.double() - scale).abs() <= scale * 2.0 ** -19).all()
        wide = sf.double().repeat_interleave(128, dim=1)[:, :inter]
        step = torch.maximum(y.abs() * 2.0 ** -4, wide * 2.0 ** -10)
        assert ((q.double() * wide - y).abs() <= step * 1.001 + y.abs() * 2.0 ** -18).all()


def test_a_gate_at_the_end_of_the_exponential(dg):
    """-87.5 and 1e36: the denominator of the sigmoid is finite, its reciprocal no normal number; the product is about -0.87."""
    for g in (-87.0, -87.5, -88.0, -88.5, -89.0, -104.0):
        x = torch.tensor([[g] * 8 + [1e36] * 8], dtype=torch.float64)
        want = g * torch.exp(torch.tensor(g, dtype=torch.float64)) * float(x.bfloat16()[0, 8])
        x = x.bfloat16().cuda()
        assert abs(float(dg.swiglu(x)[0, 0]) - float(want)) <= abs(float(want)) * 2.0 ** -7
        q, sf = dg.swiglu_per_token_cast_to_fp8(x)
        assert abs(float(q.float()[0, 0] * sf[0, 0]) - float(want)) <= max(abs(float(want)) * 2.0 ** -4, 1e-4 / 448 * 2.0 ** -10) * 1.01
    x = torch.tensor([[-float('inf')] * 8 + [2.0] * 8], device='cuda').bfloat16()
    assert torch.isnan(dg.swiglu(x)).all() and torch.isnan(dg.swiglu_per_token_cast_to_fp8(x)[0].float()).all()  # infinity times zero


def test_a_clamp_that_fp32_rounds_to_zero_is_refused(dg):
    x = torch.ones(2, 32, dtype=torch.bfloat16, device='cuda')
    for call in (lambda c: dg.swiglu(x, activation_clamp=c), lambda c: dg.swiglu_backward(x[:, :16], x, activation_clamp=c),
                 lambda c: dg.swiglu_per_token_cast_to_fp8(x, activation_clamp=c)):
        for c in (1e-46, 1e-300):
            with pytest.raises(RuntimeError, match='positive'):
                call(c)
    assert (dg.swiglu(x, activation_clamp=1e-44).float() == 0).all()  # the smallest clamps still hold
    assert torch.equal(dg.swiglu(x, activation_clamp=1e300), dg.swiglu(x))


def test_expected_rows_beyond_32_bits_only_steer(dg):
    g = torch.Generator(device='cuda').manual_seed(5)
    a = torch.randint(0, 0x70, (3, 40, 256), generator=g, device='cuda', dtype=torch.uint8).view(torch.float8_e4m3fn)
    b = torch.randint(0, 0x70, (3, 128, 256), generator=g, device='cuda', dtype=torch.uint8).view(torch.float8_e4m3fn)
    sfa, sfb = torch.rand(3, 40, 2, generator=g, device='cuda'), torch.rand(3, 1, 2, generator=g, device='cuda')
    counts = torch.tensor([40, 0, 7], dtype=torch.int32, device='cuda')
    outs = []
    for expected in (40, 2 ** 31, 2 ** 40):
        d = torch.zeros(3, 40, 128, dtype=torch.bfloat16, device='cuda')
        dg.m_grouped_fp8_gemm_nt_masked((a, sfa), (b, sfb), d, counts, expected, disable_ue8m0_cast=True)
        outs.append(d)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]) and (outs[0][0] != 0).any()


@pytest.mark.parametrize('special', ['inf', '-inf', 'nan'])
def test_special_values_in_blocks_with_a_power_of_two_scale(dg, special):
    """As the per-token quantiser with power-of-two scales: a block with an infinity has the largest scale, 2^127, and its infinities the largest
    code, whose product with the scale is infinite; NaN stays NaN and is passed over by the maximum."""
    x = torch.ones(130, 272, dtype=torch.bfloat16, device='cuda')
    x[5, 130] = float(special)
    q, sf = dg.utils.per_block_cast_to_fp8(x, use_ue8m0=True)
    if special == 'nan':
        assert torch.isnan(q[5, 130].float()) and (sf == 2.0 ** -8).all()
        q.view(torch.uint8)[5, 130] = q.view(torch.uint8)[5, 131]
        assert (q.float() == 256).all()
        return
    assert float(sf[0, 1]) == 2.0 ** 127 and float(q[5, 130].float()) == (448 if special == 'inf' else -448)
    assert torch.isinf(q[5, 130].float() * sf[0, 1])
    block = q[:128, 128:256].float().clone()
    block[5, 2] = 0
    assert (block == 0).all()
    sf[0, 1] = 2.0 ** -8
    assert (sf == 2.0 ** -8).all() and (q[:, :128].float() == 256).all() and (q[128:].float() == 256).all() and (q[:, 256:].float() == 256).all()
    t, t_sf = dg.utils.per_token_cast_to_fp8(x[5:6, 128:256], use_ue8m0=True)
    assert float(t_sf[0, 0]) == 2.0 ** 127 and torch.equal(t.view(torch.uint8)[0], q.view(torch.uint8)[5, 128:256])


def test_the_plan_with_the_most_chunks(dg):
    """128 chunks, the last one full, short by one entry and of one entry."""
    from deepgemm_b200 import _lib
    experts, alignment = 300, 16
    for entries in (6 * 131072, 6 * 131072 - 1, 127 * 6144 + 1):
        assert _lib.lib().dgb200_moe_dispatch_plan_workspace_bytes(entries, 1, experts) == 128 * experts * 4
        g = torch.Generator(device='cuda').manual_seed(entries)
        flat = torch.randint(-1, experts, (entries,), generator=g, device='cuda')
        plan = dg.moe_dispatch_plan(flat[:, None], experts, alignment=alignment)
        order = torch.argsort(torch.where(flat < 0, experts, flat), stable=True)
        counts = torch.bincount(flat[flat >= 0], minlength=experts)
        padded = (counts + alignment - 1) // alignment * alignment
        start, first = padded.cumsum(0) - padded, counts.cumsum(0) - counts
        want = torch.full((entries,), -1, dtype=torch.int64, device='cuda')
        kept = order[:int(counts.sum())]
        want[kept] = start[flat[kept]] + torch.arange(kept.numel(), device='cuda') - first[flat[kept]]
        assert torch.equal(plan.dest_row.flatten().long(), want)
        assert torch.equal(plan.expert_start.long(), start) and torch.equal(plan.expert_end.long(), start + counts)


@pytest.mark.parametrize('rows, inter', [(7, 264), (2500, 2048)])
def test_rows_beside_special_ones_keep_their_bits(dg, rows, inter):
    """NaN, infinities, far gates and products near the end of FP32 in some rows: the others' codes and scales are what they are without."""
    g = torch.Generator(device='cuda').manual_seed(7)
    x = (torch.randn(rows, 2 * inter, generator=g, device='cuda') * 2).bfloat16()
    q, sf = dg.swiglu_per_token_cast_to_fp8(x)
    special = x.clone()
    for row, (gate, up) in zip(range(1, rows, 2), ((float('nan'), 1.0), (-100.0, 1e36), (1e19, 2e19))):
        special[row, 3], special[row, inter + 3] = gate, up
    changed = [r for r in range(1, rows, 2)][:3]
    got_q, got_sf = dg.swiglu_per_token_cast_to_fp8(special)
    kept = torch.ones(rows, dtype=torch.bool, device='cuda')
    kept[changed] = False
    assert torch.equal(got_q.view(torch.uint8)[kept], q.view(torch.uint8)[kept]) and torch.equal(got_sf[kept], sf[kept])
    assert torch.equal(got_q.view(torch.uint8)[:, 128:], q.view(torch.uint8)[:, 128:]) and torch.equal(got_sf[:, 1:], sf[:, 1:])
    assert torch.isnan(got_q.float()[1, 3]) and torch.isfinite(got_q.float()[2:]).all() and torch.isfinite(got_sf).all()
    # 1e19 and 2e19: the product is finite, four times it is not
    product = special[5, 3].double() * special[5, inter + 3].double()
    assert abs(float(got_sf[5, 0]) / float(product / 448) - 1) <= 2.0 ** -20 and float(got_q.float()[5, 3]) == 448
