"""SwiGLU of the experts' rows, its FP8 form and its gradient, against FP64.

Tolerances: the FP32 arithmetic (an exponential and a reciprocal of the hardware, 2 ulp each, and four to seven roundings) is within 2^-20 of the
value, or of the sum of the magnitudes of the terms where terms cancel (the gate's gradient); one rounding to BF16 (2^-8). FP8: scales within 2^-20 relatively;
values within half a step of E4M3 (2^-4 of the value, 2^-10 of the scale below the normal range), give or take the scale's error."""
import pytest
import torch

pytestmark = pytest.mark.gpu

ARITHMETIC = 2.0 ** -20


@pytest.fixture(scope='module')
def dg():
    import deepgemm_b200
    yield deepgemm_b200
    from deepgemm_b200 import _lib
    assert _lib.device_status()[0] == 0


def case(rows, inter, pad, seed, scale=2.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    x = (torch.randn(rows, 2 * inter + pad, generator=g, device='cuda') * scale).bfloat16()[:, :2 * inter]
    dy = torch.randn(rows, inter + pad, generator=g, device='cuda').bfloat16()[:, :inter]
    return x, dy


def reference(x, dy, clamp):
    inter = x.shape[1] // 2
    gate, up = x[:, :inter].double(), x[:, inter:].double()
    limit = clamp if clamp is not None else float('inf')
    g, u, dy = gate.clamp(max=limit), up.clamp(-limit, limit), dy.double()
    s = torch.sigmoid(g)
    d_gate = torch.where(gate > limit, 0.0, dy * u * s * (1 + g * (1 - s)))
    d_up = torch.where(up.abs() > limit, 0.0, dy * g * s)
    magnitude = torch.cat([dy.abs() * u.abs() * s * (1 + g.abs() * (1 - s)), d_up.abs()], dim=1)
    return g * s * u, torch.cat([d_gate, d_up], dim=1), magnitude


SIZES = [(1, 1, 0), (1, 2048, 0), (3, 7, 1), (5, 8, 8), (33, 40, 4), (129, 520, 0), (64, 2304, 16), (257, 128, 0)]


@pytest.mark.parametrize('rows, inter, pad', SIZES)
@pytest.mark.parametrize('clamp', [None, 1.5])
def test_forward_and_gradient(dg, rows, inter, pad, clamp):
    x, dy = case(rows, inter, pad, seed=1)
    y, dx, magnitude = reference(x, dy, clamp)
    got = dg.swiglu(x, activation_clamp=clamp)
    assert got.shape == (rows, inter) and ((got.double() - y).abs() <= y.abs() * (2.0 ** -8 + 2 * ARITHMETIC)).all()
    got = dg.swiglu_backward(dy, x, activation_clamp=clamp)
    assert ((got.double() - dx).abs() <= dx.abs() * 2.0 ** -8 * 1.01 + magnitude * 2 * ARITHMETIC).all()


def check_fp8(q, sf, y):
    rows, inter = y.shape
    blocks = -(-inter // 128)
    padded = torch.nn.functional.pad(y, (0, blocks * 128 - inter)).view(rows, blocks, 128)
    scale = padded.abs().amax(dim=-1).clamp(min=1e-4) / 448
    assert ((sf.double() - scale).abs() <= scale * 2 * ARITHMETIC).all()
    wide = sf.double().repeat_interleave(128, dim=1)[:, :inter]
    step = torch.maximum(y.abs() * 2.0 ** -4, wide * 2.0 ** -10)
    assert ((q.double() * wide - y).abs() <= step * 1.001 + y.abs() * 4 * ARITHMETIC).all()


@pytest.mark.parametrize('rows, inter, pad', [s for s in SIZES if s[1] % 8 == 0 and s[2] % 8 == 0])
@pytest.mark.parametrize('clamp', [None, 1.5])
def test_forward_to_fp8(dg, rows, inter, pad, clamp):
    x, dy = case(rows, inter, pad, seed=2)
    q, sf = dg.swiglu_per_token_cast_to_fp8(x, activation_clamp=clamp)
    check_fp8(q, sf, reference(x, dy, clamp)[0])


@pytest.mark.parametrize('ends', [[0], [1], [5, 130, 128], [128, 128, 128], [100, 256, 300]])
def test_rows_behind_the_last_segment_are_left_alone(dg, ends):
    rows, inter = 700, 136
    x, dy = case(rows, inter, 0, seed=3)
    total = -(-ends[-1] // 128) * 128
    x[total:], dy[total:] = float('nan'), float('nan')
    layout = torch.tensor(ends, dtype=torch.int32, device='cuda')
    y, dx, _ = reference(x[:total], dy[:total], None)
    out = torch.full((rows, inter), 5.0, dtype=torch.bfloat16, device='cuda')
    dg.swiglu(x, grouped_layout=layout, out=out)
    assert (out[total:] == 5).all() and ((out[:total].double() - y).abs() <= y.abs() * 2.0 ** -7).all()
    out = torch.full((rows, 2 * inter), 5.0, dtype=torch.bfloat16, device='cuda')
    dg.swiglu_backward(dy, x, grouped_layout=layout, out=out)
    assert (out[total:] == 5).all() and torch.isfinite(out.float()).all()
    q, sf = torch.full((rows, inter), 5.0, device='cuda').to(torch.float8_e4m3fn), torch.full((rows, 2), 5.0, device='cuda')
    dg.swiglu_per_token_cast_to_fp8(x, grouped_layout=layout, out=(q, sf))
    assert (q[total:].float() == 5).all() and (sf[total:] == 5).all()
    if total:
        check_fp8(q[:total], sf[:total], y)


def test_a_layout_past_the_buffer_is_cut_off(dg):
    x, dy = case(40, 16, 0, seed=4)
    store = torch.full((60, 16), 5.0, dtype=torch.bfloat16, device='cuda')
    for words in ([3, 2 ** 31 - 1], [3, -7]):
        store.fill_(5.0)
        dg.swiglu(x, grouped_layout=torch.tensor(words, dtype=torch.int32, device='cuda'), out=store[:40])
        assert (store[40:] == 5).all() and bool((store[:40] == 5).all()) == (words[1] < 0)


def test_zero_rows_and_extremes(dg):
    assert dg.swiglu(torch.empty((0, 32), dtype=torch.bfloat16, device='cuda')).shape == (0, 16)
    inf, nan = float('inf'), float('nan')
    gate = torch.tensor([0.0, 100.0, -100.0, 3e38, -3e38, nan, inf, 1.0], device='cuda')
    up = torch.tensor([3.0, 2.0, 2.0, 0.0, 2.0, 1.0, 1.0, nan], device='cuda')
    x = torch.cat([gate, up]).bfloat16().view(1, 16)
    for clamp in (None, 10.0):
        y = dg.swiglu(x, activation_clamp=clamp)[0].float()
        assert torch.equal(y[:5], torch.tensor([0.0, 200.0 if clamp is None else 20.0, 0.0, 0.0, 0.0], device='cuda') + y[:5] * 0)
        assert torch.isnan(y[5]) and torch.isnan(y[7])
        q, sf = dg.swiglu_per_token_cast_to_fp8(x, activation_clamp=clamp)
        assert torch.isnan(q.float()[0, 5]) and torch.isnan(q.float()[0, 7])
    zero = torch.zeros((2, 256), dtype=torch.bfloat16, device='cuda')
    q, sf = dg.swiglu_per_token_cast_to_fp8(zero)
    assert (q.float() == 0).all() and torch.equal(sf, torch.full((2, 1), 1e-4, device='cuda') / torch.full((2, 1), 448.0, device='cuda'))


def test_gradient_against_differences(dg):
    """Central differences of the FP64 formula around the same BF16 inputs, step 2^-10: the third derivative of silu is below 1/2, so the
    quotient is within 2^-22 |u dy| of the derivative; the kernel's own rounding adds 2^-8."""
    x, dy = case(4, 24, 0, seed=5, scale=1.0)
    got = dg.swiglu_backward(dy, x).double()
    h = 2.0 ** -10
    for col in (0, 11, 23, 24, 40, 47):
        step = torch.zeros(48, dtype=torch.float64, device='cuda')
        step[col] = h

        def f(v):
            return (v[:, :24] * torch.sigmoid(v[:, :24]) * v[:, 24:] * dy.double()).sum(dim=1)

        quotient = (f(x.double() + step) - f(x.double() - step)) / (2 * h)
        bound = (x[:, col % 24 + 24].double() * dy[:, col % 24].double()).abs() * 2.0 ** -19 + 2.0 ** -30
        assert ((got[:, col] - quotient).abs() <= quotient.abs() * 2.0 ** -8 * 1.01 + bound).all()


def test_graph_and_side_stream(dg):
    x, dy = case(300, 256, 0, seed=6)
    want = dg.swiglu_backward(dy, x), dg.swiglu(x), *dg.swiglu_per_token_cast_to_fp8(x)
    static, graph = torch.zeros_like(x), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = dg.swiglu_backward(dy, static), dg.swiglu(static), *dg.swiglu_per_token_cast_to_fp8(static)
    static.copy_(x)
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = dg.swiglu_backward(dy, x), dg.swiglu(x), *dg.swiglu_per_token_cast_to_fp8(x)
    torch.cuda.synchronize()
    for a, b, c in zip(got, want, beside):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and torch.equal(c.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize('rows, inter', [(3, 520), (300, 2048)])
def test_fp8_arithmetic_is_that_of_fp32_operations(dg, rows, inter):
    """The scales and codes are those of the formula in single FP32 operations. The kernel's reciprocal comes from one Newton step on one
    that is at most 2^-22 off: 2^-44 and a rounding, another value than the division's for one in 2^20 (none or one of the values here). That
    reaches one scale, and the codes of its block only where a quotient lies at a tie."""
    x, _ = case(rows, inter, 0, seed=9)
    gate, up = x[:, :inter].float(), x[:, inter:].float()
    y = gate * (1.0 / (1.0 + torch.exp(-gate))) * up
    blocks = -(-inter // 128)
    amax = torch.nn.functional.pad(y, (0, blocks * 128 - inter)).view(rows, blocks, 128).abs().amax(dim=-1)
    scale = amax.clamp(min=1e-4) / torch.full_like(amax, 448.0)
    codes = (y / scale.repeat_interleave(128, dim=1)[:, :inter]).to(torch.float8_e4m3fn)
    q, sf = dg.swiglu_per_token_cast_to_fp8(x)
    assert (sf != scale).sum() <= 1 and (q.view(torch.uint8) != codes.view(torch.uint8)).sum() <= 1
