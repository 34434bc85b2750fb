"""Tokens sorted by expert and back, with gradients, against plain loops on the CPU and against differences.

Tolerances: a copy is exact; a sum of topk products in FP32 is off by at most topk half steps (2^-24) of the sum of magnitudes per operation, two
operations a term, then rounded once to its type (bf16 half step 2^-8); a dot product over H has H additions instead."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def dg():
    import deepgemm_b200
    yield deepgemm_b200
    from deepgemm_b200 import _lib
    assert _lib.device_status()[0] == 0


def plan_on_cpu(idx, experts, alignment):
    tokens, topk = idx.shape
    dest, counts = torch.full((tokens, topk), -1, dtype=torch.int32), [0] * experts
    for row in idx.tolist():
        for e in row:
            if 0 <= e < experts:
                counts[e] += 1
    start, at = [], 0
    for c in counts:
        start.append(at)
        at += -(-c // alignment) * alignment
    after = list(start)
    for t, row in enumerate(idx.tolist()):
        for k, e in enumerate(row):
            if 0 <= e < experts:
                dest[t, k] = after[e]
                after[e] += 1
    return dest, torch.tensor(start, dtype=torch.int32), torch.tensor(after, dtype=torch.int32), at


def routing(tokens, topk, experts, seed, kind='spread'):
    g = torch.Generator().manual_seed(seed)
    if kind == 'one expert':
        return torch.full((tokens, topk), experts - 1)
    if kind == 'all masked':
        return torch.full((tokens, topk), -1)
    idx = torch.randint(0, experts, (tokens, topk), generator=g)  # the same expert twice for a token happens
    if kind == 'masked':
        idx[torch.rand(tokens, topk, generator=g) < 0.4] = -1
        idx[torch.rand(tokens, topk, generator=g) < 0.1] = experts + 3
        idx[torch.rand(tokens, topk, generator=g) < 0.1] = -2 ** 40
    return idx


PLANS = [(0, 2, 4, 128, 'spread'), (1, 1, 1, 1, 'spread'), (1, 8, 256, 16, 'spread'), (13, 8, 256, 128, 'masked'), (100, 3, 7, 5, 'spread'),
         (128, 32, 60, 8, 'masked'), (513, 8, 1024, 4, 'spread'), (700, 6, 33, 128, 'one expert'), (700, 6, 33, 16, 'all masked'),
         (4099, 8, 256, 128, 'masked'), (20000, 8, 128, 128, 'spread'), (70000, 2, 1000, 8, 'masked')]


@pytest.mark.parametrize('tokens, topk, experts, alignment, kind', PLANS)
def test_plan(dg, tokens, topk, experts, alignment, kind):
    idx = routing(tokens, topk, experts, seed=1, kind=kind)
    plan = dg.moe_dispatch_plan(idx.cuda(), experts, alignment=alignment)
    dest, start, end, rows = plan_on_cpu(idx, experts, alignment)
    assert torch.equal(plan.dest_row.cpu(), dest)
    assert torch.equal(plan.expert_start.cpu(), start) and torch.equal(plan.expert_end.cpu(), end)
    assert rows <= plan.capacity and plan.num_experts == experts and plan.alignment == alignment


def rows_case(shape, dtype, seed, pad=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    t = torch.randn(shape[0], shape[1] + pad, generator=g, device='cuda').to(dtype)
    return t[:, :shape[1]]


SIZES = [(1, 1, 3, 1), (1, 8, 16, 7168), (5, 2, 4, 33), (37, 8, 60, 264), (300, 4, 8, 1030), (600, 8, 32, 512), (9, 11, 40, 100), (3, 32, 8, 4104)]


@pytest.mark.parametrize('tokens, topk, experts, hidden', SIZES)
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('pad', [0, 3, 8])
def test_permute_and_gradient(dg, tokens, topk, experts, hidden, dtype, pad):
    idx = routing(tokens, topk, experts, seed=2, kind='masked')
    plan = dg.moe_dispatch_plan(idx.cuda(), experts, alignment=16)
    dest, start, end, _ = plan_on_cpu(idx, experts, 16)
    x = rows_case((tokens, hidden), dtype, 3, pad)
    for zero_padding in (True, False):
        out = rows_case((plan.capacity + 5, hidden), dtype, 4, pad).fill_(7.5)
        rows = dg.moe_permute(x, plan, out=out, zero_padding=zero_padding)
        want = torch.full((plan.capacity + 5, hidden), 7.5, dtype=dtype)
        if zero_padding:
            for e in range(experts):
                want[end[e]:-(-int(end[e]) // 16) * 16] = 0
        for k in range(topk):
            there = dest[:, k] >= 0
            want[dest[there, k].long()] = x.cpu()[there]
        assert rows is out and torch.equal(rows.cpu(), want)
    d_rows = rows_case((plan.capacity, hidden), dtype, 5, pad)
    got = dg.moe_permute_backward(d_rows, plan)
    picked = torch.where((dest >= 0)[..., None], d_rows.cpu().double()[dest.clamp(min=0).long()], torch.zeros((), dtype=torch.float64))
    check_sum(got, picked, dtype, topk)


def check_sum(got, terms, dtype, topk, operations=2):
    want, magnitude = terms.sum(dim=1), terms.abs().sum(dim=1)
    tol = magnitude * operations * topk * 2.0 ** -24 + want.abs() * (2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8)
    assert ((got.cpu().double() - want).abs() <= tol * 1.01).all()


@pytest.mark.parametrize('tokens, topk, experts, hidden', SIZES)
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('pad', [0, 3])
@pytest.mark.parametrize('weighted', [True, False])
def test_unpermute_and_gradients(dg, tokens, topk, experts, hidden, dtype, pad, weighted):
    idx = routing(tokens, topk, experts, seed=6, kind='masked')
    plan = dg.moe_dispatch_plan(idx.cuda(), experts, alignment=8)
    dest, start, end, _ = plan_on_cpu(idx, experts, 8)
    rows = rows_case((plan.capacity + 2, hidden), dtype, 7, pad)
    used = torch.zeros(rows.shape[0], dtype=torch.bool)
    used[dest[dest >= 0].long()] = True
    rows[~used.cuda()] = float('nan')  # rows of no entry are never read
    weights = torch.rand(tokens, topk, device='cuda')
    weights[(dest < 0).cuda()] = float('inf')  # nor are the weights of masked entries
    w = weights.cpu().double() if weighted else torch.ones(tokens, topk, dtype=torch.float64)
    given = weights if weighted else None
    masked = (dest < 0)[..., None]
    picked = torch.where(masked, torch.zeros((), dtype=torch.float64), rows.cpu().double()[dest.clamp(min=0).long()])
    w = torch.where(masked[..., 0], torch.zeros((), dtype=torch.float64), w)
    y = dg.moe_unpermute(rows, plan, given)
    assert y.shape == (tokens, hidden) and y.dtype == dtype
    check_sum(y, picked * w[..., None], dtype, topk)

    dy = rows_case((tokens, hidden), dtype, 8, pad)
    out = rows_case((plan.capacity + 2, hidden), dtype, 9, pad).fill_(-3.0)
    d_rows, d_weights = dg.moe_unpermute_backward(dy, rows, plan, given, out=out)
    half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    want = torch.full((plan.capacity + 2, hidden), -3.0, dtype=torch.float64)
    for e in range(experts):
        want[end[e]:-(-int(end[e]) // 8) * 8] = 0
    for k in range(topk):
        there = dest[:, k] >= 0
        want[dest[there, k].long()] = w[there, k:k + 1] * dy.cpu().double()[there]
    assert d_rows is out and ((out.cpu().double() - want).abs() <= want.abs() * (half + 2.0 ** -24)).all()
    terms = picked * dy.cpu().double()[:, None, :]
    tol = terms.abs().sum(dim=-1) * (hidden + 1) * 2.0 ** -24 * 1.01
    assert ((d_weights.cpu().double() - terms.sum(dim=-1)).abs() <= tol).all()
    assert (d_weights.cpu()[dest < 0] == 0).all()


def test_gradients_against_differences(dg):
    """Central differences of <y, dy> in the weights and in x (float32 rows; the map is linear in each, so the difference quotient is the
    gradient but for rounding: 2^-24 of each of the sums' magnitudes over the step)."""
    tokens, topk, experts, hidden = 6, 3, 5, 40
    idx = routing(tokens, topk, experts, seed=10, kind='masked').cuda()
    plan = dg.moe_dispatch_plan(idx, experts, alignment=8)
    x, dy, w = (torch.randn(tokens, n, device='cuda') for n in (hidden, hidden, topk))

    def forward(x, w):
        return (dg.moe_unpermute(dg.moe_permute(x, plan), plan, w).double() * dy.double()).sum()

    rows = dg.moe_permute(x, plan)
    d_rows, d_w = dg.moe_unpermute_backward(dy, rows, plan, w)
    dx = dg.moe_permute_backward(d_rows, plan)
    tol = 2 * (x.abs().max() * w.abs().max() * dy.abs().max()).item() * tokens * hidden * topk * 2.0 ** -22
    for t, grad, which in ((w, d_w, 1), (x, dx, 0)):
        for at in ((0, 0), (2, 1), (5, 2), (3, 0)):
            step = torch.zeros_like(t)
            step[at] = 1.0
            plus, minus = (forward(*((x, t + s * step) if which else (t + s * step, w))) for s in (1, -1))
            assert abs(float((plus - minus) / 2) - float(grad[at])) <= tol


@pytest.mark.parametrize('tokens, hidden, blocks', [(1, 128, 1), (40, 640, 5), (333, 1000, 8), (20, 17, 1)])
def test_permute_fp8_rows_with_their_scales(dg, tokens, hidden, blocks):
    topk, experts = 4, 9
    idx = routing(tokens, topk, experts, seed=12, kind='masked')
    plan = dg.moe_dispatch_plan(idx.cuda(), experts, alignment=128)
    dest, start, end, rows = plan_on_cpu(idx, experts, 128)
    codes = torch.randint(0, 256, (tokens, hidden), dtype=torch.uint8, device='cuda')
    sf = torch.rand(tokens, blocks, device='cuda')
    q, s = dg.moe_permute((codes.view(torch.float8_e4m3fn), sf), plan)
    assert q.shape == (plan.capacity, hidden) and s.shape == (plan.capacity, blocks)
    want_q, want_s = torch.zeros(rows, hidden, dtype=torch.uint8), torch.zeros(rows, blocks)
    for k in range(topk):
        there = dest[:, k] >= 0
        want_q[dest[there, k].long()] = codes.cpu()[there]
        want_s[dest[there, k].long()] = sf.cpu()[there]
    assert torch.equal(q.view(torch.uint8)[:rows].cpu(), want_q) and torch.equal(s[:rows].cpu(), want_s)


def test_no_tokens(dg):
    plan = dg.moe_dispatch_plan(torch.empty((0, 4), dtype=torch.int64, device='cuda'), 6)
    assert plan.capacity == 0 and (plan.expert_end == 0).all()
    x = torch.empty((0, 64), dtype=torch.bfloat16, device='cuda')
    rows = dg.moe_permute(x, plan)
    assert rows.shape == (0, 64)
    assert dg.moe_unpermute(rows, plan).shape == (0, 64)
    d_rows, d_w = dg.moe_unpermute_backward(x, rows, plan)
    assert d_rows.shape == (0, 64) and d_w.shape == (0, 4)


def test_a_plan_that_names_rows_past_the_buffer_is_reported(dg):
    from deepgemm_b200 import _lib
    dest = torch.tensor([[0, 1000]], dtype=torch.int32, device='cuda')
    zero = torch.zeros(2, dtype=torch.int32, device='cuda')
    plan = dg.MoeDispatchPlan(dest, zero, zero + 1, 1)
    x = torch.ones((1, 64), dtype=torch.bfloat16, device='cuda')
    guard = torch.full((4096, 64), 2.0, dtype=torch.bfloat16, device='cuda')
    dg.moe_permute(x, plan, out=guard[:plan.capacity])
    with pytest.raises(RuntimeError, match='code 6'):
        _lib.device_status()
    assert (guard[0] == 1).all() and (guard[1:] == 2).all()
    assert torch.equal(dg.moe_unpermute(guard[:plan.capacity], plan), x)
    with pytest.raises(RuntimeError, match='code 6'):
        _lib.device_status()


def test_graphs_and_side_streams(dg):
    """The whole round trip captured and replayed with new routing, beside an eager run on another stream."""
    tokens, topk, experts, hidden = 3000, 4, 16, 256
    idx = [routing(tokens, topk, experts, seed=20 + i, kind='masked').cuda() for i in range(2)]
    x, dy = (rows_case((tokens, hidden), torch.bfloat16, 30 + i) for i in range(2))
    w = torch.rand(tokens, topk, device='cuda')

    def step(idx):
        plan = dg.moe_dispatch_plan(idx, experts, alignment=16)
        rows = dg.moe_permute(x, plan)
        d_rows, d_w = dg.moe_unpermute_backward(dy, rows, plan, w)
        return dg.moe_unpermute(rows, plan, w), d_w, dg.moe_permute_backward(d_rows, plan)

    want = [[t.clone() for t in step(i)] for i in idx]
    static, graph = idx[0].clone(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = step(static)
    side = torch.cuda.Stream()
    for i in (1, 0, 1):
        static.copy_(idx[i])
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = step(idx[1 - i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
        assert all(torch.equal(a, b) for a, b in zip(beside, want[1 - i]))
