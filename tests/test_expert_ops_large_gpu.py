"""The operators around the experts' GEMMs where offsets pass 32 bits, with the sort's most chunks, and as one captured chain.

Large results are compared with the same operator on a part of the rows, bit for bit (a row's result does not depend on where the row
lies), or with a gather of torch's."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def dg():
    import deepgemm_b200
    yield deepgemm_b200
    from deepgemm_b200 import _lib
    assert _lib.device_status()[0] == 0


@pytest.fixture(autouse=True)
def give_memory_back():
    yield
    torch.cuda.empty_cache()


def bits(t):
    return t.contiguous().view(torch.uint8)


def quantised(*shape, seed, block_rows):
    g = torch.Generator(device='cuda').manual_seed(seed)
    q = torch.randint(0, 120, shape, generator=g, device='cuda', dtype=torch.uint8).view(torch.float8_e4m3fn)
    rows = -(-shape[-2] // block_rows)
    sf = torch.rand(*shape[:-2], rows, -(-shape[-1] // 128), generator=g, device='cuda') + 0.5
    return q, sf


def test_the_plan_of_many_entries(dg):
    """More entries than 128 chunks of 4096."""
    tokens, topk, experts, alignment = 90001, 8, 384, 128
    g = torch.Generator(device='cuda').manual_seed(1)
    idx = torch.randint(-1, experts, (tokens, topk), generator=g, device='cuda')
    plan = dg.moe_dispatch_plan(idx, experts, alignment=alignment)
    flat = idx.flatten()
    order = torch.argsort(torch.where(flat < 0, experts, flat), stable=True)
    counts = torch.bincount(flat[flat >= 0], minlength=experts)
    padded = (counts + alignment - 1) // alignment * alignment
    start = padded.cumsum(0) - padded
    first = counts.cumsum(0) - counts
    want = torch.full((tokens * topk,), -1, dtype=torch.int64, device='cuda')
    kept = order[:int(counts.sum())]
    of = flat[kept]
    want[kept] = start[of] + torch.arange(kept.numel(), device='cuda') - first[of]
    assert torch.equal(plan.dest_row.flatten().long(), want)
    assert torch.equal(plan.expert_start.long(), start) and torch.equal(plan.expert_end.long(), start + counts)


def test_rows_past_four_gigabytes(dg):
    tokens, topk, experts, hidden = 40000, 8, 64, 7168  # 320000 rows of 14 KB
    g = torch.Generator(device='cuda').manual_seed(2)
    idx = torch.rand(tokens, experts, generator=g, device='cuda').topk(topk, dim=1).indices
    x = torch.randn(tokens, hidden, generator=g, device='cuda').bfloat16()
    w = torch.rand(tokens, topk, generator=g, device='cuda')
    plan = dg.moe_dispatch_plan(idx, experts, alignment=16)
    rows = dg.moe_permute(x, plan)
    assert rows.numel() > 2 ** 31
    for k in range(topk):
        assert torch.equal(rows[plan.dest_row[:, k].long()], x)
    y = dg.moe_unpermute(rows, plan, None)
    assert torch.equal(y, (x.float() * topk).bfloat16())  # the sum of eight equal values is exact
    d_rows, d_w = dg.moe_unpermute_backward(x, rows, plan, w)
    for k in (0, topk - 1):
        assert torch.equal(d_rows[plan.dest_row[:, k].long()], (w[:, k:k + 1] * x.float()).bfloat16())
    norm = torch.stack([x[i:i + 4000].double().square().sum(dim=1) for i in range(0, tokens, 4000)]).flatten()
    assert ((d_w.double() - norm[:, None]).abs() <= norm[:, None] * hidden * 2.0 ** -24).all()


def test_swiglu_past_four_gigabytes(dg):
    rows, inter = 300000, 4096
    x = torch.empty(rows, 2 * inter, dtype=torch.bfloat16, device='cuda')
    g = torch.Generator(device='cuda').manual_seed(3)
    part = torch.randn(1000, 2 * inter, generator=g, device='cuda').bfloat16()
    for at in (0, 150000, rows - 1000):
        x[at:at + 1000] = part
    dy = torch.empty(rows, inter, dtype=torch.bfloat16, device='cuda')
    dy[-1000:] = part[:, :inter]
    y, (q, sf) = dg.swiglu(x), dg.swiglu_per_token_cast_to_fp8(x)
    want, (want_q, want_sf) = dg.swiglu(part), dg.swiglu_per_token_cast_to_fp8(part)
    for at in (0, 150000, rows - 1000):
        assert torch.equal(y[at:at + 1000], want)
        assert torch.equal(bits(q[at:at + 1000]), bits(want_q)) and torch.equal(sf[at:at + 1000], want_sf)
    assert torch.equal(dg.swiglu_backward(dy, x)[-1000:], dg.swiglu_backward(part[:, :inter], part))


def test_quantisers_past_four_gigabytes(dg):
    g = torch.Generator(device='cuda').manual_seed(4)
    part = torch.randn(640, 8192, generator=g, device='cuda').bfloat16()
    x = torch.empty(300000, 8192, dtype=torch.bfloat16, device='cuda')
    x[-640:] = part
    for gran_k in (32, 128):
        q, sf = dg.utils.per_token_cast_to_fp8(x, use_ue8m0=False, gran_k=gran_k)
        want_q, want_sf = dg.utils.per_token_cast_to_fp8(part, use_ue8m0=False, gran_k=gran_k)
        assert torch.equal(bits(q[-640:]), bits(want_q)) and torch.equal(sf[-640:], want_sf)
    w = x.flatten()[:80 * 4096 * 7168].view(80, 4096, 7168)
    w[79, -640:] = part[:, :7168]
    q, sf = dg.utils.per_block_cast_to_fp8(w, use_ue8m0=False)
    want_q, want_sf = dg.utils.per_block_cast_to_fp8(part[:, :7168], use_ue8m0=False)
    assert torch.equal(bits(q[79, -640:]), bits(want_q)) and torch.equal(sf[79, -5:], want_sf)


def test_gemm_results_past_four_gigabytes(dg):
    k, n = 144, 8192
    a, b = quantised(300000, k, seed=5, block_rows=1), quantised(n, k, seed=6, block_rows=128)
    d = torch.empty(300000, n, dtype=torch.bfloat16, device='cuda')
    dg.fp8_gemm_nt(a, b, d, disable_ue8m0_cast=True)
    few = torch.empty(500, n, dtype=torch.bfloat16, device='cuda')
    dg.fp8_gemm_nt((a[0][-500:].clone(), a[1][-500:].clone()), b, few, disable_ue8m0_cast=True)
    assert torch.equal(d[-500:], few)
    del d
    groups, max_m = 72, 4096
    a, b = quantised(groups, max_m, k, seed=7, block_rows=1), quantised(groups, n, k, seed=8, block_rows=128)
    d = torch.empty(groups, max_m, n, dtype=torch.bfloat16, device='cuda')
    counts = torch.full((groups,), 100, dtype=torch.int32, device='cuda')
    counts[-1] = max_m
    dg.m_grouped_fp8_gemm_nt_masked(a, b, d, counts, 100, disable_ue8m0_cast=True)
    dg.fp8_gemm_nt((a[0][-1, -500:].clone(), a[1][-1, -500:].clone()), (b[0][-1], b[1][-1]), few, disable_ue8m0_cast=True)
    assert torch.equal(d[-1, -500:], few)


def test_a_chain_in_a_graph_beside_an_eager_one(dg):
    """Quantise, sort, multiply, SwiGLU to FP8, multiply, sum back: captured and replayed on new tokens and routes, beside the same on a
    second stream; the same bits as alone."""
    tokens, topk, experts, hidden, inter = 300, 4, 8, 512, 384
    g = torch.Generator(device='cuda').manual_seed(9)
    w1, w2 = ((torch.randn(experts, *s, generator=g, device='cuda') * 0.05).bfloat16() for s in ((2 * inter, hidden), (hidden, inter)))
    w1, w2 = (dg.utils.per_block_cast_to_fp8(w, use_ue8m0=False) for w in (w1, w2))
    xs = [torch.randn(tokens, hidden, generator=g, device='cuda').bfloat16() for _ in range(2)]
    routes = [torch.randint(-1, experts, (tokens, topk), generator=g, device='cuda') for _ in range(2)]
    weights = torch.rand(tokens, topk, generator=g, device='cuda')

    def step(x, idx):
        plan = dg.moe_dispatch_plan(idx, experts)
        rows = dg.moe_permute(dg.utils.per_token_cast_to_fp8(x, use_ue8m0=False), plan)
        gate_up = x.new_empty((plan.capacity, 2 * inter))
        dg.m_grouped_fp8_gemm_nt_contiguous(rows, w1, gate_up, plan.expert_end, disable_ue8m0_cast=True, use_psum_layout=True)
        act = dg.swiglu_per_token_cast_to_fp8(gate_up, grouped_layout=plan.expert_end, activation_clamp=7.0)
        out = x.new_empty((plan.capacity, hidden))
        dg.m_grouped_fp8_gemm_nt_contiguous(act, w2, out, plan.expert_end, disable_ue8m0_cast=True, use_psum_layout=True)
        return dg.moe_unpermute(out, plan, weights)

    want = [step(x, r).clone() for x, r in zip(xs, routes)]
    assert all(torch.isfinite(y).all() and (y != 0).any() for y in want)
    x, idx, graph, side = xs[0].clone(), routes[0].clone(), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = step(x, idx)
    for i in (1, 0, 1):
        x.copy_(xs[i])
        idx.copy_(routes[i])
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            beside = step(xs[1 - i], routes[1 - i])
        torch.cuda.synchronize()
        assert torch.equal(y, want[i]) and torch.equal(beside, want[1 - i])
