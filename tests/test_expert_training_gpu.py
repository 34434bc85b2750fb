"""The operators together, as a training step of the experts uses them: plan, permutation, FP8 products, SwiGLU, the weighted sum back, and
the whole backward pass with the weight gradients of the K-grouped GEMM, against FP64 on the same quantised operands."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def wide(q, sf, block_rows):
    full = sf.double().repeat_interleave(128, dim=-1)[..., :q.shape[-1]]
    return q.double() * (full.repeat_interleave(128, dim=-2)[..., :q.shape[-2], :] if block_rows == 128 else full)


def near(got, want, steps):
    """Within `steps` half steps of BF16 of each value, or of the root mean square where values cancel."""
    got, want = got.double(), want.double()
    scale = want.abs() + want.square().mean().sqrt()
    assert ((got - want).abs() <= scale * steps * 2.0 ** -8).all(), float(((got - want).abs() / scale).max()) * 2 ** 8


def test_forward_and_backward():
    import deepgemm_b200 as dg
    from deepgemm_b200 import _lib
    tokens, topk, experts, hidden, inter = 777, 4, 6, 512, 384
    g = torch.Generator(device='cuda').manual_seed(1)
    randn = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device='cuda') * scale).bfloat16()
    x, dy = randn(tokens, hidden), randn(tokens, hidden, scale=0.1)
    w1, w2 = randn(experts, 2 * inter, hidden, scale=0.05), randn(experts, hidden, inter, scale=0.05)
    logits = torch.randn(tokens, experts, generator=g, device='cuda')
    idx, weights = dg.route_sigmoid_topk(logits, topk)
    idx[::7, 2] = -1  # an entry that another rank computes
    w1_q, w2_q = (dg.utils.per_block_cast_to_fp8(w, use_ue8m0=False) for w in (w1, w2))

    # forward
    plan = dg.moe_dispatch_plan(idx, experts)
    layout, m = plan.expert_end, plan.capacity
    x_q = dg.moe_permute(dg.utils.per_token_cast_to_fp8(x, use_ue8m0=False), plan)
    gate_up = torch.zeros(m, 2 * inter, dtype=torch.bfloat16, device='cuda')
    dg.m_grouped_fp8_gemm_nt_contiguous(x_q, w1_q, gate_up, layout, disable_ue8m0_cast=True, use_psum_layout=True)
    act_q = dg.swiglu_per_token_cast_to_fp8(gate_up, grouped_layout=layout)
    out = torch.zeros(m, hidden, dtype=torch.bfloat16, device='cuda')
    dg.m_grouped_fp8_gemm_nt_contiguous(act_q, w2_q, out, layout, disable_ue8m0_cast=True, use_psum_layout=True)
    y = dg.moe_unpermute(out, plan, weights)
    # backward
    d_out, d_weights = dg.moe_unpermute_backward(dy, out, plan, weights)
    d_out_q = dg.utils.per_token_cast_to_fp8(d_out, use_ue8m0=False)
    d_act = torch.zeros(m, inter, dtype=torch.bfloat16, device='cuda')
    dg.m_grouped_fp8_gemm_nn_contiguous(d_out_q, w2_q, d_act, layout, disable_ue8m0_cast=True, use_psum_layout=True)
    d_gate_up = dg.swiglu_backward(d_act, gate_up, grouped_layout=layout)
    d_gate_up_q = dg.utils.per_token_cast_to_fp8(d_gate_up, use_ue8m0=False)
    d_rows = torch.zeros(m, hidden, dtype=torch.bfloat16, device='cuda')
    dg.m_grouped_fp8_gemm_nn_contiguous(d_gate_up_q, w1_q, d_rows, layout, disable_ue8m0_cast=True, use_psum_layout=True)
    dx = dg.moe_permute_backward(d_rows, plan)
    # weight gradients: the BF16 K-grouped GEMM over the permuted rows, whose padding rows the operators have left zero
    total = -(-int(layout[-1]) // 128) * 128
    x_rows, act = dg.moe_permute(x, plan), dg.swiglu(gate_up, grouped_layout=layout)
    dw1 = torch.zeros(experts, 2 * inter, hidden, device='cuda')
    dw2 = torch.zeros(experts, hidden, inter, device='cuda')
    dg.k_grouped_bf16_gemm_tn_contiguous(d_gate_up[:total], x_rows[:total], dw1, None, layout, dw1, use_psum_layout=True)
    dg.k_grouped_bf16_gemm_tn_contiguous(d_out[:total], act[:total], dw2, None, layout, dw2, use_psum_layout=True)
    assert _lib.device_status()[0] == 0

    # the same step in FP64 from the same quantised operands, stage by stage
    want_y = torch.zeros(tokens, hidden, dtype=torch.float64, device='cuda')
    want_dx, want_dw = torch.zeros_like(want_y), torch.zeros(tokens, topk, dtype=torch.float64, device='cuda')
    w1_w, w2_w = wide(*w1_q, 128), wide(*w2_q, 128)
    for e in range(experts):
        s, t = int(plan.expert_start[e]), int(plan.expert_end[e])
        if s == t:
            continue
        tok, slot = torch.nonzero(idx == e, as_tuple=True)
        rows = plan.dest_row[tok, slot].long()
        assert sorted(rows.tolist()) == list(range(s, t))
        gu = wide(x_q[0][rows], x_q[1][rows], 1) @ w1_w[e].T
        near(gate_up[rows], gu, 1.1)
        a = torch.sigmoid(gate_up[rows, :inter].double()) * gate_up[rows, :inter].double() * gate_up[rows, inter:].double()
        near(act[rows], a, 1.1)
        assert ((wide(act_q[0][rows], act_q[1][rows], 1) - a).abs() <= a.abs() * 2.0 ** -3.99 + act_q[1][rows].double().max() * 2.0 ** -9).all()
        o = wide(act_q[0][rows], act_q[1][rows], 1) @ w2_w[e].T
        near(out[rows], o, 1.1)
        w = weights[tok, slot].double()[:, None]
        want_y.index_add_(0, tok, w * out[rows].double())
        want_dw[tok, slot] = (out[rows].double() * dy[tok].double()).sum(dim=1)
        near(d_out[rows], w * dy[tok].double(), 1.1)
        near(d_act[rows], wide(d_out_q[0][rows], d_out_q[1][rows], 1) @ w2_w[e], 1.1)
        near(d_rows[rows], wide(d_gate_up_q[0][rows], d_gate_up_q[1][rows], 1) @ w1_w[e], 1.1)
        want_dx.index_add_(0, tok, d_rows[rows].double())
        near(dw1[e], d_gate_up[rows].double().T @ x[tok].double(), 0.1)
        near(dw2[e], d_out[rows].double().T @ act[rows].double(), 0.1)
    near(y, want_y, 1.1)
    near(dx, want_dx, 1.1)
    assert torch.allclose(d_weights.double(), want_dw, rtol=1e-4, atol=1e-4 * float(want_dw.abs().max()))
    assert torch.isfinite(dw1).all() and torch.isfinite(dw2).all()
