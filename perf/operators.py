"""Cases that time and check the operators around FP8 experts whose scales are FP32 numbers, one for each block of 128: the
matrix products, the quantisers of their operands, the sort of tokens by expert with its way back and its gradients, and SwiGLU
of the experts' rows with its gradient.

``run`` computes an operator either from elementary torch operations in FP32 (``own`` false) or through the framework's public
entry points (``own`` true); ``exact`` computes it in FP64, written apart from both."""
import torch

own = False

E4M3_MAX = 448.0


# ------------------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # A handful of tokens against a dense layer's gate and up projection: bound by the weights, and by the launch.
        dict(name='gemm_dense_7', kind='dense', m=7, n=4096, k=7168, f32=False),
        # A ragged chunk of a prefill against a projection whose width is no multiple of 128, added to an FP32 accumulator.
        dict(name='gemm_dense_1999_acc', kind='dense', m=1999, n=2112, k=7168, f32=True),
        # Prefill through 32 experts of a rank: gate and up products, uneven groups, free rows at the buffer's end.
        dict(name='gemm_grouped_32', kind='grouped', groups=32, rows=7900, n=4096, k=7168, nn=False, psum=True),
        # The gradient of the experts' inputs: the weights as they are stored, their rows summed over.
        dict(name='gemm_grouped_nn_8', kind='grouped', groups=8, rows=7200, n=7168, k=4096, nn=True, psum=True),
        # Decode: a fixed buffer for each expert, a few valid rows in it; the down products.
        dict(name='gemm_masked_32', kind='masked', groups=32, max_m=128, mean=24, n=7168, k=2048),
        # A decode step's tokens to 256 experts.
        dict(name='permute_13', kind='permute', tokens=13, hidden=7168, topk=8, experts=256, alignment=16, masked=0.0, fp8=False, grad=False),
        # A training step's tokens to their experts and their gradients back; an expert-parallel rank masks what others compute.
        dict(name='permute_grad_4099', kind='permute', tokens=4099, hidden=7168, topk=8, experts=256, alignment=128, masked=0.1,
             fp8=False, grad=True),
        # The experts' rows back to the tokens with the routing weights, and the gradients of both.
        dict(name='unpermute_grad_8192', kind='unpermute', tokens=8192, hidden=4096, topk=8, experts=64, alignment=128, masked=0.0, grad=True),
        # Between the two FP8 products of a prefill chunk.
        dict(name='swiglu_fp8_5000', kind='swiglu', rows=5000, groups=32, inter=2048, clamp=0.0, fp8=True, grad=False),
        # A training step: activations and their gradients.
        dict(name='swiglu_grad_32768', kind='swiglu', rows=32768, groups=64, inter=2048, clamp=10.0, fp8=False, grad=True),
        # One decode step's tokens, quantised.
        dict(name='cast_tokens_31', kind='cast', rows=31, k=7168, groups=0, block=False),
        # The weights of a rank's experts, quantised once a training step.
        dict(name='cast_weights_32', kind='cast', rows=4096, k=7168, groups=32, block=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(['dense', 'dense', 'grouped', 'grouped', 'masked', 'permute', 'permute', 'unpermute', 'unpermute', 'swiglu',
                       'swiglu', 'cast', 'cast'])
    if kind == 'dense':
        n, k = 8 * _log_int(rng, 8, 1024), 16 * _log_int(rng, 6, 448)
        m = _log_int(rng, 1, max(1, min(8192, int(2.2e11 / (n * k)))))
        return dict(kind=kind, m=m, n=n, k=k, f32=rng.random() < 0.4)
    if kind == 'grouped':
        groups = rng.choice([1, 3, 8, 16, 32])
        n, k = 16 * _log_int(rng, 8, 448), 16 * _log_int(rng, 8, 448)
        rows = _log_int(rng, 1, max(1, min(32768, int(2.2e11 / (n * k)))))
        return dict(kind=kind, groups=groups, rows=rows, n=n, k=k, nn=rng.random() < 0.4, psum=rng.random() < 0.6)
    if kind == 'masked':
        max_m = 4 * _log_int(rng, 4, 64)
        return dict(kind=kind, groups=_log_int(rng, 2, 32), max_m=max_m, mean=_log_int(rng, 1, max_m), n=8 * _log_int(rng, 16, 896),
                    k=16 * _log_int(rng, 16, 256))
    if kind in ('permute', 'unpermute'):
        hidden = rng.choice([128 * _log_int(rng, 4, 56), 8 * _log_int(rng, 16, 900), _log_int(rng, 33, 5000)])
        topk = rng.choice([1, 2, 4, 6, 8])
        tokens = _log_int(rng, 1, max(1, min(16384, int(2.3e8 / (hidden * topk)))))
        case = dict(kind=kind, tokens=tokens, hidden=hidden, topk=topk, experts=rng.choice([8, 32, 60, 128, 256]),
                    alignment=rng.choice([8, 16, 128]) if tokens > 256 else 8, masked=rng.choice([0.0, 0.0, 0.3]), grad=rng.random() < 0.5)
        if kind == 'permute':
            case['fp8'] = hidden % 128 == 0 and not case['grad'] and rng.random() < 0.5
        return case
    if kind == 'swiglu':
        grad = rng.random() < 0.5
        inter = 128 * _log_int(rng, 2, 32) if rng.random() < 0.5 else 16 * _log_int(rng, 16, 256)
        return dict(kind=kind, rows=_log_int(rng, 1, max(1, int(6.0e7 / inter))), groups=rng.choice([0, 4, 32, 64]), inter=inter,
                    clamp=rng.choice([0.0, 2.0, 10.0]), fp8=not grad and rng.random() < 0.7, grad=grad)
    block = rng.random() < 0.4
    k = 16 * _log_int(rng, 8, 448)
    groups = rng.choice([0, 2, 8]) if block else 0
    return dict(kind='cast', rows=_log_int(rng, 1, max(1, min(16384, int(4.0e8 / (k * max(groups, 1)))))), k=k, groups=groups, block=block)


# ------------------------------------------------------------------------------------------------------------ the inputs

def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _randn(gen, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen, device='cuda') * scale).bfloat16()


def _tokens(gen, rows, width):
    """Activations as they come out of a norm: most channels near one, a few an order of magnitude larger."""
    channel = 1.0 + 12.0 * (torch.rand(width, generator=gen, device='cuda') > 0.997).float()
    return (torch.randn(rows, width, generator=gen, device='cuda') * channel).bfloat16()


def _pad_last(x, multiple):
    pad = -x.shape[-1] % multiple
    return torch.nn.functional.pad(x, (0, pad)) if pad else x


def _scale(amax):
    """FP32 scale of a block, correctly rounded (a tensor divided by a number is a product with its rounded inverse)."""
    amax = amax.clamp(min=1e-4)
    return amax / torch.full_like(amax, E4M3_MAX)


def _cast_tokens(x):
    blocks = _pad_last(x.float(), 128).unflatten(-1, (-1, 128))
    sf = _scale(blocks.abs().amax(dim=-1))
    q = (blocks / sf.unsqueeze(-1)).flatten(-2)[..., :x.shape[-1]]
    return q.to(torch.float8_e4m3fn), sf


def _cast_blocks(x):
    n, k = x.shape[-2:]
    padded = torch.nn.functional.pad(x.float(), (0, -k % 128, 0, -n % 128))
    blocks = padded.unflatten(-1, (-1, 128)).unflatten(-3, (-1, 128))  # [..., N / 128, 128, K / 128, 128]
    sf = _scale(blocks.abs().amax(dim=(-3, -1)))
    q = (blocks / sf[..., :, None, :, None]).flatten(-2).flatten(-3, -2)[..., :n, :k]
    return q.to(torch.float8_e4m3fn).contiguous(), sf


def _weights(gen, groups, n, k):
    """[groups, n, k] weights in FP8 with a scale for each 128 x 128 block, a few groups at a time."""
    q = torch.empty((groups, n, k), dtype=torch.float8_e4m3fn, device='cuda')
    sf = torch.empty((groups, -(-n // 128), -(-k // 128)), device='cuda')
    for g in range(groups):
        q[g], sf[g] = _cast_blocks(_randn(gen, n, k, scale=0.02))
    return q, sf


def _group_rows(gen, groups, rows):
    """`rows` rows dealt out to the groups unevenly: with few rows some groups have none. Returns the rows of each, their ends
    (groups begin at multiples of 128) and the rows of a buffer that holds them whatever the deal."""
    share = torch.rand(groups, generator=gen, device='cuda') ** 2 + 0.1
    ms = (share / share.sum() * rows).int().tolist()
    ms[int(share.argmax())] += rows - sum(ms)
    ends, start = [], 0
    for m in ms:
        ends.append(start + m)
        start += -(-m // 128) * 128
    return ms, ends, -(-(rows + 127 * groups) // 128) * 128


def prepare(case, seed):
    gen = _generator(seed)
    s = dict(case)
    kind = case['kind']
    if kind == 'dense':
        s['a'], s['sfa'] = _cast_tokens(_tokens(gen, case['m'], case['k']))
        q, sf = _weights(gen, 1, case['n'], case['k'])
        s['b'], s['sfb'] = q[0], sf[0]
        s['c'] = torch.randn(case['m'], case['n'], generator=gen, device='cuda') if case['f32'] else None
        s['d'] = torch.zeros((case['m'], case['n']), dtype=torch.float32 if case['f32'] else torch.bfloat16, device='cuda')
    elif kind == 'grouped':
        ms, ends, rows = _group_rows(gen, case['groups'], case['rows'])
        x, ids = _tokens(gen, rows, case['k']), torch.full((rows,), -1, dtype=torch.int32)
        for g, end in enumerate(ends):
            x[end:-(-end // 128) * 128] = 0
            ids[end - ms[g]:end] = g
        s['a'], s['sfa'] = _cast_tokens(x)
        s['psum_ends'] = torch.tensor(ends, dtype=torch.int32, device='cuda')
        s['layout'] = s['psum_ends'] if case['psum'] else ids.cuda()
        if case['nn']:
            s['b'], s['sfb'] = _weights(gen, case['groups'], case['k'], case['n'])
        else:
            s['b'], s['sfb'] = _weights(gen, case['groups'], case['n'], case['k'])
        s['d'] = torch.zeros((rows, case['n']), dtype=torch.bfloat16, device='cuda')
    elif kind == 'masked':
        g, max_m = case['groups'], case['max_m']
        q, sf = _cast_tokens(_tokens(gen, g * max_m, case['k']))
        s['a'], s['sfa'] = q.view(g, max_m, -1), sf.view(g, max_m, -1)
        s['b'], s['sfb'] = _weights(gen, g, case['n'], case['k'])
        s['masked_m'] = torch.poisson(torch.full((g,), float(case['mean']), device='cuda'), generator=gen).clamp(max=max_m).int()
        s['d'] = torch.zeros((g, max_m, case['n']), dtype=torch.bfloat16, device='cuda')
    elif kind in ('permute', 'unpermute'):
        t, h, k, e = case['tokens'], case['hidden'], case['topk'], case['experts']
        scores = torch.rand(t, e, generator=gen, device='cuda') * torch.rand(e, generator=gen, device='cuda').add(0.3)  # some experts are popular
        weights, idx = scores.topk(k, dim=1)
        idx = torch.where(torch.rand(t, k, generator=gen, device='cuda') < case['masked'], torch.full_like(idx, -1), idx)
        s['topk_idx'], s['topk_weights'] = idx, (weights / weights.sum(dim=1, keepdim=True)).contiguous()
        al = case['alignment']
        s['capacity'] = -(-(t * k + min(e, t * k) * (al - 1)) // al) * al
        if kind == 'permute':
            x = _tokens(gen, t, h)
            s['x'] = _cast_tokens(x) if case['fp8'] else x
            s['out'] = torch.zeros((s['capacity'], h), dtype=torch.float8_e4m3fn if case['fp8'] else torch.bfloat16, device='cuda')
            s['out_sf'] = torch.zeros((s['capacity'], h // 128), device='cuda') if case['fp8'] else None
        if kind == 'unpermute' or case['grad']:
            s['rows'] = _randn(gen, s['capacity'], h)
            s['dy'] = _randn(gen, t, h, scale=0.1)
            s['d_rows'] = torch.zeros((s['capacity'], h), dtype=torch.bfloat16, device='cuda')
        if kind == 'unpermute':  # the plan was made where the rows were sorted, earlier in the step
            s['dest_row'], s['expert_start'], s['expert_end'] = (p.int() for p in _plain_plan(s))
    elif kind == 'swiglu':
        r, inter, g = case['rows'], case['inter'], case['groups']
        if g:
            _, ends, s['buffer_rows'] = _group_rows(gen, g, r)
            s['layout'], s['total'] = torch.tensor(ends, dtype=torch.int32, device='cuda'), -(-ends[-1] // 128) * 128
        else:
            s['layout'], s['buffer_rows'], s['total'], ends = None, r, r, []
        s['gate_up'] = _randn(gen, s['buffer_rows'], 2 * inter, scale=1.5)
        s['dy'] = _randn(gen, s['buffer_rows'], inter, scale=0.1)
        for end in ends:
            s['gate_up'][end:-(-end // 128) * 128] = 0
        s['y'] = torch.zeros((s['buffer_rows'], inter), dtype=torch.float8_e4m3fn if case['fp8'] else torch.bfloat16, device='cuda')
        s['y_sf'] = torch.zeros((s['buffer_rows'], -(-inter // 128)), device='cuda')
        s['d_gate_up'] = torch.zeros_like(s['gate_up'])
    else:
        shape = ((case['groups'],) if case['groups'] else ()) + (case['rows'], case['k'])
        s['x'] = _randn(gen, *shape, scale=0.02) if case['block'] else _tokens(gen, case['rows'], case['k'])
    return s


# ------------------------------------------------------------------------------------------------------- the plain forms

def _wide(q, sf, rows_per_scale):
    """FP8 values times their scales, in FP32: a scale covers `rows_per_scale` x 128 values."""
    n, k = q.shape[-2:]
    sf = sf.repeat_interleave(rows_per_scale, dim=-2)[..., :n, :] if rows_per_scale > 1 else sf
    return q.float() * sf.repeat_interleave(128, dim=-1)[..., :k]


def _plain_grouped(s):
    """Tiles of 128 rows, each against its group's weights: a group's rows begin at a multiple of 128."""
    rows = s['a'].shape[0]
    a = _wide(s['a'], s['sfa'], 1).view(rows // 128, 128, -1)
    b = _wide(s['b'], s['sfb'], 128)
    b = b if s['nn'] else b.transpose(1, 2)
    aligned_ends = (s['psum_ends'] + 127) // 128
    tile_group = torch.searchsorted(aligned_ends, torch.arange(rows // 128, device='cuda', dtype=torch.int32), right=True)
    used = tile_group < s['groups']
    d = torch.bmm(a, b[tile_group.clamp(max=s['groups'] - 1)])
    return torch.where(used[:, None, None], d, torch.zeros((), device='cuda')).bfloat16().view(rows, -1)


def _plain_plan(s):
    t, k, e, al = s['tokens'], s['topk'], s['experts'], s['alignment']
    flat = s['topk_idx'].reshape(-1)
    key = torch.where((flat >= 0) & (flat < e), flat, e)
    counts = torch.zeros(e + 1, dtype=torch.int64, device='cuda').scatter_add_(0, key, torch.ones_like(key))
    padded = (counts + al - 1) // al * al
    start = padded.cumsum(0) - padded
    order = torch.argsort(key, stable=True)
    sorted_key = key[order]
    place = torch.arange(t * k, device='cuda') - (counts.cumsum(0) - counts)[sorted_key] + start[sorted_key]
    dest = torch.empty_like(key)
    dest[order] = torch.where(sorted_key < e, place, -1)
    return dest.view(t, k), start[:e], (start + counts)[:e]


def _gathered(rows, dest):
    """rows[dest] in FP32 with zeros where an entry is masked: [tokens, topk, hidden]."""
    return torch.where((dest >= 0).unsqueeze(-1), rows[dest.clamp(min=0)].float(), torch.zeros((), device='cuda'))


def _scattered(values, dest, capacity):
    """values [tokens, topk, hidden] to rows `dest` of a zeroed buffer; masked entries go to a row behind it."""
    out = torch.zeros((capacity + 1,) + values.shape[2:], dtype=values.dtype, device='cuda')
    out[torch.where(dest < 0, capacity, dest).reshape(-1)] = values.flatten(0, 1)
    return out[:capacity]


def _plain_swiglu(s):
    x = s['gate_up'].float()
    gate, up = x[:, :s['inter']], x[:, s['inter']:]
    if s['clamp'] > 0:
        gate_c, up_c = gate.clamp(max=s['clamp']), up.clamp(-s['clamp'], s['clamp'])
    else:
        gate_c, up_c = gate, up
    sig = 1.0 / (1.0 + torch.exp(-gate_c))
    used = (torch.arange(x.shape[0], device='cuda') < s['total']).unsqueeze(1)
    zero = torch.zeros((), device='cuda')
    act = torch.where(used, gate_c * sig * up_c, zero)
    if s['fp8']:
        q, sf = _cast_tokens(act)
        return {'q': q, 'sf': torch.where(used, sf, zero)}
    out = {'y': act.bfloat16()}
    if s['grad']:
        dy = s['dy'].float()
        d_gate = dy * up_c * sig * (1.0 + gate_c * (1.0 - sig))
        d_up = dy * gate_c * sig
        if s['clamp'] > 0:
            d_gate = torch.where(gate > s['clamp'], zero, d_gate)
            d_up = torch.where(up.abs() > s['clamp'], zero, d_up)
        out['d_gate_up'] = torch.where(used, torch.cat([d_gate, d_up], dim=1), zero).bfloat16()
    return out


def _run_plain(s):
    kind = s['kind']
    if kind == 'dense':
        d = _wide(s['a'], s['sfa'], 1) @ _wide(s['b'], s['sfb'], 128).T
        return {'d': d + s['c'] if s['f32'] else d.bfloat16()}
    if kind == 'grouped':
        return {'d': _plain_grouped(s)}
    if kind == 'masked':
        d = torch.bmm(_wide(s['a'], s['sfa'], 1), _wide(s['b'], s['sfb'], 128).transpose(1, 2))
        valid = torch.arange(s['max_m'], device='cuda') < s['masked_m'].unsqueeze(1)
        return {'d': torch.where(valid.unsqueeze(-1), d, torch.zeros((), device='cuda')).bfloat16()}
    if kind == 'permute':
        dest, _, ends = _plain_plan(s)
        out = {'dest_row': dest.int(), 'expert_end': ends.int()}
        parts = s['x'] if s['fp8'] else (s['x'],)
        for name, x in zip(('rows', 'rows_sf'), parts):
            out[name] = _scattered(x.float().unsqueeze(1).expand(-1, s['topk'], -1), dest, s['capacity']).to(x.dtype)
        if s['grad']:
            out['dx'] = _gathered(s['rows'], dest).sum(dim=1).bfloat16()
        return out
    if kind == 'unpermute':
        dest = s['dest_row'].long()
        picked = _gathered(s['rows'], dest)
        out = {'y': (picked * s['topk_weights'].unsqueeze(-1)).sum(dim=1).bfloat16()}
        if s['grad']:
            dy = s['dy'].float().unsqueeze(1)
            out['d_rows'] = _scattered((dy * s['topk_weights'].unsqueeze(-1)).bfloat16(), dest, s['capacity'])
            out['d_weights'] = (picked * dy).sum(dim=-1)
        return out
    if kind == 'swiglu':
        return _plain_swiglu(s)
    q, sf = (_cast_blocks if s['block'] else _cast_tokens)(s['x'])
    return {'q': q, 'sf': sf}


def _run_own(s):
    import deepgemm_b200 as dg
    kind = s['kind']
    if kind == 'dense':
        dg.fp8_gemm_nt((s['a'], s['sfa']), (s['b'], s['sfb']), s['d'], c=s['c'], disable_ue8m0_cast=True)
        return {'d': s['d']}
    if kind == 'grouped':
        gemm = dg.m_grouped_fp8_gemm_nn_contiguous if s['nn'] else dg.m_grouped_fp8_gemm_nt_contiguous
        gemm((s['a'], s['sfa']), (s['b'], s['sfb']), s['d'], s['layout'], disable_ue8m0_cast=True, use_psum_layout=s['psum'])
        return {'d': s['d']}
    if kind == 'masked':
        dg.m_grouped_fp8_gemm_nt_masked((s['a'], s['sfa']), (s['b'], s['sfb']), s['d'], s['masked_m'], s['mean'], disable_ue8m0_cast=True)
        return {'d': s['d']}
    if kind == 'permute':
        plan = dg.moe_dispatch_plan(s['topk_idx'], s['experts'], alignment=s['alignment'])
        out = {'dest_row': plan.dest_row, 'expert_end': plan.expert_end}
        if s['fp8']:
            out['rows'], out['rows_sf'] = dg.moe_permute(s['x'], plan, out=(s['out'], s['out_sf']))
        else:
            out['rows'] = dg.moe_permute(s['x'], plan, out=s['out'])
        if s['grad']:
            out['dx'] = dg.moe_permute_backward(s['rows'], plan)
        return out
    if kind == 'unpermute':
        plan = dg.MoeDispatchPlan(s['dest_row'], s['expert_start'], s['expert_end'], s['alignment'])
        out = {'y': dg.moe_unpermute(s['rows'], plan, s['topk_weights'])}
        if s['grad']:
            out['d_rows'], out['d_weights'] = dg.moe_unpermute_backward(s['dy'], s['rows'], plan, s['topk_weights'], out=s['d_rows'])
        return out
    if kind == 'swiglu':
        clamp = s['clamp'] if s['clamp'] > 0 else None
        if s['fp8']:
            q, sf = dg.swiglu_per_token_cast_to_fp8(s['gate_up'], grouped_layout=s['layout'], activation_clamp=clamp, out=(s['y'], s['y_sf']))
            return {'q': q, 'sf': sf}
        out = {'y': dg.swiglu(s['gate_up'], grouped_layout=s['layout'], activation_clamp=clamp, out=s['y'])}
        if s['grad']:
            out['d_gate_up'] = dg.swiglu_backward(s['dy'], s['gate_up'], grouped_layout=s['layout'], activation_clamp=clamp, out=s['d_gate_up'])
        return out
    cast = dg.utils.per_block_cast_to_fp8 if s['block'] else dg.utils.per_token_cast_to_fp8
    q, sf = cast(s['x'], use_ue8m0=False)
    return {'q': q, 'sf': sf}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------------- the least work

def work(case):
    kind = case['kind']
    if kind in ('dense', 'grouped', 'masked'):
        n, k = case['n'], case['k']
        if kind == 'dense':
            m, groups = case['m'], 1
        elif kind == 'grouped':
            m, groups = case['rows'], case['groups']
        else:
            m, groups = max(1, round(case['groups'] * min(case['mean'], case['max_m']))), case['groups']
        out = m * n * (8 if case.get('f32') else 2)
        return {'bytes': m * k * (1 + 4 / 128) + groups * n * k * (1 + 4 / 16384) + out, 'flops': 2.0 * m * n * k}
    if kind in ('permute', 'unpermute'):
        t, h, size = case['tokens'], case['hidden'], 1.03125 if case.get('fp8') else 2
        moved = t * case['topk'] * (1 - case['masked'])
        one_way = (t + moved) * h * size
        if kind == 'permute':
            return {'bytes': one_way * (2 if case['grad'] else 1) + 8 * t * case['topk'], 'flops': moved * h if case['grad'] else 0}
        both = one_way + (t + 2 * moved) * h * size if case['grad'] else one_way
        return {'bytes': both + 8 * t * case['topk'], 'flops': moved * h * (5 if case['grad'] else 2)}
    if kind == 'swiglu':
        values = case['rows'] * case['inter']
        forward = values * (4 + (1.03125 if case['fp8'] else 2))
        return {'bytes': forward + (values * 10 if case['grad'] else 0), 'flops': values * (20 if case['grad'] else 8)}
    values = case['rows'] * case['k'] * max(case['groups'], 1)
    return {'bytes': values * (3 + (4 / 16384 if case['block'] else 4 / 128)), 'flops': values * 2}


# ------------------------------------------------------------------------------------------------- the definition in FP64

def _exact_matrix(q, sf, rows_per_scale):
    out = q.double()
    for r in range(0, q.shape[0], rows_per_scale):
        for c in range(sf.shape[1]):
            out[r:r + rows_per_scale, c * 128:(c + 1) * 128] *= sf[r // rows_per_scale, c].double()
    return out


def _exact_tokens(q, sf):
    out = q.double()
    for c in range(sf.shape[1]):
        out[:, c * 128:(c + 1) * 128] *= sf[:, c:c + 1].double()
    return out


def _exact_codes(x, sf):
    """E4M3 values nearest to x / sf (FP64), ties to the even mantissa, as float8: torch rounds a double once."""
    v = x / sf
    exponent = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))).clamp(min=-6)
    step = torch.exp2(exponent - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _exact_cast_rows(x):
    """x [rows, k] double -> (q, sf) with a scale for each 128 values of a row, the scale rounded to FP32 as it is stored."""
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    sf = torch.empty((x.shape[0], -(-x.shape[1] // 128)), device=x.device)
    for c in range(sf.shape[1]):
        part = x[:, c * 128:(c + 1) * 128]
        sf[:, c] = (part.abs().amax(dim=1).clamp(min=1e-4) / E4M3_MAX).float()
        q[:, c * 128:(c + 1) * 128] = _exact_codes(part, sf[:, c:c + 1].double())
    return q, sf


def _exact_plan(s):
    idx, e, al = s['topk_idx'].cpu().tolist(), s['experts'], s['alignment']
    counts = [0] * e
    for row in idx:
        for x in row:
            if 0 <= x < e:
                counts[x] += 1
    start, ends, total = [], [], 0
    for c in counts:
        start.append(total)
        ends.append(total + c)
        total += -(-c // al) * al
    following, dest = list(start), []
    for row in idx:
        for x in row:
            if 0 <= x < e:
                dest.append(following[x])
                following[x] += 1
            else:
                dest.append(-1)
    return torch.tensor(dest, device='cuda').view(s['tokens'], s['topk']), torch.tensor(ends, dtype=torch.int32, device='cuda')


def exact(case, seed):
    s = prepare(case, seed)
    kind = case['kind']
    if kind == 'dense':
        d = _exact_tokens(s['a'], s['sfa']) @ _exact_matrix(s['b'], s['sfb'], 128).T
        return {'d': d + s['c'].double() if case['f32'] else d}
    if kind == 'grouped':
        d = torch.zeros(s['d'].shape, dtype=torch.float64, device='cuda')
        start = 0
        for g, end in enumerate(s['psum_ends'].tolist()):
            b = _exact_matrix(s['b'][g], s['sfb'][g], 128)
            d[start:end] = _exact_tokens(s['a'][start:end], s['sfa'][start:end]) @ (b if case['nn'] else b.T)
            start = -(-end // 128) * 128
        return {'d': d}
    if kind == 'masked':
        d = torch.zeros(s['d'].shape, dtype=torch.float64, device='cuda')
        for g, m in enumerate(s['masked_m'].tolist()):
            d[g, :m] = _exact_tokens(s['a'][g, :m], s['sfa'][g, :m]) @ _exact_matrix(s['b'][g], s['sfb'][g], 128).T
        return {'d': d}
    if kind in ('permute', 'unpermute'):
        dest, ends = _exact_plan(s)
        t, h, cap = case['tokens'], case['hidden'], s['capacity']
        if kind == 'permute':
            out = {'dest_row': dest.int(), 'expert_end': ends}
            for name, x in zip(('rows', 'rows_sf'), s['x'] if case['fp8'] else (s['x'],)):
                rows = torch.zeros((cap, x.shape[1]), dtype=torch.float64, device='cuda')
                for k in range(case['topk']):
                    there = dest[:, k] >= 0
                    rows[dest[there, k]] = x[there].double() if x.dtype != torch.float8_e4m3fn else x.double()[there]
                out[name] = rows
            if case['grad']:
                dx = torch.zeros((t, h), dtype=torch.float64, device='cuda')
                for k in range(case['topk']):
                    there = dest[:, k] >= 0
                    dx[there] += s['rows'][dest[there, k]].double()
                out['dx'] = dx
            return out
        w = s['topk_weights'].double()
        y = torch.zeros((t, h), dtype=torch.float64, device='cuda')
        d_rows = torch.zeros((cap, h), dtype=torch.float64, device='cuda')
        d_weights = torch.zeros((t, case['topk']), dtype=torch.float64, device='cuda')
        for k in range(case['topk']):
            there = dest[:, k] >= 0
            picked = s['rows'][dest[there, k]].double()
            y[there] += w[there, k:k + 1] * picked
            d_rows[dest[there, k]] = w[there, k:k + 1] * s['dy'][there].double()
            d_weights[there, k] = torch.einsum('th,th->t', picked, s['dy'][there].double())
        return {'y': y, 'd_rows': d_rows, 'd_weights': d_weights} if case['grad'] else {'y': y}
    if kind == 'swiglu':
        n, inter, limit = s['total'], case['inter'], case['clamp'] if case['clamp'] > 0 else float('inf')
        gate, up = s['gate_up'][:n, :inter].double(), s['gate_up'][:n, inter:].double()
        g, u = gate.clamp(max=limit), up.clamp(-limit, limit)
        sig = torch.sigmoid(g)
        if case['fp8']:
            q = torch.zeros((s['buffer_rows'], inter), dtype=torch.float64, device='cuda')
            sf = torch.zeros((s['buffer_rows'], -(-inter // 128)), dtype=torch.float64, device='cuda')
            codes, scales = _exact_cast_rows(g * sig * u)
            q[:n], sf[:n] = codes.double(), scales.double()
            return {'q': q, 'sf': sf}
        y = torch.zeros((s['buffer_rows'], inter), dtype=torch.float64, device='cuda')
        y[:n] = g * sig * u
        out = {'y': y}
        if case['grad']:
            dy = s['dy'][:n].double()
            grad = torch.zeros((s['buffer_rows'], 2 * inter), dtype=torch.float64, device='cuda')
            grad[:n, :inter] = dy * u * (sig + g * sig * (1 - sig)) * (gate <= limit)
            grad[:n, inter:] = dy * g * sig * (up.abs() <= limit)
            out['d_gate_up'] = grad
        return out
    x = s['x']
    if not case['block']:
        return dict(zip(('q', 'sf'), _exact_cast_rows(x.double())))
    parts = x if x.dim() == 3 else x.unsqueeze(0)
    q = torch.empty(parts.shape, dtype=torch.float8_e4m3fn, device='cuda')
    sf = torch.empty((parts.shape[0], -(-parts.shape[1] // 128), -(-parts.shape[2] // 128)), device='cuda')
    for g in range(parts.shape[0]):
        for r in range(sf.shape[1]):
            block = parts[g, r * 128:(r + 1) * 128].double()
            for c in range(sf.shape[2]):
                sf[g, r, c] = (block[:, c * 128:(c + 1) * 128].abs().amax().clamp(min=1e-4) / E4M3_MAX).float()
            wide = sf[g, r].double().repeat_interleave(128)[:block.shape[1]]
            q[g, r * 128:(r + 1) * 128] = _exact_codes(block, wide)
    return {'q': q.view(x.shape), 'sf': sf if x.dim() == 3 else sf[0]}
