"""Operators of the expert path, timed one pass at a time: routing of tokens to
experts (scores, balance bias, groups, top-k, renormalised weights), MXFP4
quantisation and its inverse, and the routed experts' SwiGLU over MXFP4
weights.

`own` False: the plain form of each operator in elementary torch operations.
`own` True: the calls a user makes of ferry_b200.expert_ops.
"""
import math

import numpy as np
import torch

own = False

# the values of the 16 e2m1 codes (sign, two exponent bits, one mantissa bit)
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
BYTES = {'bf16': 2, 'fp16': 2, 'fp32': 4}


def _route(name, tokens, experts, topk, score, dtype, groups=1, kept=1, group_score='max', bias=False,
           norm=True, scaling=1.0, out='bf16'):
    return {'op': 'route', 'name': name, 'tokens': tokens, 'experts': experts, 'topk': topk, 'score': score,
            'dtype': dtype, 'groups': groups, 'kept': kept, 'group_score': group_score, 'bias': bias,
            'norm': norm, 'scaling': scaling, 'out': out}


def _quant(name, rows, width, dtype, gap=0):
    return {'op': 'quantize', 'name': name, 'rows': rows, 'width': width, 'dtype': dtype, 'gap': gap}


def _experts(name, tokens, topk, experts, hidden, inter, weights='bf16'):
    return {'op': 'experts', 'name': name, 'tokens': tokens, 'topk': topk, 'experts': experts,
            'hidden': hidden, 'inter': inter, 'weights': weights}


def listed():
    return [
        # one decode step of 64 sequences over 128 experts: the routing call is latency alone
        _route('route decode 64', 64, 128, 8, 'softmax', 'bf16'),
        # one token of a group-limited softmax router whose weights are scaled, not renormalised
        _route('route grouped 1', 1, 160, 6, 'softmax', 'fp32', 8, 3, 'max', False, False, 16.0),
        # a long prompt batch through a sigmoid router with a balance bias and groups
        _route('route sigmoid 16381', 16381, 256, 8, 'sigmoid', 'fp32', 8, 4, 'top2', True, True, 2.5, 'fp32'),
        # one expert's weights quantised and read back (a checkpoint loaded expert by expert)
        _quant('quantize expert row', 1, 3 * 2048 * 768, 'bf16'),
        # a matrix of odd height cut out of a wider one, in fp16
        _quant('quantize strided fp16', 1409, 2048, 'fp16', 96),
        # sixteen wider experts of a float32 checkpoint at once
        _quant('quantize 16 rows fp32', 16, 3 * 2048 * 1408, 'fp32'),
        # a tiny layer with odd token count and float32 routing weights (groups left empty)
        _experts('experts small', 33, 4, 32, 256, 128, 'fp32'),
        # one token of one sequence: eight experts, one route each
        _experts('experts decode 1', 1, 8, 128, 2048, 768),
        # the decode batch of the benchmark: 64 tokens, about forty experts active
        _experts('experts decode 64', 64, 8, 128, 2048, 768),
        # the wider experts, 16 tokens of top 6
        _experts('experts wide decode 16', 16, 6, 64, 2048, 1408),
        # a short prompt batch of odd length
        _experts('experts prompt 509', 509, 8, 128, 2048, 768),
        # a prompt batch large enough for the tensor cores to bound it
        _experts('experts prompt 4096', 4096, 8, 128, 2048, 768),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(('route', 'quantize', 'experts'))
    if kind == 'route':
        groups = rng.choice((1, 1, 2, 4, 8))
        experts = groups * _log_int(rng, 8, 64)
        kept = rng.randint(1, groups)
        topk = rng.randint(1, min(16, kept * experts // groups))
        case = _route('', _log_int(rng, 1, 16000), experts, topk, rng.choice(('softmax', 'sigmoid')),
                      rng.choice(('bf16', 'fp16', 'fp32')), groups, kept, rng.choice(('max', 'top2')),
                      rng.random() < 0.5, rng.random() < 0.5, rng.choice((1.0, 2.5, 16.0)),
                      rng.choice(('bf16', 'fp32')))
    elif kind == 'quantize':
        width = 32 * _log_int(rng, 1, 8192)
        rows = _log_int(rng, 1, max(1, min(20000, 130000000 // width)))
        case = _quant('', rows, width, rng.choice(('bf16', 'fp16', 'fp32')), rng.choice((0, 0, 32, 8)))
    else:
        hidden, inter = 128 * _log_int(rng, 1, 32), 128 * _log_int(rng, 1, 14)
        experts = _log_int(rng, 4, max(4, min(128, 128 * 2048 * 1408 // (hidden * inter))))
        topk = rng.randint(1, min(8, experts))
        most = max(1, min(4000, 4096 * 8 * 2048 * 768 // (topk * hidden * inter)))
        case = _experts('', _log_int(rng, 1, most), topk, experts, hidden, inter, rng.choice(('bf16', 'fp32')))
    del case['name']
    return case


# ---------------------------------------------------------------------------
# inputs


def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _popularity(experts, g):
    """log p of a Zipf(1.1) popularity over a random order of the experts."""
    p = torch.arange(1, experts + 1, dtype=torch.float32, device='cuda') ** -1.1
    return torch.log(p / p.sum())[torch.randperm(experts, generator=g, device='cuda')]


def _logits(tokens, experts, g):
    """Router logits of N(0, 1) hidden states and N(0, 0.02) gates of 2048 columns, with a popularity bias."""
    return 0.9 * torch.randn(tokens, experts, generator=g, device='cuda') + _popularity(experts, g)


def prepare(case, seed):
    g = _generator(seed)
    if case['op'] == 'route':
        logits = _logits(case['tokens'], case['experts'], g).to(DTYPES[case['dtype']])
        bias = 0.1 * torch.randn(case['experts'], generator=g, device='cuda') if case['bias'] else None
        return {'case': case, 'logits': logits, 'bias': bias}
    if case['op'] == 'quantize':
        wide = torch.randn(case['rows'], case['width'] + case['gap'], generator=g, device='cuda').mul_(0.02)
        return {'case': case, 'x': wide.to(DTYPES[case['dtype']])[:, :case['width']]}
    E, H, I, K, T = (case[k] for k in ('experts', 'hidden', 'inter', 'topk', 'tokens'))
    # every expert's weights, quantised: a row is [gate I x H | up I x H | down H x I] codes, then their scales
    n = 3 * H * I
    cache = torch.empty(E, n // 2 + n // 32, dtype=torch.uint8, device='cuda')
    w = torch.randn(E, n, generator=g, device='cuda').mul_(0.02)
    byte, q = _mx_parts(w.view(E, n // 32, 32))
    code = _code(q).view(E, n)
    cache[:, :n // 2] = code[:, 0::2] | (code[:, 1::2] << 4)
    cache[:, n // 2:] = byte
    del w, q, code, byte
    sel = torch.topk(_logits(T, E, g), K, dim=1).indices
    weights = torch.rand(T, K, generator=g, device='cuda').add_(0.1)
    weights = (weights / weights.sum(1, keepdim=True)).to(DTYPES[case['weights']])
    flat = sel.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    starts = torch.zeros(E + 1, dtype=torch.int64, device='cuda')
    starts[1:] = torch.bincount(flat, minlength=E).cumsum(0)
    return {'case': case, 'cache': cache, 'x': torch.randn(T, H, generator=g, device='cuda').to(torch.bfloat16),
            'weights': weights, 'slots': torch.randperm(E, generator=g, device='cuda'), 'starts': starts,
            'rows': order // K, 'cols': order % K, 'longest': int((starts[1:] - starts[:-1]).max()),
            'err': torch.zeros(1, dtype=torch.int32, device='cuda')}


# ---------------------------------------------------------------------------
# the plain forms


def _plain_route(s):
    """Selection in 64 bits (two scores may lie next to each other), ties to the lower id."""
    c = s['case']
    x = s['logits'].double()
    if c['score'] == 'softmax':
        e = torch.exp(x - x.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    key = score if s['bias'] is None else score + s['bias'].double()
    T, E = key.shape
    if c['groups'] > 1:
        by_group = torch.sort(key.view(T, c['groups'], E // c['groups']), dim=2, descending=True).values
        of_group = by_group[:, :, 0] if c['group_score'] == 'max' else by_group[:, :, 0] + by_group[:, :, 1]
        best = torch.sort(of_group, dim=1, descending=True, stable=True).indices[:, :c['kept']]
        keep = torch.zeros_like(of_group, dtype=torch.bool).scatter_(1, best, True)
        key = torch.where(keep.repeat_interleave(E // c['groups'], 1), key, -math.inf)
    selected = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :c['topk']]
    w = score.gather(1, selected)
    if c['norm']:
        w = w / w.sum(1, keepdim=True)
    return {'selected': selected, 'weights': (w * c['scaling']).to(DTYPES[c['out']])}


def _power(n):
    """2^n in float64 for integer tensors n."""
    return torch.pow(torch.full((), 2.0, dtype=torch.float64, device=n.device), n.double())


def _mx_parts(x):
    """x [..., 32] float32 -> scale bytes [...] and signed e2m1 values [..., 32] (round half to even, at most 6)."""
    top = x.abs().amax(-1)
    field = top.view(torch.int32) >> 23
    byte = torch.where(field == 255, field, (field - 2).clamp_min(0))
    y = x.abs() * _power(127 - byte).float().unsqueeze(-1)
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    q = (torch.round(y / step) * step).clamp_max(6.0)
    return byte.to(torch.uint8), torch.copysign(q, x)


def _code(q):
    """The 4-bit codes of e2m1 values."""
    m = q.abs()
    code = torch.where(m <= 2, 2 * m, torch.where(m <= 4, m + 2, 7.0)).to(torch.uint8)
    return code | (torch.signbit(q).to(torch.uint8) << 3)


def _plain_quantize(s):
    x = s['x']
    v = x.float().reshape(x.shape[0], -1, 32)
    byte, q = _mx_parts(v)
    scale = _power(byte.int() - 127).float().unsqueeze(-1)
    scale = torch.where(byte.unsqueeze(-1) == 255, math.nan, scale)
    return (q * scale).view(x.shape).to(torch.float32 if x.dtype == torch.float32 else torch.bfloat16)


def _plain_weights(s):
    """gate and up [G, I, H] and down [G, H, I] in float32."""
    c = s['case']
    H, I, n = c['hidden'], c['inter'], 3 * c['hidden'] * c['inter']
    rows = s['cache'][s['slots']]
    table = torch.tensor(E2M1, device='cuda')
    codes = rows[:, :n // 2]
    w = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), 2).view(rows.shape[0], n // 32, 32)
    w = (w * _power(rows[:, n // 2:].int() - 127).float().unsqueeze(-1)).view(rows.shape[0], n)
    return (w[:, :I * H].view(-1, I, H), w[:, I * H:2 * I * H].view(-1, I, H), w[:, 2 * I * H:].view(-1, H, I))


def _plain_experts(s):
    gate, up, down = _plain_weights(s)
    routes = s['rows'].numel()
    at = torch.arange(routes, device='cuda')
    group = torch.bucketize(at, s['starts'][1:], right=True)
    place = at - s['starts'][group]
    x = torch.zeros(gate.shape[0], s['longest'], gate.shape[2], device='cuda')
    x[group, place] = s['x'].float()[s['rows']]
    g = torch.bmm(x, gate.transpose(1, 2))
    a = g / (1.0 + torch.exp(-g)) * torch.bmm(x, up.transpose(1, 2))
    y = torch.bmm(a, down.transpose(1, 2))[group, place]
    return (y * s['weights'].float()[s['rows'], s['cols']].unsqueeze(1)).to(torch.bfloat16)


def run(state):
    c = state['case']
    if own:
        from ferry_b200 import expert_ops as ops
        if c['op'] == 'route':
            selected, weights = ops.route_experts(
                state['logits'], c['topk'], score=c['score'], bias=state['bias'], n_group=c['groups'],
                topk_group=c['kept'], group_score=c['group_score'], norm_topk_prob=c['norm'],
                scaling=c['scaling'], weights_dtype=DTYPES[c['out']])
            return {'selected': selected, 'weights': weights}
        if c['op'] == 'quantize':
            codes, scales = ops.quantize_mxfp4(state['x'])
            kind = torch.float32 if state['x'].dtype == torch.float32 else torch.bfloat16
            return ops.dequantize_mxfp4(codes, scales, kind)
        return ops.execute_experts_mxfp4(state['cache'], state['x'], state['weights'], state['slots'],
                                         state['starts'], state['rows'], state['cols'], c['hidden'],
                                         c['inter'], err=state['err'])
    if c['op'] == 'route':
        return _plain_route(state)
    return _plain_quantize(state) if c['op'] == 'quantize' else _plain_experts(state)


# ---------------------------------------------------------------------------
# what one pass cannot do without


def work(case):
    if case['op'] == 'route':
        T, E, K = case['tokens'], case['experts'], case['topk']
        return {'bytes': T * E * BYTES[case['dtype']] + T * K * (8 + BYTES[case['out']]) + (4 * E if case['bias'] else 0),
                'flops': 4 * T * E}
    if case['op'] == 'quantize':
        n = case['rows'] * case['width']
        # read the values, write codes and scales; read those, write the values they stand for
        back = 4 if case['dtype'] == 'fp32' else 2
        return {'bytes': n * (BYTES[case['dtype']] + back) + 2 * (n // 2 + n // 32), 'flops': 4 * n}
    T, K, E, H, I = (case[k] for k in ('tokens', 'topk', 'experts', 'hidden', 'inter'))
    rng = np.random.RandomState(0)
    p = np.arange(1, E + 1) ** -1.1
    pick = np.argpartition(-(0.9 * rng.randn(T, E) + np.log(p / p.sum())), K - 1, axis=1)[:, :K]
    routes, active = T * K, len(np.unique(pick))
    weights = active * (3 * H * I // 2 + 3 * H * I // 32)
    return {'bytes': weights + 2 * T * H + 2 * routes * H + routes * (16 + BYTES[case['weights']]),
            'flops': 6 * routes * H * I}


# ---------------------------------------------------------------------------
# the definitions in 64 bits


def _exact_route(case, seed):
    s = prepare(case, seed)
    x = s['logits'].double().cpu().numpy()
    if case['score'] == 'softmax':
        score = np.exp(x - x.max(1, keepdims=True))
        score /= score.sum(1, keepdims=True)
    else:
        score = np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))
    key = score if s['bias'] is None else score + s['bias'].double().cpu().numpy()
    T, E = x.shape
    if case['groups'] > 1:
        parts = np.partition(key.reshape(T, case['groups'], -1), -2, axis=2)
        worth = parts[:, :, -1] if case['group_score'] == 'max' else parts[:, :, -1] + parts[:, :, -2]
        rank = np.argsort(np.argsort(-worth, axis=1, kind='stable'), axis=1, kind='stable')
        key = np.where(np.repeat(rank < case['kept'], E // case['groups'], axis=1), key, -np.inf)
    sel = np.argsort(-key, axis=1, kind='stable')[:, :case['topk']]
    w = np.take_along_axis(score, sel, 1)
    if case['norm']:
        w = w / w.sum(1, keepdims=True)
    return {'selected': torch.from_numpy(sel), 'weights': torch.from_numpy(w * case['scaling'])}


def _exact_quantize(case, seed):
    x = prepare(case, seed)['x'].double()
    out = torch.empty(x.shape, dtype=torch.float64, device='cuda')
    grid = torch.tensor(E2M1[:8], dtype=torch.float64, device='cuda')
    border = (grid[1:] + grid[:-1]) / 2
    for r in range(0, x.shape[0], max(1, (1 << 24) // x.shape[1])):
        b = x[r:r + max(1, (1 << 24) // x.shape[1])].reshape(-1, 32)
        top = b.abs().amax(1)
        power = torch.frexp(top).exponent - 3  # floor(log2 top) - 2
        power = torch.where(top == 0, -127, power).clamp_min(-127)
        y = torch.ldexp(b.abs(), -power.unsqueeze(1))
        low = torch.bucketize(y, border)                # a value on a border goes down ...
        high = torch.bucketize(y, border, right=True)   # ... or up: to the even code
        code = torch.where(low % 2 == 0, low, high)
        out[r:r + max(1, (1 << 24) // x.shape[1])] = torch.copysign(
            torch.ldexp(grid[code], power.unsqueeze(1)), b).view(-1, x.shape[1])
    return out


def _exact_experts(case, seed):
    s = prepare(case, seed)
    H, I = case['hidden'], case['inter']
    n = 3 * H * I
    starts, slots = s['starts'].tolist(), s['slots'].tolist()
    table = torch.tensor(E2M1, dtype=torch.float64, device='cuda')
    out = torch.empty(s['rows'].numel(), H, dtype=torch.float64, device='cuda')
    for e in range(case['experts']):
        a, b = starts[e], starts[e + 1]
        if a == b:
            continue
        row = s['cache'][slots[e]]
        w = torch.empty(n, dtype=torch.float64, device='cuda')
        w[0::2], w[1::2] = table[(row[:n // 2] % 16).long()], table[(row[:n // 2] // 16).long()]
        w = torch.ldexp(w.view(-1, 32), row[n // 2:].double().unsqueeze(1) - 127).view(-1)
        x = s['x'][s['rows'][a:b]].double()
        g, u = x @ w[:I * H].view(I, H).T, x @ w[I * H:2 * I * H].view(I, H).T
        y = (g * torch.sigmoid(g) * u) @ w[2 * I * H:].view(H, I).T
        out[a:b] = y * s['weights'][s['rows'][a:b], s['cols'][a:b]].double().unsqueeze(1)
    return out


def exact(case, seed):
    return {'route': _exact_route, 'quantize': _exact_quantize, 'experts': _exact_experts}[case['op']](case, seed)
