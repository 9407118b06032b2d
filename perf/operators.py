"""What the operators in front of the MoE layer cost: their cases, their plain forms, their work.

Three operators, in the order in which a decoder layer calls them before ``fp8_fp4_gc_moe``:

* ``norm``:  residual addition, RMS norm, e4m3 output with one UE8M0 scale per 32 channels
             (``rms_norm_for_gc_moe``);
* ``logits``: the router's product, BF16 activations against BF16 or FP32 router weights, FP32
             result (``router_logits_for_gc_moe``);
* ``route``: scores, balance bias, expert groups, top-k and weights (``route_for_gc_moe``).

``own`` selects what ``run`` does: the framework's calls, or the same formulas in elementary torch
operations.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
MAX_ELEMENTS = 4096 * 7168          # of a drawn activation: the largest listed one


def listed() -> list:
    return [
        # decoding a single sequence: one launch, latency is all there is
        _norm('norm 1 x 7168', 1, 7168, 'bf16', 'bf16', True),
        # an odd decode batch of a model that keeps its residual stream and norm weights in FP32
        _norm('norm 37 x 5120 f32 residual', 37, 5120, 'f32', 'f32', True),
        # a decode batch of the single-GPU configuration whose residual was added elsewhere; the router reads nothing from it
        _norm('norm 256 x 4096 no residual', 256, 4096, 'none', 'bf16', False),
        # a prefill chunk of the large-token configuration
        _norm('norm 4096 x 7168', 4096, 7168, 'bf16', 'bf16', True),
        # the router of the expert-parallel decode configuration: one token, then an odd batch of another width
        _logits('logits 1 x 7168 x 256', 1, 7168, 256, 'bf16'),
        _logits('logits 33 x 5120 x 384', 33, 5120, 384, 'bf16'),
        # FP32 router weights, a full decode batch
        _logits('logits 128 x 6144 x 256 f32', 128, 6144, 256, 'f32'),
        # prefill chunk
        _logits('logits 4096 x 7168 x 256', 4096, 7168, 256, 'bf16'),
        # one token, sigmoid scores with a balance bias, 4 of 8 groups
        _route('route 1 x 256 groups', 1, 256, 8, 'sigmoid', True, 8, 4, 'top2', True, 'f32', 0),
        # the plain softmax router of the single-GPU configuration
        _route('route 256 x 64 softmax', 256, 64, 8, 'softmax', False, 1, 1, 'top2', True, 'f32', 0),
        # BF16 logits (many exact ties), an odd batch padded to a captured size with masked rows
        _route('route 131 x 384 bf16', 131, 384, 6, 'sigmoid', True, 1, 1, 'top2', True, 'bf16', 3),
        # several prefill chunks routed at once
        _route('route 16384 x 256 groups', 16384, 256, 8, 'sigmoid', True, 8, 4, 'top2', True, 'f32', 0),
    ]


def _norm(name, tokens, hidden, residual, weight, normed):
    return {'name': name, 'op': 'norm', 'tokens': tokens, 'hidden': hidden, 'residual': residual, 'weight': weight,
            'normed': normed}


def _logits(name, tokens, hidden, experts, weight):
    return {'name': name, 'op': 'logits', 'tokens': tokens, 'hidden': hidden, 'experts': experts, 'weight': weight}


def _route(name, tokens, experts, topk, scoring, bias, groups, topk_groups, group_score, renormalize, dtype, padded):
    return {'name': name, 'op': 'route', 'tokens': tokens, 'experts': experts, 'topk': topk, 'scoring': scoring,
            'bias': bias, 'groups': groups, 'topk_groups': topk_groups, 'group_score': group_score,
            'renormalize': renormalize, 'dtype': dtype, 'padded': padded}


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng) -> dict:
    """One more case: token counts over their logarithm, hidden sizes in whole scale groups, expert
    counts that need not be round."""
    op = rng.choice(('norm', 'logits', 'route'))
    if op == 'norm':
        hidden = 32 * rng.randint(32, 256)
        tokens = _log_uniform(rng, 1, min(4096, MAX_ELEMENTS // hidden))
        case = _norm('', tokens, hidden, rng.choice(('none', 'bf16', 'f32')), rng.choice(('bf16', 'f32')),
                     rng.random() < 0.7)
        if tokens * hidden > MAX_ELEMENTS // 2 and case['residual'] == 'f32':
            case['residual'] = 'bf16'
    elif op == 'logits':
        hidden = 32 * rng.randint(32, 224)
        experts = rng.choice((8, 64, 128, 160, 256, 384, rng.randint(8, 256)))
        tokens = _log_uniform(rng, 1, min(4096, 4096 * 7168 * 256 // (hidden * experts)))
        case = _logits('', tokens, hidden, experts, rng.choice(('bf16', 'f32')))
        if tokens > 2048:
            case['weight'] = 'bf16'
    else:
        groups = rng.choice((1, 1, 2, 4, 8))
        experts = groups * rng.randint(max(4, 16 // groups), 512 // groups)
        topk_groups = rng.randint(max(1, groups // 2), groups)
        topk = rng.randint(1, min(10, topk_groups * (experts // groups)))
        tokens = _log_uniform(rng, 1, min(16384, 16384 * 256 // experts))
        case = _route('', tokens, experts, topk, rng.choice(('sigmoid', 'softmax')), rng.random() < 0.6, groups,
                      topk_groups, rng.choice(('top2', 'max')), rng.random() < 0.8, rng.choice(('f32', 'bf16')),
                      rng.randint(0, tokens // 8))
    del case['name']
    return case


_DTYPES = {'bf16': torch.bfloat16, 'f32': torch.float32}


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device='cuda').manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device='cuda')

    t, state = case['tokens'], {'case': case}
    if own:
        import gc_moe_b200
        state['G'] = gc_moe_b200
    if case['op'] == 'norm':
        h = case['hidden']
        state['x'] = normal(t, h).to(torch.bfloat16)
        state['weight'] = (1 + 0.2 * normal(h)).to(_DTYPES[case['weight']])
        state['residual'] = None
        if case['residual'] != 'none':
            # a residual stream is much larger than what a layer adds, and a few of its channels dominate
            channel = torch.where(torch.rand(h, generator=g, device='cuda') < 0.01, 40.0, 3.0)
            state['residual'] = (normal(t, h) * channel).to(_DTYPES[case['residual']])
    elif case['op'] == 'logits':
        h, e = case['hidden'], case['experts']
        state['x'] = normal(t, h).to(torch.bfloat16)
        state['weight'] = (normal(e, h) * h ** -0.5).to(_DTYPES[case['weight']])
        if own:
            state['router_weight'] = gc_moe_b200.transform_router_weight_for_gc_moe(state['weight'])
    else:
        e = case['experts']
        logits = normal(t, e) * 1.5
        if case['padded']:
            logits[t - case['padded']:] = float('-inf')
        state['logits'] = logits.to(_DTYPES[case['dtype']])
        # balance biases are of the size of the gaps between the scores that they reorder
        spread = 0.05 if case['scoring'] == 'sigmoid' else 0.5 / e
        state['bias'] = normal(e) * spread if case['bias'] else None
    return state


def run(state: dict) -> dict:
    case = state['case']
    if case['op'] == 'norm':
        return _run_norm(case, state)
    if case['op'] == 'logits':
        if own:
            return {'logits': state['G'].router_logits_for_gc_moe(state['x'], state['router_weight'])}
        return {'logits': state['x'].float() @ state['weight'].float().T}
    return _run_route(case, state)


def _run_norm(case: dict, state: dict) -> dict:
    x, weight, residual = state['x'], state['weight'], state['residual']
    if own:
        r = state['G'].rms_norm_for_gc_moe(x, weight, residual, eps=EPS, normed=case['normed'])
        q, scales, normed, h = r.x, r.x_sf.view(torch.float8_e8m0fnu), r.normed, r.residual
    else:
        h32 = x.float() if residual is None else x.float() + residual.float()
        v = h32 * torch.rsqrt(h32.square().mean(-1, keepdim=True) + EPS) * weight.float()
        groups = v.view(v.shape[0], -1, 32)
        mantissa, exponent = torch.frexp(groups.abs().amax(-1))       # 448 = 0.875 * 2^9
        code = exponent - 9 + (mantissa > 0.875) + 127
        code = torch.where(mantissa == 0, 0, code.clamp(0, 254)).to(torch.int32)
        inverse = ((254 - code) << 23).view(torch.float32)            # 2^(127 - code)
        q = (groups * inverse[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(v.shape)
        code = torch.nn.functional.pad(code.to(torch.uint8), (0, -code.shape[1] % 4), value=127)
        scales = code.view(torch.float8_e8m0fnu)
        normed = v.to(torch.bfloat16) if case['normed'] else None
        h = None if residual is None else h32.to(residual.dtype)
    out = {'x': q, 'scales': scales}
    if normed is not None:
        out['normed'] = normed
    if h is not None:
        out['residual'] = h
    return out


def _run_route(case: dict, state: dict) -> dict:
    logits, bias, k = state['logits'], state['bias'], case['topk']
    if own:
        idx, weights = state['G'].route_for_gc_moe(
            logits, k, scoring=case['scoring'], bias=bias, num_groups=case['groups'], topk_groups=case['topk_groups'],
            group_score=case['group_score'], renormalize=case['renormalize'], scale=2.5)
        return {'topk_idx': idx, 'topk_weights': weights}
    # 64 bits for the scores: experts next to the border between chosen and not chosen
    low = float('-inf')
    l64 = logits.double()
    open_ = l64 > low                                                  # an expert that is masked is never chosen
    top = l64.amax(-1, keepdim=True)
    exps = torch.where(open_, (l64 - torch.where(top > low, top, 0.0)).exp(), 0.0)
    if case['scoring'] == 'sigmoid':
        score = 1 / (1 + (-l64).exp())
    else:
        score = exps / exps.sum(-1, keepdim=True).clamp_min(1e-300)
    biased = score if bias is None else score + bias.double()
    key = torch.where(open_, l64 if bias is None else biased, low)
    t, e, groups = logits.shape[0], case['experts'], case['groups']
    if groups > 1:
        by_max = case['group_score'] == 'max'
        members = key if by_max else torch.where(open_, biased, low)
        best = members.view(t, groups, e // groups).sort(dim=-1, descending=True).values
        value = best[..., 0] if by_max else best[..., 0] + best[..., 1]
        kept = value.sort(dim=-1, descending=True, stable=True).indices[:, :case['topk_groups']]
        stays = torch.zeros_like(value, dtype=torch.bool).scatter_(1, kept, True)
        key = torch.where(stays.repeat_interleave(e // groups, 1), key, low)
    key, idx = key.sort(dim=-1, descending=True, stable=True)
    key, idx = key[:, :k], idx[:, :k]
    chosen = key > low
    weights = torch.where(chosen, score.gather(1, idx), 0.0)
    if case['renormalize']:
        weights = weights / weights.sum(-1, keepdim=True).clamp_min(1e-300)
    return {'topk_idx': torch.where(chosen, idx, -1), 'topk_weights': (weights * 2.5).float()}


def work(case: dict) -> dict:
    t = case['tokens']
    size = {'none': 0, 'bf16': 2, 'f32': 4}
    if case['op'] == 'norm':
        h = case['hidden']
        per_element = 2 + 2 * size[case['residual']] + 1 + 1 / 32 + 2 * case['normed']
        return {'bytes': t * h * per_element + h * size[case['weight']], 'flops': 6 * t * h}
    e = case['experts']
    if case['op'] == 'logits':
        h = case['hidden']
        return {'bytes': t * h * 2 + e * h * size[case['weight']] + t * e * 4, 'flops': 2 * t * e * h}
    return {'bytes': t * (e * size[case['dtype']] + case['topk'] * 12) + e * 4 * case['bias'], 'flops': 4 * t * e}


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case['op'] == 'norm':
        return _exact_norm(case, state)
    if case['op'] == 'logits':
        return {'logits': torch.einsum('th,eh->te', state['x'].double(), state['weight'].double())}
    return _exact_route(case, state)


def _exact_norm(case: dict, state: dict) -> dict:
    h = state['x'].double()
    if state['residual'] is not None:
        h = h + state['residual'].double()
    v = h / (h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).sqrt() * state['weight'].double()
    top = v.unflatten(1, (-1, 32)).abs().max(2).values
    code = torch.ceil(torch.log2(top / 448)).clamp(-127, 127)
    code = torch.where(top > 448 * torch.exp2(code), code + 1, code)
    code = torch.where(448 * torch.exp2(code - 1) >= top, code - 1, code).clamp_min(-127)
    pad = -code.shape[1] % 4
    scales = torch.cat([torch.exp2(code), torch.ones((code.shape[0], pad), dtype=torch.float64, device=code.device)], 1)
    # like the other outputs, before it is rounded to its type
    out = {'x': v / torch.exp2(code).repeat_interleave(32, 1), 'scales': scales}
    if case['normed']:
        out['normed'] = v
    if state['residual'] is not None:
        out['residual'] = h
    return out


def _exact_route(case: dict, state: dict) -> dict:
    """Row by row on the experts that are left, choosing one expert at a time."""
    logits = state['logits'].double().cpu()
    bias = None if state['bias'] is None else state['bias'].double().cpu()
    t, e, k = logits.shape[0], case['experts'], case['topk']
    minus = -math.inf
    dead = logits == minus
    if case['scoring'] == 'sigmoid':
        score = torch.sigmoid(logits)
    else:
        score = torch.softmax(logits.masked_fill(dead.all(1, keepdim=True), 0.0), 1)
    biased = score if bias is None else score + bias
    key = (logits if bias is None else biased).masked_fill(dead, minus)
    if case['groups'] > 1:
        size = e // case['groups']
        member = (key if case['group_score'] == 'max' else biased.masked_fill(dead, minus)).reshape(t, -1, size)
        value = member.amax(2) if case['group_score'] == 'max' else member.topk(2, 2).values.sum(2)
        out_of = torch.ones_like(value, dtype=torch.bool)
        for _ in range(case['topk_groups']):
            best = value.masked_fill(~out_of, minus)
            first = torch.where(out_of & (best == best.amax(1, keepdim=True)), 0, 1).argmin(1, keepdim=True)
            out_of.scatter_(1, first, False)
        key = key.masked_fill(out_of.repeat_interleave(size, 1), minus)
    key = key.clone()
    ids, weights = [], []
    for _ in range(k):
        value = key.amax(1, keepdim=True)
        first = (key < value).to(torch.int8).argmin(1, keepdim=True)
        ids.append(torch.where(value > minus, first, -1))
        weights.append(torch.where(value > minus, score.gather(1, first), 0.0))
        key.scatter_(1, first, minus)
    weights = torch.cat(weights, 1)
    if case['renormalize']:
        weights = weights / weights.sum(1, keepdim=True).clamp_min(1e-300)
    return {'topk_idx': torch.cat(ids, 1), 'topk_weights': weights * 2.5}
