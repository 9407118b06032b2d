"""GPU parity of ``router_logits_for_gc_moe`` and ``route_for_gc_moe`` against
their formulas in 64 bits.

Expert ids are exact.  Tolerances:
* logits: the products are exact; an element takes part in fewer than 256
  additions, each of which loses at most 2^-23 of a partial sum that is at most
  sum |x w|: 2^-15 * sum |x w|;
* weights: the exponent's argument is rounded once (at most 64 * 2^-24 here),
  the exponential, the sum over at most 2048 experts (69 additions one after the
  other) and the quotient add less than 2^-17.6: 2^-16.5 relative.
"""
import itertools

import pytest
import torch

import gc_moe_b200 as G

pytestmark = pytest.mark.gpu

WEIGHT_REL = 2.0 ** -16.5
INF = float('inf')


# ------------------------------------------------------------------ logits
def _logits_case(tokens, hidden, experts, weight, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((tokens, hidden), generator=g).to(torch.bfloat16)
    w = (torch.randn((experts, hidden), generator=g) * hidden ** -0.5).to(weight)
    return x, w


def _check_logits(got, x, w):
    x, w = x.cuda().double(), w.cuda().double()
    want, size = x @ w.T, x.abs() @ w.abs().T
    assert got.dtype == torch.float32 and got.shape == want.shape
    assert bool(((got.double() - want).abs() <= size * 2.0 ** -15).all())


@pytest.mark.parametrize('weight', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('tokens,hidden,experts', [
    (1, 8, 1), (1, 7168, 256), (2, 1024, 8), (3, 1032, 7), (4, 5120, 384), (7, 2056, 33), (8, 4096, 64), (13, 6144, 255),
    (16, 7168, 256), (17, 7168, 256), (31, 4104, 65), (64, 512, 130), (129, 7168, 256), (200, 64, 300), (257, 1064, 257),
    (1000, 5120, 384), (40, 2048, 2048), (2100, 2048, 256), (700, 1096, 250), (4097, 136, 40), (130, 7168, 512),
    (300, 7168, 384), (96, 7168, 256), (63, 72, 500), (65, 1000, 129)])
def test_logits_against_the_formula(tokens, hidden, experts, weight):
    x, w = _logits_case(tokens, hidden, experts, weight, seed=tokens + experts)
    planes = G.transform_router_weight_for_gc_moe(w.cuda())
    assert planes.shape[0] == (1 if weight == torch.bfloat16 else 3)
    got = G.router_logits_for_gc_moe(x.cuda(), planes)
    _check_logits(got, x, w)
    assert torch.equal(got, G.router_logits_for_gc_moe(x.cuda(), planes))      # the same bits every time


# Few tokens: rows of one, two and four rounds of loads and longer ones, and as many experts as are
# computed with one, two and four tokens at a time, and more.
@pytest.mark.parametrize('weight', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('hidden,experts', [
    (2048, 129), (4096, 256), (4104, 296), (4104, 297), (5120, 384), (5120, 385), (8192, 592), (8200, 593), (16384, 64),
    (1032, 888), (1032, 889), (520, 2048), (8, 2047)])
def test_logits_of_few_tokens(hidden, experts, weight):
    x, w = _logits_case(8, hidden, experts, weight, seed=hidden + experts)
    planes = G.transform_router_weight_for_gc_moe(w.cuda())
    for tokens in range(1, 9):
        guard = torch.full((tokens + 2, experts), 7.0, device='cuda')
        got = G.router_logits_for_gc_moe(x[:tokens].cuda(), planes, out=guard[1:-1])
        _check_logits(got, x[:tokens], w)
        assert bool((guard[0] == 7).all()) and bool((guard[-1] == 7).all())
        same = G.router_logits_for_gc_moe(x[:1].cuda().expand(tokens, hidden), planes)     # rows that overlap
        _check_logits(same, x[:1].expand(tokens, hidden), w)


@pytest.mark.parametrize('tokens', [1, 5, 40, 300])
def test_logits_of_strided_rows_into_a_given_tensor(tokens):
    x, w = _logits_case(tokens, 1024, 100, torch.bfloat16, seed=tokens)
    planes = G.transform_router_weight_for_gc_moe(w.cuda())
    wide = torch.full((tokens, 1048), float('nan'), dtype=torch.bfloat16, device='cuda')
    wide[:, 8:1032] = x.cuda()
    guard = torch.full((tokens + 2, 100), 7.0, device='cuda')
    got = G.router_logits_for_gc_moe(wide[:, 8:1032], planes, out=guard[1:-1])
    assert got.data_ptr() == guard[1:].data_ptr()
    _check_logits(got, x, w)
    assert bool((guard[0] == 7).all()) and bool((guard[-1] == 7).all())
    same = G.router_logits_for_gc_moe(x[:1].cuda().expand(tokens, 1024), planes)
    assert torch.equal(same, same[:1].expand(tokens, 100))


@pytest.mark.parametrize('tokens', [3, 150])
def test_a_nan_or_infinity_stays_in_its_row_and_column(tokens):
    x, w = _logits_case(tokens, 2048, 70, torch.bfloat16, seed=3)
    x[1, 100] = float('nan')
    x[2, 5] = INF
    w[6, 9] = float('nan')
    got = G.router_logits_for_gc_moe(x.cuda(), G.transform_router_weight_for_gc_moe(w.cuda()))
    assert bool(torch.isnan(got[1]).all()) and bool(torch.isnan(got[:, 6]).all())
    assert not bool(torch.isfinite(got[2]).any())
    rows = [t for t in range(tokens) if t not in (1, 2)]
    columns = [e for e in range(70) if e != 6]
    _check_logits(got[rows][:, columns], x[rows], w[columns])


def test_no_tokens_and_logits_argument_errors():
    x, w = (t.cuda() for t in _logits_case(4, 1024, 16, torch.bfloat16, seed=4))
    planes = G.transform_router_weight_for_gc_moe(w)
    call = G.router_logits_for_gc_moe
    assert call(x[:0], planes).shape == (0, 16)
    for bad in (lambda: call(x.float(), planes), lambda: call(x[0], planes), lambda: call(x.T, planes),
                lambda: call(x, w), lambda: call(x, planes.float()), lambda: call(x, planes.cpu()),
                lambda: call(x[:, :512], planes), lambda: call(x, planes[:, ::2]),
                lambda: call(x, planes.expand(2, 16, 1024).contiguous()), lambda: call(x[:, 4:1004], planes[:, :, :1000].contiguous()),
                lambda: call(x[:, :1004], planes[:, :, :1004].contiguous()),
                lambda: call(x, planes, out=torch.empty((4, 16), dtype=torch.bfloat16, device='cuda')),
                lambda: call(x, planes, out=torch.empty((4, 17), device='cuda')),
                lambda: call(x, planes, out=torch.empty((16, 4), device='cuda').T),
                lambda: call(x, torch.zeros((1, 2049, 1024), dtype=torch.bfloat16, device='cuda'))):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------ routing
def _route_reference(logits, topk, scoring, bias, groups, topk_groups, group_score, renormalize, scale):
    """Row by row, one choice at a time, in Python's 64-bit floats."""
    import math
    l32 = logits.float()
    ids, weights = [], []
    for row in l32.tolist():
        b = [0.0] * len(row) if bias is None else bias.tolist()
        alive = [v == v and v > -INF and c == c and c > -INF for v, c in zip(row, b)]
        row = [min(v, 3.4028234663852886e38) if v == v else v for v in row]
        experts = [e for e, a in enumerate(alive) if a]
        score = [0.0] * len(row)
        if scoring == 'sigmoid':
            for e in experts:
                z = math.exp(-abs(row[e]))
                score[e] = (1.0 if row[e] >= 0 else z) / (1.0 + z)
        elif experts:
            top = max(row[e] for e in experts)
            ex = {e: math.exp(row[e] - top) for e in experts}
            total = math.fsum(ex.values())
            for e in experts:
                score[e] = ex[e] / total
        # the kernel's formula for keys: 1 / (1 + exp(-l))
        raw = list(score)
        if scoring == 'sigmoid':
            for e in experts:
                raw[e] = 1.0 / (1.0 + math.exp(min(-row[e], 709.0))) if row[e] > -709 else 0.0
        biased = [raw[e] + b[e] for e in range(len(row))]
        key = list(row) if bias is None else biased
        if groups > 1:
            size = len(row) // groups
            values = []
            for g in range(groups):
                members = sorted(((key if group_score == 'max' else biased)[e] for e in range(g * size, (g + 1) * size) if alive[e]),
                                 reverse=True)
                if not members:
                    values.append(-INF)
                elif group_score == 'max':
                    values.append(members[0])
                else:
                    values.append(sum(members[:2]))
            kept = sorted(range(groups), key=lambda g: (-values[g], g))[:topk_groups]
            experts = [e for e in experts if e // size in kept]
        order = sorted(experts, key=lambda e: (-key[e], e))[:topk]
        w = [score[e] for e in order]
        if renormalize and order:
            if scoring == 'sigmoid':
                m = min(0.0, max(row[e] for e in order))
                w = [1 / (1 + math.exp(-row[e])) if row[e] > 0 else math.exp(row[e] - m) / (1 + math.exp(row[e])) for e in order]
            else:
                m = max(row[e] for e in order)
                w = [math.exp(row[e] - m) for e in order]
            total = math.fsum(w)
            w = [v / total for v in w]
        ids.append(order + [-1] * (topk - len(order)))
        weights.append([v * scale for v in w] + [0.0] * (topk - len(order)))
    return torch.tensor(ids).view(len(l32), topk), torch.tensor(weights, dtype=torch.float64).view(len(l32), topk)


def _check_route(logits, topk, scoring='softmax', bias=None, groups=1, topk_groups=None, group_score='top2',
                 renormalize=True, scale=1.0):
    topk_groups = groups if topk_groups is None else topk_groups
    idx, w = G.route_for_gc_moe(logits.cuda(), topk, scoring=scoring, bias=None if bias is None else bias.cuda(),
                                num_groups=groups, topk_groups=topk_groups, group_score=group_score,
                                renormalize=renormalize, scale=scale)
    want_idx, want_w = _route_reference(logits, topk, scoring, bias, groups, topk_groups, group_score, renormalize, scale)
    assert torch.equal(idx.cpu(), want_idx)
    # results below f32's normal range are rounded to multiples of 2^-149
    assert bool(((w.cpu().double() - want_w).abs() <= want_w.abs() * WEIGHT_REL + 2.0 ** -126).all())
    return idx, w


def _logits(tokens, experts, seed, dtype=torch.float32, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((tokens, experts), generator=g) * spread).to(dtype)


def _bias(experts, seed, spread=0.1):
    return torch.randn(experts, generator=torch.Generator().manual_seed(seed)) * spread


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('scoring,biased', list(itertools.product(('softmax', 'sigmoid'), (False, True))))
@pytest.mark.parametrize('tokens,experts,topk', [(1, 1, 1), (1, 256, 8), (3, 2, 2), (5, 64, 8), (33, 257, 7), (6, 384, 6),
                                                 (2, 2048, 32), (4, 33, 32), (9, 1023, 10)])
def test_routing_without_groups(tokens, experts, topk, scoring, biased, dtype):
    _check_route(_logits(tokens, experts, tokens + experts, dtype), topk, scoring, _bias(experts, 3) if biased else None)


@pytest.mark.parametrize('group_score', ['top2', 'max'])
@pytest.mark.parametrize('scoring,biased', list(itertools.product(('softmax', 'sigmoid'), (False, True))))
@pytest.mark.parametrize('experts,topk,groups,topk_groups', [
    (256, 8, 8, 4), (256, 8, 8, 1), (160, 6, 8, 3), (384, 6, 3, 2), (64, 8, 4, 4), (32, 4, 32, 4), (66, 9, 33 // 3, 5),
    (85, 5, 17, 3), (2048, 20, 8, 5), (1024, 8, 16, 7), (6, 2, 2, 1)])
def test_routing_with_groups(experts, topk, groups, topk_groups, scoring, biased, group_score):
    _check_route(_logits(17, experts, experts + groups), topk, scoring, _bias(experts, 4) if biased else None, groups,
                 topk_groups, group_score, scale=2.5)


@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('groups', [1, 8])
def test_weights_without_renormalisation(scoring, groups):
    _check_route(_logits(21, 128, 5), 6, scoring, None, groups, max(1, groups // 2), 'max', renormalize=False, scale=16.0)
    _check_route(_logits(21, 128, 6), 6, scoring, _bias(128, 6), groups, max(1, groups // 2), renormalize=False)


@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lower_expert_and_group(scoring, dtype):
    zero = torch.zeros((2, 64), dtype=dtype)
    zero[1] = (torch.arange(64) // 4).to(dtype)
    zero[1, 3] = -0.0                                   # equal to the other zeros
    for bias in (None, torch.zeros(64), torch.full((64,), -0.25)):
        idx, _ = _check_route(zero, 8, scoring, bias)
        assert idx[0].tolist() == list(range(8)) and idx[1].tolist() == [60, 61, 62, 63, 56, 57, 58, 59]
        for group_score in ('top2', 'max'):
            idx, _ = _check_route(zero, 8, scoring, bias, 8, 2, group_score)
            assert idx[0].tolist() == list(range(8))


def test_near_ties_follow_the_64_bit_order():
    """Keys that f32 cannot tell apart: biases that differ by far less than f32's step at the key, logits one
    step apart whose scores round to the same f32."""
    g = torch.Generator().manual_seed(11)
    logits = torch.full((16, 128), 1.5)
    logits[:, ::3] = torch.nextafter(torch.tensor(1.5), torch.tensor(2.0))
    logits[8:] = 1.5 + torch.randint(0, 3, (8, 128), generator=g) * 2.0 ** -23
    bias = torch.randint(-3, 4, (128,), generator=g).float() * 2.0 ** -45
    for scoring, groups in itertools.product(('sigmoid', 'softmax'), (1, 8)):
        _check_route(logits, 8, scoring, bias, groups, max(1, groups // 2))
        _check_route(logits, 8, scoring, None, groups, max(1, groups // 2))
    large = _logits(8, 128, 12, spread=0.01)             # a bias that swallows the scores' low bits in f32
    _check_route(large, 8, 'sigmoid', torch.full((128,), 4096.0))


@pytest.mark.parametrize('scoring,biased', list(itertools.product(('softmax', 'sigmoid'), (False, True))))
@pytest.mark.parametrize('groups', [1, 4])
def test_masked_experts_and_empty_rows(scoring, biased, groups):
    logits = _logits(10, 64, 21)
    logits[0] = -INF                                     # a row that pads the batch
    logits[1] = float('nan')
    logits[2, 1:] = -INF                                 # one expert left
    logits[3, 5:] = float('nan')                         # fewer left than asked for
    logits[4, ::2] = -INF
    logits[5, 16:32] = -INF                              # a whole group
    logits[6, 7] = INF
    logits[7, [3, 40]] = INF
    logits[8] = torch.finfo(torch.float32).min           # the type's lowest value is a value
    logits[9, :60] = torch.finfo(torch.float32).min
    bias = None
    if biased:
        bias = _bias(64, 22)
        bias[10], bias[11] = -INF, float('nan')
    for renormalize in (True, False):
        idx, w = _check_route(logits, 8, scoring, bias, groups, max(1, groups // 2), renormalize=renormalize)
        assert bool((idx[:2] == -1).all()) and bool((w[:2] == 0).all()) and bool(torch.isfinite(w).all())
        if biased:
            assert not bool(((idx == 10) | (idx == 11)).any())


def test_scores_that_underflow_still_have_weights():
    logits = torch.tensor([[-200.0, -201.0, -300.0, -1000.0], [-1e30, -1e30, -2e30, -3e30], [90.0, 80.0, -90.0, -800.0]])
    _, w = _check_route(logits, 2, 'sigmoid')
    assert bool(((w.sum(-1) - 1).abs() < 1e-6).all())
    _check_route(logits, 2, 'softmax')
    _check_route(logits, 2, 'softmax', renormalize=False)


@pytest.mark.parametrize('tokens', [1, 3, 4, 5, 127, 2000])
def test_token_counts_strides_and_given_outputs(tokens):
    wide = torch.full((tokens, 80), 50.0, device='cuda')
    logits = _logits(tokens, 64, 31)
    wide[:, 8:72] = logits.cuda()
    idx = torch.full((tokens + 2, 8), -7, device='cuda')
    w = torch.full((tokens + 2, 8), 7.0, device='cuda')
    bias = _bias(64, 32)
    got = G.route_for_gc_moe(wide[:, 8:72], 8, scoring='sigmoid', bias=bias.cuda(), out=(idx[1:-1], w[1:-1]))
    want_idx, want_w = G.route_for_gc_moe(logits.cuda(), 8, scoring='sigmoid', bias=bias.cuda())
    assert got[0].data_ptr() == idx[1:].data_ptr() and torch.equal(got[0], want_idx) and torch.equal(got[1], want_w)
    for guard, value in ((idx, -7), (w, 7.0)):
        assert bool((guard[0] == value).all()) and bool((guard[-1] == value).all())
    n = min(tokens, 40)
    ref_idx, _ = _route_reference(logits[:n], 8, 'sigmoid', bias, 1, 1, 'top2', True, 1.0)
    assert torch.equal(want_idx[:n].cpu(), ref_idx)
    odd = torch.zeros((tokens, 67), device='cuda')        # rows that start at every alignment
    odd[:, :64] = logits.cuda()
    assert torch.equal(G.route_for_gc_moe(odd[:, :64], 8, scoring='sigmoid', bias=bias.cuda())[0], want_idx)


def test_no_tokens_and_routing_argument_errors():
    logits = _logits(4, 64, 41).cuda()
    idx, w = G.route_for_gc_moe(logits[:0], 8)
    assert idx.shape == (0, 8) and w.shape == (0, 8)
    call = G.route_for_gc_moe
    good = (torch.empty((4, 8), dtype=torch.int64, device='cuda'), torch.empty((4, 8), device='cuda'))
    for bad in (lambda: call(logits.double(), 8), lambda: call(logits[0], 8), lambda: call(logits.T, 8), lambda: call(logits.cpu(), 8),
                lambda: call(logits, 0), lambda: call(logits, 33), lambda: call(logits[:, :4], 8), lambda: call(logits, 8, scoring='relu'),
                lambda: call(logits, 8, group_score='sum'), lambda: call(logits, 8, num_groups=3),
                lambda: call(logits, 8, num_groups=16, topk_groups=1), lambda: call(logits, 8, bias=torch.zeros(64)),
                lambda: call(logits, 8, bias=torch.zeros(63, device='cuda')), lambda: call(logits, 8, scale=INF),
                lambda: call(logits, 8, out=(good[0].int(), good[1])), lambda: call(logits, 8, out=(good[0], good[1][:3])),
                lambda: call(logits, 7, out=good), lambda: call(logits, 8, out=(None, good[1])),
                lambda: call(logits, 8, out=(good[0], None)), lambda: call(None, 8), lambda: call(logits, 8, bias=[0.0] * 64)):
        with pytest.raises(ValueError):
            bad()
