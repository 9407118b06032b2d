"""GPU tests of ``router_logits_for_gc_moe`` and ``route_for_gc_moe`` where an
address, a plane, an infinity or a launch in flight decides.

Logits are compared as in ``test_gpu_router``: the products are exact, an element
takes part in fewer than 256 additions, each of which loses at most 2^-23 of a
partial sum that is at most sum |x w|: 2^-15 * sum |x w|.
"""
import pytest
import torch

import gc_moe_b200 as G

pytestmark = pytest.mark.gpu

INF = float('inf')


def _case(tokens, experts, hidden, weight, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((tokens, hidden), generator=g).to(torch.bfloat16)
    return x, (torch.randn((experts, hidden), generator=g) * hidden ** -0.5).to(weight)


def _close(got, x, w):
    x, w = x.cuda().double(), w.cuda().double()
    return bool(((got.double() - x @ w.T).abs() <= (x.abs() @ w.abs().T) * 2.0 ** -15).all())


@pytest.mark.parametrize('weight', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('experts', [4, 100, 256, 255])
@pytest.mark.parametrize('tokens', [1, 4, 8, 9, 64, 300])
def test_logits_into_a_view_at_any_address(tokens, experts, weight):
    """A contiguous ``out`` may start at any element of its storage: the values are those of an aligned one, and what
    lies on either side stays."""
    x, w = (t.cuda() for t in _case(tokens, experts, 1024, weight, seed=tokens + experts))
    planes = G.transform_router_weight_for_gc_moe(w)
    want = G.router_logits_for_gc_moe(x, planes)
    assert want.data_ptr() % 16 == 0 and _close(want, x, w)
    size = tokens * experts
    for shift in (1, 2, 3, 4):
        flat = torch.full((size + 8,), 7.0, device='cuda')
        got = G.router_logits_for_gc_moe(x, planes, out=flat[shift:shift + size].view(tokens, experts))
        assert got.data_ptr() == flat.data_ptr() + 4 * shift
        assert torch.equal(got, want)
        assert bool((flat[:shift] == 7).all()) and bool((flat[shift + size:] == 7).all())


@pytest.mark.parametrize('weight', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('tokens,experts,hidden', [(3, 70, 2048), (8, 70, 2048), (9, 70, 2048), (150, 70, 2048), (150, 384, 512),
                                                   (300, 384, 2048), (1000, 384, 2048), (40, 65, 1000)])
def test_an_infinity_gives_what_the_formula_gives(tokens, experts, hidden, weight):
    """Whatever the number of tokens and the weight's planes: an infinite activation times the weight is an infinity of
    the weight's sign, NaN where the weight is zero or where both infinities meet.  Weights with one, two and three
    planes that are not zero, and planes of both signs."""
    x, w = _case(tokens, experts, hidden, weight, seed=tokens)
    w[:, 5:9] = torch.tensor([1.0, -2.0, 1 + 2.0 ** -10, -(1 + 2.0 ** -10 - 2.0 ** -18)])
    w[3, 5] = 0.0
    w[4, 6] = -0.0
    w[5:9, 11] = torch.tensor([2.0 ** -40, -2.0 ** -40, 1 - 2.0 ** -9, -1 + 2.0 ** -20])
    x[0, 5] = INF
    x[1, 6] = -INF
    x[2, [7, 8]] = INF                                    # infinities of both signs meet
    if tokens > 3:
        x[3, [5, 7]] = INF                                # of one sign
        x[4, 11] = INF
        x[5, hidden - 1] = -INF
        x[6, 8], x[6, 9] = INF, float('nan')
        x[7] = INF
    rows = min(tokens, 8)
    got = G.router_logits_for_gc_moe(x.cuda(), G.transform_router_weight_for_gc_moe(w.cuda())).cpu()
    # element by element: a library product need not keep infinities apart
    want = (x[:rows, None, :].double() * w[None].double()).sum(-1)
    special = ~torch.isfinite(want)
    assert bool(special.any(1).all())
    assert torch.equal(torch.isnan(got[:rows]), torch.isnan(want))
    assert torch.equal(got[:rows][special & ~torch.isnan(want)].double(), want[special & ~torch.isnan(want)])
    assert bool(torch.isfinite(got[rows:]).all())
    if tokens > rows:
        assert _close(got[rows:].cuda(), x[rows:], w)


def test_sizes_past_32_bits_are_refused():
    """Counts that do not fit the library's 32 bits must not lose their upper half (views of one row: nothing large is
    read, and a refusal allocates nothing)."""
    rows = 2 ** 32 + 3
    x = torch.zeros((1, 32), dtype=torch.bfloat16, device='cuda').expand(rows, 32)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(ValueError, match='tokens'):
        G.router_logits_for_gc_moe(x, torch.zeros((1, 1, 32), dtype=torch.bfloat16, device='cuda'))
    with pytest.raises(ValueError, match='tokens'):
        G.route_for_gc_moe(x[:, :4], 1)
    with pytest.raises(ValueError, match='tokens'):
        G.rms_norm_for_gc_moe(x, torch.ones(32, device='cuda'), normed=False)
    assert torch.cuda.max_memory_allocated() < before + 2 ** 20


def test_a_row_past_32_bits_is_refused():
    wide = torch.empty((1, 2 ** 32 + 8), dtype=torch.bfloat16, device='cuda')
    try:
        with pytest.raises(ValueError, match='hidden'):
            G.router_logits_for_gc_moe(wide, wide[None])
    finally:
        del wide
        torch.cuda.empty_cache()


@pytest.mark.parametrize('tokens', [1, 4, 8, 40])
@pytest.mark.parametrize('experts', [64, 256])
def test_launches_in_flight_read_what_the_launch_before_wrote(tokens, experts):
    """Products and routings one behind the other over ONE tensor of logits, each launched while those before it still
    run: every routing reads the product directly before it, not an earlier content of the tensor."""
    steps = 60
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn((steps, tokens, 1024), generator=g).to(torch.bfloat16).cuda()
    planes = G.transform_router_weight_for_gc_moe(torch.randn((experts, 1024), generator=g).cuda() * 0.03)
    weight = torch.ones(1024, device='cuda')
    want = []
    for step in range(steps):
        normed = G.rms_norm_for_gc_moe(x[step], weight).normed
        torch.cuda.synchronize()
        logits = G.router_logits_for_gc_moe(normed, planes)
        torch.cuda.synchronize()
        want.append([t.clone() for t in G.route_for_gc_moe(logits, 8)])
        torch.cuda.synchronize()
    logits = torch.zeros((tokens, experts), device='cuda')
    normed = torch.zeros((tokens, 1024), dtype=torch.bfloat16, device='cuda')
    out = [tuple(torch.zeros_like(t) for t in pair) for pair in want]

    def chain(with_norm):
        for step in range(steps):
            rows = x[step]
            if with_norm:
                rows = G.rms_norm_for_gc_moe(x[step], weight, normed=normed).normed
            else:
                rows = ready[step]
            G.router_logits_for_gc_moe(rows, planes, out=logits)
            G.route_for_gc_moe(logits, 8, out=out[step])

    ready = [G.rms_norm_for_gc_moe(x[step], weight).normed for step in range(steps)]
    for with_norm in (True, False):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            chain(with_norm)
        for run in (graph.replay, lambda: chain(with_norm)):
            for _ in range(20):
                for pair in out:
                    for t in pair:
                        t.zero_()
                run()
                torch.cuda.synchronize()
                for got, ref in zip(out, want):
                    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


# Tokens, experts, H: the form for few tokens with one, two and four of them a CTA and rows of one,
# two and four rounds of loads, then each tile of the tensor-core form with each split of the K range.
SIZES = [(1, 8, 2048), (2, 256, 4096), (3, 100, 7168), (8, 64, 4104), (8, 384, 2048),
         (9, 8, 64), (64, 8, 512), (9, 8, 1024), (9, 512, 1024), (150, 384, 512), (300, 384, 2048), (700, 512, 64),
         (512, 512, 512), (65, 512, 512), (65, 256, 1024), (2048, 384, 64), (700, 512, 1024), (300, 512, 2048),
         (96, 512, 7168), (1000, 384, 2048), (300, 512, 7168), (64, 256, 7168), (33, 4, 1032)]


@pytest.mark.parametrize('tokens,experts,hidden', SIZES)
def test_each_plane_takes_part_in_full(tokens, experts, hidden):
    """Planes of one size, one at a time and all together: in a real FP32 weight the third is below 2^-17 of the first,
    and its loss would drown in the bound of the sum."""
    g = torch.Generator(device='cuda').manual_seed(tokens + hidden)
    x = torch.randn((tokens, hidden), generator=g, device='cuda').to(torch.bfloat16)
    planes = torch.randn((3, experts, hidden), generator=g, device='cuda').to(torch.bfloat16)
    for kept in ((0,), (1,), (2,), (0, 1, 2)):
        some = torch.zeros_like(planes)
        some[list(kept)] = planes[list(kept)]
        got = G.router_logits_for_gc_moe(x, some)
        want = sum(x.double() @ p.double().T for p in some)
        size = sum(x.double().abs() @ p.double().abs().T for p in some)
        assert bool(((got.double() - want).abs() <= size * 2.0 ** -15).all()), kept


@pytest.mark.parametrize('weight', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('tokens,experts,hidden', [(9, 8, 65536), (64, 256, 65536), (150, 384, 65536), (300, 256, 65536),
                                                   (2048, 384, 7168), (4096, 256, 7168)])
def test_truncation_does_not_grow_with_the_row(tokens, experts, hidden, weight):
    """Terms of one sign, whose partial sums only grow.  A tensor core's addition loses less than 2^-23 of its partial
    sum; in a chain of 512 channels, 32 additions, the partial sums are i/32 of the chain's: less than 16.5 * 2^-23
    = 2.0e-6 of it, half of that on average.  The sums of the chains are rounded to nearest, which favours no side.
    One chain over these rows (at least 3584 channels a CTA) would lose 3.9e-6 to 9e-6 on average."""
    g = torch.Generator(device='cuda').manual_seed(experts)
    x = (torch.rand((tokens, hidden), generator=g, device='cuda') + 0.5).to(torch.bfloat16)
    w = (torch.rand((experts, hidden), generator=g, device='cuda') + 0.5).to(weight)
    got = G.router_logits_for_gc_moe(x, G.transform_router_weight_for_gc_moe(w))
    want = torch.cat([rows.double() @ w.double().T for rows in x.split(256)])
    bias = float(((got.double() - want) / want).mean())
    assert abs(bias) < 16.5 * 2.0 ** -23, bias
