"""The operators in front of the layer together: norm, router logits and routing
into a workspace, then the layer call, eagerly and captured in one CUDA graph."""
import pytest
import torch

import gc_moe_b200 as G
from oracle import gcmoe_oracle as O

from _cases import LayerCase
from test_gpu_norm import _check as check_norm, _inputs as norm_inputs
from test_gpu_router import _check_logits, _route_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('tokens', [1, 37, 200])
@pytest.mark.parametrize('weight', [torch.bfloat16, torch.float32])
def test_staged_inputs_feed_the_layer(single_rank_group, tokens, weight):
    e, h, i, k = 16, 1024, 512, 4
    options = dict(scoring='sigmoid', num_groups=4, topk_groups=2, scale=2.5)
    case = LayerCase(single_rank_group, e, h, i, k, seed=18)
    try:
        x, w, r = norm_inputs(tokens, h, torch.bfloat16, torch.bfloat16, seed=60 + tokens)
        g = torch.Generator().manual_seed(61)
        router = (torch.randn((e, h), generator=g) * h ** -0.5).to(weight)
        bias = torch.randn(e, generator=g) * 0.05
        planes = G.transform_router_weight_for_gc_moe(router.cuda())
        xd, wd, rd, bd = x.cuda(), w.cuda(), r.cuda(), bias.cuda()
        out = torch.empty_like(rd)
        y = torch.full((tokens, h), float('nan'), dtype=torch.bfloat16, device='cuda')

        def call():
            staged = G.stage_normed_inputs_for_gc_moe(case.buf, xd, wd, planes, rd, 1e-6, residual_out=out, bias=bd, **options)
            G.fp8_fp4_gc_moe(y, case.l1, case.l2, case.buf, activation_clamp=10.0)
            return staged

        staged = call()
        torch.cuda.synchronize()
        case.buf.raise_on_device_error()
        assert staged.block_m == case.block_m(tokens) and staged.residual is out
        check_norm(G.NormedInputs(case.buf.x[:tokens], case.buf.x_sf[:tokens], staged.normed, out), x, w, r, 1e-6)
        _check_logits(staged.logits, staged.normed, router)
        idx, wts = case.buf.topk_idx[:tokens].cpu(), case.buf.topk_weights[:tokens].cpu()
        want_idx, want_w = _route_reference(staged.logits.cpu(), k, 'sigmoid', bias, 4, 2, 'top2', True, 2.5)
        assert torch.equal(idx, want_idx) and float((wts.double() - want_w).abs().max()) <= 2.5 * 2.0 ** -16
        ref = O.moe_layer([case.buf.x[:tokens].cpu()], [case.buf.x_sf[:tokens].cpu()], [idx], [wts], case.q1, case.c1,
                          case.q2, case.c2, [staged.block_m], clamp=10.0)
        first = y.cpu().clone()
        assert torch.isfinite(first.float()).all()
        assert O.cosine(first, ref.y[0]) >= 0.9999 and O.max_rel_err(first, ref.y[0]) <= 2.0 ** -6
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            with torch.cuda.graph(graph, stream=side):
                call()
        other = norm_inputs(tokens, h, torch.bfloat16, torch.bfloat16, seed=70 + tokens)[0].cuda()
        keep = xd.clone()
        for _ in range(3):
            xd.copy_(other)                               # new inputs in the captured tensors ...
            graph.replay()
            xd.copy_(keep)                                # ... and the first ones again
            y.fill_(float('nan'))
            graph.replay()
        torch.cuda.synchronize()
        case.buf.raise_on_device_error()
        assert torch.equal(y.cpu(), first)
    finally:
        case.close()


def test_a_batch_padded_with_masked_rows(single_rank_group):
    """Routing with masked logits stages rows without routes: the layer answers zero for them."""
    case = LayerCase(single_rank_group, 8, 1024, 512, 2, seed=19)
    try:
        x, logits = torch.randn((12, 1024)).to(torch.bfloat16), torch.randn((12, 8))
        logits[7:] = float('-inf')
        rows = G.rms_norm_for_gc_moe(x.cuda(), torch.ones(1024, device='cuda'), normed=False, sym_buffer=case.buf)
        G.route_for_gc_moe(logits.cuda(), 2, out=(case.buf.topk_idx[:12], case.buf.topk_weights[:12]))
        y = torch.full((12, 1024), float('nan'), dtype=torch.bfloat16, device='cuda')
        G.fp8_fp4_gc_moe(y, case.l1, case.l2, case.buf, activation_clamp=10.0)
        torch.cuda.synchronize()
        case.buf.raise_on_device_error()
        assert rows.normed is None and bool((y[7:] == 0).all()) and bool((y[:7] != 0).any(-1).all())
    finally:
        case.close()


def test_results_do_not_depend_on_the_stream():
    """Two streams at once, each with its own tensors, give what one gives."""
    x, w, r = (t.cuda() for t in norm_inputs(300, 2048, torch.bfloat16, torch.bfloat16, seed=80))
    planes = G.transform_router_weight_for_gc_moe(torch.randn((96, 2048), device='cuda') * 0.02)

    def chain(rows):
        n = G.rms_norm_for_gc_moe(rows, w, r)
        logits = G.router_logits_for_gc_moe(n.normed, planes)
        return (n.normed, n.residual, logits, *G.route_for_gc_moe(logits, 6, scoring='sigmoid', num_groups=4, topk_groups=2))

    inputs = [x, x.flip(0).contiguous()]
    want = [chain(rows) for rows in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    got = [None, None]
    for _ in range(10):
        for s, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[s] = chain(inputs[s])
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_refusals_come_before_the_residual_is_touched(single_rank_group):
    buf = G.get_symm_buffer_for_gc_moe(single_rank_group, 8, 256, 2, 1024, 512)
    try:
        x, w, r = (t.cuda() for t in norm_inputs(4, 1024, torch.bfloat16, torch.bfloat16, seed=90))
        planes = G.transform_router_weight_for_gc_moe(torch.zeros((8, 1024), dtype=torch.bfloat16, device='cuda'))
        before = r.clone()
        for bad in (dict(scoring='tanh'), dict(num_groups=3), dict(bias=torch.zeros(7, device='cuda')), dict(scale=float('nan')),
                    dict(num_groups=8, topk_groups=1), dict(router_weight=planes[:, :4].contiguous()),
                    dict(router_weight=planes.float()), dict(x=x.float())):
            args = {**dict(x=x, router_weight=planes), **bad}
            with pytest.raises(ValueError):
                G.stage_normed_inputs_for_gc_moe(buf, args.pop('x'), w, args.pop('router_weight'), r, residual_out=r, **args)
        torch.cuda.synchronize()
        assert torch.equal(r, before)
    finally:
        buf.destroy()


def test_a_wait_that_gives_up_is_reported_once(single_rank_group):
    """The router's launches have no plan: their status is the library's, and the workspace's check reads it."""
    import ctypes
    from gc_moe_b200 import _native
    lib = _native.library()
    buf = G.get_symm_buffer_for_gc_moe(single_rank_group, 8, 256, 2, 1024, 512)
    try:
        buf.raise_on_device_error()
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        _native.raise_for(lib.gcmoe_debug_expire_producer_wait(200, stream))
        with pytest.raises(RuntimeError, match='gave up: code 1 kernel 5'):
            buf.raise_on_device_error()
        buf.raise_on_device_error()
        # and the next product is right
        x, w = torch.randn((130, 512), device='cuda').to(torch.bfloat16), torch.randn((20, 512), device='cuda').to(torch.bfloat16)
        _check_logits(G.router_logits_for_gc_moe(x, G.transform_router_weight_for_gc_moe(w)), x, w)
        buf.raise_on_device_error()
    finally:
        buf.destroy()


def test_no_tokens_are_staged(single_rank_group):
    buf = G.get_symm_buffer_for_gc_moe(single_rank_group, 8, 256, 2, 1024, 512)
    try:
        planes = G.transform_router_weight_for_gc_moe(torch.zeros((8, 1024), device='cuda'))
        x = torch.empty((0, 1024), dtype=torch.bfloat16, device='cuda')
        staged = G.stage_normed_inputs_for_gc_moe(buf, x, torch.ones(1024, device='cuda'), planes, x)
        assert staged.normed.shape == (0, 1024) and staged.residual.shape == (0, 1024) and staged.logits.shape == (0, 8)
    finally:
        buf.destroy()


def test_first_calls_of_a_process_can_be_captured():
    """No call before the capture: nothing is set up lazily that a capture forbids."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch, gc_moe_b200 as G
g = torch.Generator(device='cuda').manual_seed(1)
x = {t: torch.randn((t, 1024), device='cuda', generator=g).to(torch.bfloat16) for t in (2, 40, 300)}
w = torch.ones(1024, device='cuda')
planes = G.transform_router_weight_for_gc_moe(torch.randn((64, 1024), device='cuda', generator=g) * 0.03)
bias = torch.zeros(64, device='cuda')
def call(t):
    n = G.rms_norm_for_gc_moe(x[t], w, x[t])
    logits = G.router_logits_for_gc_moe(n.normed, planes)
    return (n.x_sf, n.normed, n.residual, logits, *G.route_for_gc_moe(logits, 4, scoring='sigmoid', bias=bias, num_groups=8, topk_groups=4))
torch.cuda.synchronize()
graphs = {}
for t in x:
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphs[t] = (graph, call(t))
for t, (graph, out) in graphs.items():
    graph.replay()
torch.cuda.synchronize()
for t, (graph, out) in graphs.items():
    assert all(torch.equal(a, b) for a, b in zip(out, call(t))), t
print('captured')
"""
    got = subprocess.run([sys.executable, '-c', code], cwd=root, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and 'captured' in got.stdout, got.stderr[-2000:]


def test_capture_with_two_streams_that_join():
    """Norm and product of one half of a batch on a side stream, of the other on the capturing one; routing after both."""
    x, w, r = (t.cuda() for t in norm_inputs(200, 1024, torch.bfloat16, torch.bfloat16, seed=95))
    planes = G.transform_router_weight_for_gc_moe(torch.randn((64, 1024), device='cuda') * 0.03)
    logits = torch.zeros((200, 64), device='cuda')

    def half(rows):
        return G.router_logits_for_gc_moe(G.rms_norm_for_gc_moe(x[rows], w, r[rows]).normed, planes, out=logits[rows])

    def both(main, side):
        side.wait_stream(main)
        with torch.cuda.stream(side):
            half(slice(0, 100))
        half(slice(100, 200))
        main.wait_stream(side)
        return G.route_for_gc_moe(logits, 4, scoring='sigmoid')

    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(main):
        want = [t.clone() for t in both(main, side)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        got = both(main, side)
    for _ in range(5):
        logits.fill_(float('nan'))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_offsets_past_32_bits():
    """Rows 2^29 + 8 elements apart: the last ones start past 2^32 elements."""
    rows, stride = 12, 2 ** 29 + 8
    big = torch.zeros((rows - 1) * stride + 1024, dtype=torch.bfloat16, device='cuda')
    x = big.as_strided((rows, 1024), (stride, 1))
    x.copy_(torch.randn((rows, 1024)).to(torch.bfloat16))
    near = x.contiguous()
    w = torch.rand(1024, device='cuda')
    planes = G.transform_router_weight_for_gc_moe(torch.randn((32, 1024), device='cuda').to(torch.bfloat16))
    assert torch.equal(G.router_logits_for_gc_moe(x, planes), G.router_logits_for_gc_moe(near, planes))      # tensor cores
    assert torch.equal(G.router_logits_for_gc_moe(x[5::3], planes), G.router_logits_for_gc_moe(near[5::3].contiguous(), planes))
    for a, b in zip(G.route_for_gc_moe(x[:, :64], 8), G.route_for_gc_moe(near[:, :64], 8)):
        assert torch.equal(a, b)
    want = G.rms_norm_for_gc_moe(near, w, near)
    got = G.rms_norm_for_gc_moe(x, w, x, residual_out=x)
    assert torch.equal(got.normed, want.normed) and torch.equal(x, want.residual) and torch.equal(got.x_sf, want.x_sf)
    del big, x, got
    torch.cuda.empty_cache()


def test_another_device_than_the_current_one_is_refused():
    import ctypes
    from gc_moe_b200 import _native
    lib = _native.library()
    x = torch.zeros((4, 1024), dtype=torch.bfloat16, device='cuda')
    p, other = x.data_ptr(), torch.cuda.current_device() + 1
    calls = ((lib.gcmoe_rms_norm, _native.NormArgs(x=p, weight=p, x_q=p, x_sf=p, x_stride=1024, num_tokens=1, hidden=1024, device=other)),
             (lib.gcmoe_router_logits, _native.LogitsArgs(x=p, weight=p, out=p, x_stride=1024, num_tokens=1, hidden=1024, num_experts=1, planes=1, device=other)),
             (lib.gcmoe_route, _native.RouteArgs(logits=p, topk_idx=p, topk_weights=p, logits_stride=8, num_tokens=1, num_experts=8, topk=1,
                                                 num_groups=1, topk_groups=1, scale=1.0, device=other)))
    for fn, args in calls:
        assert fn(ctypes.byref(args), None) == _native.ERR_INVALID
        assert 'current device' in _native.last_error()
