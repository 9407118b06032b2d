"""What the operators in front of the layer refuse before anything runs; only the
test marked ``gpu`` needs a GPU."""
import ctypes

import pytest
import torch

import gc_moe_b200 as G
from gc_moe_b200 import _native, build
from gc_moe_b200.router import check_routing


@pytest.fixture(scope='module')
def lib():
    build.build()
    return _native.library()


def test_counts_beyond_the_kernels_reach(lib):
    """A grid counts blocks of four rows in 32 bits, and a tensor map's coordinates are signed."""
    route = dict(logits=0x1000, topk_idx=0x2000, topk_weights=0x3000, logits_stride=0, num_experts=8, topk=2,
                 num_groups=1, topk_groups=1, scale=1.0, device=-1)
    logits = dict(x=0x1000, weight=0x2000, out=0x3000, x_stride=0, num_experts=8, planes=1, device=-1)
    norm = dict(x=0x1000, weight=0x2000, x_q=0x3000, x_sf=0x4000, hidden=32, eps=1e-6, device=-1)
    for fn, struct, good, bad, word in (
            (lib.gcmoe_route, _native.RouteArgs, route, dict(num_tokens=2 ** 31), 'tokens'),
            (lib.gcmoe_route, _native.RouteArgs, route, dict(num_tokens=2 ** 32 - 1), 'tokens'),
            (lib.gcmoe_rms_norm, _native.NormArgs, norm, dict(num_tokens=2 ** 31), 'tokens'),
            (lib.gcmoe_router_logits, _native.LogitsArgs, logits, dict(num_tokens=262141, hidden=1024), 'tokens'),
            (lib.gcmoe_router_logits, _native.LogitsArgs, logits, dict(num_tokens=1, hidden=2 ** 30 + 8), 'hidden'),
            (lib.gcmoe_router_logits, _native.LogitsArgs, logits, dict(num_tokens=1, hidden=2 ** 32 - 8), 'hidden')):
        assert fn(ctypes.byref(struct(**{**good, **bad})), None) == _native.ERR_INVALID, bad
        assert word in _native.last_error(), _native.last_error()


@pytest.mark.parametrize('change', [dict(topk=8.0), dict(num_groups=8.0), dict(topk_groups=4.0), dict(topk_groups='4'),
                                    dict(num_groups=None), dict(scale='1'), dict(scale=None)])
def test_options_of_another_kind(change):
    """The check that stands in front of the norm refuses what the routing's call behind it would refuse."""
    good = dict(experts=256, topk=8, scoring='sigmoid', bias=None, num_groups=8, topk_groups=4, group_score='top2',
                scale=1.0, device=-1)
    check_routing(**good)
    with pytest.raises(TypeError):
        check_routing(**{**good, **change})


@pytest.mark.gpu
def test_options_of_another_kind_leave_the_residual_alone(single_rank_group):
    buf = G.get_symm_buffer_for_gc_moe(single_rank_group, 8, 256, 2, 1024, 512)
    try:
        x = torch.randn((4, 1024), device='cuda').to(torch.bfloat16)
        residual, w = x * 2, torch.ones(1024, device='cuda')
        planes = G.transform_router_weight_for_gc_moe(torch.zeros((8, 1024), dtype=torch.bfloat16, device='cuda'))
        before = residual.clone()
        for bad in (dict(num_groups=4, topk_groups=2.0), dict(num_groups=4.0), dict(scale='2'),
                    dict(renormalize=torch.ones(2))):
            with pytest.raises((TypeError, RuntimeError)):
                G.stage_normed_inputs_for_gc_moe(buf, x, w, planes, residual, residual_out=residual, **bad)
        torch.cuda.synchronize()
        assert torch.equal(residual, before)
    finally:
        buf.destroy()
