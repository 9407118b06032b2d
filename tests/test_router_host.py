"""Host side of the operators in front of the layer (norm with 8-bit output,
router logits, routing): struct layouts, argument errors and the router weight's
planes, none of which needs a GPU."""
import ctypes
import os
import subprocess

import pytest
import torch

import gc_moe_b200 as G
from gc_moe_b200 import _native, build
from gc_moe_b200.router import check_routing

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope='module')
def lib():
    build.build()
    return _native.library()


def test_structs_match_the_header(tmp_path):
    structs = {'gcmoe_norm_args': (_native.NormArgs, ('shared_sf', 'hidden', 'eps', 'device')),
               'gcmoe_logits_args': (_native.LogitsArgs, ('x_stride', 'planes', 'device')),
               'gcmoe_route_args': (_native.RouteArgs, ('logits_stride', 'renormalize', 'scale', 'device'))}
    lines = [f'printf("%zu\\n", sizeof({c}));' + ''.join(f'printf("%zu\\n", offsetof({c}, {m}));' for m in members)
             for c, (_, members) in structs.items()]
    src = tmp_path / 'sizes.c'
    src.write_text('#include <stdio.h>\n#include "gcmoe.h"\nint main(void){' + ''.join(lines) + 'return 0;}\n')
    exe = tmp_path / 'sizes'
    subprocess.run(['gcc', '-I', os.path.join(ROOT, 'include'), str(src), '-o', str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = [v for s, members in structs.values()
            for v in (ctypes.sizeof(s), *(getattr(s, m).offset for m in members))]
    assert got == want


def _refused(fn, struct, good, bad):
    for change in bad:
        args = struct(**{**good, **change})
        assert fn(ctypes.byref(args), None) in (_native.ERR_INVALID, _native.ERR_UNSUPPORTED), change
        assert _native.last_error()
    # nothing to do: nothing is launched, no device is asked for
    assert fn(ctypes.byref(struct(**{**good, 'num_tokens': 0})), None) == 0
    assert fn(None, None) == _native.ERR_INVALID


def test_norm_argument_errors(lib):
    good = dict(x=0x1000, weight=0x2000, x_q=0x3000, x_sf=0x4000, normed=0x5000, residual=0x6000, residual_out=0x6000,
                x_stride=1024, residual_stride=1024, normed_stride=1024, residual_out_stride=1024, num_tokens=4,
                hidden=1024, eps=1e-6)
    _refused(lib.gcmoe_rms_norm, _native.NormArgs, good, (
        dict(hidden=0), dict(hidden=1000), dict(hidden=32800), dict(x=0), dict(x=0x1008), dict(x_stride=1028),
        dict(weight=0), dict(weight=0x2004), dict(x_q=0), dict(x_q=0x3004), dict(x_sf=0), dict(x_sf=0x4002),
        dict(residual=0), dict(residual_out=0), dict(residual=0x6008), dict(residual_stride=1026),
        dict(residual_f32=1, residual_out_stride=1026), dict(normed=0x5008), dict(normed_stride=1028),
        dict(normed_stride=512), dict(residual_out_stride=0), dict(eps=-1.0), dict(eps=float('nan')),
        dict(eps=float('inf')), dict(shared_sf=0x7000, shared_sf_rows=64, block_m=16, num_tokens=200),
        dict(shared_sf=0x7000, shared_sf_rows=4096, block_m=0), dict(shared_sf=0x7000, shared_sf_rows=4096, block_m=24),
        dict(shared_sf=0x7000, shared_sf_rows=4096, block_m=16, hidden=1056)))


def test_logits_argument_errors(lib):
    good = dict(x=0x1000, weight=0x2000, out=0x3000, x_stride=1024, num_tokens=4, hidden=1024, num_experts=8, planes=1)
    _refused(lib.gcmoe_router_logits, _native.LogitsArgs, good, (
        dict(hidden=0), dict(hidden=1004), dict(num_experts=0), dict(num_experts=2049), dict(planes=0), dict(planes=2),
        dict(x=0), dict(x=0x1008), dict(x_stride=1028), dict(weight=0), dict(weight=0x2008), dict(out=0), dict(out=0x3002)))


def test_route_argument_errors(lib):
    good = dict(logits=0x1000, topk_idx=0x2000, topk_weights=0x3000, logits_stride=256, num_tokens=4, num_experts=256,
                topk=8, num_groups=8, topk_groups=4, sigmoid=1, scale=1.0)
    _refused(lib.gcmoe_route, _native.RouteArgs, good, (
        dict(topk=0), dict(topk=33), dict(num_experts=0), dict(num_experts=2056), dict(num_groups=0), dict(num_groups=33),
        dict(num_groups=7), dict(topk_groups=0), dict(topk_groups=9), dict(num_experts=16, topk=9), dict(logit_type=3),
        dict(logits=0), dict(logits=0x1002), dict(bias=0x4002), dict(topk_idx=0), dict(topk_idx=0x2004),
        dict(topk_weights=0), dict(topk_weights=0x3002), dict(scale=float('inf')), dict(scale=float('nan')),
        dict(num_experts=2040, num_groups=17, topk_groups=17)))


def test_python_refusals_without_a_gpu(lib):
    x = torch.zeros((4, 1024), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match='CUDA'):
        G.rms_norm_for_gc_moe(x, torch.ones(1024))
    with pytest.raises(ValueError, match='CUDA'):
        G.router_logits_for_gc_moe(x, torch.zeros((1, 8, 1024), dtype=torch.bfloat16))
    with pytest.raises(ValueError, match='CUDA'):
        G.route_for_gc_moe(torch.zeros((4, 8)), 2)


@pytest.mark.parametrize('change,error', [
    (dict(scoring='tanh'), ValueError), (dict(group_score='mean'), ValueError), (dict(topk=0), ValueError),
    (dict(topk=33), ValueError), (dict(num_groups=0), ValueError), (dict(num_groups=7), ValueError),
    (dict(num_groups=64), ValueError), (dict(topk_groups=9), ValueError), (dict(topk_groups=0), ValueError),
    (dict(experts=0), ValueError), (dict(experts=2056), ValueError), (dict(experts=16, topk_groups=2), ValueError),
    (dict(experts=2040, num_groups=17), NotImplementedError), (dict(scale=float('inf')), ValueError),
    (dict(scale=float('nan')), ValueError), (dict(bias=torch.zeros(255)), ValueError),
    (dict(bias=torch.zeros(256, dtype=torch.float64)), ValueError), (dict(bias=torch.zeros(512)[::2]), ValueError),
    (dict(bias=torch.zeros(256), device=0), ValueError)])
def test_routing_options(change, error):
    good = dict(experts=256, topk=8, scoring='sigmoid', bias=None, num_groups=8, topk_groups=4, group_score='top2',
                scale=1.0, device=-1)
    check_routing(**good)
    check_routing(**{**good, 'bias': torch.zeros(256)})
    with pytest.raises(error):
        check_routing(**{**good, **change})


def test_every_group_count_that_the_host_accepts_fits_a_warp():
    """The host's limit is the kernel's: groups x lanes within a warp, at most 64 experts a lane."""
    for groups in range(1, 33):
        lanes = 1
        while lanes * 2 * groups <= 32:
            lanes *= 2
        assert lanes == 1 << (32 // groups).bit_length() - 1
        most = min(2048 // groups, 64 * lanes)
        check_routing(most * groups, 1, 'softmax', None, groups, groups, 'max', 1.0, -1)
        if (most + 1) * groups <= 2048:
            with pytest.raises(NotImplementedError):
                check_routing((most + 1) * groups, 1, 'softmax', None, groups, groups, 'max', 1.0, -1)


def test_router_weight_planes_sum_to_the_weight():
    g = torch.Generator().manual_seed(1)
    w = torch.randn((5, 64), generator=g) * torch.exp2(torch.randint(-60, 60, (5, 64), generator=g).float())
    w[0, :4] = torch.tensor([0.0, -0.0, 1 + 2.0 ** -23, -(2 - 2.0 ** -23)])
    planes = G.transform_router_weight_for_gc_moe(w)
    assert planes.shape == (3, 5, 64) and planes.dtype == torch.bfloat16 and planes.is_contiguous()
    assert torch.equal(planes.double().sum(0), w.double())
    # in the kernel's order the sums are exact in f32 too
    assert torch.equal(planes[0].float() + (planes[1].float() + planes[2].float()), w)
    half = torch.randn((3, 16), generator=g).half()
    assert torch.equal(G.transform_router_weight_for_gc_moe(half).double().sum(0), half.double())


def test_router_weight_of_bf16_values_is_one_plane():
    w = torch.randn((4, 32)).to(torch.bfloat16)
    planes = G.transform_router_weight_for_gc_moe(w)
    assert planes.shape == (1, 4, 32) and planes.data_ptr() == w.data_ptr()
    stored = G.transform_router_weight_for_gc_moe(w.float())
    assert stored.shape == (1, 4, 32) and torch.equal(stored, planes)
    strided = torch.randn((32, 4)).to(torch.bfloat16).T
    assert torch.equal(G.transform_router_weight_for_gc_moe(strided)[0], strided)


def test_router_weight_refusals():
    for bad in (torch.zeros(4), torch.zeros((2, 4, 4)), torch.zeros((4, 4), dtype=torch.float64)):
        with pytest.raises(ValueError):
            G.transform_router_weight_for_gc_moe(bad)
    for value in (float('inf'), float('nan'), 3.4e38):
        with pytest.raises(ValueError, match='finite'):
            G.transform_router_weight_for_gc_moe(torch.full((1, 8), value))
