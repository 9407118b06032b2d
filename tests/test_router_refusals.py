"""What the operators in front of the layer refuse before anything runs; no GPU
needed."""
import ctypes

import pytest

from gc_moe_b200 import _native, build


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
