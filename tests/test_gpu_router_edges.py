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
