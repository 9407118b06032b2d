"""GPU parity of ``rms_norm_for_gc_moe`` against the formula in 64 bits.

Tolerances, derived from the roundings on the way (u = 2^-24, a half step of f32):
* v: one rounding of h, at most 70 additions of the sum of squares (half of its
  relative error survives the root), a handful of products and quotients: below
  48 u < 2^-18 relative; 2^-16 is allowed;
* BF16 outputs: half a step, 2^-8, more;
* e4m3: half a step, 2^-4 of the value, or half of the smallest step, 2^-10 of the
  scale, below the normal range; the scale is the smallest power of two that
  holds amax / 448, where an amax within 2^-16 of the border may go either way.
"""
import numpy as np
import pytest
import torch

import gc_moe_b200 as G
from gc_moe_b200.layout import sf_row_in_block
from oracle import gcmoe_oracle as O

pytestmark = pytest.mark.gpu

V_REL = 2.0 ** -16


def _inputs(tokens, hidden, residual, weight, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((tokens, hidden), generator=g).to(torch.bfloat16)
    w = (1 + 0.3 * torch.randn(hidden, generator=g)).to(weight)
    r = None
    if residual is not None:
        r = (torch.randn((tokens, hidden), generator=g) * torch.where(torch.rand(hidden, generator=g) < 0.02, 50.0, 2.0)).to(residual)
    return x, w, r


def _reference(x, w, r, eps):
    h = x.double() + (0 if r is None else r.double())
    return h, h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w.double()


def _scale_bytes(x_sf):
    return x_sf.cpu().contiguous().view(torch.uint8)


def _check(got, x, w, r, eps, normed=True):
    tokens, hidden = x.shape
    h, v = _reference(x, w, r, eps)
    codes = _scale_bytes(got.x_sf).to(torch.int64)
    assert codes.shape == (tokens, -(-hidden // 128) * 4)
    assert bool((codes[:, hidden // 32:] == 127).all())
    codes = codes[:, :hidden // 32]
    scale = torch.exp2(codes.double() - 127)
    amax = v.view(tokens, -1, 32).abs().amax(-1)
    assert bool((amax <= 448 * scale * (1 + V_REL)).all())
    assert bool(((codes == 0) | (amax > 224 * scale * (1 - V_REL))).all())
    wide = scale.repeat_interleave(32, -1)
    q = got.x.cpu().float().double() * wide
    assert bool(((q - v).abs() <= v.abs() * (2.0 ** -4 + V_REL) + wide * 2.0 ** -10).all())
    if normed:
        n = got.normed.cpu().double()
        assert bool(((n - v).abs() <= v.abs() * (2.0 ** -8 + 2 * V_REL)).all())
    else:
        assert got.normed is None
    if r is None:
        assert got.residual is None
    else:
        assert got.residual.dtype == r.dtype
        half = 2.0 ** -24 if r.dtype == torch.float32 else 2.0 ** -8 + 2.0 ** -23
        assert bool(((got.residual.cpu().double() - h).abs() <= h.abs() * half).all())


@pytest.mark.parametrize('tokens,hidden,residual,weight', [
    (1, 32, None, torch.bfloat16), (3, 96, torch.bfloat16, torch.float32), (1, 7168, torch.bfloat16, torch.bfloat16),
    (37, 5120, torch.float32, torch.float32), (5, 1056, torch.float32, torch.bfloat16),
    (130, 4096, None, torch.float32), (2, 4128, torch.bfloat16, torch.bfloat16), (9, 6144, torch.bfloat16, torch.float32),
    (4, 8192, torch.float32, torch.bfloat16), (3, 8224, torch.bfloat16, torch.bfloat16), (2, 16384, None, torch.bfloat16),
    (2, 16416, torch.bfloat16, torch.float32), (2, 32768, torch.float32, torch.float32), (700, 2048, torch.bfloat16, torch.bfloat16)])
def test_against_the_formula(tokens, hidden, residual, weight):
    x, w, r = _inputs(tokens, hidden, residual, weight, seed=tokens + hidden)
    got = G.rms_norm_for_gc_moe(x.cuda(), w.cuda(), None if r is None else r.cuda(), 1e-5)
    _check(got, x, w, r, 1e-5)
    only = G.rms_norm_for_gc_moe(x.cuda(), w.cuda(), None if r is None else r.cuda(), 1e-5, normed=False)
    _check(only, x, w, r, 1e-5, normed=False)
    assert torch.equal(only.x.view(torch.uint8), got.x.view(torch.uint8)) and torch.equal(only.x_sf, got.x_sf)


@pytest.mark.parametrize('residual', [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('hidden', [1024, 1056, 2560, 4096, 4128, 8192, 8224, 16416, 32768])
def test_a_row_has_the_same_bits_in_a_batch_of_any_size(hidden, residual):
    x, w, r = _inputs(3, hidden, residual, torch.bfloat16, seed=hidden)
    x, w, r = x.cuda(), w.cuda(), None if r is None else r.cuda()
    one = G.rms_norm_for_gc_moe(x, w, r)
    _check(one, x.cpu(), w.cpu(), None if r is None else r.cpu(), 1e-6)
    for tokens in (148, 149, 1023, 1024):
        rows = torch.arange(tokens, device='cuda') % 3
        got = G.rms_norm_for_gc_moe(x[rows], w, None if r is None else r[rows])
        assert torch.equal(got.normed, one.normed[rows]) and torch.equal(got.x_sf, one.x_sf[rows])
        assert torch.equal(got.x.view(torch.uint8), one.x.view(torch.uint8)[rows])
        assert r is None or torch.equal(got.residual, one.residual[rows])


def test_rows_that_exercise_the_scale_rule():
    """Zero rows and groups (scale byte 0 and zeros, no NaN), a row of equal values, one hot channel, tiny and
    large magnitudes."""
    x, w, _ = _inputs(8, 1024, None, torch.bfloat16, seed=5)
    x[0] = 0
    x[1, 32:64] = 0
    x[2] = 1.75
    x[3, 100] = 3e4
    x[4] *= 1e-18                      # mean square 1e-36, far below eps
    x[5] *= 1e15
    w[64:96] = 0
    got = G.rms_norm_for_gc_moe(x.cuda(), w.cuda(), eps=1e-6)
    _check(got, x, w, None, 1e-6)
    assert bool((_scale_bytes(got.x_sf)[0] == 0).all()) and bool((got.x[0].float() == 0).all())
    assert bool((_scale_bytes(got.x_sf)[:, 2] == 0).all())
    # without eps a zero row is 0 / 0, as the formula says
    nan = G.rms_norm_for_gc_moe(x[:1].cuda(), w.cuda(), eps=0.0)
    assert bool(torch.isnan(nan.normed.float()).all())


def test_a_row_with_a_nan_leaves_its_neighbours_alone():
    x, w, r = _inputs(3, 2048, torch.bfloat16, torch.bfloat16, seed=6)
    clean = G.rms_norm_for_gc_moe(x.cuda(), w.cuda(), r.cuda())
    x[1, 700] = float('nan')
    got = G.rms_norm_for_gc_moe(x.cuda(), w.cuda(), r.cuda())
    assert bool(torch.isnan(got.normed[1].float()).all()) and bool(torch.isnan(got.x[1].float()).all())
    for row in (0, 2):
        assert torch.equal(got.normed[row], clean.normed[row]) and torch.equal(got.x_sf[row], clean.x_sf[row])
        assert torch.equal(got.x[row].view(torch.uint8), clean.x[row].view(torch.uint8))


def test_strides_outputs_given_and_the_residual_in_place():
    x, w, r = _inputs(21, 1024, torch.bfloat16, torch.bfloat16, seed=7)
    plain = G.rms_norm_for_gc_moe(x.cuda(), w.cuda(), r.cuda())
    wide = torch.full((21, 3 * 1024), 7.0, dtype=torch.bfloat16, device='cuda')
    wide[:, :1024], wide[:, 1024:2048] = x.cuda(), r.cuda()
    out = torch.full((23, 1040), 7.0, dtype=torch.bfloat16, device='cuda')
    got = G.rms_norm_for_gc_moe(wide[:, :1024], w.cuda(), wide[:, 1024:2048], normed=out[1:22, 8:1032],
                                residual_out=wide[:, 1024:2048])
    assert torch.equal(got.normed, plain.normed) and torch.equal(got.residual, plain.residual)
    assert torch.equal(got.x.view(torch.uint8), plain.x.view(torch.uint8)) and torch.equal(got.x_sf, plain.x_sf)
    assert torch.equal(wide[:, :1024], x.cuda()) and bool((wide[:, 2048:] == 7).all())
    assert bool((out[0] == 7).all()) and bool((out[22] == 7).all()) and bool((out[:, :8] == 7).all()) and bool((out[:, 1032:] == 7).all())
    # one row broadcast over the batch, and a residual in place in f32
    same = G.rms_norm_for_gc_moe(x[:1].cuda().expand(21, 1024), w.cuda(), r.cuda())
    assert torch.equal(same.normed[0], plain.normed[0])
    f = r.float().cuda()
    inplace = G.rms_norm_for_gc_moe(x.cuda(), w.cuda(), f, residual_out=f)
    assert inplace.residual is f and torch.equal(f, (x.float() + r.float()).cuda())


def test_no_tokens():
    x = torch.empty((0, 1024), dtype=torch.bfloat16, device='cuda')
    got = G.rms_norm_for_gc_moe(x, torch.ones(1024, device='cuda'))
    assert got.x.shape == (0, 1024) and got.x_sf.shape == (0, 8) and got.normed.shape == (0, 1024)


@pytest.mark.parametrize('shared', [0, 1])
def test_into_a_workspace(single_rank_group, shared):
    tokens = 200
    buf = G.get_symm_buffer_for_gc_moe(single_rank_group, 8, 256, 2, 1024, 512, shared)
    try:
        x, w, r = _inputs(tokens, 1024, torch.bfloat16, torch.bfloat16, seed=8)
        buf.x.view(torch.uint8).fill_(0xAA)
        buf.x_sf.fill_(-1)
        got = G.rms_norm_for_gc_moe(x.cuda(), w.cuda(), r.cuda(), sym_buffer=buf)
        assert got.x.data_ptr() == buf.x.data_ptr() and got.x_sf.data_ptr() == buf.x_sf.data_ptr()
        _check(got, x, w, r, 1e-6)
        assert int(buf.x[tokens:].view(torch.uint8).min()) == 0xAA and bool((buf.x_sf[tokens:] == -1).all())
        if shared:
            bm = G.get_block_m_for_gc_moe(1, 8, buf.num_max_tokens_per_rank, tokens, 2)
            want, rows = O.stage_shared_sf(got.x_sf.cpu(), bm, buf.shared_l1_acts_sf.shape[0])
            assert torch.equal(buf.shared_l1_acts_sf.cpu()[rows], want[rows])
    finally:
        buf.destroy()


def test_argument_errors(single_rank_group):
    x, w, r = (t.cuda() for t in _inputs(4, 1024, torch.bfloat16, torch.bfloat16, seed=9))
    call = G.rms_norm_for_gc_moe
    for bad in (lambda: call(x.float(), w), lambda: call(x[0], w), lambda: call(x.T, w), lambda: call(x[:, :1000], w[:1000]),
                lambda: call(x, w[:512]), lambda: call(x, w.double()), lambda: call(x, w.cpu()),
                lambda: call(x, torch.ones(2048, device='cuda')[::2]), lambda: call(x, w, r.half()),
                lambda: call(x, w, r[:3]), lambda: call(x, w, r.cpu()), lambda: call(x, w, residual_out=r),
                lambda: call(x, w, r, residual_out=r.float()), lambda: call(x, w, r, normed=r.float()),
                lambda: call(x, w, r, normed=r[:2]), lambda: call(x, w, eps=-1e-6), lambda: call(x, w, eps=float('nan')),
                lambda: call(x[:, 1:993], w[:992]), lambda: call(x, w, r, normed=r[:1].expand(4, 1024)),
                lambda: call(torch.zeros((1, 32800), dtype=torch.bfloat16, device='cuda'), torch.ones(32800, device='cuda'))):
        with pytest.raises(ValueError):
            bad()
    buf = G.get_symm_buffer_for_gc_moe(single_rank_group, 8, 256, 2, 2048, 512)
    with pytest.raises(ValueError, match='hidden'):
        call(x, w, sym_buffer=buf)
    buf.destroy()
    with pytest.raises(ValueError, match='destroyed'):
        call(x, w, sym_buffer=buf)
