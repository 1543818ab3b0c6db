"""Corners of the gradient norm, clipping and the AdamW step that need a device: coefficients below fp32's normal range,
the norm that an optimizer shows, empty lists at the C entry.  Tolerances as counted in test_gpu_optimizer."""
import ctypes

import pytest
import torch

from tests.test_gpu_optimizer import (DTYPES, HALF_STEP, NORMS, SIZES, TINY, U, check_step, gen, make, make_state,
                                      near_norm, norm64, optimizer, params_of, snapshot)

pytestmark = pytest.mark.gpu


# ---- coefficients below the normal range of fp32 ------------------------------------------------------------------

def huge(dtype, n=4099):
    """Entries of the size of the type's largest; their norm is beyond fp32 (but for fp16)."""
    x = torch.rand(n, device='cuda', generator=gen(9)) * 0.5 + 0.5
    x[::3] *= -1
    return (x.double() * 0.99 * torch.finfo(dtype).max).to(dtype)


# the coefficient itself: normal, on both sides of 2^-126, subnormal, below the smallest subnormal, and far below
COEFFICIENTS = [2.0 ** -100, 2.0 ** -126 * (1 + 2.0 ** -10), 2.0 ** -126 * (1 - 2.0 ** -10), 2.0 ** -133, 1.1e-43, 2.0 ** -151,
                3e-48, 1e-60, 1e-200]


@pytest.mark.parametrize('coefficient', COEFFICIENTS)
@pytest.mark.parametrize('norm_type', NORMS)
@pytest.mark.parametrize('dtype', DTYPES)
def test_clip_by_a_coefficient_below_the_normal_range(dtype, norm_type, coefficient):
    from nerf_amd import ops
    t = huge(dtype)
    was, norm = t.double(), norm64([t], norm_type)
    got = ops.clip_grad_norm_(t, coefficient * norm, norm_type)
    assert float(got) == float(torch.tensor(norm, dtype=torch.float64).float())
    want = was * (coefficient * norm / (norm + 1e-6))
    # the coefficient, the product, the rounding to the type; below the normal ranges half a smallest step of both types
    tol = want.abs() * (2 * U + HALF_STEP[dtype]) * (1 + U) + TINY[dtype] + 2.0 ** -150
    off = (t.double() - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize('coefficient', COEFFICIENTS)
@pytest.mark.parametrize('dtype', DTYPES)
def test_adamw_with_a_coefficient_below_the_normal_range(dtype, coefficient):
    p = torch.nn.Parameter(make([4099], dtype, scale=0.3)[0].clone())
    p.grad = huge(dtype)
    norm = norm64([p.grad], 2.0)
    states = make_state([p], 0)             # (moments of zero: what the gradient adds is all there is)
    was = snapshot([p], states)
    opt = optimizer([p], states, max_norm=coefficient * norm)
    opt.step()
    check_step([p], was, states, 1, coefficient * norm / (norm + 1e-6))


# ---- the norm that an optimizer shows -----------------------------------------------------------------------------

def test_grad_norm_after_eager_and_captured_steps():
    """Whatever ran last, an eager step or a replay of either graph: grad_norm is its norm."""
    from nerf_amd import optim
    ps = params_of(SIZES['network'], torch.float32)
    opt = optim.AdamW(ps, lr=1e-4, max_norm=0.5)
    kept = []
    for k in range(2):
        ps[0].grad.mul_(1.5)
        opt.step()
        kept.append((opt.grad_norm, norm64([p.grad for p in ps], 2.0)))
    graphs = []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            opt.step()
    for k, run in enumerate((graphs[0].replay, opt.step, graphs[0].replay, graphs[1].replay, graphs[0].replay, opt.step, opt.step,
                             graphs[1].replay)):
        for p in ps:
            p.grad.copy_(torch.randn(p.shape, device='cuda', generator=gen(50 + k)) * (0.1 + 0.05 * k))
        run()
        torch.cuda.synchronize()
        near_norm(opt.grad_norm, norm64([p.grad for p in ps], 2.0))
    for got, want in kept:          # eager steps ahead of a capture: a tensor each, which nothing writes again
        near_norm(got, want)
    for p in ps:
        p.grad = None
    opt.step()
    assert float(opt.grad_norm) == 0


# ---- the C entry with nothing to update ---------------------------------------------------------------------------

@pytest.mark.parametrize('kind', [1, 2, 3])
def test_c_adamw_of_an_empty_list_writes_the_norm(kind):
    from nerf_amd import _lib
    L = _lib.lib()
    norm = torch.full((3,), 5.0, device='cuda')
    torch.cuda.synchronize()
    t = _lib.AdamwTensors(0, *([None] * 8))
    assert L.nerf_adamw_step(ctypes.byref(t), None, 0, kind, 1.0, 0, None, 0, norm[1:].data_ptr(), None) == 0
    torch.cuda.synchronize()
    assert norm.tolist() == [5.0, 0.0, 5.0]
