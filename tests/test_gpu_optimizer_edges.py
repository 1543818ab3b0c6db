"""Corners of the gradient norm, clipping and the AdamW step that need a device: the norm that an optimizer shows.
Tolerances as counted in test_gpu_optimizer."""
import pytest
import torch

from tests.test_gpu_optimizer import (SIZES, gen, near_norm, norm64, params_of)

pytestmark = pytest.mark.gpu


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
