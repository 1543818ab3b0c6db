"""The SAR scatter inside a captured graph: every replay clears its work buffers by itself."""
import ctypes

import pytest
import torch

from tests.test_zz_no_alloc import _call, _inputs

pytestmark = pytest.mark.gpu


def test_replays_clear_the_winners():
    """Between the replays the winner buffer holds the last ray's index in every bin (what a tensor that shares the
    memory might leave): a bin that no ray reaches must come out empty, and a bin's winner is among the rays in it."""
    from nerf_amd import _lib
    L = _lib.lib()
    R, S, nsam = 200, 24, 512
    P = lambda t: ctypes.c_void_p(t.data_ptr())         # noqa: E731
    dev = 'cuda'
    ins = _inputs(R, S, nsam, 4)
    _call(False, ins, R, S, nsam)
    f = lambda *s: torch.zeros(*s, device=dev)          # noqa: E731
    pulse, dist, acc, w, alpha, comp, ray_ret = f(nsam, 2), f(R), f(R), f(R, S), f(R, S), f(R, 5), f(R, 2)
    i = lambda n: torch.zeros(n, device=dev, dtype=torch.int32)     # noqa: E731
    ray_bin, winner, status = i(R), i(nsam), i(1)
    act = _lib.NerfActivation(1, 1e-4, -1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rc = L.nerf_scatter_fwd(*[P(x) for x in ins], R, S, nsam, 0.03, ctypes.byref(act), P(pulse), P(dist), P(acc), P(w),
                                P(alpha), P(ray_ret), P(ray_bin), P(comp), P(winner), P(status),
                                ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    for seed in (4, 5, 6, 7):
        for dst, src in zip(ins, _inputs(R, S, nsam, seed)):
            dst.copy_(src)
        winner.fill_(R - 1)
        status.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        want = _call(False, ins, R, S, nsam)
        assert torch.equal(pulse, want['pulse']) and int(status) == 0
        empty = torch.ones(nsam, dtype=torch.bool, device=dev)
        empty[ray_bin.long()] = False
        assert bool(empty.any()) and bool((winner[empty] == -1).all()) and not pulse[empty].any()
