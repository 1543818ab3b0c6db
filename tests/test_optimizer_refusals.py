"""Arguments that the gradient-norm, clipping and AdamW entry points refuse ahead of any launch (no GPU needed)."""
import ctypes
import math
from array import array

import pytest
import torch

from nerf_amd import _lib, ops, optim

ARG, SIZE = -1, -3
CPU = torch.zeros(8)


def _list(ptrs=(0x10000,), numels=(4,), dtypes=(0,)):
    return array('Q', ptrs), array('q', numels), array('i', dtypes)


def _norm(ptrs=(0x10000,), numels=(4,), dtypes=(0,), kind=2, ws=0x20000, bytes_=1 << 20, norm=0x30000, n=None, clip=None):
    a = _list(ptrs, numels, dtypes)
    L = _lib.lib()
    args = [x.buffer_info()[0] for x in a] + [len(ptrs) if n is None else n, kind]
    if clip is not None:
        return L.nerf_clip_grad_norm(*args, clip, ws, bytes_, norm, None)
    return L.nerf_grad_norm(*args, ws, bytes_, norm, None)


@pytest.mark.parametrize('clip', [None, 1.0])
@pytest.mark.parametrize('bad', [
    dict(n=-1), dict(kind=0), dict(kind=4), dict(ws=0), dict(ws=0x20004), dict(bytes_=64), dict(norm=0), dict(ptrs=(0,)),
    dict(numels=(-1,)), dict(dtypes=(3,)), dict(dtypes=(-1,)), dict(ptrs=(0x10002,)), dict(ptrs=(0x10001,), dtypes=(1,)),
])
def test_c_list_arguments(bad, clip):
    assert _norm(clip=clip, **bad) == ARG


@pytest.mark.parametrize('numels', [((1 << 46) + 1,), (1 << 46, 1)])
def test_c_list_too_large(numels):
    assert _norm(ptrs=(0x10000,) * len(numels), numels=numels, dtypes=(0,) * len(numels)) == SIZE


@pytest.mark.parametrize('max_norm', [-1.0, math.nan])
def test_c_max_norm(max_norm):
    assert _norm(clip=max_norm) == ARG


@pytest.mark.parametrize('ptrs,numels,dtypes', [
    ((0x10000, 0x10000), (4, 4), (0, 0)),               # the same tensor twice
    ((0x10000, 0x1000c), (4, 4), (0, 0)),               # the last entry of one is the first of the other
    ((0x10020, 0x10000, 0x10004), (4, 4, 1), (0, 0, 0)),    # one inside another, not ascending
    ((0x10008, 0x10000), (4, 5), (1, 1)),
])
def test_c_shared_memory(ptrs, numels, dtypes):
    assert _norm(ptrs=ptrs, numels=numels, dtypes=dtypes, clip=1.0) == ARG


def _adamw(n=1, numels=None, dtypes=None, param=0x10000, step=0x60000, master=None, moments=0x30000, groups=None, kind=0,
           max_norm=1.0, skip=0, ws=0x20000, bytes_=1 << 20):
    numels, dtypes = array('q', numels or [4] * n), array('i', dtypes or [0] * n)
    far = lambda base: array('Q', [base + 0x1000 * i if base else 0 for i in range(n)])    # noqa: E731
    arrays = [far(param), far(0x80000), far(moments), far(0xa0000), far(master or 0), far(step), numels, dtypes]
    addr = [a.buffer_info()[0] for a in arrays]
    if master is None:
        addr[4] = None
    t = _lib.AdamwTensors(n, *addr)
    groups = groups or [(n, 0.1, 0.9, 0.99, 1e-8, 0.0)]
    gs = (_lib.AdamwGroup * len(groups))(*[_lib.AdamwGroup(c, None, *rest) for c, *rest in groups])
    return _lib.lib().nerf_adamw_step(ctypes.byref(t), gs, len(groups), kind, max_norm, skip, ws, bytes_, None, None)


@pytest.mark.parametrize('bad', [
    dict(n=-1), dict(numels=[-1]), dict(dtypes=[7]), dict(param=0), dict(param=0x10002), dict(step=0), dict(step=0x60002),
    dict(moments=0), dict(moments=0x30002), dict(dtypes=[1]), dict(dtypes=[2], master=0x50002), dict(kind=9),
    dict(kind=2, max_norm=-0.5), dict(kind=2, max_norm=math.nan), dict(skip=1), dict(ws=0), dict(bytes_=8),
    dict(groups=[(0, 0.1, 0.9, 0.99, 1e-8, 0.0)]), dict(groups=[(2, 0.1, 0.9, 0.99, 1e-8, 0.0)]),
    dict(groups=[(-1, 0.1, 0.9, 0.99, 1e-8, 0.0)]), dict(groups=[(1, 0.1, 1.0, 0.99, 1e-8, 0.0)]),
    dict(groups=[(1, 0.1, 0.9, -0.1, 1e-8, 0.0)]), dict(groups=[(1, 0.1, 0.9, 0.99, -1.0, 0.0)]),
    dict(groups=[(1, 0.1, math.nan, 0.99, 1e-8, 0.0)]),
])
def test_c_adamw_arguments(bad):
    assert _adamw(**bad) == ARG


def test_c_adamw_nothing_to_do():
    assert _adamw(n=0, groups=[(0, 0.1, 0.9, 0.99, 1e-8, 0.0)]) == 0


@pytest.mark.parametrize('norm_type', [0, 3, 0.5, -1, math.nan, -math.inf])
def test_norm_type(norm_type):
    for call in (lambda: ops.grad_norm([CPU], norm_type), lambda: ops.clip_grad_norm_([CPU], 1.0, norm_type),
                 lambda: optim.AdamW([CPU], norm_type=norm_type)):
        with pytest.raises(ValueError, match='norm_type'):
            call()


@pytest.mark.parametrize('max_norm', [-1.0, math.nan])
def test_max_norm(max_norm):
    for call in (lambda: ops.clip_grad_norm_([CPU], max_norm), lambda: optim.AdamW([CPU], max_norm=max_norm)):
        with pytest.raises(ValueError, match='max_norm'):
            call()


@pytest.mark.parametrize('bad', [dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8),
                                 dict(weight_decay=-0.1), dict(lr=math.nan), dict(eps=math.nan)])
def test_adamw_settings(bad):
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(CPU.clone())], **bad)


def test_host_tensors():
    p = torch.nn.Parameter(CPU.clone())
    p.grad = torch.ones(8)
    for call in (lambda: ops.grad_norm([CPU]), lambda: ops.grad_norm(CPU), lambda: ops.clip_grad_norm_([CPU], 1.0),
                 lambda: optim.clip_grad_norm_(p, 1.0), lambda: optim.AdamW([p]).step()):
        with pytest.raises(RuntimeError, match='HIP device'):
            call()
    assert torch.equal(p.detach(), CPU) and torch.equal(p.grad, torch.ones(8))


@pytest.mark.parametrize('t,dense', [
    (torch.zeros(4, 6).t(), True), (torch.zeros(2, 3, 4).permute(2, 0, 1), True), (torch.zeros(1, 5)[:, ::1], True),
    (torch.zeros(2, 3, 4, 5).contiguous(memory_format=torch.channels_last), True), (torch.zeros(0, 3).t(), True),
    (torch.zeros(()), True), (torch.zeros(4, 6)[:, :3], False), (torch.zeros(1, 3).expand(4, 3), False),
    (torch.zeros(5, 1).expand(5, 1).t(), True), (torch.zeros(6, 4)[::2].t(), False),
])
def test_is_dense(t, dense):
    assert _lib.lists().is_dense(t) is dense


def test_list_reader():
    L = _lib.lists()
    for bad in (CPU, (CPU,), [3], [None], None):
        with pytest.raises(TypeError):
            L.describe(bad)
    assert L.describe([]) == (-1, b'', b'', b'', True)
    with pytest.raises(RuntimeError, match='HIP device'):
        L.describe([CPU])
    with pytest.raises(RuntimeError, match='strided'):
        L.describe([torch.zeros(3, 3).to_sparse()])
    with pytest.raises(RuntimeError, match='strided'):
        L.describe([torch.zeros(3, dtype=torch.complex64).conj().imag])
    for bad in ((), ([], {}, 1), ((), {}), ([()], {}), ([3], {})):
        with pytest.raises(TypeError):
            L.optimizer(*bad)
    p = torch.nn.Parameter(CPU.clone())
    assert L.optimizer([[p], []], {}) == (-1, [], [], b'\0' * 8, b'', b'', b'', b'', None, b'', b'', b'')
    p.grad = torch.ones(8)
    with pytest.raises(RuntimeError, match='HIP device'):
        L.optimizer([[p]], {})


def test_unsupported_optimizer_states():
    p = torch.nn.Parameter(CPU.clone())
    other = torch.optim.AdamW([p], amsgrad=True)
    with pytest.raises(ValueError, match='amsgrad'):
        optim.AdamW([p]).load_state_dict(other.state_dict())


def test_state_dict_of_the_other_optimizer():
    """torch.optim.AdamW's state loads, with its settings; fp32 moments stay fp32 beside 16-bit parameters."""
    a, b = torch.nn.Parameter(torch.randn(3, 4)), torch.nn.Parameter(torch.randn(5).bfloat16())
    other = torch.optim.AdamW([{'params': [a], 'lr': 0.5}, {'params': [b], 'weight_decay': 0.25}])
    a.grad, b.grad = torch.randn(3, 4), torch.randn(5).bfloat16()
    other.step()
    mine = optim.AdamW([{'params': [a]}, {'params': [b]}], max_norm=1.0)
    mine.load_state_dict(other.state_dict())
    assert mine.param_groups[0]['lr'] == 0.5 and mine.param_groups[1]['weight_decay'] == 0.25
    assert all(g['capturable'] and 'foreach' not in g for g in mine.param_groups)
    for p in (a, b):
        st = mine.state[p]
        assert st['exp_avg'].dtype == st['exp_avg_sq'].dtype == st['step'].dtype == torch.float32
        assert float(st['step']) == 1.0
        assert torch.equal(st['exp_avg'], other.state[p]['exp_avg'].float())
        assert st['exp_avg'].data_ptr() != other.state[p]['exp_avg'].data_ptr()
    moments = mine.state_dict()
    moments['state'][1]['exp_avg'] = torch.full((5,), 1.0 + 2.0 ** -20)
    mine.load_state_dict(moments)
    assert torch.equal(mine.state[b]['exp_avg'], torch.full((5,), 1.0 + 2.0 ** -20))


def test_copies_of_an_optimizer():
    import copy
    import pickle
    p = torch.nn.Parameter(CPU.clone())
    opt = optim.AdamW([p], lr=0.25, max_norm=2.0, norm_type=1, skip_nonfinite=True)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert (other.max_norm, other.norm_type, other.skip_nonfinite, other.grad_norm) == (2.0, 1.0, True, None)
        assert other._kind == opt._kind and other.param_groups[0]['lr'] == 0.25
        assert optim.own_max_norm(other) == 2.0
    assert optim.own_max_norm(torch.optim.AdamW([p])) is None
