"""Loading the AdamW step's state: hooks, the groups' own options, extra entries, and the settings that it accepts (no GPU
needed)."""
import pytest
import torch

from nerf_amd import optim


def two():
    return [torch.nn.Parameter(torch.zeros(4)), torch.nn.Parameter(torch.zeros(4))]


def saved(a, b):
    """The state dict of an optimizer whose two parameters' moments are `a` and `b` throughout."""
    ps = two()
    opt = torch.optim.AdamW(ps)
    for p, x in zip(ps, (a, b)):
        opt.state[p] = dict(step=torch.tensor(3.0), exp_avg=torch.full((4,), x), exp_avg_sq=torch.full((4,), x * x))
    return opt.state_dict()


def swapped(state_dict):
    """The same state dict for the parameters in the other order."""
    state = state_dict['state']
    return dict(state_dict, state={0: state[1], 1: state[0]})


@pytest.mark.parametrize('cls', [optim.AdamW, torch.optim.AdamW])
def test_a_pre_hook_decides_what_is_loaded(cls):
    ps = two()
    opt = cls(ps)
    opt.register_load_state_dict_pre_hook(lambda _, sd: swapped(sd))
    given = saved(0.2, 0.1)
    opt.load_state_dict(given)
    for p, x in zip(ps, (0.1, 0.2)):
        assert torch.equal(opt.state[p]['exp_avg'], torch.full((4,), x))
        assert torch.equal(opt.state[p]['exp_avg_sq'], torch.full((4,), x * x))
        assert float(opt.state[p]['step']) == 3.0
    opt.load_state_dict(given)              # (a second time: nothing of the first is left behind)
    assert torch.equal(opt.state[ps[0]]['exp_avg'], torch.full((4,), 0.1))


def test_a_pre_hook_on_16_bit_parameters_keeps_the_moments_in_32():
    ps = [torch.nn.Parameter(torch.zeros(4, dtype=torch.bfloat16)) for _ in range(2)]
    opt = optim.AdamW(ps)
    opt.register_load_state_dict_pre_hook(lambda _, sd: swapped(sd))
    opt.load_state_dict(saved(1.0 + 2.0 ** -20, 3.0))
    assert torch.equal(opt.state[ps[1]]['exp_avg'], torch.full((4,), 1.0 + 2.0 ** -20))


def test_a_pre_hook_may_bring_what_is_refused():
    opt = optim.AdamW(two())
    other = torch.optim.AdamW(two(), amsgrad=True).state_dict()
    opt.register_load_state_dict_pre_hook(lambda _, sd: other)
    before = opt.state_dict()
    with pytest.raises(ValueError, match='amsgrad'):
        opt.load_state_dict(saved(0.1, 0.2))
    assert opt.state_dict() == before


@pytest.mark.parametrize('cls', [optim.AdamW, torch.optim.AdamW])
def test_a_post_hook_has_the_last_word(cls):
    ps = two()
    opt = cls(ps)

    def halve(o):
        for st in o.state.values():
            st['exp_avg'].mul_(0.5)
    opt.register_load_state_dict_post_hook(halve)
    opt.load_state_dict(saved(0.5, 0.25))
    assert float(opt.state[ps[0]]['exp_avg'][0]) == 0.25 and float(opt.state[ps[1]]['exp_avg'][0]) == 0.125


@pytest.mark.parametrize('cls', [optim.AdamW, torch.optim.AdamW])
def test_a_scheduler_goes_on_after_loading(cls):
    ps = two()
    opt = cls(ps, lr=0.1)
    sched = torch.optim.lr_scheduler.OneCycleLR(opt, max_lr=0.1, total_steps=10)
    opt.load_state_dict(opt.state_dict())
    was = opt.param_groups[0]['lr']
    opt._opt_called = True                  # (no step was taken: there is no device here)
    sched.step()
    assert opt.param_groups[0]['lr'] != was and opt.param_groups[0]['max_lr'] == 0.1


def test_a_groups_own_options_are_kept_and_the_other_optimizers_settings_are_not():
    ps = two()
    groups = [dict(params=[ps[0]], name='trunk', lr_scale=0.5), dict(params=[ps[1]], name='heads')]
    opt = optim.AdamW(groups)
    opt.load_state_dict(opt.state_dict())
    assert opt.param_groups[0]['name'] == 'trunk' and opt.param_groups[0]['lr_scale'] == 0.5
    assert opt.param_groups[1]['name'] == 'heads' and 'lr_scale' not in opt.param_groups[1]
    other = torch.optim.AdamW([dict(params=[ps[0]], name='a'), dict(params=[ps[1]], name='b')], foreach=True)
    opt.load_state_dict(other.state_dict())
    for g, name in zip(opt.param_groups, 'ab'):
        assert g['name'] == name and g['capturable'] is True
        assert not {'foreach', 'fused', 'amsgrad', 'maximize', 'differentiable', 'decoupled_weight_decay'} & set(g)


def test_extra_entries_of_a_state_are_kept():
    ps = two()
    opt = optim.AdamW(ps)
    state = saved(0.1, 0.2)
    state['state'][0]['seen'] = 7
    state['state'][0]['trace'] = torch.arange(4.0)
    opt.load_state_dict(state)
    assert opt.state[ps[0]]['seen'] == 7 and torch.equal(opt.state[ps[0]]['trace'], torch.arange(4.0))
    assert 'seen' not in opt.state[ps[1]]


def test_settings_of_the_other_optimizer():
    """What asks for nothing, or for one of the other optimizer's ways to the same result, is taken; the rest is refused."""
    for kw in (dict(amsgrad=False), dict(maximize=False), dict(differentiable=False), dict(foreach=False), dict(foreach=True),
               dict(foreach=None), dict(fused=True), dict(fused=False), dict(capturable=False), dict(capturable=True)):
        opt = optim.AdamW(two(), lr=0.5, **kw)
        assert opt.param_groups[0]['lr'] == 0.5 and opt.param_groups[0]['capturable'] is True and opt.max_norm is None
    for kw in (dict(amsgrad=True), dict(maximize=True), dict(differentiable=True)):
        with pytest.raises(ValueError, match=next(iter(kw))):
            optim.AdamW(two(), **kw)
        with pytest.raises(ValueError, match=next(iter(kw))):
            optim.AdamW([dict(params=two(), **kw)])


@pytest.mark.parametrize('value', [True, False])
def test_a_truth_value_is_no_max_norm(value):
    """The other optimizer's sixth argument is amsgrad: in its place here stands a number."""
    with pytest.raises(ValueError, match='max_norm'):
        optim.AdamW(two(), 1e-3, (0.9, 0.999), 1e-8, 0.01, value)


def test_a_copy_made_before_there_was_one_norm_for_all_replays():
    state = optim.AdamW(two(), max_norm=2.0).__getstate__()
    assert state.pop('_graph_norm') is None
    other = optim.AdamW.__new__(optim.AdamW)
    other.__setstate__(state)
    assert other._graph_norm is None and other.max_norm == 2.0
