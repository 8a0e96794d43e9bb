"""What spmm_cpp.AdamW takes over from saved states and refuses, on the host: no step is taken."""
import copy

import pytest
import torch


def _optimiser(dtype=torch.bfloat16, **options):
    import spmm_cpp
    params = [torch.nn.Parameter(torch.ones(300, dtype=dtype)), torch.nn.Parameter(torch.ones(5, 7, dtype=dtype))]
    return spmm_cpp.AdamW(params, **options), params


def _state(bits, params):
    out = {}
    for i, p in enumerate(params):
        small = dict(dtype=torch.float8_e4m3fn) if bits == 8 else dict(dtype=torch.float32)
        out[i] = dict(step=torch.tensor(3 + i), exp_avg=(torch.randn(p.shape) / 8).to(**small))
        if bits == 8:
            blocks = (p.numel() + 255) // 256
            out[i].update(root=torch.rand(p.shape).to(**small), exp_avg_scale=torch.rand(blocks), root_scale=torch.rand(blocks))
        else:
            out[i]['exp_avg_sq'] = torch.rand(p.shape)
    return out


@pytest.mark.parametrize('bits', [32, 8])
def test_hooks_around_loading(bits):
    """A hook before loading may hand over another state; a hook after it sees the state as steps read it, and what it puts there stays."""
    opt, params = _optimiser(state_bits=bits)
    given = dict(opt.state_dict(), state=_state(bits, params))
    other = copy.deepcopy(given)
    other['state'][0]['step'] = torch.tensor(77)
    seen = {}

    def after(o):
        seen.update({name: value.dtype for name, value in o.state[params[0]].items()})
        o.state[params[1]]['step'] = torch.tensor(1000)

    opt.register_load_state_dict_pre_hook(lambda o, state: other)
    opt.register_load_state_dict_post_hook(after)
    opt.load_state_dict(given)
    assert int(opt.state[params[0]]['step']) == 77 and int(opt.state[params[1]]['step']) == 1000
    assert seen == {name: value.dtype for name, value in given['state'][0].items()}
    for name, value in given['state'][0].items():
        got = opt.state[params[0]][name]
        assert got.dtype == value.dtype and (name == 'step' or torch.equal(got.float(), value.float()))
    assert opt.state[params[0]]['exp_avg'].data_ptr() != other['state'][0]['exp_avg'].data_ptr()
    opt.load_state_dict(given)                                     # the hooks of the first call are gone, the user's are not
    assert len(opt._optimizer_load_state_dict_pre_hooks) == 1 and len(opt._optimizer_load_state_dict_post_hooks) == 1


def test_states_of_other_steps_are_refused():
    """Nothing has changed after a refusal; what differs in nothing but its name is taken."""
    opt, params = _optimiser(torch.float32, lr=0.5)

    def saved(kind, **options):
        twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
        other = kind(twins, **options)
        for p in twins:
            p.grad = torch.ones_like(p)
        other.step()
        return other.state_dict()

    for bad in (saved(torch.optim.AdamW, amsgrad=True), saved(torch.optim.AdamW, maximize=True), saved(torch.optim.Adam, weight_decay=0.1)):
        with pytest.raises(ValueError, match='cannot be taken over'):
            opt.load_state_dict(bad)
        assert opt.param_groups[0]['lr'] == 0.5 and not opt.state
    bad = saved(torch.optim.AdamW)
    bad['param_groups'][0]['betas'] = (1.5, 0.9)
    with pytest.raises(ValueError, match='betas'):
        opt.load_state_dict(bad)
    assert opt.param_groups[0]['betas'] == (0.9, 0.999) and not opt.state
    for good in (saved(torch.optim.AdamW, lr=0.25), saved(torch.optim.Adam, lr=0.25), saved(torch.optim.AdamW, lr=torch.tensor(0.25), foreach=False)):
        opt.load_state_dict(good)
        assert opt.param_groups[0]['lr'] == 0.25 and type(opt.param_groups[0]['lr']) is float and int(opt.state[params[0]]['step']) == 1
        assert opt.state[params[0]]['step'].dtype == torch.int64


def test_a_refused_group_is_not_kept():
    opt, params = _optimiser()
    more = torch.nn.Parameter(torch.ones(3))
    for bad in (dict(betas=(2.0, 0.9)), dict(lr=-1.0), dict(eps=float('nan')), dict(lr=torch.tensor(0.1))):
        with pytest.raises(ValueError):
            opt.add_param_group(dict(params=[more], **bad))
        assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[more], lr=0.1))
    assert len(opt.param_groups) == 2 and opt.param_groups[1]['lr'] == 0.1
