"""Muon's parameter groups: what a group takes from the optimizer, whenever it is added (CPU; steps on the GPU)."""
import pytest
import torch

from igr.optim import Adam, Muon

SETTINGS = ('lr', 'momentum', 'nesterov', 'ns_steps', 'ns_coeffs')


def weight(r, c, device='cpu'):
    return torch.nn.Parameter(torch.randn(r, c, device=device))


def test_a_group_added_later_is_as_one_given_at_first():
    given = [{'params': [weight(8, 8)], 'orthogonal': True}, {'params': [weight(3, 4)]}]
    kw = dict(lr=1e-3, orthogonal_lr=0.07, momentum=0.8, nesterov=False, ns_steps=3, ns_coeffs=[1.5, -0.5, 0.0])
    at_once = Muon(given, **kw)
    later = Muon([{'params': [weight(2, 2)]}], **kw)
    later.add_param_group({'params': weight(8, 8), 'orthogonal': True})
    later.add_param_group({'params': [weight(3, 4)]})
    for a, b in zip(at_once.param_groups, later.param_groups[1:]):
        assert {k: v for k, v in a.items() if k != 'params'} == {k: v for k, v in b.items() if k != 'params'}
    assert [later.param_groups[1][k] for k in SETTINGS] == [0.07, 0.8, False, 3, (1.5, -0.5, 0.0)]
    assert later.param_groups[2]['orthogonal'] is False and later.param_groups[2]['lr'] == 1e-3
    later.add_param_group({'params': [weight(5, 5)], 'orthogonal': True, 'lr': 0.5, 'momentum': 0.1})
    assert later.param_groups[3]['lr'] == 0.5 and later.param_groups[3]['momentum'] == 0.1


def test_a_group_added_later_is_checked():
    opt = Muon([weight(4, 4)])
    for bad in (torch.nn.Parameter(torch.zeros(4)), torch.nn.Parameter(torch.zeros(4, 4, dtype=torch.float64))):
        with pytest.raises(ValueError, match='2-D float32'):
            opt.add_param_group({'params': [bad], 'orthogonal': True})
    assert len(opt.param_groups) == 1


def test_a_state_saved_under_another_rule_is_refused():
    p, q = weight(4, 4), weight(4, 4)
    with pytest.raises(ValueError, match='another rule'):
        Muon([p]).load_state_dict(Adam([q]).state_dict())
    with pytest.raises(ValueError, match='another rule'):
        Muon([{'params': [p]}]).load_state_dict(Muon([q]).state_dict())
    with pytest.raises(ValueError, match='number of parameter groups'):
        Muon([p]).load_state_dict(Muon([{'params': [q], 'orthogonal': True}, {'params': [weight(2, 2)]}]).state_dict())


def test_an_adam_state_and_older_settings_load():
    opt = Muon([{'params': [weight(4, 4)]}], lr=0.5)
    opt.load_state_dict(Adam([weight(4, 4)], lr=0.25).state_dict())
    assert opt.param_groups[0]['orthogonal'] is False and opt.param_groups[0]['lr'] == 0.25
    state = Muon([weight(4, 4)], momentum=0.7).state_dict()
    del state['param_groups'][0]['ns_steps']
    kept = {k: v for k, v in state['param_groups'][0].items()}
    opt = Muon([weight(4, 4)], ns_steps=2)
    opt.load_state_dict(state)
    assert opt.param_groups[0]['ns_steps'] == 2 and opt.param_groups[0]['momentum'] == 0.7
    assert state['param_groups'][0] == kept


@pytest.mark.gpu
def test_groups_added_later_step():
    torch.manual_seed(0)
    a, b, c = weight(16, 8, 'cuda'), weight(8, 24, 'cuda'), torch.nn.Parameter(torch.randn(5, device='cuda'))
    twins = [torch.nn.Parameter(p.detach().clone()) for p in (a, b, c)]
    later = Muon([{'params': [a], 'orthogonal': True}])
    later.add_param_group({'params': [b], 'orthogonal': True})
    later.add_param_group({'params': [c]})
    at_once = Muon([{'params': twins[:1], 'orthogonal': True}, {'params': twins[1:2], 'orthogonal': True}, {'params': twins[2:]}])
    for _ in range(2):
        for p, q in zip((a, b, c), twins):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.clone()
        later.step()
        at_once.step()
    for p, q in zip((a, b, c), twins):
        assert torch.equal(p, q)
