"""The eval-mode fold of the router's BatchNorm follows whatever changes the statistics.  No GPU: the fold is torch code."""
import copy

import pytest
import torch


def layer():
    from omni_moe_b200.modules import OmniMoE, OmniMoEConfig
    m = OmniMoE(OmniMoEConfig(16, 32, "silu", 64, 2)).eval()
    for bn in (m.router_norm_x, m.router_norm_y):
        bn.running_mean.copy_(torch.linspace(-1, 1, 8))
        bn.running_var.copy_(torch.linspace(0.5, 2, 8))
    return m


def check(m):
    bx, by = m.router_norm_x, m.router_norm_y
    z = torch.linspace(-2, 2, 16)
    want = torch.cat([(z[s] - bn.running_mean) / torch.sqrt(bn.running_var + bn.eps) for bn, s in ((bx, slice(0, 8)), (by, slice(8, 16)))])
    scale, shift = m._bn_fold_eval()
    # an rsqrt, a product with the mean (at most 1.5 scales of magnitude 2) and the two roundings of either side
    assert ((z * scale + shift) - want).abs().max() <= 16 * 2.0 ** -23


def assign(name, value):
    def change(m):
        for bn in (m.router_norm_x, m.router_norm_y):
            setattr(bn, name, value(bn))
    return change


def in_place(m):
    m.router_norm_y.running_var.mul_(3)


def data_of(m):
    m.router_norm_y.running_var.data = m.router_norm_y.running_var * 2


CHANGES = {
    "new running_var": assign("running_var", lambda bn: torch.full((8,), 3.0)),
    "new running_mean": assign("running_mean", lambda bn: torch.full((8,), 0.25)),
    "eps": assign("eps", lambda bn: 0.5),
    "in place": in_place,
    "storage": data_of,
    "loaded": lambda m: m.load_state_dict({**m.state_dict(), "router_norm_x.running_var": torch.full((8,), 0.7)}),
}


@pytest.mark.parametrize("name", CHANGES)
def test_every_change_is_followed(name):
    m = layer()
    check(m)
    with torch.no_grad():
        # assigned tensors have their own version counters: the old ones stand where the new ones start
        for bn in (m.router_norm_x, m.router_norm_y):
            bn.running_mean, bn.running_var = bn.running_mean.clone(), bn.running_var.clone()
        check(m)
        CHANGES[name](m)
    check(m)


def test_kept_while_nothing_changes():
    m = layer()
    a, b = m._bn_fold_eval(), m._bn_fold_eval()
    assert a[0] is b[0] and a[1] is b[1]


def test_a_copy_has_its_own():
    m = layer()
    m._bn_fold_eval()
    other = copy.deepcopy(m)
    other.router_norm_x.running_var.fill_(5)
    check(other), check(m)
