"""What `optim.Muon` says to a schedule and to parameters before it touches a device."""
import pytest
import torch


@pytest.mark.parametrize("bad", [dict(ns_coefficients=(100.0, 0.0, 0.0)), dict(ns_coefficients=(float("nan"), 0.0, 0.0)), dict(ns_steps=4, ns_coefficients=(3.0, 0.0, 0.0)),
                                 dict(ns_coefficients=(0.01, 0.0, 0.0)), dict(ns_eps=1e-60), dict(ns_eps=float("inf"))])
def test_a_schedule_that_no_step_takes_fails_at_once(bad):
    from nerf_amd.optim import Muon
    with pytest.raises(ValueError):
        Muon([torch.nn.Parameter(torch.zeros(32, 32))], **bad)


@pytest.mark.parametrize("bad", [dict(ns_steps=0), dict(momentum=1.0), dict(weight_decay=-1.0), dict(adjust_lr="other"), dict(ns_eps=0.0),
                                 dict(ns_coefficients=(100.0, 0.0, 0.0)), dict(weight_decay=float("nan"))])
def test_what_a_group_names_for_itself_is_checked_too(bad):
    from nerf_amd.optim import Muon
    for kind in (True, None):
        with pytest.raises(ValueError):
            Muon([{"params": [torch.nn.Parameter(torch.zeros(32, 32))], "muon": kind, **bad}])
