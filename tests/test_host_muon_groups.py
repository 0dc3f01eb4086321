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


def test_named_parameters_are_split_as_plain_ones_are(monkeypatch):
    """torch's optimisers, and so `Adam`, take (name, parameter) pairs too; here up to where the device is looked at."""
    from nerf_amd.optim import Adam, Muon
    model = torch.nn.Sequential(torch.nn.Linear(40, 32), torch.nn.Linear(32, 3))
    monkeypatch.setattr(Adam, "_flatten", lambda self, group: None)
    monkeypatch.setattr(Muon, "_flatten", lambda self, group: None)
    assert len(Adam(model.named_parameters()).param_groups[0]["params"]) == 4
    plain, named = Muon(model.parameters()), Muon(model.named_parameters())
    in_groups = Muon([{"params": list(model.named_parameters())}])
    for other in (named, in_groups):
        assert [[id(p) for p in g["params"]] for g in other.param_groups] == [[id(p) for p in g["params"]] for g in plain.param_groups]
        assert [g["param_names"] for g in other.param_groups] == [["0.weight"], ["0.bias", "1.weight", "1.bias"]]
    assert [g["muon"] for g in plain.param_groups] == [True, False]
    with pytest.raises(ValueError, match="2-D"):
        Muon([{"params": [("0.bias", model[0].bias)], "muon": True}])


def test_a_side_that_no_step_takes_fails_at_once():
    from nerf_amd.optim import Muon
    long = torch.nn.Parameter(torch.zeros(32769, 16))
    for group in ([long], [{"params": [long], "muon": True}], [("table", long)]):
        with pytest.raises(ValueError, match="32768"):
            Muon(group)
    with pytest.raises(RuntimeError, match="ROCm"):                       # Adam's may be of any size
        Muon([{"params": [long], "muon": False}])
