"""`ops.orthogonalize` answers in the form that it is asked in."""
import pytest


def test_no_matrices_in_either_form():
    import nerf_amd.ops as ops
    assert ops.orthogonalize(()) == () and ops.orthogonalize([]) == []


@pytest.mark.gpu
def test_a_tuple_gives_a_tuple():
    import torch

    import nerf_amd.ops as ops
    a, b = torch.randn(20, 30, device="cuda"), torch.randn(70, 40, device="cuda")
    listed, paired = ops.orthogonalize([a, b]), ops.orthogonalize((a, b))
    assert isinstance(listed, list) and isinstance(paired, tuple)
    assert all(torch.equal(x, y) for x, y in zip(listed, paired))
