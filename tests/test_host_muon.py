"""What the orthogonalisation and its optimiser refuse, checked without a GPU: the C ABI's argument checks run
before any HIP call, the Python layer's before any launch."""
import ctypes as C

import pytest
import torch

COEF = (3.4445, -4.7750, 2.0315)


@pytest.fixture()
def ops():
    import nerf_amd.ops as ops_
    return ops_


def _table(_lib, *shapes, ptr=0):
    return (_lib.Matrix * len(shapes))(*[_lib.Matrix(ptr, ptr, ptr, ptr, *s) for s in shapes])


def test_workspace_bytes():
    from nerf_amd import _lib
    size = _lib.lib.nerfx_orthogonalize_workspace_bytes
    assert size(None, 0) == 0 and size(_table(_lib, (0, 5), (5, 0)), 2) == 0
    assert size(_table(_lib, (300, 300)), 1) >= 5 * 300 * 300 * 4
    # matrices of one group lie side by side; a 33rd starts a group that reuses the space
    three = size(_table(_lib, *[(300, 300)] * 3), 3)
    assert size(_table(_lib, (300, 300)), 1) < three < size(_table(_lib, *[(300, 300)] * 32), 32)
    assert size(_table(_lib, *[(300, 300)] * 32), 32) == size(_table(_lib, *[(300, 300)] * 33), 33)
    # small matrices by themselves stay inside their workgroups
    assert size(_table(_lib, (64, 256), (1, 1)), 2) == 0 and size(_table(_lib, (65, 65)), 1) > 0
    assert size(_table(_lib, (256, 39)), 1) == size(_table(_lib, (39, 256)), 1)
    assert size(None, 1) == -1
    assert size(_table(_lib, (-1, 4)), 1) == -1 and size(_table(_lib, (4, 32769)), 1) == -1
    assert b"32769" in _lib.lib.nerfx_last_error()


@pytest.mark.parametrize("change,text", [
    (dict(steps=0), b"steps 0"), (dict(steps=33), b"steps 33"), (dict(coef=None), b"coefficients"), (dict(eps=0.0), b"eps"),
    (dict(eps=float("nan")), b"eps"), (dict(coef=[float("inf"), 0, 0]), b"not finite"), (dict(coef=[100.0, 0, 0]), b"grow"),
    (dict(dtype=7), b"type"), (dict(ptr=0), b"NULL"), (dict(ws=0), b"workspace"), (dict(ws=8), b"aligned"), (dict(bytes=10), b"needed"),
])
def test_c_refusals_of_orthogonalize(change, text):
    from nerf_amd import _lib
    lib = _lib.lib
    coef = change.get("coef", COEF * change.get("steps", 1) or COEF)
    arr = None if coef is None else (C.c_float * max(3, len(coef)))(*coef)
    rc = lib.nerfx_orthogonalize(_table(_lib, (80, 80), ptr=change.get("ptr", 4096)), 1, change.get("dtype", 0), arr, change.get("steps", 1),
                                 change.get("eps", 1e-7), C.c_void_p(change.get("ws", 4096)), change.get("bytes", 1 << 40), None)
    assert rc == -1 and text in lib.nerfx_last_error(), lib.nerfx_last_error()


@pytest.mark.parametrize("change,text", [
    (dict(momentum=1.0), b"momentum"), (dict(momentum=-0.1), b"momentum"), (dict(lr=-1.0), b"lr"), (dict(lr=float("nan")), b"lr"),
    (dict(decay=-1.0), b"weight_decay"), (dict(adjust=5), b"rule"), (dict(ptr=0), b"NULL"),
])
def test_c_refusals_of_muon_step(change, text):
    from nerf_amd import _lib
    lib = _lib.lib
    rc = lib.nerfx_muon_step(_table(_lib, (8, 8), ptr=change.get("ptr", 4096)), 1, change.get("lr", 0.1), change.get("momentum", 0.9), 1,
                             change.get("decay", 0.0), change.get("adjust", 0), (C.c_float * 3)(*COEF), 1, 1e-7, None, None,
                             C.c_void_p(4096), 1 << 40, None)
    assert rc == -1 and text in lib.nerfx_last_error(), lib.nerfx_last_error()


def test_python_refusals(ops):
    with pytest.raises(RuntimeError, match="ROCm"):
        ops.orthogonalize(torch.zeros(4, 4))
    with pytest.raises(TypeError):
        ops.orthogonalize([None])
    with pytest.raises(ValueError, match="steps"):
        ops.orthogonalize(torch.zeros(4, 4), steps=0)
    for bad in ((1.0, 2.0), [COEF] * 3, [(1.0, 2.0)] * 5):
        with pytest.raises(ValueError, match="coefficients"):
            ops.orthogonalize(torch.zeros(4, 4), steps=5, coefficients=bad)
    assert ops.orthogonalize([]) == []
    w = [torch.zeros(4, 4)]
    with pytest.raises(RuntimeError, match="ROCm"):
        ops.muon_step(w, w, w, lr=0.1)
    with pytest.raises(ValueError, match="pair up"):
        ops.muon_step(w, [], w, lr=0.1)
    with pytest.raises(ValueError, match="adjust_lr"):
        ops.muon_step(w, w, w, lr=0.1, adjust_lr="other")
    ops.muon_step([], [], [], lr=0.1)


def test_optimizer_refusals():
    from nerf_amd.optim import Muon
    w = torch.nn.Parameter(torch.zeros(32, 32))
    for bad in (dict(momentum=1.0), dict(ns_eps=0.0), dict(weight_decay=-1.0), dict(adjust_lr="other"), dict(ns_steps=0),
                dict(ns_coefficients=(1.0,)), dict(lr=-1.0)):
        with pytest.raises(ValueError):
            Muon([w], **bad)
    with pytest.raises(ValueError, match="2-D"):
        Muon([{"params": [torch.nn.Parameter(torch.zeros(32))], "muon": True}])
    with pytest.raises(RuntimeError, match="ROCm"):
        Muon([w])
