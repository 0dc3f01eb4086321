"""How near orthogonalised matrices come to float64 where nothing is at its worst: what test_gpu_muon's bound, which holds for
any matrix, is too wide to see.

The tolerance is worked out for each matrix.  X, A and B are stored with 22 significand bits; the same steps in float64 with
just these rounded are some 6e-7 to 1.2e-6 off.  What that leaves out are the sums, fp32 and of K / 16 additions: rounding like a
random walk they are off by sqrt(K / 16) 2^-24 of their size, for K up to 4,096 at most 2^-20, on average of the longest as much as
four of the roundings that are simulated, and for K up to 256 as much as one.  So twice the simulated error, and for longer rows
sqrt(K / 256) times the second part, with half as much again for the scatter between the two."""
import math

import numpy as np
import pytest
import torch

from test_gpu_muon import COEF, exact, matrix

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ops():
    import nerf_amd.ops as ops_
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    return ops_


def rounded(v, bits=22):
    m, e = np.frexp(v)
    return np.ldexp(np.round(m * 2.0 ** bits) * 2.0 ** -bits, e)


def simulated(g, stored):
    x = g.T if g.shape[0] > g.shape[1] else g
    x = stored(x / math.sqrt(float((x * x).sum())))
    for k in range(5):
        gram = stored(x @ x.T)
        x = COEF[0] * x + stored(COEF[1] * gram + COEF[2] * (gram @ gram)) @ x
        if k < 4:
            x = stored(x)
    return x.T if g.shape[0] > g.shape[1] else x


def allowed(m):
    g = m.double().cpu().numpy()
    plain = simulated(g, lambda v: v)
    off = float(np.linalg.norm(simulated(g, rounded) - plain) / np.linalg.norm(plain))
    return 1.5 * off * (1 + math.sqrt(max(1.0, max(g.shape) / 256)))


SHAPES = [(2, 1500), (8, 60), (4, 400), (16, 16), (17, 17), (17, 60), (32, 39), (64, 64), (77, 77), (48, 700), (17, 2048), (64, 2000), (256, 39),
          (256, 256), (256, 295), (129, 1000), (515, 1027), (1024, 1024), (1030, 4100)]


@pytest.mark.parametrize("beside", [None, (70, 300), (2100, 1600)])
def test_orthogonalize_is_as_near_as_its_numbers_are(ops, beside):
    """By themselves, in launches they share, and in the large tiles that a large matrix brings with it."""
    mats = [matrix(s, 31 + i) for i, s in enumerate(SHAPES)]
    outs = [ops.orthogonalize(m) for m in mats] if beside is None else ops.orthogonalize(mats + [matrix(beside, 99)])
    for m, out in zip(mats, outs):
        want = exact(m)
        off = float((out.double().cpu() - want).norm() / want.norm())
        assert off <= allowed(m), f"{tuple(m.shape)}: {off:.2e} of {allowed(m):.2e}"
