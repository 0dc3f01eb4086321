"""Every code under every scale, as a stored matrix may have them: the quantiser itself never makes scales above 2^125."""
import pytest
import torch

from test_gpu_mx4 import TYPES, values

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ops():
    import nerf_amd.ops as ops_
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    yield ops_


def every():
    """-> codes (256, 1, 32) and scales (256, 1): row s has scale s, all 16 codes twice."""
    return (torch.arange(32) % 16).expand(256, 1, 32).contiguous(), torch.arange(256).view(256, 1)


def stored(ops, code, scale, k):
    flat = code.view(code.shape[0], -1).to(torch.uint8)
    return ops.Mx4((flat[:, 0::2] | flat[:, 1::2] << 4).contiguous().cuda(), scale.to(torch.uint8).cuda(), k)


@pytest.mark.parametrize("k", [32, 31, 30, 17])
def test_every_code_with_every_scale(ops, k):
    code, scale = every()
    q = stored(ops, code, scale, k)
    for dtype in TYPES:
        want, got = values(code, scale, k).to(dtype), q.dequantize(dtype).cpu()
        same = (got == want) & (torch.signbit(got) == torch.signbit(want)) | torch.isnan(got) & torch.isnan(want)
        assert bool(same.all()), f"{dtype}: scales {torch.nonzero(~same)[:, 0].unique().tolist()}"


@pytest.mark.parametrize("m", [3, 100])
def test_every_code_with_every_scale_in_a_product(ops, m):
    """Rows of ones times a single code: the code's value, to the bit, by way of each kernel."""
    for k in (32, 320, 1024):
        code, scale = torch.zeros(16 * 256, k // 32, 32, dtype=torch.int64), torch.full((16 * 256, k // 32), 127)
        for c in range(16):
            code[256 * c:256 * (c + 1), 0, 5] = c
        scale[:, 0] = torch.arange(256).repeat(16)
        want = values(code, scale, k).sum(1).float()
        x = torch.ones(m, k, device="cuda")
        got = ops.mx4_linear(x, stored(ops, code, scale, k)).cpu()
        same = (got == want) | torch.isnan(got) & torch.isnan(want)
        assert bool(same.all()), f"k {k}: scales {(torch.nonzero(~same)[:, 1] % 256).unique().tolist()}"
