"""A result in blocks is a matrix of blocks like any other: of 1 to 2^20 columns."""
import pytest
import torch


@pytest.mark.parametrize("n", [0, (1 << 20) + 1, 1 << 24])
def test_c_refuses_results_that_no_call_takes(n):
    from nerf_amd import _lib
    lib, p = _lib.lib, 4096
    assert lib.nerfx_mx4_linear_workspace_bytes(4, n, 64, _lib.TYPE_F32, _lib.TYPE_MX4) == -1
    rc = lib.nerfx_mx4_linear(p, _lib.TYPE_F32, None, 4, 64, p, p, n, None, -1, p, _lib.TYPE_MX4, p, p, 1 << 40, None)
    assert rc == -1 and b"n %d" % n in lib.nerfx_last_error(), lib.nerfx_last_error()
    assert lib.nerfx_mx4_linear_workspace_bytes(4, n, 64, _lib.TYPE_F32, _lib.TYPE_F32) >= 0          # of floats it may have them


@pytest.mark.parametrize("k", [0, (1 << 20) + 1])
def test_no_unwritten_one_beyond_the_constructors_bounds(k):
    import nerf_amd.ops as ops
    like = torch.zeros(1)
    with pytest.raises(ValueError, match="2.20"):
        ops.Mx4._new(3, k, like)
    assert ops.Mx4._new(3, 1 << 20, like).codes.shape == (3, 1 << 19)
    assert ops.Mx4._new(0, 5, like).scales.shape == (0, 1)


@pytest.mark.gpu
def test_linear_refuses_results_that_no_call_takes():
    import nerf_amd.ops as ops
    x = torch.randn(4, 64, device="cuda")
    none = ops.mx4_quantize(torch.empty(0, 64, device="cuda"))
    many = ops.mx4_quantize(torch.zeros((1 << 20) + 1, 64, device="cuda"))
    for w in (none, many):
        with pytest.raises(ValueError, match="2.20"):
            ops.mx4_linear(x, w, out_dtype="mx4")
        assert ops.mx4_linear(x, w).shape == (4, w.shape[0])
    last = ops.mx4_linear(x, ops.Mx4(many.codes[1:], many.scales[1:], 64), out_dtype="mx4")
    assert last.shape == (4, 1 << 20) and not bool(last.dequantize().any())
