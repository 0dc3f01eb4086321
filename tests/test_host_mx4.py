"""What the microscaled 4-bit operators refuse, checked without a GPU."""
import pytest
import torch


@pytest.fixture()
def ops():
    import nerf_amd.ops as ops_
    return ops_


def _mx4(ops, rows=4, k=64):
    return ops.Mx4(torch.zeros(rows, 16 * ((k + 31) // 32), dtype=torch.uint8), torch.zeros(rows, (k + 31) // 32, dtype=torch.uint8), k)


def test_workspace_bytes():
    from nerf_amd import _lib
    size = _lib.lib.nerfx_mx4_linear_workspace_bytes
    assert size(10, 4, 33, _lib.TYPE_MX4, 0) == 0
    assert size(-1, 4, 4, 0, 0) == size(4, -1, 4, 0, 0) == size(4, 4, 0, 0, 0) == size(4, 4, (1 << 20) + 1, 0, 0) == -1
    assert size(4, 4, 4, 9, 0) == size(4, 4, 4, 0, 9) == size(1 << 31, 4, 4, 0, 0) == -1
    assert size(524288, 256, 256, _lib.TYPE_BF16, _lib.TYPE_BF16) == 0          # quantised in registers
    assert size(524288, 300, 295, _lib.TYPE_BF16, _lib.TYPE_MX4) >= 524288 * 10 * 17


def test_c_refusals():
    from nerf_amd import _lib
    lib = _lib.lib
    p = 4096

    def refused(rc, text):
        assert rc == -1 and text in lib.nerfx_last_error(), lib.nerfx_last_error()

    refused(lib.nerfx_mx4_quantize(p, 0, -1, 8, p, p, None), b"rows")
    refused(lib.nerfx_mx4_quantize(p, 0, 4, 0, p, p, None), b"k 0")
    refused(lib.nerfx_mx4_quantize(p, 3, 4, 8, p, p, None), b"type")
    refused(lib.nerfx_mx4_quantize(p, 0, 4, 8, None, p, None), b"NULL")
    refused(lib.nerfx_mx4_quantize(p, 0, 4, 8, p + 2, p, None), b"aligned")
    assert lib.nerfx_mx4_quantize(None, 0, 0, 8, None, None, None) == 0
    refused(lib.nerfx_mx4_dequantize(p, p, 4, 8, 3, p, None), b"type")
    refused(lib.nerfx_mx4_dequantize(p, None, 4, 8, 0, p, None), b"NULL")
    refused(lib.nerfx_mx4_dequantize(p, p, 4, (1 << 20) + 1, 0, p, None), b"k ")
    refused(lib.nerfx_mx4_dequantize(p + 1, p, 4, 8, 0, p, None), b"aligned")

    def linear(x=p, xt=0, xs=None, m=4, k=64, w=p, ws=p, n=4, act=0, y=p, yt=0, ys=None, work=p, size=1 << 40):
        return lib.nerfx_mx4_linear(x, xt, xs, m, k, w, ws, n, None, act, y, yt, ys, work, size, None)

    refused(linear(m=-1), b"rows")
    refused(linear(n=-1), b"n -1")
    refused(linear(n=(1 << 24) + 1), b"n 16777217")
    refused(linear(k=0), b"k 0")
    refused(linear(xt=4), b"of x")
    refused(linear(yt=4), b"of y")
    refused(linear(yt=3), b"NULL")                                     # codes without scales
    refused(linear(yt=3, ys=p, y=p + 8), b"aligned")
    refused(linear(m=100, n=300, k=600, size=0), b"workspace")
    refused(linear(m=100, n=300, k=600, work=None), b"workspace")
    refused(linear(m=100, n=300, k=600, work=p + 8), b"workspace")
    refused(linear(act=3), b"activation")
    refused(linear(act=-2), b"activation")
    for name in ("x", "w", "ws", "y"):
        refused(linear(**{name: None}), b"NULL")
    refused(linear(xt=3), b"NULL")                                     # codes without scales
    refused(linear(w=p + 8), b"aligned")
    refused(linear(x=p + 4, xt=3, xs=p), b"aligned")
    assert linear(m=0, x=None) == 0 and linear(n=0, w=None) == 0


def test_mx4_checks_its_parts(ops):
    t = _mx4(ops)
    assert t.shape == (4, 64)
    codes, scales = t.codes, t.scales
    for bad in ((codes, scales, 65), (codes, scales, 32), (codes, scales, 0), (codes.int(), scales, 64), (codes, scales.float(), 64),
                (codes[0], scales, 64), (codes, scales[:3], 64), (codes.t(), scales, 64), (codes[:, :16], scales, 32)):
        with pytest.raises(ValueError):
            ops.Mx4(*bad)
    both = ops.Mx4.cat([t, _mx4(ops, 4, 39)])
    assert both.shape == (4, 103) and both.codes.shape == (4, 64)
    with pytest.raises(ValueError, match="32"):
        ops.Mx4.cat([_mx4(ops, 4, 39), t])
    flat = torch.zeros(200, dtype=torch.uint8)
    start = next(i for i in range(16) if (flat.data_ptr() + i) % 16 == 8)
    with pytest.raises(ValueError, match="aligned"):
        ops.Mx4(flat[start:start + 128].view(4, 32), torch.zeros(4, 2, dtype=torch.uint8), 64)


def test_python_refusals(ops):
    w = _mx4(ops)
    with pytest.raises(RuntimeError, match="ROCm"):
        ops.mx4_quantize(torch.zeros(4, 4))
    with pytest.raises(TypeError):
        ops.mx4_quantize([1.0])
    with pytest.raises(RuntimeError, match="ROCm"):
        w.dequantize()
    with pytest.raises(TypeError):
        w.dequantize(torch.float64)
    with pytest.raises(RuntimeError, match="ROCm"):
        ops.mx4_linear(torch.zeros(2, 64), w)
    with pytest.raises(RuntimeError, match="ROCm"):
        ops.mx4_linear(w, w)
    with pytest.raises(TypeError, match="Mx4"):
        ops.mx4_linear(torch.zeros(2, 64), torch.zeros(4, 64))
    with pytest.raises(ValueError, match="activation"):
        ops.mx4_linear(torch.zeros(2, 64), w, activation="gelu")
