"""The microscaled product where its kernels are largest: whole workgroups of eight waves, rows of W for 256 columns in LDS (more
than 64 KB of it), float rows of up to 512 values quantised in registers.  Every result is held against float64 on the values of
the quantised operands, with test_gpu_mx4's tolerance: K + 1 additions, each off by at most 2^-23 of what has been added up, and the
result's own half step; SiLU adds four roundings and passes an error on at most 1.1-fold.  That quantising is exact is tested there."""
import pytest
import torch

from test_gpu_mx4 import HALF_STEP, TYPES, activated, pair

pytestmark = pytest.mark.gpu


@pytest.fixture()
def ops():
    import nerf_amd.ops as ops_
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    ops_.set_precision(None)
    yield ops_
    ops_.set_precision(None)


def check(ops, x, w, bias, act, out_dtype=None, what=""):
    k = w.shape[1]
    qw = ops.mx4_quantize(w)
    got = ops.mx4_linear(x, qw, bias, act, out_dtype)
    xv, wv = ops.mx4_quantize(x).dequantize().double(), qw.dequantize().double()
    pre = xv @ wv.t().contiguous() + bias.double()
    want = activated(pre, act)
    room = xv.abs() @ wv.abs().t().contiguous() + bias.double().abs()
    tol = 1.1 * (k + 1) * 2.0 ** -23 * room + (HALF_STEP[got.dtype] + 4 * 2.0 ** -24) * want.abs()
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    over = (got.double() - want).abs() - tol
    assert got.shape == want.shape and bool((over <= 0).all()), f"{what}: {float(over.max()):.3e} beyond the tolerance"
    return got


# steps of 64 values: 8, 7, 6, 5, 4, 1; whole blocks and rows that end inside of one
ROWS = [(50000, 256, 512), (50000, 255, 511), (50000, 256, 448), (50000, 250, 400), (50000, 256, 384), (50000, 200, 330), (50000, 256, 295),
        (50000, 256, 256), (50000, 256, 39), (300, 256, 512), (300, 200, 333), (66, 31, 449), (1000, 129, 385)]


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_of_every_length(ops, dtype):
    """Longer rows, which take more LDS, before shorter ones: each length has a kernel of its own."""
    for m, n, k in ROWS:
        x, w, bias = pair(m, n, k, dtype, 12)
        check(ops, x, w, bias, "silu", what=f"{m} x {n} by {k}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_rows_that_begin_inside_a_word(ops, dtype):
    for m, n, k in ROWS:
        x, w, bias = pair(m, n, k, dtype, 13)
        odd = torch.empty(m * k + 1, device="cuda", dtype=dtype)[1:].view(m, k)
        odd.copy_(x)
        assert odd.data_ptr() % 4 == 2
        got = check(ops, odd, w, bias, "relu", what=f"{m} x {n} by {k}")
        assert torch.equal(got, ops.mx4_linear(x, ops.mx4_quantize(w), bias, "relu"))


@pytest.mark.parametrize("m,n,k", [(50000, 256, 512), (50000, 256, 400), (50000, 256, 256), (300, 256, 512), (5000, 1000, 200)])
def test_results_of_every_type(ops, m, n, k):
    """Lines of each width leave by way of LDS, between lanes of a wave; blocks are the fp32 result, quantised."""
    x, w, bias = pair(m, n, k, torch.bfloat16, 14)
    for out in TYPES:
        check(ops, x, w, bias, "leaky_relu", out, what=f"{m} x {n} by {k} to {out}")
    q, qw = ops.mx4_quantize(x), ops.mx4_quantize(w)
    blocks = ops.mx4_linear(q, qw, bias, "leaky_relu", "mx4")
    want = ops.mx4_quantize(ops.mx4_linear(q, qw, bias, "leaky_relu", torch.float32))
    assert torch.equal(blocks.codes, want.codes) and torch.equal(blocks.scales, want.scales)
