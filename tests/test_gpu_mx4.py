"""Microscaled 4-bit numbers and their product against float64.

Quantising is exact: codes and scales have to be equal, byte for byte, to those found by distances in float64.  In the product
every term is exact (a code has at most two significand bits), so that only sums round: K + 1 additions, each off by at
most 2^-23 of what has been added up (sums inside a matrix instruction may truncate), and the result's own
half step; SiLU adds four roundings and passes an error on at most 1.1-fold.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


@pytest.fixture()
def ops():
    import nerf_amd.ops as ops_
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    ops_.set_precision(None)
    yield ops_
    ops_.set_precision(None)


def quantized(x):
    """-> codes (rows, blocks, 32), scales (rows, blocks): the definition in float64 on the CPU."""
    x = x.detach().double().cpu()
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).view(x.shape[0], -1, 32)
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(-127, 127)
    v = torch.ldexp(x, -e.unsqueeze(-1))
    d = (v.abs().unsqueeze(-1) - GRID).abs()
    best = d.amin(-1, keepdim=True)
    near = d == best                                                   # one or two neighbours: of two, the even code
    even = near & (torch.arange(8) % 2 == 0)
    code = torch.where(near.sum(-1) == 2, even.int().argmax(-1), near.int().argmax(-1)) + 8 * torch.signbit(v)
    code = torch.where(bad.unsqueeze(-1), 0, code)
    return code, torch.where(bad, 255, e + 127)


def values(code, scale, k):
    v = torch.cat((GRID, -GRID))[code] * torch.exp2(scale.double() - 127).unsqueeze(-1)
    v = torch.where((scale == 255).unsqueeze(-1), float("nan"), v)
    return v.view(code.shape[0], -1)[:, :k]


def check_quantize(ops, x, what):
    q = ops.mx4_quantize(x)
    code, scale = quantized(x)
    flat = code.view(x.shape[0], -1)
    assert torch.equal(q.scales.cpu().long(), scale), f"{what}: scales"
    assert torch.equal(q.codes.cpu().long(), flat[:, 0::2] | flat[:, 1::2] << 4), f"{what}: codes"
    for dtype in TYPES:
        want = values(code, scale, x.shape[1]).to(dtype)
        got = q.dequantize(dtype).cpu()
        assert torch.equal(torch.nan_to_num(got, 7.0), torch.nan_to_num(want, 7.0)), f"{what}: values in {dtype}"
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.signbit(got) | torch.isnan(got), torch.signbit(want) | torch.isnan(want)), f"{what}: signs of zeros"
    return q


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 31), (1, 32), (5, 33), (2, 8), (7, 39), (64, 256), (100, 295), (3, 4096), (513, 72)])
def test_quantize(ops, dtype, rows, k):
    g = torch.Generator().manual_seed(rows * 1000 + k)
    x = torch.randn(rows, k, generator=g) * torch.exp2(torch.randint(-20, 12, (rows, k), generator=g))
    check_quantize(ops, x.to(dtype).cuda(), f"{rows} x {k}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantize_every_16_bit_number(ops, dtype):
    """Each alone in a block, and beside a largest value that puts it on every place of the grid."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    alone = torch.zeros(65536, 32, dtype=dtype)
    alone[torch.arange(65536), torch.arange(65536) % 32] = every
    check_quantize(ops, alone.cuda(), "alone")
    finite = every[torch.isfinite(every)]
    for top in (6.0, 7.5, 1.0, 2.0 ** -14):
        beside = torch.full((finite.numel() // 8, 32), 0.0, dtype=dtype)
        beside[:, 0] = top
        beside[:, 8:16] = finite[:finite.numel() // 8 * 8].view(-1, 8)
        check_quantize(ops, beside.cuda(), f"beside {top}")


def test_quantize_fp32_edges(ops):
    tiny, huge = 2.0 ** -149, 3.4028234663852886e38
    rows = [[0.0, -0.0], [tiny, -tiny], [2.0 ** -126, 2.0 ** -127], [2.0 ** -125, 2.0 ** -128 * 1.5], [huge, -huge], [huge, 1.0],
            [float("inf"), 1.0], [1.0, float("nan")], [-float("inf"), 0.0], [7.9999995, 0.25], [8.0, 0.5], [5.0, 2.5], [5.0000005, 0.74999994]]
    x = torch.zeros(len(rows), 40)
    for i, (a, b) in enumerate(rows):
        x[i, 3], x[i, 17], x[i, 39] = a, b, b
    q = check_quantize(ops, x.cuda(), "edges")
    assert bool(torch.isnan(q.dequantize()[6, :32]).all())


def test_quantize_takes_views_and_empty_matrices(ops):
    x = torch.randn(50, 70, device="cuda")
    check_quantize(ops, x[:, 1:66], "columns from an odd place")
    check_quantize(ops, x.t(), "transposed")
    flat = torch.randn(64 * 8 + 1, device="cuda").to(torch.bfloat16)
    check_quantize(ops, flat[1:].view(8, 64), "a start that is not aligned")
    q = ops.mx4_quantize(torch.empty(0, 64, device="cuda"))
    assert q.shape == (0, 64) and q.dequantize().shape == (0, 64)
    for bad in (torch.randn(3, device="cuda"), torch.randn(2, 2, 2, device="cuda"), torch.empty(3, 0, device="cuda")):
        with pytest.raises(ValueError):
            ops.mx4_quantize(bad)
    with pytest.raises(TypeError):
        ops.mx4_quantize(x.double())
    with pytest.raises(RuntimeError, match="gradient"):
        ops.mx4_quantize(x.requires_grad_(True))


# ---- the product ----------------------------------------------------------------------------------------------------
def activated(y, act):
    if act == "relu":
        return torch.where(y < 0, torch.zeros_like(y), y)
    if act == "leaky_relu":
        return torch.where(y < 0, 0.01 * y, y)
    return y / (1 + torch.exp(-y)) if act == "silu" else y


def check_linear(ops, x, w, bias, act, out_dtype=None, x_form=None, what=""):
    """x, w fp32/16-bit tensors on the device; the product of their 4-bit forms against float64."""
    qw = ops.mx4_quantize(w)
    got = ops.mx4_linear(x if x_form is None else x_form, qw, bias, act, out_dtype)
    k = w.shape[1]
    xv, wv = values(*quantized(x.reshape(-1, k)), k).cuda(), values(*quantized(w), k).cuda()
    b = torch.zeros(w.shape[0], dtype=torch.float64, device="cuda") if bias is None else bias.double()
    pre = xv @ wv.t().contiguous() + b
    want = activated(pre, act)
    room = xv.abs() @ wv.abs().t().contiguous() + b.abs()
    tol = 1.1 * (k + 1) * 2.0 ** -23 * room + (HALF_STEP[got.dtype] + 4 * 2.0 ** -24) * want.abs()
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert got.shape == (*x.shape[:-1], w.shape[0]) and got.is_contiguous()
    d = (got.double().reshape(want.shape) - want).abs()
    worst = (d - tol).flatten().argmax() if d.numel() else None
    assert bool((d <= tol).all()), f"{what}: off by {float(d.flatten()[worst]):.3e}, allowed {float(tol.flatten()[worst]):.3e} at {int(worst)}"
    return got


def pair(m, n, k, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + m * 7 + n * 3 + k)
    x = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    w = torch.randn(n, k, generator=g, device="cuda") / k ** 0.5
    return x, w, 0.1 * torch.randn(n, generator=g, device="cuda")


SIZES = [(1, 1, 1), (1, 3, 32), (1, 256, 256), (2, 130, 95), (16, 64, 4096), (17, 16, 40), (33, 1, 256), (64, 4096, 512), (65, 31, 64),
         (129, 3, 128), (200, 128, 295), (256, 256, 39), (300, 256, 319), (1000, 128, 295), (257, 129, 1025), (515, 700, 1032), (4100, 256, 256),
         (130, 520, 96)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear(ops, dtype, m, n, k):
    x, w, bias = pair(m, n, k, dtype)
    for act in (None, "silu"):
        check_linear(ops, x, w, bias, act, what=f"{m} x {n} x {k} {act}")


# Columns in several groups; tiles of each size, with rows of one stage and more, and too long for their scales to be in LDS.
@pytest.mark.parametrize("m,n,k", [(70, 300, 200), (300, 1000, 256), (5000, 520, 33), (600, 2100, 64), (20000, 257, 256), (70, 100, 30000),
                                   (100, 70, 8200), (65, 65, 513), (2100, 1600, 300), (1700, 2500, 1100), (2100, 1600, 520), (6200, 2050, 290),
                                   (5000, 3000, 700), (12300, 1030, 545), (16, 20, 8200),
                                   (3, 5, 60000), (33, 100, 4096)])
def test_linear_many_columns_and_tiles(ops, m, n, k):
    x, w, bias = pair(m, n, k, torch.bfloat16, 8)
    check_linear(ops, x, w, bias, "relu", what=f"{m} x {n} by {k}")


@pytest.mark.parametrize("act", [None, "relu", "leaky_relu", "silu"])
@pytest.mark.parametrize("m,n,k", [(5, 96, 64), (300, 256, 256), (700, 640, 416)])
def test_linear_activations_and_types(ops, m, n, k, act):
    for dtype in TYPES:
        for out in TYPES:
            x, w, bias = pair(m, n, k, dtype, 1)
            check_linear(ops, x, w, bias, act, out, what=f"{dtype} to {out}")
            check_linear(ops, x, w, None, act, out, what=f"{dtype} to {out}, no bias")


@pytest.mark.parametrize("m,n,k", [(1, 100, 256), (40, 48, 300), (500, 256, 256), (500, 700, 600)])
def test_linear_of_a_quantized_input(ops, m, n, k):
    x, w, bias = pair(m, n, k, torch.bfloat16, 2)
    q = ops.mx4_quantize(x)
    a = check_linear(ops, x, w, bias, "relu", torch.bfloat16, x_form=q)
    assert torch.equal(a, ops.mx4_linear(x, ops.mx4_quantize(w), bias, "relu")), "the two forms of x take the same products"
    assert ops.mx4_linear(q, ops.mx4_quantize(w)).dtype == torch.float32


@pytest.mark.parametrize("act", [None, "relu", "silu"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (3, 40, 39), (64, 256, 256), (129, 256, 295), (300, 31, 96), (300, 256, 256), (500, 300, 64),
                                   (33, 600, 200), (2100, 1600, 300), (515, 700, 1032), (200, 64, 600)])
def test_linear_into_blocks(ops, m, n, k, act):
    """A result quantised on its way out is the fp32 result, which the same product gives, quantised."""
    for dtype in TYPES:
        x, w, bias = pair(m, n, k, dtype, 8)
        x[m // 2, k // 2] = float("nan") if m > 100 else 1.0
        qw, qx = ops.mx4_quantize(w), ops.mx4_quantize(x)
        got = ops.mx4_linear(qx, qw, bias, act, "mx4")
        assert got.shape == (m, n)
        plain = ops.mx4_linear(torch.cat((qx.dequantize(), torch.zeros(100, k, device="cuda"))), qw, bias, act)[:m]
        want = ops.mx4_quantize(plain)                                  # more rows: the same kernels as for blocks
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
        again = ops.mx4_linear(x, qw, bias, act, "mx4")
        assert torch.equal(got.codes, again.codes) and torch.equal(got.scales, again.scales)
    assert ops.mx4_linear(x.view(1, m, k), qw, bias, act, "mx4").shape == (m, n)


def test_linear_shapes_views_and_empty(ops):
    x, w, bias = pair(24, 40, 64, torch.float32, 3)
    qw = ops.mx4_quantize(w)
    flat = ops.mx4_linear(x, qw, bias)
    assert torch.equal(ops.mx4_linear(x.view(2, 3, 4, 64), qw, bias), flat.view(2, 3, 4, 40))
    assert torch.equal(ops.mx4_linear(x[0], qw, bias), flat[0])
    wide = torch.randn(24, 130, device="cuda")
    check_linear(ops, wide[:, 1:65], w, bias, None, what="a strided x")
    assert torch.equal(ops.mx4_linear(x, ops.Mx4(qw.codes[8:], qw.scales[8:], 64), bias[8:]), flat[:, 8:]), "a slice of the weight's rows"
    assert ops.mx4_linear(x[:0], qw).shape == (0, 40)
    assert ops.mx4_linear(x, ops.mx4_quantize(w[:0])).shape == (24, 0)
    odd = torch.randn(24 * 64 + 1, device="cuda").to(torch.bfloat16)[1:].view(24, 64)
    check_linear(ops, odd, w, bias, None, what="a start that is not aligned")


@pytest.mark.parametrize("m,n,k", [(3, 70, 96), (300, 256, 256), (300, 300, 600)])
def test_linear_extremes(ops, m, n, k):
    """NaN rows stay in their rows and columns; the largest and smallest scales multiply as their powers of two do."""
    x, w, bias = pair(m, n, k, torch.float32, 4)
    clean = check_linear(ops, x, w, bias, None)
    for poison in (float("nan"), float("inf")):
        y = x.clone()
        y[1, k - 1] = poison
        got = ops.mx4_linear(y, ops.mx4_quantize(w), bias)
        assert bool(torch.isnan(got[1]).all())
        keep = [i for i in range(m) if i != 1]
        assert torch.equal(got[keep], clean[keep])
        v = w.clone()
        v[n - 1, 0] = poison
        got = ops.mx4_linear(x, ops.mx4_quantize(v), bias)
        assert bool(torch.isnan(got[:, n - 1]).all()) and torch.equal(got[:, :n - 1], clean[:, :n - 1])
    check_linear(ops, x * 2.0 ** 100, w * 2.0 ** -110, bias, None, what="far scales")
    check_linear(ops, x * 2.0 ** -126, w * 2.0 ** 120, bias, None, what="subnormal inputs")
    zero = check_linear(ops, x * 0, w, bias, None, what="zeros")
    assert torch.equal(zero, bias.expand(m, n))


def test_linear_writes_nothing_beside_its_result(ops):
    """The rows behind the last one keep what they hold: the C entry writes into the middle of a larger buffer."""
    import ctypes as C
    from nerf_amd import _lib
    for m, n, k, dt, code in ((1, 5, 40, torch.float32, 0), (70, 20, 64, torch.bfloat16, 1), (130, 256, 256, torch.bfloat16, 1),
                              (300, 333, 320, torch.float16, 2)):
        x, w, bias = pair(m, n, k, dt, 5)
        qw = ops.mx4_quantize(w)
        buf = torch.full((m * n + 512,), 3.0, device="cuda", dtype=dt)
        y = buf[256:256 + m * n]
        need = _lib.lib.nerfx_mx4_linear_workspace_bytes(m, n, k, code, code)
        ws = torch.empty(max(need, 1), device="cuda", dtype=torch.uint8)
        p = lambda t: C.c_void_p(t.data_ptr())
        _lib.check(_lib.lib.nerfx_mx4_linear(p(x), code, None, m, k, p(qw.codes), p(qw.scales), n, p(bias), 0, p(y), code, None, p(ws), need,
                                             C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        assert bool((buf[:256] == 3).all()) and bool((buf[256 + m * n:] == 3).all())
        assert torch.equal(y.view(m, n), ops.mx4_linear(x, qw, bias, "relu"))


@pytest.mark.parametrize("m,n,k", [(7, 37, 43), (90, 37, 43), (90, 3, 31), (200, 301, 333), (90, 65, 96)])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_from_and_to_any_place(ops, dtype, m, n, k):
    """x amid NaNs and y amid other numbers, each from any value of a buffer on: nothing from beside x counts, nothing beside y changes."""
    import ctypes as C
    from nerf_amd import _lib
    x, w, bias = pair(m, n, k, dtype, 7)
    qw = ops.mx4_quantize(w)
    code = TYPES.index(dtype)
    p = lambda t: C.c_void_p(t.data_ptr())
    need = _lib.lib.nerfx_mx4_linear_workspace_bytes(m, n, k, code, code)
    ws = torch.empty(max(need, 16), device="cuda", dtype=torch.uint8)
    want = check_linear(ops, x, w, bias, None)
    for at in range(9):
        src = torch.full((m * k + 64,), float("nan"), device="cuda", dtype=dtype)
        buf = torch.full((m * n + 64,), 3.0, device="cuda", dtype=dtype)
        src[at:at + m * k] = x.flatten()
        y = buf[8 - at:8 - at + m * n]
        _lib.check(_lib.lib.nerfx_mx4_linear(p(src[at:]), code, None, m, k, p(qw.codes), p(qw.scales), n, p(bias), -1, p(y), code, None, p(ws),
                                             need, C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        assert torch.equal(y.view(m, n), want), at
        assert bool((buf[:8 - at] == 3).all()) and bool((buf[8 - at + m * n:] == 3).all()), at
        q = ops.mx4_quantize(src[at:at + m * k].view(m, k))
        assert torch.equal(q.scales, ops.mx4_quantize(x).scales) and torch.equal(q.codes, ops.mx4_quantize(x).codes), at


@pytest.mark.parametrize("m,n,k", [(9_000_000, 256, 64), (9_000_000, 257, 33), (280_000, 8200, 290)])
def test_linear_past_32_bits(ops, m, n, k):
    """Results of more than 2^32 bytes: the last rows are those of a call of their own."""
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(m, k, generator=g, device="cuda").to(torch.bfloat16)
    w = ops.mx4_quantize(torch.randn(n, k, generator=g, device="cuda"))
    y = ops.mx4_linear(x, w, None, "relu")
    for rows in (slice(m - 3000, m), slice(m // 2 - 11, m // 2 + 2989), slice(0, 3000)):
        assert torch.equal(y[rows], ops.mx4_linear(x[rows].clone(), w, None, "relu"))
    del y
    q = ops.mx4_quantize(x)
    back = q.dequantize(torch.bfloat16)
    tail = ops.mx4_quantize(x[m - 3000:].clone())
    assert torch.equal(q.codes[m - 3000:], tail.codes) and torch.equal(q.scales[m - 3000:], tail.scales)
    assert torch.equal(back[m - 3000:], tail.dequantize(torch.bfloat16))


def test_linear_refuses(ops):
    x, w, bias = pair(4, 8, 64, torch.float32, 6)
    qw = ops.mx4_quantize(w)
    with pytest.raises(ValueError, match="columns"):
        ops.mx4_linear(x[:, :32], qw)
    with pytest.raises(ValueError, match="bias"):
        ops.mx4_linear(x, qw, bias[:4])
    with pytest.raises(TypeError):
        ops.mx4_linear(x.double(), qw)
    with pytest.raises(TypeError):
        ops.mx4_linear(x, qw, out_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.mx4_linear(x.clone().requires_grad_(True), qw)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.mx4_linear(x, qw, bias.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="weight on"):
        ops.mx4_linear(x, qw.to("cpu"))


def test_linear_on_streams_and_in_graphs(ops):
    for m, n, k in ((1, 512, 512), (400, 256, 256), (400, 600, 512)):
        x, w, bias = pair(m, n, k, torch.bfloat16, 7)
        qw = ops.mx4_quantize(w)
        want = ops.mx4_linear(x, qw, bias, "silu")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = ops.mx4_linear(x, qw, bias, "silu")
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = ops.mx4_linear(x, qw, bias, "silu")
            back = ops.mx4_quantize(got).dequantize()
        for i in range(4):
            x.mul_(1.5)
            graph.replay()
            torch.cuda.synchronize()
            want = ops.mx4_linear(x, qw, bias, "silu")
            assert torch.equal(got, want) and torch.equal(back, ops.mx4_quantize(want).dequantize()), f"replay {i}"


def test_two_products_of_one_weight_at_once(ops):
    """Workspaces are each call's own: two streams go over the same weight with inputs of their own."""
    x, w, bias = pair(700, 900, 600, torch.float32, 9)
    qw = ops.mx4_quantize(w)
    inputs = [x, x.flip(0).contiguous()]
    want = [ops.mx4_linear(v, qw, bias, "silu") for v in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, side in enumerate(streams):
            with torch.cuda.stream(side):
                got[i].append(ops.mx4_linear(inputs[i], qw, bias, "silu"))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
