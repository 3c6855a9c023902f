"""MXFP4 quantisation and product against plain 64-bit implementations.

Quantisation is exact: codes, scales and values equal the definition's.  The
product's tolerance: one bf16 rounding of the result (half an ulp: 2^-8 of it) plus the f32
accumulation, 2^-22 of sum |x||w| for each 64 columns and four for the
epilogue (act' is at most 1.13)."""
import math

import pytest
import torch

import qwen_imager_b200 as qib
from qwen_imager_b200 import _lib

pytestmark = pytest.mark.gpu

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def definition(x):
    """(values f64 [rows, k], scales [rows, blocks]) of a CPU tensor by search over the grid."""
    x = x.double()
    rows, k = x.shape
    blocks = -(-k // 32)
    b = torch.zeros((rows, blocks * 32), dtype=torch.float64)
    b[:, :k] = x
    b = b.view(rows, blocks, 32)
    scales = torch.zeros((rows, blocks), dtype=torch.int64)
    values = torch.zeros_like(b)
    for r in range(rows):
        for j in range(blocks):
            v = b[r, j]
            top = v.abs().max().item()
            if not math.isfinite(top):
                scales[r, j] = 255
                values[r, j] = math.nan
                continue
            e = max(math.frexp(top)[1] - 1 - 2 + 127, 0) if top else 0
            scales[r, j] = e
            y = v.abs() / 2.0 ** (e - 127)
            d = (y[:, None] - GRID).abs()
            best = d.min(-1, keepdim=True).values
            tie = d == best  # at most two neighbours; ties go to the even code
            code = torch.tensor([next(c for c in sorted(range(8), key=lambda c: (c & 1)) if t[c]) if t.sum() > 1 else int(t.nonzero()[0])
                                 for t in tie])
            values[r, j] = torch.copysign(GRID[code], v) * 2.0 ** (e - 127)
    return values.view(rows, -1)[:, :k], scales


def randn(shape, seed, std=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype)


def awkward(rows, k, dtype, seed=0):
    """Every tie and neighbour of a tie of the grid, in blocks of several magnitudes, with zeros and a short last block."""
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.96875])
    pool = torch.cat([ties, ties * (1 + 2.0**-7), ties * (1 - 2.0**-8), torch.zeros(3), torch.tensor([4.0, 6.0])])
    g = torch.Generator().manual_seed(seed)
    x = pool[torch.randint(len(pool), (rows, k), generator=g)]
    x = x * (torch.randint(0, 2, (rows, k), generator=g) * 2 - 1)
    span = 6 if dtype == torch.float16 else 60
    power = torch.randint(-span, span, (rows, -(-k // 32)), generator=g).repeat_interleave(32, 1)[:, :k]
    x = torch.ldexp(x, power)
    x[rows // 2] = 0.0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 32), (3, 31), (2, 33), (33, 64), (5, 264), (130, 40), (2, 1001)])
def test_quantize_is_the_definition(rows, k, dtype):
    x = awkward(rows, k, dtype, rows + k)
    values, scales = definition(x)
    t = qib.mx_quantize(x.cuda())
    assert torch.equal(t.row_scales().cpu().long(), scales)
    for out in (torch.bfloat16, torch.float32):
        assert torch.equal(t.dequantize(out).cpu().double(), values)
    assert t.shape == (rows, k)


@pytest.mark.parametrize("rows,k", [(257, 4307), (1, 12288), (1000, 96)])
def test_quantize_of_ordinary_values(rows, k):
    x = randn((rows, k), 3, 2.0, torch.bfloat16)
    got = qib.mx_quantize(x.cuda()).dequantize(torch.float32).cpu()
    # within half a step: 1/16 of the value from half the scale on, a quarter scale below; saturation loses up to a quarter
    pad = torch.nn.functional.pad(x.float(), (0, -k % 32)).view(rows, -1, 32)
    scale = torch.exp2(torch.floor(torch.log2(pad.abs().amax(-1, keepdim=True))) - 2).expand_as(pad).reshape(rows, -1)[:, :k]
    assert ((got - x.float()).abs() <= torch.maximum(x.float().abs() * 0.25, scale * 0.25)).all()


def test_extremes_and_non_finite_blocks():
    x = torch.zeros((6, 64))
    x[0, :32] = torch.finfo(torch.float32).max
    x[1, 3] = 2.0**-149                # smallest subnormal: below half a code of the smallest scale
    x[1, 40] = 2.0**-126
    x[2, 5], x[2, 6] = math.inf, 1.0
    x[3, 37] = math.nan
    x[4, 0] = -0.0
    x[5] = 2.0**-127 * torch.tensor([0.5, 1.5, 6.0, 0.25] * 16)
    t = qib.mx_quantize(x.cuda())
    values, scales = definition(x)
    assert torch.equal(t.row_scales().cpu().long(), scales)
    got = t.dequantize(torch.float32).cpu()
    torch.testing.assert_close(got.double(), values, rtol=0, atol=0, equal_nan=True)
    assert scales[2, 0] == 255 and not torch.isnan(got[2, 32:]).any() and torch.isnan(got[3, 32:]).all()
    half = qib.mx_quantize(torch.full((1, 32), 1e6).cuda()).dequantize(torch.float16)
    assert torch.isinf(half).all()     # past f16's range


def test_strided_rows_leading_dims_and_odd_addresses():
    base = randn((2, 9, 200), 5, dtype=torch.bfloat16).cuda()
    x = base[:, :, 3:100]              # rows 200 apart from an odd column
    t = qib.mx_quantize(x)
    assert t.shape == (2, 9, 97) and t.dequantize().shape == (2, 9, 97)
    assert torch.equal(t.dequantize(), qib.mx_quantize(x.contiguous()).dequantize())
    y = base[0].t()                    # columns apart: copied
    assert torch.equal(qib.mx_quantize(y).dequantize(), qib.mx_quantize(y.contiguous()).dequantize())


def test_packed_round_trip_and_empty():
    x = randn((130, 100), 9).cuda()
    t = qib.mx_quantize(x)
    u = qib.MxTensor.from_packed(t.codes, t.row_scales(), 100)
    assert torch.equal(u.dequantize(), t.dequantize()) and torch.equal(u.row_scales(), t.row_scales())
    e = qib.mx_quantize(x[:0])
    assert e.dequantize().shape == (0, 100) and e.row_scales().shape == (0, 4)
    with pytest.raises(qib.QmmError):
        qib.mx_quantize(x[:, :0])
    with pytest.raises(qib.QmmError):
        qib.mx_quantize(x.double())


# ---------------------------------------------------------------- product


def layer(n, k, seed, bias=True):
    w = randn((n, k), seed, 0.05)
    b = randn((n,), seed + 1, 0.3, torch.bfloat16) if bias else None
    return qib.MxLinear.from_dense(w.cuda(), None if b is None else b.cuda())


def reference(lin, x, act="none", gate=None, residual=None, mul=False, bias="own"):
    """(result, tolerance) in 64 bits from the values that the operands stand for."""
    xv = qib.mx_quantize(x).dequantize(torch.float32).double()
    wv = lin.weight.dequantize(torch.float32).double()
    t, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    b = lin.bias if isinstance(bias, str) else bias
    if b is not None:
        t, size = t + b.double(), size + b.double().abs()
    if act == "gelu_tanh":
        t = torch.nn.functional.gelu(t, approximate="tanh")
    elif act == "silu":
        t = torch.nn.functional.silu(t)
    if gate is not None:
        t, size = t * gate.double(), size * gate.double().abs()
    if residual is not None:
        r = residual.double().view(t.shape)
        t, size = (r * t, r.abs() * size) if mul else (r + t, size + r.abs())
    return t, 2.0**-8 * 1.01 * t.abs() + 2.0**-22 * (lin.input / 64 + 4) * size


def close(y, ref):
    want, tol = ref
    d = (y.double().view(want.shape) - want).abs()
    assert (d <= tol).all(), float((d - tol).max())


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 64, 127, 129, 300])
@pytest.mark.parametrize("k,n", [(32, 8), (33, 7), (64, 192), (100, 193), (256, 64), (257, 500), (1152, 333), (3072, 128)])
def test_product_at_odd_sizes(m, k, n):
    lin = layer(n, k, m + k)
    x = randn((m, k), n, dtype=torch.bfloat16).cuda()
    y = lin.forward(x)
    assert y.dtype == torch.bfloat16 and y.shape == (m, n)
    close(y, reference(lin, x))
    assert qib.device_error() == 0


@pytest.mark.parametrize("m,k,n", [(1, 12288, 9601), (3, 6400, 9728), (1, 20000, 9600), (2, 9000, 200), (17, 5000, 4800)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_deep_products_of_few_tokens(m, k, n, dtype):
    # more stages than the ring holds, several times over, with and without a split of k
    lin = layer(n, k, 1)
    x = randn((m, k), 2, dtype=dtype).cuda()
    y = lin.forward(x)
    close(y, reference(lin, x))
    assert torch.equal(y, lin.forward(qib.mx_quantize(x))) and qib.device_error() == 0


@pytest.mark.parametrize("m,k,n", [(1, 512, 640), (9, 320, 96), (40, 1000, 1000), (513, 768, 2304), (2100, 512, 384)])
@pytest.mark.parametrize("act,gated,residual,mul", [("gelu_tanh", False, False, False), ("none", True, True, False),
                                                    ("silu", False, True, True), ("gelu_tanh", True, True, True), (None, True, False, False)])
def test_epilogues(m, k, n, act, gated, residual, mul):
    lin = layer(n, k, 1)
    x = randn((m, k), 2, dtype=torch.float16).cuda()
    gate = randn((n,), 3, dtype=torch.bfloat16).cuda() if gated else None
    res = randn((m, n), 4, 2.0, torch.bfloat16).cuda() if residual else None
    y = lin.forward_fused(x, activation=act, gate=gate, residual=res, residual_mul=mul)
    close(y, reference(lin, x, act or "none", gate, res, mul))


@pytest.mark.parametrize("m", [3, 200])
@pytest.mark.parametrize("n", [96, 101])
def test_residual_in_place_bias_override_and_out(m, n):
    lin = layer(n, 256, 1)
    x = randn((m, 256), 2).cuda()
    res = randn((m, n), 4, 2.0, torch.bfloat16).cuda()
    want = lin.forward_fused(x, residual=res, bias=None)
    close(want, reference(lin, x, residual=res, bias=None))
    acc = res.clone()
    assert lin.forward_fused(x, residual=acc, bias=None, out=acc) is acc and torch.equal(acc, want)
    odd = torch.empty((m * n + 1,), dtype=torch.bfloat16, device="cuda")[1:].view(m, n)  # not 16-byte aligned
    lin.forward_fused(x, residual=res, bias=None, out=odd)
    assert torch.equal(odd, want)


@pytest.mark.parametrize("k", [300, 2401])  # single CTAs, pairs
@pytest.mark.parametrize("n", [3501, 3502, 3504, 3517, 3551])  # rows of y that begin at any element; a last chunk of any width
def test_wide_rows_at_any_alignment(k, n):
    m = 1100
    lin = layer(n, k, 1)
    x = qib.mx_quantize(randn((m, k), 2).cuda())
    xv = x.dequantize(torch.float32)
    close(lin.forward(x), reference(lin, xv))
    res = randn((m, n), 4, 2.0, torch.bfloat16).cuda()
    gate = randn((n,), 3, dtype=torch.bfloat16).cuda()
    want = lin.forward_fused(x, activation="silu", gate=gate, residual=res)
    close(want, reference(lin, xv, "silu", gate, res))
    close(lin.forward_fused(x, residual=res, residual_mul=True), reference(lin, xv, residual=res, mul=True))
    guard = torch.full((m * n + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
    acc = guard[: m * n].view(m, n)
    acc.copy_(res)
    lin.forward_fused(x, activation="silu", gate=gate, residual=acc, out=acc)
    assert torch.equal(acc, want) and (guard[m * n :] == 7.0).all() and qib.device_error() == 0


def test_quantised_input_strides_batches_and_order_of_rows():
    lin = layer(300, 200, 1)
    x = randn((2, 70, 260), 2, dtype=torch.bfloat16).cuda()[:, :, 40:240]
    y = lin.forward(x)
    assert y.shape == (2, 70, 300)
    assert torch.equal(y, lin.forward(x.contiguous())) and torch.equal(y, lin.forward(qib.mx_quantize(x)))
    # rows do not meet: any order and number of them gives the same bits on the same path
    flip = torch.arange(139, -1, -1, device="cuda")
    assert torch.equal(lin.forward(x.reshape(140, 200)[flip]), y.view(140, 300)[flip])
    assert lin.forward(x[:0]).shape == (0, 70, 300)


@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_non_finite_rows_stay_in_their_row(m):
    lin = layer(200, 512, 1)
    x = randn((m, 512), 2, dtype=torch.bfloat16).cuda()
    want = lin.forward(x)
    x[m // 2, 100] = math.nan
    y = lin.forward(x)
    assert torch.isnan(y[m // 2]).all()
    keep = torch.arange(m, device="cuda") != m // 2
    assert torch.equal(y[keep], want[keep])
    x[m // 2] = 0.0
    assert torch.equal(lin.forward(x)[m // 2], lin.bias)


@pytest.mark.parametrize("m", [1, 33, 400])
def test_repeats_streams_and_graphs(m):
    lin = layer(1000, 1000, 1)
    x = randn((m, 1000), 2, dtype=torch.bfloat16).cuda()
    want = lin.forward(x)
    for _ in range(3):
        assert torch.equal(lin.forward(x), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys = [lin.forward(x * s) for s in (1.0, 2.0, 1.0)]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(ys[0], want) and torch.equal(ys[2], want)
    buf = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = lin.forward(buf)
    buf.copy_(x * 2)
    graph.replay()
    assert torch.equal(y, ys[1])
    buf.copy_(x)
    graph.replay()
    graph.replay()
    assert torch.equal(y, want)


def test_back_to_back_calls_read_fresh_inputs():
    # each call's input is written by the kernel before it, and its output feeds the next
    lin = layer(512, 512, 1, bias=False)
    x = randn((4, 512), 2, dtype=torch.bfloat16).cuda()
    want = x
    for _ in range(6):
        want = (lin.forward(want.clone()).float() * 0.5).to(torch.bfloat16)
        torch.cuda.synchronize()
    got = x
    for _ in range(6):
        got = (lin.forward(got).float() * 0.5).to(torch.bfloat16)
    assert torch.equal(got, want)


def test_python_refusals():
    lin = layer(64, 64, 1)
    x = randn((4, 64), 2, dtype=torch.bfloat16).cuda()
    for call, status in (
            (lambda: lin.forward(x[:, :63]), _lib.QMM_ERR_BAD_SHAPE),
            (lambda: lin.forward(x.double()), _lib.QMM_ERR_INVALID_ARGUMENT),
            (lambda: lin.forward(x.cpu()), _lib.QMM_ERR_CUDA),
            (lambda: lin.forward_fused(x, activation="tanh"), _lib.QMM_ERR_INVALID_ARGUMENT),
            (lambda: lin.forward_fused(x, gate=x), _lib.QMM_ERR_BAD_SHAPE),
            (lambda: lin.forward_fused(x, residual=x[:3]), _lib.QMM_ERR_BAD_SHAPE),
            (lambda: lin.forward_fused(x, out=torch.empty((4, 64), device="cuda")), _lib.QMM_ERR_INVALID_ARGUMENT),
            (lambda: qib.MxLinear(lin.weight, torch.zeros(63).cuda()), _lib.QMM_ERR_BAD_SHAPE),
            (lambda: qib.mx_quantize(x).dequantize(torch.int32), _lib.QMM_ERR_INVALID_ARGUMENT)):
        with pytest.raises(qib.QmmError) as e:
            call()
        assert e.value.status == status
