"""Block operators under an SM budget, on wide rows at any alignment, and with vectors of
mixed alignment in every width's kernel.  Tolerances are those of the operators' own
tests (test_gpu_gated_norm, test_gpu_mxfp4); a budget changes which CTA works, and only
the few-token product's split of k, so everything else keeps its bits."""
import math

import pytest
import torch

import qwen_imager_b200 as qib
from qwen_imager_b200 import _lib
from test_gpu_gated_norm import BF, close, make, reference
from test_gpu_mxfp4 import close as product_close
from test_gpu_mxfp4 import layer, randn
from test_gpu_mxfp4 import reference as product_reference

pytestmark = pytest.mark.gpu


@pytest.fixture
def budget():
    lib = _lib.load()
    yield lib.qmm_set_sm_budget
    lib.qmm_set_sm_budget(0)


@pytest.mark.parametrize("sms", [1, 2, 3, 37, 147])
@pytest.mark.parametrize("m,k,n", [(1, 6400, 500), (3, 12288, 3000), (40, 2048, 640), (128, 1100, 333), (600, 300, 3504), (1100, 2401, 3500), (1100, 2401, 3501)])
def test_products_under_a_budget(budget, sms, m, k, n):
    lin = layer(n, k, 1)
    x = randn((m, k), 2, dtype=torch.bfloat16).cuda()
    res = randn((m, n), 4, 2.0, torch.bfloat16).cuda()
    budget(sms)
    y = lin.forward(x)
    z = lin.forward_fused(x, activation="silu", residual=res)
    codes = lin.forward(qib.mx_quantize(x))
    assert qib.device_error() == 0
    budget(0)
    product_close(y, product_reference(lin, x))
    product_close(z, product_reference(lin, x, "silu", None, res))
    product_close(codes, product_reference(lin, x))


@pytest.mark.parametrize("sms", [1, 5, 100])
def test_norm_and_rotary_under_a_budget(budget, sms):
    axes, pos = qib.RotaryAxes((10, 12)), torch.randint(0, 99, (301, 2), device="cuda")
    q = randn((301, 6, 64), 1, dtype=torch.bfloat16).cuda()
    w = torch.ones((64,), dtype=torch.bfloat16, device="cuda")

    def everything():
        out = list(qib.qk_norm_rotary(q[:, :4], q[:, 4:], pos, axes, q_weight=w, k_weight=w))
        for hidden in (100, 250, 500, 1001, 5000, 20000):
            x, b, s = make(301 if hidden < 5000 else 7, hidden, BF, BF, seed=hidden, groups=7)
            out += qib.gated_residual_norm(x, b, post="rms", pre="layer", **s)
            out.append(qib.gated_residual_norm(x, b, post="rms", pre="layer", quantize=True, **s)[1].dequantize())
        return out

    want = everything()
    budget(sms)
    got = everything()
    budget(0)
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), i


@pytest.mark.parametrize("xt,bt", [(BF, BF), (torch.float32, BF), (torch.float32, torch.float32), (torch.float16, torch.float32)])
@pytest.mark.parametrize("rows,hidden", [(5, 8193), (3, 10007), (4, 12288), (3, 16383), (3, 16384), (2, 16385), (2, 32767)])
@pytest.mark.parametrize("at,gap", [(1, 0), (3, 2), (0, 4)])
def test_wide_rows_at_any_alignment_among_nan(rows, hidden, xt, bt, at, gap):
    x, b, s = make(rows, hidden, xt, bt)

    def slot(t, dtype, fill):
        buf = torch.full((at + rows * (hidden + gap) + 5,), fill, dtype=dtype, device="cuda")
        view = torch.as_strided(buf, (rows, hidden), (hidden + gap, 1), at)
        if t is not None:
            view.copy_(t)
        return buf, view

    _, xv = slot(x, xt, math.nan)
    _, bv = slot(b, bt, math.nan)
    (xb, xo), (nb, no) = slot(None, xt, 7.0), slot(None, xt, 7.0)
    qib.gated_residual_norm(xv, bv, post="layer", pre="rms", residual_scale=0.75, x_out=xo, n_out=no, **s)
    ref = reference(x, b, s, "layer", "rms", 0.75)
    close(xo, ref[0])
    close(no, ref[1])
    _, mx = qib.gated_residual_norm(xv, bv, post="layer", pre="rms", residual_scale=0.75, quantize=True, **s)
    assert torch.isfinite(mx.dequantize(torch.float32)).all()
    for buf, view in ((xb, xo), (nb, no)):
        view.fill_(7.0)
        assert (buf == 7.0).all()


@pytest.mark.parametrize("vt", [BF, torch.float32])
@pytest.mark.parametrize("rows,hidden", [(35, 96), (35, 99), (21, 128), (21, 121), (14, 248), (14, 480), (7, 1024), (7, 1030), (7, 9000)])
@pytest.mark.parametrize("off", [("gate",), ("post_weight",), ("scale", "shift"), ("pre_weight", "gate", "scale", "shift", "post_weight")])
def test_vectors_of_mixed_alignment_and_groups(rows, hidden, vt, off):
    x, b, s = make(rows, hidden, BF, BF, groups=7, vt=vt)
    moved = dict(s)
    for name in off:  # one element behind a boundary, groups a stride apart that is no multiple of eight
        v = s[name].view(-1, hidden)
        buf = torch.full((v.shape[0] * (hidden + 3) + 1,), math.nan, dtype=vt, device="cuda")
        view = torch.as_strided(buf, v.shape, (hidden + 3, 1), 1)
        view.copy_(v)
        moved[name] = view if s[name].dim() == 2 else view[0]
    got = qib.gated_residual_norm(x, b, post="rms", pre="layer", **moved)
    want = qib.gated_residual_norm(x, b, post="rms", pre="layer", **s)
    ref = reference(x, b, s, "rms", "layer", 1.0)
    close(got[0], ref[0])
    close(got[1], ref[1])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])  # the vectors' values do not depend on how they are read
    q = qib.gated_residual_norm(x, b, post="rms", pre="layer", quantize=True, **moved)[1]
    assert torch.equal(q.codes, qib.gated_residual_norm(x, b, post="rms", pre="layer", quantize=True, **s)[1].codes)
