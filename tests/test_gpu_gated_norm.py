"""Norms before and after a sublayer with gate and residual against 64 bits.

Tolerances: one rounding to the output type (half an ulp: 2^-p of the value with p
significant bits, 8, 11 or 24) plus f32 arithmetic.
Sums of up to 32768 columns go through at most 32 terms a thread and two trees:
2^-18 relative covers them; a layer norm's mean is off by at most 2^-22 of the
row's largest magnitude, which 1 / std magnifies."""
import itertools
import math

import pytest
import torch

import qwen_imager_b200 as qib
from qwen_imager_b200 import _lib

pytestmark = pytest.mark.gpu

ROUND = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
BF = torch.bfloat16


def normed(v, how, eps):
    """(norm, magnification of the row's largest magnitude)"""
    if how == "layer":
        v = v - v.mean(-1, keepdim=True)
    elif how != "rms":
        return v, torch.ones_like(v[..., :1])
    r = 1 / (v.square().mean(-1, keepdim=True) + eps).sqrt()
    return v * r, r


def reference(x, branch, s, post, pre, c, eps=1e-6):
    """((x', tolerance), (n, tolerance))"""
    rows, hidden = x.shape
    def per_row(name):
        v = s.get(name)
        if v is None:
            return None
        v = v.double().reshape(-1, hidden)
        return v.repeat_interleave(rows // v.shape[0], 0)
    size = (x.double() * c).abs()
    y = x.double() * c
    if branch is not None:
        b = branch.double()
        h, r = normed(b, post, eps)
        hs = h.abs() + b.abs().amax(-1, keepdim=True) * r * 2.0**-3
        for name in ("post_weight", "gate"):
            if s.get(name) is not None:
                h, hs = h * per_row(name), hs * per_row(name).abs()
        y, size = y + h, size + hs
    out = x.dtype
    xt = y.abs() * ROUND[out] * 1.01 + size * 2.0**-18 + (2.0**-25 if out == torch.float16 else 0.0)
    n, r = normed(y, pre, eps)
    ns = n.abs() + (size.amax(-1, keepdim=True) * r if pre not in (None, "none") else size)
    if s.get("pre_weight") is not None:
        n, ns = n * per_row("pre_weight"), ns * per_row("pre_weight").abs()
    if s.get("scale") is not None:
        n, ns = n * (1 + per_row("scale")), ns * (1 + per_row("scale")).abs()
    if s.get("shift") is not None:
        n, ns = n + per_row("shift"), ns + per_row("shift").abs()
    return (y, xt), (n, n.abs() * ROUND[out] * 1.01 + ns * 2.0**-18 + (2.0**-25 if out == torch.float16 else 0.0))


def close(got, ref):
    want, tol = ref
    d = (got.double() - want).abs()
    assert (d <= tol).all(), float((d - tol).max())


def make(rows, hidden, xt, bt, groups=1, seed=0, vt=BF):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, sd=1.0, mean=0.0: torch.randn(s, generator=g, device="cuda") * sd + mean  # noqa: E731
    x, b = r(rows, hidden, sd=2.0, mean=0.3).to(xt), r(rows, hidden, mean=0.5).to(bt)
    s = dict(post_weight=r(hidden, sd=0.1, mean=1.0).to(vt), pre_weight=r(hidden, sd=0.1, mean=1.0).to(vt),
             gate=r(groups, hidden, sd=0.5).to(vt), scale=r(groups, hidden, sd=0.2).to(vt), shift=r(groups, hidden, sd=0.3).to(vt))
    return x, b, s


@pytest.mark.parametrize("hidden", [1, 7, 8, 31, 64, 250, 768, 1000, 1024, 1025, 1160, 3072, 4096, 5000, 8192, 8200, 16384, 20001, 32768])
@pytest.mark.parametrize("rows", [1, 5])
def test_widths(rows, hidden):
    for xt, bt in ((BF, BF), (torch.float32, BF), (torch.float16, torch.float32)):
        x, b, s = make(rows, hidden, xt, bt, seed=hidden)
        xn, n = qib.gated_residual_norm(x, b, post="rms", pre="layer", residual_scale=0.75, **s)
        assert xn.dtype == n.dtype == xt
        rx, rn = reference(x, b, s, "rms", "layer", 0.75)
        close(xn, rx)
        if hidden > 1:  # a layer norm of one column is rounding alone
            close(n, rn)


@pytest.mark.parametrize("post,pre", list(itertools.product([None, "rms", "layer"], ["none", "rms", "layer"])))
@pytest.mark.parametrize("keep", [(), ("gate",), ("post_weight", "pre_weight"), ("scale", "shift"), ("gate", "shift"),
                                  ("post_weight", "pre_weight", "gate", "scale", "shift")])
@pytest.mark.parametrize("hidden", [512, 333])
def test_every_combination(post, pre, keep, hidden):
    x, b, s = make(6, hidden, BF, torch.float16, groups=3, vt=torch.float32)
    s = {k: v for k, v in s.items() if k in keep}
    xn, n = qib.gated_residual_norm(x, b, post=post, pre=pre, **s)
    rx, rn = reference(x, b, s, post, pre, 1.0)
    close(xn, rx)
    close(n, rn)


def test_no_branch_mixed_vectors_and_broadcast_groups():
    x, _, s = make(12, 640, torch.float32, BF, groups=4)
    s = dict(pre_weight=s["pre_weight"].float(), scale=s["scale"][:, None], shift=s["shift"][:1])  # f32, [4, 1, h], one row
    xn, n = qib.gated_residual_norm(x, pre="rms", residual_scale=0.5, **s)
    rx, rn = reference(x, None, s, None, "rms", 0.5)
    close(xn, rx)
    close(n, rn)
    y, m = qib.gated_residual_norm(x.view(4, 3, 640), pre="rms", residual_scale=0.5, **s)
    assert torch.equal(m.view(12, 640), n) and m.shape == (4, 3, 640)


@pytest.mark.parametrize("hidden", [1024, 1001])
def test_in_place_and_strided_rows(hidden):
    x, b, s = make(40, hidden, BF, BF)
    want = qib.gated_residual_norm(x, b, post="rms", pre="layer", **s)
    wide_x, wide_b = (torch.zeros((40, hidden + 13), dtype=BF, device="cuda") for _ in range(2))
    wide_x[:, 5:5 + hidden], wide_b[:, :hidden] = x, b
    got = qib.gated_residual_norm(wide_x[:, 5:5 + hidden], wide_b[:, :hidden], post="rms", pre="layer", **s)
    # the order of a sum depends on alignment: equal up to the tolerance of each
    ref = reference(x, b, s, "rms", "layer", 1.0)
    close(got[0], ref[0])
    close(got[1], ref[1])
    x2, b2 = x.clone(), b.clone()
    r = qib.gated_residual_norm(x2, b2, post="rms", pre="layer", x_out=x2, n_out=b2, **s)
    assert r[0] is x2 and r[1] is b2 and torch.equal(x2, want[0]) and torch.equal(b2, want[1])


@pytest.mark.parametrize("xt,bt", [(BF, BF), (torch.float16, BF), (torch.float32, BF), (torch.float32, torch.float32), (BF, torch.float32)])
@pytest.mark.parametrize("rows,hidden", [(1, 1), (9, 3), (30, 84), (31, 127), (5, 129), (40, 201), (12, 257), (6, 511), (7, 1677), (3, 5001), (2, 9001)])
@pytest.mark.parametrize("at,gap", [(0, 0), (1, 0), (3, 2), (6, 10)])  # first column, columns between rows
def test_rows_at_any_alignment_among_nan(rows, hidden, xt, bt, at, gap):
    x, b, s = make(rows, hidden, xt, bt, groups=1 if rows % 2 else 2)

    def slot(t, dtype, fill):  # t as a view inside a buffer of `fill`
        buf = torch.full((at + rows * (hidden + gap) + 5,), fill, dtype=dtype, device="cuda")
        view = torch.as_strided(buf, (rows, hidden), (hidden + gap, 1), at)
        if t is not None:
            view.copy_(t)
        return buf, view

    _, xv = slot(x, xt, math.nan)
    _, bv = slot(b, bt, math.nan)
    (xb, xo), (nb, no) = slot(None, xt, 7.0), slot(None, xt, 7.0)
    qib.gated_residual_norm(xv, bv, post="rms", pre="layer", residual_scale=0.75, x_out=xo, n_out=no, **s)
    ref = reference(x, b, s, "rms", "layer", 0.75)
    close(xo, ref[0])
    close(no, ref[1])
    for buf, view in ((xb, xo), (nb, no)):
        view.fill_(7.0)
        assert (buf == 7.0).all()  # nothing written beside the rows


@pytest.mark.parametrize("rows,hidden", [(33, 100), (50, 128), (7, 129), (3, 5), (129, 120)])
def test_mxfp4_of_narrow_rows(rows, hidden):
    x, b, s = make(rows, hidden, torch.float32, BF)
    _, n = qib.gated_residual_norm(x, b, post="rms", pre="layer", **s)
    _, q = qib.gated_residual_norm(x, b, post="rms", pre="layer", quantize=True, **s)
    want = qib.mx_quantize(n)
    assert torch.equal(q.row_scales(), want.row_scales()) and torch.equal(q.codes, want.codes)
    lin = qib.MxLinear.from_dense(torch.randn((96, hidden), device="cuda"))
    assert torch.equal(lin.forward(q), lin.forward(n))


@pytest.mark.parametrize("rows,hidden", [(1, 64), (3, 40), (130, 3072), (33, 1000), (5, 761), (2, 9000)])
def test_mxfp4_result_is_the_quantised_norm(rows, hidden):
    x, b, s = make(rows, hidden, torch.float32, BF)
    xn, n = qib.gated_residual_norm(x, b, post="rms", pre="layer", **s)
    xq, q = qib.gated_residual_norm(x, b, post="rms", pre="layer", quantize=True, **s)
    want = qib.mx_quantize(n)  # f32 n: nothing is rounded in between
    assert torch.equal(xq, xn) and q.shape == (rows, hidden)
    assert torch.equal(q.row_scales(), want.row_scales()) and torch.equal(q.codes, want.codes)
    lin = qib.MxLinear.from_dense(torch.randn((96, hidden), device="cuda"))
    assert torch.equal(lin.forward(q), lin.forward(n))


def test_constant_rows_large_means_and_non_finite_rows():
    x, b, s = make(6, 512, torch.float32, torch.float32)
    b[0], x[0] = 0.0, 0.0
    x[1] = x[1] + 1000.0
    xn, n = qib.gated_residual_norm(x, b, post="rms", pre="layer", scale=s["scale"], shift=s["shift"])
    rx, rn = reference(x, b, dict(scale=s["scale"], shift=s["shift"]), "rms", "layer", 1.0)
    close(xn, rx)
    close(n, rn)
    assert torch.equal(n[0], s["shift"][0].float())  # variance 0: eps keeps it finite
    x[2, 3], b[3, 4] = math.nan, math.inf
    xm, m = qib.gated_residual_norm(x, b, post="rms", pre="layer", scale=s["scale"], shift=s["shift"])
    assert torch.isnan(m[2]).all() and torch.isnan(m[3]).any()
    keep = [0, 1, 4, 5]
    assert torch.equal(m[keep], n[keep]) and torch.equal(xm[keep], xn[keep])


def test_repeats_empty_and_streams():
    x, b, s = make(100, 3072, BF, BF)
    want = qib.gated_residual_norm(x, b, post="rms", pre="layer", **s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = qib.gated_residual_norm(x, b, post="rms", pre="layer", **s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    e = qib.gated_residual_norm(x[:0], b[:0], pre="rms")
    assert e[0].shape == e[1].shape == (0, 3072)
    e = qib.gated_residual_norm(x[:0], b[:0], pre="rms", quantize=True)
    assert e[1].shape == (0, 3072)


def test_python_refusals():
    x, b, s = make(12, 64, BF, BF, groups=3)
    g = qib.gated_residual_norm
    for call, status in (
            (lambda: g(x, b[:, :63]), _lib.QMM_ERR_BAD_SHAPE),
            (lambda: g(x.double()), _lib.QMM_ERR_INVALID_ARGUMENT),
            (lambda: g(x, b, post="batch"), _lib.QMM_ERR_INVALID_ARGUMENT),
            (lambda: g(x, gate=s["gate"]), _lib.QMM_ERR_INVALID_ARGUMENT),   # a gate without a branch
            (lambda: g(x[:10], b[:10], gate=s["gate"]), _lib.QMM_ERR_BAD_SHAPE),  # 10 rows, 3 groups
            (lambda: g(x, b, post_weight=s["gate"]), _lib.QMM_ERR_BAD_SHAPE),
            (lambda: g(x, b, pre_weight=s["pre_weight"].cpu()), _lib.QMM_ERR_INVALID_ARGUMENT),
            (lambda: g(x, b, x_out=torch.empty_like(x, dtype=torch.float32)), _lib.QMM_ERR_BAD_SHAPE),
            (lambda: g(x, b, n_out=x.clone(), quantize=True), _lib.QMM_ERR_INVALID_ARGUMENT),
            (lambda: g(x[1:], b[1:], x_out=x[:-1]), _lib.QMM_ERR_INVALID_ARGUMENT)):  # overlaps x, shifted
        with pytest.raises(qib.QmmError) as e:
            call()
        assert e.value.status == status
