"""q/k norm and multi-axis rotary positions against a 64-bit implementation.

Tolerance: one rounding to the output type (half an ulp: 2^-8, 2^-11, 2^-24 of
the value) plus f32 arithmetic on a pair: 2^-20 of the pair's length covers the
norm's sum over at most 256 columns (2^-21 in relative error), the angle's
2^-22 turns and the products."""
import math

import pytest
import torch

import qwen_imager_b200 as qib
from qwen_imager_b200 import _lib

pytestmark = pytest.mark.gpu

ROUND = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def reference(x, positions, dims, theta, pairs, ladder, weight, eps=1e-6):
    """(values, tolerance) f64; x [batch, tokens, heads, dim], positions [batch, tokens, axes]."""
    v = x.double()
    if weight is not None:
        v = v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    total = sum(dims)
    freq = [theta ** (-i / n) for n in dims for i in range(n)] if ladder == "own" else [theta ** (-i / total) for i in range(total)]
    axis = [a for a, n in enumerate(dims) for _ in range(n)]
    angle = positions.double()[..., axis] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    c, s = angle.cos()[..., None, :], angle.sin()[..., None, :]
    a, b = (v[..., 0:2 * total:2], v[..., 1:2 * total:2]) if pairs == "adjacent" else (v[..., :total], v[..., total:2 * total])
    out, size = v.clone(), v.abs()
    length = (a.square() + b.square()).sqrt()
    if pairs == "adjacent":
        out[..., 0:2 * total:2], out[..., 1:2 * total:2] = a * c - b * s, a * s + b * c
        size[..., 0:2 * total:2], size[..., 1:2 * total:2] = length, length
    else:
        out[..., :total], out[..., total:2 * total] = a * c - b * s, a * s + b * c
        size[..., :total], size[..., total:2 * total] = length, length
    return out, out.abs() * ROUND[x.dtype] * 1.01 + size * 2.0**-20 + (2.0**-25 if x.dtype == torch.float16 else 0.0)


def close(got, ref):
    want, tol = ref
    d = (got.double() - want).abs()
    assert (d <= tol).all(), float((d - tol).max())


def make(batch, tokens, hq, hk, dim, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (torch.randn((batch, tokens, hq, dim), generator=g, device="cuda") * 1.5).to(dtype)
    k = (torch.randn((batch, tokens, hk, dim), generator=g, device="cuda") * 1.5).to(dtype)
    w = lambda: (1 + 0.1 * torch.randn((dim,), generator=g, device="cuda")).to(dtype)  # noqa: E731
    return q, k, w(), w()


def grid(tokens, axes, seed=1, lo=-64, hi=2000):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(lo, hi, (tokens, axes), generator=g, dtype=torch.int32).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("dim,dims", [(128, (8, 28, 28)), (64, (32,)), (72, (8, 12, 12)), (80, (7, 13, 11)), (96, (16, 17, 15)),
                                      (256, (64, 32, 32)), (32, (4, 4)), (30, (5, 5, 5)), (7, (1, 1, 1)), (2, (1,)), (256, (43, 43, 42))])
def test_matches_64_bits(dim, dims, pairs, dtype):
    for batch, tokens, hq, hk, ladder, norm in ((1, 1, 4, 1, "own", True), (2, 37, 6, 2, "shared", True), (1, 300, 3, 3, "own", False)):
        q, k, wq, wk = make(batch, tokens, hq, hk, dim, dtype, tokens)
        pos = grid(tokens, len(dims))
        axes = qib.RotaryAxes(dims, 10000.0, pairs, ladder)
        if not norm:
            wq = wk = None
        a, b = qib.qk_norm_rotary(q, k, pos, axes, q_weight=wq, k_weight=wk)
        close(a, reference(q, pos[None], dims, 10000.0, pairs, ladder, wq))
        close(b, reference(k, pos[None], dims, 10000.0, pairs, ladder, wk))


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_far_and_fractional_positions_lose_nothing(kind):
    q, k, wq, wk = make(1, 64, 2, 2, 128, torch.float32)
    pos = torch.randint(-2**24, 2**24, (64, 3), generator=torch.Generator().manual_seed(2)).cuda()
    pos = pos.to(kind) if kind != torch.float32 else pos.float() / 64
    axes = qib.RotaryAxes((24, 20, 20), 1e6)
    a, b = qib.qk_norm_rotary(q, k, pos, axes, q_weight=wq, k_weight=wk)
    # the frequency itself is held to 2^-48: 2^24 positions turn it by at most 2^-24 more
    close(a, reference(q, pos[None], (24, 20, 20), 1e6, "adjacent", "own", wq))
    close(b, reference(k, pos[None], (24, 20, 20), 1e6, "adjacent", "own", wk))


def test_positions_of_each_batch_one_weight_and_q_alone():
    q, k, wq, _ = make(3, 50, 4, 2, 64, torch.bfloat16)
    pos = torch.stack([grid(50, 2, s) for s in range(3)])
    axes = qib.RotaryAxes((10, 22), pairs="halves")
    a, b = qib.qk_norm_rotary(q, k, pos, axes, q_weight=wq)
    close(a, reference(q, pos, (10, 22), 10000.0, "halves", "own", wq))
    close(b, reference(k, pos, (10, 22), 10000.0, "halves", "own", None))
    c, none = qib.qk_norm_rotary(q, None, pos, axes, q_weight=wq)
    assert none is None and torch.equal(c, a)
    d, _ = qib.qk_norm_rotary(q[0], k[0], pos[0], axes, q_weight=wq)
    assert torch.equal(d, a[0])


@pytest.mark.parametrize("dim,dims", [(128, (8, 28, 28)), (40, (5, 7))])
@pytest.mark.parametrize("tokens", [1, 129])
def test_fused_projection_in_place_and_into_head_major(dim, dims, tokens):
    qkv = torch.randn((2, tokens, 8, dim), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(torch.bfloat16)
    q, k, v = qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]
    w = torch.ones((dim,), dtype=torch.bfloat16, device="cuda")
    pos = grid(tokens, len(dims))
    axes = qib.RotaryAxes(dims)
    a, b = qib.qk_norm_rotary(q, k, pos, axes, q_weight=w, k_weight=w)
    assert a.is_contiguous() and a.shape == q.shape
    close(a, reference(q, pos[None], dims, 10000.0, "adjacent", "own", w))
    heads = torch.empty((2, 4, tokens, dim), dtype=torch.bfloat16, device="cuda")
    kheads = torch.empty((2, 2, tokens, dim), dtype=torch.bfloat16, device="cuda")
    qib.qk_norm_rotary(q, k, pos, axes, q_weight=w, k_weight=w, q_out=heads.transpose(1, 2), k_out=kheads.transpose(1, 2))
    assert torch.equal(heads.transpose(1, 2), a) and torch.equal(kheads.transpose(1, 2), b)
    keep = v.clone()
    qib.qk_norm_rotary(q, k, pos, axes, q_weight=w, k_weight=w, q_out=q, k_out=k)
    assert torch.equal(q, a) and torch.equal(k, b) and torch.equal(v, keep)


def test_odd_addresses_and_strides_take_the_general_path():
    flat = torch.randn((3 + 20 * 5 * 131,), device="cuda").to(torch.float16)
    q = flat[3:].view(20, 5, 131)[:, :, 1:129]
    pos = grid(20, 3)
    axes = qib.RotaryAxes((8, 28, 28), pairs="halves")
    a, _ = qib.qk_norm_rotary(q, None, pos, axes)
    b, _ = qib.qk_norm_rotary(q.contiguous(), None, pos, axes)
    close(a[None], reference(q[None], pos[None], (8, 28, 28), 10000.0, "halves", "own", None))
    assert torch.equal(a, b)


def test_no_pairs_no_tokens_and_other_frequencies():
    q, k, wq, wk = make(1, 9, 2, 2, 64, torch.float32)
    none = qib.RotaryAxes.from_pairs([], [], 1)
    a, b = qib.qk_norm_rotary(q, k, torch.zeros((9, 1), dtype=torch.int32, device="cuda"), none, q_weight=wq, k_weight=wk)
    want = q.double() / (q.double().square().mean(-1, keepdim=True) + 1e-6).sqrt() * wq.double()
    close(a, (want, want.abs() * 2.0**-20))
    e, _ = qib.qk_norm_rotary(q[:, :0], k[:, :0], torch.zeros((0, 1), dtype=torch.int32, device="cuda"), none)
    assert e.shape == (1, 0, 2, 64)
    # pairs dealt to the axes in turn, one ladder
    order = [p % 3 for p in range(32)]
    freq = [1e4 ** (-p / 32) for p in range(32)]
    axes = qib.RotaryAxes.from_pairs(order, freq, 3)
    pos = grid(9, 3)
    c, _ = qib.qk_norm_rotary(q, None, pos, axes)
    angle = pos.double()[:, order] * torch.tensor(freq, dtype=torch.float64, device="cuda")
    z = torch.view_as_complex(q.double().view(1, 9, 2, 32, 2).contiguous()) * torch.polar(torch.ones_like(angle), angle)[None, :, None]
    want = torch.view_as_real(z).reshape(1, 9, 2, 64)
    assert ((c.double() - want).abs() <= z.abs().repeat_interleave(2, -1) * 2.0**-20).all()


def test_zeros_infinities_and_nan_stay_in_their_head():
    q, _, wq, _ = make(1, 5, 4, 1, 64, torch.bfloat16)
    pos = grid(5, 1)
    axes = qib.RotaryAxes((32,))
    want, _ = qib.qk_norm_rotary(q, None, pos, axes, q_weight=wq)
    q[0, 2, 1] = 0.0
    q[0, 3, 2, 7] = math.nan
    q[0, 4, 0, 9] = math.inf
    got, _ = qib.qk_norm_rotary(q, None, pos, axes, q_weight=wq)
    assert (got[0, 2, 1] == 0).all() and torch.isnan(got[0, 3, 2]).all() and torch.isnan(got[0, 4, 0]).any()
    same = torch.ones((5, 4), dtype=torch.bool)
    same[2, 1] = same[3, 2] = same[4, 0] = False
    assert torch.equal(got[0][same.cuda()], want[0][same.cuda()])


def test_python_refusals():
    q, k, wq, _ = make(1, 9, 4, 2, 64, torch.bfloat16)
    pos = grid(9, 3)
    axes = qib.RotaryAxes((10, 11, 11))
    for call, status in (
            (lambda: qib.qk_norm_rotary(q, k.float(), pos, axes), _lib.QMM_ERR_BAD_SHAPE),
            (lambda: qib.qk_norm_rotary(q, k[:, :8], pos, axes), _lib.QMM_ERR_BAD_SHAPE),
            (lambda: qib.qk_norm_rotary(q[0, 0], None, pos, axes), _lib.QMM_ERR_BAD_SHAPE),
            (lambda: qib.qk_norm_rotary(q, k, pos[:8], axes), _lib.QMM_ERR_BAD_SHAPE),
            (lambda: qib.qk_norm_rotary(q, k, pos[:, :2], axes), _lib.QMM_ERR_BAD_SHAPE),
            (lambda: qib.qk_norm_rotary(q, k, pos.double(), axes), _lib.QMM_ERR_INVALID_ARGUMENT),
            (lambda: qib.qk_norm_rotary(q, k, pos.cpu(), axes), _lib.QMM_ERR_INVALID_ARGUMENT),
            (lambda: qib.qk_norm_rotary(q, k, pos, qib.RotaryAxes((11, 11, 11))), _lib.QMM_ERR_BAD_SHAPE),
            (lambda: qib.qk_norm_rotary(q, k, pos, axes, q_weight=wq[:63]), _lib.QMM_ERR_BAD_SHAPE),
            (lambda: qib.qk_norm_rotary(q, k, pos, axes, q_out=k), _lib.QMM_ERR_BAD_SHAPE),
            (lambda: qib.qk_norm_rotary(q[:, :8], None, pos[:8], axes, q_out=q[:, 1:]), _lib.QMM_ERR_INVALID_ARGUMENT)):
        with pytest.raises(qib.QmmError) as e:
            call()
        assert e.value.status == status
