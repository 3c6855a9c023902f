"""Columns that rotary positions leave unturned, among infinities, NaN and signed
zeros: they are only normalised, so each goes its own way, in every layout.

Without a weight they leave with the bits they came with.  With one, and for the
turned columns, the 64-bit definition decides: finite values within one rounding
(half an ulp) and 2^-20 of the pair's length, the same infinities and NaN."""
import math

import pytest
import torch

import qwen_imager_b200 as qib

pytestmark = pytest.mark.gpu

ROUND = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
BITS = {torch.bfloat16: torch.int16, torch.float16: torch.int16, torch.float32: torch.int32}
AWKWARD = [math.inf, -math.inf, math.nan, -0.0, 0.0]


def definition(x, pos, count, pairs, weight):
    """(values, length of what each column's value comes from) f64."""
    v = x.double()
    if weight is not None:
        v = v / (v.square().mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
    freq = torch.tensor([10000.0 ** (-i / count) for i in range(count)], dtype=torch.float64, device=x.device)
    angle = (pos.double() * freq)[:, None]
    ia = torch.arange(count, device=x.device) * (2 if pairs == "adjacent" else 1)
    ib = ia + (1 if pairs == "adjacent" else count)
    a, b = v[..., ia], v[..., ib]
    out, size = v.clone(), v.abs()
    out[..., ia], out[..., ib] = a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()
    size[..., ia] = size[..., ib] = (a.square() + b.square()).sqrt()
    return out, size


def agree(got, want, size, dtype):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    ok = torch.isfinite(want)
    tol = want.abs() * ROUND[dtype] * 1.01 + size * 2.0**-20 + (2.0**-25 if dtype == torch.float16 else 0.0)
    assert ((got - want).abs()[ok] <= tol[ok]).all()


def heads(tokens, count, dim, dtype, offset):
    """[tokens, heads, dim] whose first element lies `offset` elements behind a 16-byte boundary, rows at multiples of 8."""
    g = torch.Generator(device="cuda").manual_seed(dim + count)
    pitch = -(-dim // 8) * 8 + 8
    base = torch.randn((tokens, count, pitch), generator=g, device="cuda").to(dtype)
    return base[..., offset:offset + dim]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
@pytest.mark.parametrize("dim,count", [(64, 16), (64, 17), (64, 18), (64, 19), (64, 0), (72, 32), (72, 33), (128, 20), (256, 100), (30, 5)])
@pytest.mark.parametrize("offset", [0, 4, 1])  # 16-byte accesses, 8-byte ones, the general kernel
def test_unturned_columns_keep_to_themselves(dim, count, pairs, dtype, offset):
    q = heads(6, 5, dim, dtype, offset)
    tail = 2 * count
    for h in range(5):
        for j, bad in enumerate(AWKWARD):
            q[1, h, tail + (7 * h + 3 * j) % (dim - tail)] = bad
        q[2, h, tail] = AWKWARD[h]                   # the first column behind the boundary
        q[3, h, dim - 1] = AWKWARD[h]
        if count:
            q[4, h, tail - 1] = AWKWARD[h]           # the last one before it, and its pair
    pos = torch.arange(1, 7, device="cuda", dtype=torch.int32)[:, None]
    axes = qib.RotaryAxes((count,), pairs=pairs)
    got, _ = qib.qk_norm_rotary(q, None, pos, axes)
    kind = BITS[dtype]
    nan = torch.isnan(q[..., tail:])
    assert torch.equal(torch.isnan(got[..., tail:]), nan)
    assert torch.equal(got[..., tail:].contiguous().view(kind)[~nan], q[..., tail:].contiguous().view(kind)[~nan])
    agree(got, *definition(q, pos, count, pairs, None), dtype)


@pytest.mark.parametrize("pairs,dim,count", [("adjacent", 64, 17), ("adjacent", 72, 20), ("halves", 64, 16), ("halves", 72, 20), ("halves", 64, 17)])
def test_unturned_columns_with_norm_weights(pairs, dim, count):
    dtype = torch.bfloat16
    q = heads(4, 3, dim, dtype, 0)
    pos = torch.arange(1, 5, device="cuda", dtype=torch.int32)[:, None]
    axes = qib.RotaryAxes((count,), pairs=pairs)
    w = torch.linspace(-1.5, 1.5, dim, device="cuda").to(dtype)
    got, _ = qib.qk_norm_rotary(q, None, pos, axes, q_weight=w)
    agree(got, *definition(q, pos, count, pairs, w), dtype)
    q[1, 0, dim - 2] = math.inf                      # the head's other columns become 0, this one NaN
    q[2, 1, dim - 1] = math.nan
    got, _ = qib.qk_norm_rotary(q, None, pos, axes, q_weight=w)
    agree(got, *definition(q, pos, count, pairs, w), dtype)
    w[dim - 1] = math.inf                            # a weight reaches its own column alone
    got, _ = qib.qk_norm_rotary(q, None, pos, axes, q_weight=w)
    agree(got, *definition(q, pos, count, pairs, w), dtype)


@pytest.mark.parametrize("pairs", ["adjacent", "halves"])
def test_unturned_columns_in_place_and_in_k(pairs):
    qkv = torch.randn((9, 6, 64), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.float16)
    qkv[:, :, 41] = math.inf
    qkv[3, :, 50] = math.nan
    keep = qkv.clone()
    q, k = qkv[:, :2], qkv[:, 2:4]
    pos = torch.arange(9, device="cuda", dtype=torch.int32)[:, None]
    axes = qib.RotaryAxes((16,), pairs=pairs)
    a, b = qib.qk_norm_rotary(q, k, pos, axes)
    qib.qk_norm_rotary(q, k, pos, axes, q_out=q, k_out=k)
    assert torch.equal(q.view(torch.int16), a.view(torch.int16)) and torch.equal(k.view(torch.int16), b.view(torch.int16))
    assert torch.equal(qkv[..., 32:].isnan(), keep[..., 32:].isnan())
    assert torch.equal(qkv[..., 32:].nan_to_num(0, 9, -9), keep[..., 32:].nan_to_num(0, 9, -9))
    assert torch.equal(qkv[:, 4:].nan_to_num(0, 9, -9), keep[:, 4:].nan_to_num(0, 9, -9))
