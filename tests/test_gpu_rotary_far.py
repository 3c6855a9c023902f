"""Rotary positions past 2^24, where a whole number no longer fits one f32.

Tolerance beside the rounding of the output and 2^-20 of the pair's length (as at
near positions): frequencies up to one radian are held to 2^-52 turns, and the
terms of the angle that are not reduced to a fraction first stay below 2^-27 of the
position in turns, so below 2^7 for the farthest here (2^33): rounded to 2^-18
turns, three of them.  In radians 2 pi 3 2^-18 = 7.2e-5, and per position below the
stated maximum in proportion."""
import math

import pytest
import torch

import qwen_imager_b200 as qib

pytestmark = pytest.mark.gpu


def check(got, x, pos, freq, pairs, far):
    v, count = x.double(), len(freq)
    angle = (pos.double() * torch.tensor(freq, dtype=torch.float64, device=x.device))[:, None]
    a, b = (v[..., 0:2 * count:2], v[..., 1:2 * count:2]) if pairs == "adjacent" else (v[..., :count], v[..., count:2 * count])
    length = (a.square() + b.square()).sqrt()
    tol = length * (2.0**-24 + 2.0**-20 + 7.2e-5 * far / 2.0**33)
    g = got.double()
    ga, gb = (g[..., 0:2 * count:2], g[..., 1:2 * count:2]) if pairs == "adjacent" else (g[..., :count], g[..., count:2 * count])
    assert ((ga - (a * angle.cos() - b * angle.sin())).abs() <= tol).all()
    assert ((gb - (a * angle.sin() + b * angle.cos())).abs() <= tol).all()


@pytest.mark.parametrize("pairs,count,dim", [("adjacent", 32, 64), ("halves", 32, 64), ("adjacent", 20, 64), ("halves", 5, 30)])
@pytest.mark.parametrize("kind,reach", [(torch.int32, 2**31 - 1), (torch.int64, 2**31), (torch.int64, 2**33)])
def test_whole_positions_past_24_bits(pairs, count, dim, kind, reach):
    g = torch.Generator(device="cuda").manual_seed(count)
    q = torch.randn((64, 3, dim), generator=g, device="cuda")
    far = torch.randint(-reach, reach, (52,), generator=torch.Generator().manual_seed(1))
    near = torch.tensor([2**24 + 1, -(2**24) - 1, 2**24 - 1, 2**25 + 1, 2**25 + 3, 2**30 + 1, 2**30 + 63, -reach, reach, reach - 1, 0, 1])
    pos = torch.cat([far, near]).to(kind).cuda()[:, None]
    freq = [10000.0 ** (-i / count) for i in range(count)]
    got, _ = qib.qk_norm_rotary(q, None, pos, qib.RotaryAxes((count,), pairs=pairs))
    check(got, q, pos, freq, pairs, reach)


def test_neighbours_past_24_bits_differ():
    q = torch.ones((2, 1, 2), device="cuda")
    pos = torch.tensor([[2**24], [2**24 + 1]], dtype=torch.int32, device="cuda")
    got, _ = qib.qk_norm_rotary(q, None, pos, qib.RotaryAxes((1,)))
    a = got.double().cpu()
    turn = math.atan2(a[1, 0, 1], a[1, 0, 0]) - math.atan2(a[0, 0, 1], a[0, 0, 0])
    assert abs((turn - 1.0 + math.pi) % (2 * math.pi) - math.pi) <= 2e-6
