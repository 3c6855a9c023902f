"""MxTensor takes codes and scales of exactly the sizes that the kernels read:
anything else would be read, or written, past its end."""
import pytest
import torch

import qwen_imager_b200 as qib
from qwen_imager_b200 import _lib

ROWS, K = 130, 300  # two row tiles, two 256-column chunks, a short last block


def parts(rows=ROWS, k=K):
    return torch.zeros((rows, -(-k // 32) * 16), dtype=torch.uint8), torch.zeros((-(-rows // 128) * -(-k // 256) * 1024,), dtype=torch.uint8)


def test_the_sizes_are_the_librarys():
    from qwen_imager_b200 import _block
    for rows, k in ((1, 1), (128, 256), (129, 257), (ROWS, K), (5, 33)):
        codes, scales = parts(rows, k)
        assert codes.numel() == _block.load().qmm_mx4_code_bytes(rows, k) and scales.numel() == _block.load().qmm_mx4_scale_bytes(rows, k)
        t = qib.MxTensor(codes, scales, rows, k)
        assert t.shape == (rows, k) and t.lead == (rows,)
        e = qib.MxTensor.empty(rows, k, "cpu")
        assert e.codes.shape == codes.shape and e.scales.shape == scales.shape
    codes, scales = parts()
    assert qib.MxTensor(codes, scales, ROWS, K, (2, 65)).shape == (2, 65, K)
    assert qib.MxTensor(codes[:0], scales[:0], 0, K).shape == (0, K)


def shifted(t):
    return torch.cat([t.new_zeros((4,)), t.flatten()])[4:].view(t.shape)  # 4 bytes behind a 16-byte boundary


@pytest.mark.parametrize("change,status", [
    (lambda c, s: (c, s[:-1], ROWS, K), _lib.QMM_ERR_BAD_SHAPE),               # scales end early
    (lambda c, s: (c, s[:1024], ROWS, K), _lib.QMM_ERR_BAD_SHAPE),
    (lambda c, s: (c[:-1], s, ROWS, K), _lib.QMM_ERR_BAD_SHAPE),               # so do codes
    (lambda c, s: (c, s, ROWS + 1, K), _lib.QMM_ERR_BAD_SHAPE),
    (lambda c, s: (c, s, ROWS, K + 32), _lib.QMM_ERR_BAD_SHAPE),
    (lambda c, s: (c, s, ROWS, 0), _lib.QMM_ERR_BAD_SHAPE),
    (lambda c, s: (c, s, -1, K), _lib.QMM_ERR_BAD_SHAPE),
    (lambda c, s: (c.flatten(), s, ROWS, K), _lib.QMM_ERR_BAD_SHAPE),
    (lambda c, s: (c, s, ROWS, K, (2, 64)), _lib.QMM_ERR_BAD_SHAPE),           # results would be shorter than the rows
    (lambda c, s: (c, s, ROWS, K, (-2, -65)), _lib.QMM_ERR_BAD_SHAPE),
    (lambda c, s: (c.short(), s, ROWS, K), _lib.QMM_ERR_INVALID_ARGUMENT),
    (lambda c, s: (c, s.float(), ROWS, K), _lib.QMM_ERR_INVALID_ARGUMENT),
    (lambda c, s: (c.t().contiguous().t(), s, ROWS, K), _lib.QMM_ERR_INVALID_ARGUMENT),  # columns apart
    (lambda c, s: (c, s.repeat_interleave(2)[::2], ROWS, K), _lib.QMM_ERR_INVALID_ARGUMENT),
    (lambda c, s: (c, s.to("meta"), ROWS, K), _lib.QMM_ERR_INVALID_ARGUMENT),  # another device
    (lambda c, s: (shifted(c), s, ROWS, K), _lib.QMM_ERR_MISALIGNED),
    (lambda c, s: (c, shifted(s), ROWS, K), _lib.QMM_ERR_MISALIGNED),
])
def test_refuses(change, status):
    with pytest.raises(qib.QmmError) as e:
        qib.MxTensor(*change(*parts()))
    assert e.value.status == status


@pytest.mark.gpu
def test_a_tensor_of_given_parts_is_the_quantised_one():
    x = torch.randn((ROWS, K), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    t = qib.mx_quantize(x)
    u = qib.MxTensor(t.codes, t.scales, ROWS, K, (2, 65))
    assert torch.equal(u.dequantize(), t.dequantize().view(2, 65, K))
    lin = qib.MxLinear.from_dense(torch.randn((64, K), device="cuda"))
    assert torch.equal(lin.forward(u).view(ROWS, 64), lin.forward(t))
    assert torch.equal(qib.MxLinear(qib.MxTensor(lin.weight.codes, lin.weight.scales, 64, K)).forward(t), lin.forward(t))
