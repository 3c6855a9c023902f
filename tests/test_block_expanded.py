"""Operands that are only read may repeat or share their rows (expanded batches, sliding
windows): the operators give what they give on a copy.  An output may not."""
import pytest
import torch

import qwen_imager_b200 as qib
from qwen_imager_b200 import _block, _lib


def forms(base, rows):
    """[rows, cols] views of base [1, cols] and of its neighbours whose rows overlap."""
    cols = base.shape[1]
    flat = torch.cat([base.flatten() + i for i in range(2 + 8 * rows // cols)])
    return [base.expand(rows, cols), flat.as_strided((rows, cols), (1, 1)), flat.as_strided((rows, cols), (8, 1))]


def test_rows_of_copies_rows_that_overlap():
    base = torch.arange(64.0)[None]
    for x in forms(base, 5):
        rows = _block.rows_of(x, 64)
        assert rows.stride(0) >= 64 and rows.stride(1) == 1 and torch.equal(rows, x)
    one = base.expand(1, 64)
    assert _block.rows_of(one, 64).data_ptr() == base.data_ptr()
    wide = torch.zeros((5, 80))[:, :64]
    assert _block.rows_of(wide, 64).data_ptr() == wide.data_ptr()
    column = torch.zeros((1, 1)).expand(7, 1)
    assert _block.rows_of(column, 1).stride(0) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [2, 40, 300])
def test_quantise_product_and_norm_of_repeated_rows(rows, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows)
    base = torch.randn((1, 512), generator=g, device="cuda").to(dtype)
    lin = qib.MxLinear.from_dense(torch.randn((200, 512), generator=g, device="cuda"))
    branch = torch.randn((rows, 512), generator=g, device="cuda").to(dtype)
    for x in forms(base, rows) + [base[0].expand(2, rows // 2, 512)]:
        copy = x.contiguous()
        assert torch.equal(qib.mx_quantize(x).dequantize(), qib.mx_quantize(copy).dequantize())
        assert torch.equal(lin.forward(x), lin.forward(copy))
        b = branch[: copy.numel() // 512].view(copy.shape)
        for got, want in ((qib.gated_residual_norm(x, b, post="rms"), qib.gated_residual_norm(copy, b, post="rms")),
                          (qib.gated_residual_norm(b, x, post="layer"), qib.gated_residual_norm(b, copy, post="layer"))):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        got, want = (qib.gated_residual_norm(t, b, quantize=True)[1].dequantize() for t in (x, copy))
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_an_output_with_repeated_rows_is_refused():
    x = torch.zeros((4, 64), device="cuda")
    for kw in (dict(x_out=torch.zeros((1, 64), device="cuda").expand(4, 64)), dict(n_out=torch.zeros((1, 64), device="cuda").expand(4, 64))):
        with pytest.raises(qib.QmmError) as e:
            qib.gated_residual_norm(x, x + 1, **kw)
        assert e.value.status == _lib.QMM_ERR_BAD_SHAPE
