"""An MXFP4 product right behind the kernels that make its operands: the
process-wide qmm_set_weights_immutable concerns the GEMV's affine weights, which no
kernel of the library writes, and must not let a product read the codes that a
quantisation ahead of it on the stream is still writing."""
import glob
import os

import pytest
import torch

import qwen_imager_b200 as qib
from qwen_imager_b200 import _lib

CSRC = os.path.join(os.path.dirname(os.path.abspath(qib.__file__)), "csrc")


def test_only_the_gemv_reads_its_weight_ahead_of_the_stream():
    users = [os.path.basename(f) for f in glob.glob(os.path.join(CSRC, "*.cu")) if "weights_immutable()" in open(f).read()]
    assert sorted(users) == ["qmm_api.cu", "qmm_gemv_mma.cu"]  # its definition, its one reader


@pytest.fixture
def immutable():
    lib = _lib.load()
    before = lib.qmm_set_weights_immutable(1)
    yield
    lib.qmm_set_weights_immutable(before)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 4, 40, 128, 300])
@pytest.mark.parametrize("n,k", [(640, 512), (9216, 3072), (1000, 6400)])
def test_product_right_behind_its_weights_quantisation(immutable, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m + n)
    x = torch.randn((m, k), generator=g, device="cuda").to(torch.bfloat16)
    for _ in range(3):
        w = torch.randn((n, k), generator=g, device="cuda")
        torch.cuda.synchronize()
        lin = qib.MxLinear.from_dense(w)
        got = lin.forward(x)                                 # the weight's codes were written by the kernel just ahead
        torch.cuda.synchronize()
        assert torch.equal(got, lin.forward(x))
        assert torch.equal(qib.mx_quantize(w).codes, lin.weight.codes)
    assert qib.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 300])
def test_product_right_behind_its_input(immutable, m):
    g = torch.Generator(device="cuda").manual_seed(m)
    lin = qib.MxLinear.from_dense(torch.randn((512, 512), generator=g, device="cuda"))
    x = torch.randn((m, 512), generator=g, device="cuda").to(torch.bfloat16)
    for _ in range(4):
        _, n = qib.gated_residual_norm(x, pre="rms", quantize=True)
        got = lin.forward(n)                                 # MXFP4 rows by the norm just ahead
        torch.cuda.synchronize()
        assert torch.equal(got, lin.forward(n))
        x = got
