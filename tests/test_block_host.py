"""The extension of the block operators' ordinary calls saves time and nothing else:
without it every operator gives the same results through its general way."""
import pytest
import torch

import qwen_imager_b200 as qib
from qwen_imager_b200 import _block, _lib, build


@pytest.fixture
def absent(tmp_path, monkeypatch):
    """No extension, and no compiler to build it."""
    monkeypatch.setattr(_block, "_host_module", None)
    monkeypatch.setattr(build, "HOST", str(tmp_path / "_qmm_host.so"))

    def failing(force=False):
        raise RuntimeError("no compiler")

    monkeypatch.setattr(build, "build_host", failing)


def test_the_extension_is_there_and_names_what_the_package_calls():
    host = _block.host()
    assert host is not _block._General
    for name in ("mx_quantize", "mx_dequantize", "mx_linear", "qk_norm_rotary", "gated_norm"):
        assert callable(getattr(host, name)) and getattr(_block._General, name)(1, 2) is None


def test_operators_go_their_general_way_without_it(absent):
    t = torch.zeros((4, 64), dtype=torch.bfloat16)
    with pytest.warns(RuntimeWarning, match="no compiler"):
        with pytest.raises(qib.QmmError) as e:
            qib.mx_quantize(t)
    assert e.value.status == _lib.QMM_ERR_CUDA and "CUDA only" in str(e.value)  # the operator's own refusal of a CPU tensor
    assert _block.host() is _block._General


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_results_do_not_depend_on_it(dtype, monkeypatch):
    g = torch.Generator(device="cuda").manual_seed(1)
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda").to(dtype)  # noqa: E731
    x, branch, w = randn(2, 70, 260), randn(2, 70, 260), randn(300, 260)
    bias, gate, residual = randn(300).bfloat16(), randn(300).bfloat16(), randn(2, 70, 300).bfloat16()
    q, k, qw = randn(2, 9, 4, 64), randn(2, 9, 2, 64), randn(64)
    pos = torch.randint(0, 90, (9, 2), device="cuda")
    axes = qib.RotaryAxes((12, 12))
    lin = qib.MxLinear.from_dense(w, bias)

    def everything():
        t = qib.mx_quantize(x)
        a, n = qib.gated_residual_norm(x, branch, post="rms", gate=x[0, 0], scale=x[:, 1], shift=branch[:, 2])
        b, m = qib.gated_residual_norm(x, None, residual_scale=0.5, quantize=True)
        return [t.codes, t.row_scales(), t.dequantize(), qib.mx_quantize(x[0]).dequantize(), a, n, b, m.dequantize(),
                lin.forward(x), lin.forward(t), lin.forward(m), lin.forward(x[0, :1]),
                lin.forward_fused(x, activation="silu", gate=gate, residual=residual, bias=None),
                *qib.qk_norm_rotary(q, k, pos, axes, q_weight=qw, k_weight=qw), qib.qk_norm_rotary(q, None, pos, axes)[0]]

    want = everything()
    assert _block.host() is not _block._General
    monkeypatch.setattr(_block, "_host_module", _block._General)
    for i, (a, b) in enumerate(zip(everything(), want)):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b), i
