"""include/qmm_block.h against its bindings and its host-side checks, on the CPU:
every declared symbol is exported and bound, the packed argument structs and
the Rust structs have the C layout, and each entry point refuses bad arguments
before it touches a device."""
import os
import re
import subprocess

import pytest

from qwen_imager_b200 import _block, _lib
from test_rust_binding import SCALARS, _c_param, _strip_c_comments

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "qmm_block.h")
CRATE = os.path.join(ROOT, "qmm-sys", "src", "block.rs")

TYPES = {"uint8_t": "u8", "qmm_mx4": "qmm_mx4", "qmm_mx4_linear_args": "qmm_mx4_linear_args",
         "qmm_rotary_args": "qmm_rotary_args", "qmm_gated_norm_args": "qmm_gated_norm_args"}


@pytest.fixture(autouse=True)
def block_types(monkeypatch):
    for k, v in TYPES.items():
        monkeypatch.setitem(SCALARS, k, v)


def header_text():
    return _strip_c_comments(open(HEADER).read())


def functions():
    out = {}
    for ret, name, args in re.findall(r"QMM_API\s+(\w+)\s+(qmm_\w+)\s*\(([^)]*)\)\s*;", header_text()):
        out[name] = ([_c_param(a) for a in " ".join(args.split()).split(",")], SCALARS[ret])
    return out


def test_every_declared_symbol_is_bound_and_exported():
    assert sorted(functions()) == sorted(_block.EXPORTED_SYMBOLS)
    lib = _block.load()
    for name in _block.EXPORTED_SYMBOLS:
        assert hasattr(lib, name), name


def test_rust_functions_structs_and_constants_match():
    text = re.sub(r"//.*", "", open(CRATE).read())
    block = re.search(r'extern "C" \{(.*?)\n\}', text, re.S).group(1)
    rust = {}
    for name, args, ret in re.findall(r"pub fn (qmm_\w+)\s*\(([^)]*)\)\s*->\s*([^;]+);", block):
        params = [tuple(p.strip() for p in a.split(":", 1)) for a in args.split(",") if a.strip()]
        rust[name] = (params, ret.strip())
    c = functions()
    assert sorted(rust) == sorted(c)
    for name in c:
        assert rust[name] == c[name], name
    fields = {n: [tuple(p.strip() for p in f.split(":", 1)) for f in re.findall(r"pub ([^\n]+?),\s*$", b, re.M)]
              for n, b in re.findall(r"pub struct (\w+) \{(.*?)\n\}", text, re.S)}
    mutable = {"y", "workspace", "q_out", "k_out", "x_out", "n_out", "n_codes", "n_scales"}  # written through
    for body, name in re.findall(r"typedef struct \w+ \{([^}]*)\}\s*(\w+);", header_text()):
        want = [_c_param(f) for f in body.split(";") if f.strip()]
        got = fields[name]
        assert [n for n, _ in got] == [n for n, _ in want], name
        for (n, g), (_, w) in zip(got, want):
            assert g == w, (name, n, g, w)
            assert not g.startswith("*mut") or n in mutable, (name, n)
    consts = {k: int(v) for k, v in re.findall(r"pub const (QMM_\w+): \w+ = (\d+);", text)}
    for body in re.findall(r"typedef enum \w+ \{([^}]*)\}", header_text()):
        for k, v in re.findall(r"(QMM_\w+)\s*=\s*(\d+)", body):
            assert consts.pop(k) == int(v)
    assert not consts
    assert "pub mod block;" in open(os.path.join(ROOT, "qmm-sys", "src", "lib.rs")).read()


def test_packed_structs_have_the_c_layout(tmp_path):
    names = ("qmm_mx4", "qmm_mx4_linear_args", "qmm_rotary_args", "qmm_gated_norm_args")
    src = tmp_path / "sizes.c"
    lines = ['printf("%%zu\\n", sizeof(%s));' % n for n in names]
    offsets = (("qmm_mx4_linear_args", "x_elem"), ("qmm_rotary_args", "batch"), ("qmm_rotary_args", "pos_batch_stride"),
               ("qmm_rotary_args", "eps"), ("qmm_gated_norm_args", "rows"), ("qmm_gated_norm_args", "x_elem"),
               ("qmm_gated_norm_args", "eps"))
    lines += ['printf("%%zu\\n", offsetof(%s, %s));' % o for o in offsets]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "qmm_block.h"\nint main(void) {%s return 0;}' % "".join(lines))
    exe = str(tmp_path / "sizes")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = [int(v) for v in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got[:4] == [_block.MX4.size, _block.LINEAR.size, _block.ROTARY.size, _block.NORM.size]
    assert got[4:] == [120, 72, 184, 224, 88, 168, 192]


def test_sizes_of_mxfp4_buffers():
    lib = _block.load()
    assert lib.qmm_mx4_code_bytes(5, 33) == 5 * 32          # two blocks a row
    assert lib.qmm_mx4_scale_bytes(5, 33) == 2 * 512        # one row tile, one 256-column chunk
    assert lib.qmm_mx4_scale_bytes(129, 257) == 2 * 4 * 512
    assert lib.qmm_mx4_workspace_bytes(3, 33) == 3 * 32 + 2 * 512
    # few tokens are quantised inside the product; the rest need the whole of x
    assert lib.qmm_mx4_linear_workspace_bytes(1, 18432, 3072) == lib.qmm_mx4_linear_workspace_bytes(4, 64, 64) == 0
    assert lib.qmm_mx4_linear_workspace_bytes(4096, 3072, 3072) == lib.qmm_mx4_workspace_bytes(4096, 3072)
    assert lib.qmm_mx4_linear_workspace_bytes(0, 64, 64) == 0
    assert lib.qmm_mx4_code_bytes(0, 33) == lib.qmm_mx4_scale_bytes(4, 0) == 0


A = 1 << 28  # an aligned address that nothing dereferences
NEED = 4096 * 32 + 32 * 1024


def linear(**kw):
    v = dict(codes=A, scales=2 * A, n=4096, k=64, m=4096, x=3 * A, stride=64, x_codes=0, x_scales=0, bias=0, gate=0, residual=0, y=4 * A,
             work=5 * A, bytes=NEED, elem=0, act=0)
    v.update(kw)
    return _block.load().qmm_mx4_linear(_block.LINEAR.pack(*v.values()), None)


@pytest.mark.parametrize("change,status", [
    (dict(codes=0), _lib.QMM_ERR_INVALID_ARGUMENT),
    (dict(y=0), _lib.QMM_ERR_INVALID_ARGUMENT),
    (dict(x=0), _lib.QMM_ERR_INVALID_ARGUMENT),                       # neither form of x
    (dict(x_codes=6 * A, x_scales=7 * A), _lib.QMM_ERR_INVALID_ARGUMENT),  # both
    (dict(x=0, x_codes=6 * A), _lib.QMM_ERR_INVALID_ARGUMENT),        # codes without scales
    (dict(n=0), _lib.QMM_ERR_BAD_SHAPE),
    (dict(k=-1), _lib.QMM_ERR_BAD_SHAPE),
    (dict(m=-1), _lib.QMM_ERR_BAD_SHAPE),
    (dict(m=1 << 40), _lib.QMM_ERR_UNSUPPORTED),
    (dict(stride=63), _lib.QMM_ERR_BAD_SHAPE),
    (dict(elem=3), _lib.QMM_ERR_INVALID_ARGUMENT),
    (dict(act=7), _lib.QMM_ERR_INVALID_ARGUMENT),
    (dict(act=0x200), _lib.QMM_ERR_INVALID_ARGUMENT),
    (dict(codes=A + 8), _lib.QMM_ERR_MISALIGNED),
    (dict(y=4 * A + 2), _lib.QMM_ERR_MISALIGNED),
    (dict(x=3 * A + 1), _lib.QMM_ERR_MISALIGNED),
    (dict(work=5 * A + 4), _lib.QMM_ERR_MISALIGNED),
    (dict(work=0), _lib.QMM_ERR_INVALID_ARGUMENT),
    (dict(bytes=NEED - 1), _lib.QMM_ERR_INVALID_ARGUMENT),
    (dict(y=3 * A), _lib.QMM_ERR_INVALID_ARGUMENT),                   # y overlaps x
    (dict(y=5 * A + 16), _lib.QMM_ERR_INVALID_ARGUMENT),              # y overlaps the workspace
    (dict(work=3 * A + 16), _lib.QMM_ERR_INVALID_ARGUMENT),           # the workspace overlaps x
    (dict(residual=4 * A + 16), _lib.QMM_ERR_INVALID_ARGUMENT),       # the residual overlaps y without being it
])
def test_linear_refuses(change, status):
    assert linear(**change) == status, _lib.load().qmm_last_error()


def test_no_tokens_is_a_no_op_without_a_device():
    assert linear(m=0, x=0, y=0) == _lib.QMM_OK


def rotary(**kw):
    v = dict(q=A, k=2 * A, q_out=3 * A, k_out=4 * A, q_weight=0, k_weight=0, positions=5 * A, turns=6 * A, axis=7 * A, batch=1,
             tokens=3, qs=(0, 256, 64), ks=(0, 128, 64), qo=(0, 256, 64), ko=(0, 128, 64), pos_batch=0, q_heads=4, k_heads=2, dim=64,
             pairs=32, axes=3, adjacent=1, pos_kind=0, elem=0, eps=1e-6)
    v.update(kw)
    flat = []
    for x in v.values():
        flat.extend(x if isinstance(x, tuple) else (x,))
    return _block.load().qmm_qk_norm_rotary(_block.ROTARY.pack(*flat), None)


@pytest.mark.parametrize("change,status", [
    (dict(q=0), _lib.QMM_ERR_INVALID_ARGUMENT),
    (dict(k_out=0), _lib.QMM_ERR_INVALID_ARGUMENT),
    (dict(positions=0), _lib.QMM_ERR_INVALID_ARGUMENT),
    (dict(pairs=33), _lib.QMM_ERR_BAD_SHAPE),
    (dict(axes=0), _lib.QMM_ERR_BAD_SHAPE),
    (dict(dim=264, pairs=4), _lib.QMM_ERR_UNSUPPORTED),
    (dict(elem=5), _lib.QMM_ERR_INVALID_ARGUMENT),
    (dict(pos_kind=3), _lib.QMM_ERR_INVALID_ARGUMENT),
    (dict(qs=(0, -256, 64)), _lib.QMM_ERR_BAD_SHAPE),
    (dict(qo=(0, 64, 64)), _lib.QMM_ERR_BAD_SHAPE),                   # output heads overlap
    (dict(q_out=A + 64), _lib.QMM_ERR_INVALID_ARGUMENT),              # half in place
    (dict(q_out=2 * A), _lib.QMM_ERR_INVALID_ARGUMENT),               # q's output over k
    (dict(k_out=3 * A), _lib.QMM_ERR_INVALID_ARGUMENT),               # one output over the other
    (dict(q=A + 1), _lib.QMM_ERR_MISALIGNED),
    (dict(turns=6 * A + 2), _lib.QMM_ERR_MISALIGNED),
    (dict(positions=5 * A + 4, pos_kind=1), _lib.QMM_ERR_MISALIGNED),
])
def test_rotary_refuses(change, status):
    assert rotary(**change) == status, _lib.load().qmm_last_error()


def test_rotary_accepts_q_and_k_side_by_side_in_place(monkeypatch):
    # q and k of a fused projection [tokens, 4 + 2 + 2 heads, 64], in place, and
    # alternating head by head: past every check, so only the device is missing.
    import torch
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")
    qs, ks = (0, 512, 64), (0, 512, 64)
    fused = dict(qs=qs, qo=qs, ks=ks, ko=ks, q_out=A, k=A + 4 * 128, k_out=A + 4 * 128)
    assert rotary(**fused) == _lib.QMM_ERR_CUDA
    alt = (0, 768, 192)
    assert rotary(qs=alt, qo=alt, ks=alt, ko=alt, q_out=A, k=A + 128, k_out=A + 128) == _lib.QMM_ERR_CUDA
    # one column of overlap is refused
    assert rotary(**dict(fused, k=A + 4 * 128 - 2, k_out=A + 4 * 128 - 2)) == _lib.QMM_ERR_INVALID_ARGUMENT


def norm(**kw):
    v = dict(x=A, branch=2 * A, x_out=3 * A, n_out=4 * A, codes=0, scales=0, post_weight=0, pre_weight=0, gate=0, shift=0, scale=0,
             rows=4, hidden=64, xs=64, bs=64, xo=64, no=64, gs=0, hs=0, ss=0, groups=1, xe=0, be=0, ve=0, post=1, pre=2, c=1.0, eps=1e-6)
    v.update(kw)
    return _block.load().qmm_gated_residual_norm(_block.NORM.pack(*v.values()), None)


@pytest.mark.parametrize("change,status", [
    (dict(x=0), _lib.QMM_ERR_INVALID_ARGUMENT),
    (dict(x_out=0, n_out=0, pre=0), _lib.QMM_ERR_INVALID_ARGUMENT),   # no output
    (dict(n_out=0), _lib.QMM_ERR_INVALID_ARGUMENT),                   # a norm without its output
    (dict(branch=0), _lib.QMM_ERR_INVALID_ARGUMENT),                  # a norm of no branch
    (dict(codes=5 * A), _lib.QMM_ERR_INVALID_ARGUMENT),               # codes without scales
    (dict(codes=5 * A, scales=6 * A), _lib.QMM_ERR_INVALID_ARGUMENT), # both forms of n
    (dict(rows=-1), _lib.QMM_ERR_BAD_SHAPE),
    (dict(hidden=0), _lib.QMM_ERR_BAD_SHAPE),
    (dict(groups=3), _lib.QMM_ERR_BAD_SHAPE),
    (dict(hidden=40000, xs=40000, bs=40000, xo=40000, no=40000), _lib.QMM_ERR_UNSUPPORTED),
    (dict(xs=63), _lib.QMM_ERR_BAD_SHAPE),
    (dict(xe=3), _lib.QMM_ERR_INVALID_ARGUMENT),
    (dict(post=3), _lib.QMM_ERR_INVALID_ARGUMENT),
    (dict(x=A + 1), _lib.QMM_ERR_MISALIGNED),
    (dict(gate=7 * A + 2, ve=1), _lib.QMM_ERR_MISALIGNED),
    (dict(x_out=A + 128), _lib.QMM_ERR_INVALID_ARGUMENT),             # overlaps x, not in place
    (dict(n_out=3 * A + 2), _lib.QMM_ERR_INVALID_ARGUMENT),           # overlaps x_out
    (dict(x_out=2 * A, be=1), _lib.QMM_ERR_INVALID_ARGUMENT),         # branch in place, but of another type
    (dict(n_out=0, codes=A, scales=6 * A), _lib.QMM_ERR_INVALID_ARGUMENT),  # codes over x
])
def test_norm_refuses(change, status):
    assert norm(**change) == status, _lib.load().qmm_last_error()


def test_quantize_refuses():
    lib = _block.load()
    q = lambda x=A, elem=0, rows=4, k=64, stride=64, codes=2 * A, scales=3 * A: lib.qmm_mx4_quantize(  # noqa: E731
        x, elem, rows, k, stride, codes, scales, None)
    assert q(x=0) == q(codes=0) == q(elem=9) == _lib.QMM_ERR_INVALID_ARGUMENT
    assert q(rows=-1) == q(k=0) == q(stride=63) == _lib.QMM_ERR_BAD_SHAPE
    assert q(codes=2 * A + 4) == q(x=A + 1) == _lib.QMM_ERR_MISALIGNED
    assert q(rows=0, x=0) == _lib.QMM_OK
    w = _block.MX4.pack(A, 2 * A, 4, 64)
    assert lib.qmm_mx4_dequantize(w, 3 * A, 7, None) == _lib.QMM_ERR_INVALID_ARGUMENT
    assert lib.qmm_mx4_dequantize(w, 0, 0, None) == _lib.QMM_ERR_INVALID_ARGUMENT
    assert lib.qmm_mx4_dequantize(w, 3 * A + 2, 1, None) == _lib.QMM_ERR_MISALIGNED
    assert lib.qmm_mx4_dequantize(_block.MX4.pack(A, 2 * A, 4, 0), 3 * A, 0, None) == _lib.QMM_ERR_BAD_SHAPE
    assert lib.qmm_mx4_tile_scales(0, 4, 64, A, None) == _lib.QMM_ERR_INVALID_ARGUMENT


def test_entry_points_fail_loudly_without_a_device():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")
    assert linear() == rotary() == norm() == _lib.QMM_ERR_CUDA
    assert _block.load().qmm_mx4_quantize(A, 0, 4, 64, 64, 2 * A, 3 * A, None) == _lib.QMM_ERR_CUDA


def test_python_entry_points_refuse_cpu_tensors_and_bad_axes():
    import torch

    import qwen_imager_b200 as q
    t = torch.zeros((4, 64), dtype=torch.bfloat16)
    for call in (lambda: q.mx_quantize(t), lambda: q.gated_residual_norm(t),
                 lambda: q.MxTensor.from_packed(torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((4, 2), dtype=torch.uint8))):
        with pytest.raises(q.QmmError) as e:
            call()
        assert e.value.status == _lib.QMM_ERR_CUDA
    axes = q.RotaryAxes((4, 6, 6), device="cpu")
    with pytest.raises(q.QmmError) as e:
        q.qk_norm_rotary(t.view(4, 2, 32), None, torch.zeros((4, 3), dtype=torch.int32), axes)
    assert e.value.status == _lib.QMM_ERR_CUDA
    for bad in (lambda: q.RotaryAxes((), device="cpu"), lambda: q.RotaryAxes((4,), pairs="odd", device="cpu"),
                lambda: q.RotaryAxes((4,), ladder="steep", device="cpu"), lambda: q.RotaryAxes((4, 4), theta=(1e4,), device="cpu"),
                lambda: q.RotaryAxes.from_pairs([0, 3], [1.0, 0.1], 3, device="cpu"),
                lambda: q.RotaryAxes.from_pairs([0], [float("inf")], 1, device="cpu"),
                lambda: q.MxTensor.from_packed(torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((4, 3), dtype=torch.uint8))):
        with pytest.raises(q.QmmError):
            bad()


def test_axes_turns_hold_each_frequency_in_two_terms():
    import math

    import qwen_imager_b200 as q
    axes = q.RotaryAxes((8, 28, 28), theta=10000.0, device="cpu")
    want = [10000.0 ** (-i / n) / (2 * math.pi) for n in (8, 28, 28) for i in range(n)]
    got = axes._turns.double().sum(-1)
    assert axes._axis.tolist() == [0] * 8 + [1] * 28 + [2] * 28
    # leading term to 2^-24, the rest to 2^-24 of that
    assert max(abs(g - w) / w for g, w in zip(got.tolist(), want)) <= 2.0**-48
    shared = q.RotaryAxes((24, 20, 20), ladder="shared", pairs="halves", device="cpu")
    assert shared.count == 64 and abs(shared._turns[63].double().sum().item() * 2 * math.pi - 10000.0 ** (-63 / 64)) < 1e-12
