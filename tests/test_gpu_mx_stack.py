"""The MXFP4 stack: its fused, in-place path against the same steps one at a time.

Quantisation to four bits is discontinuous, so a stack compared with 32-bit
operations differs by whole codes wherever a rounding falls the other way; each
operator is compared with 64 bits in its own tests.  Here the steps are taken apart
(separate norms on 32-bit copies, separate quantisation, new tensors, torch for the
gate and residual): every value that is rounded is rounded from the same 32-bit
result up to its own last bits, and everything linear in front of a quantisation is
the same call, so the first block's inputs must be equal bit for bit and its outputs
up to the bits that two orders of the same 32-bit sum leave."""
import pytest
import torch
import torch.nn.functional as F

import qwen_imager_b200 as qib
from qwen_imager_b200.mx_stack import MxStack, MxStackConfig, joint_positions

pytestmark = pytest.mark.gpu

CFG = MxStackConfig(height=9, width=7, text=13, blocks=2, hidden=512, heads=4, head_dim=128, ffn=1024)


def apart(stack, x, temb):
    """The module docstring's formulas with one public call, or a torch operation, a step."""
    cfg = stack.cfg
    rows = (slice(0, cfg.image), slice(cfg.image, cfg.tokens))
    pos = joint_positions(cfg)
    t = F.silu(temb.float()).to(torch.bfloat16)[None]
    mods = [[w.mod(t).view(6, cfg.hidden) for w in block] for block in stack.blocks]
    norm = lambda v, scale, shift: qib.mx_quantize(qib.gated_residual_norm(v, pre="layer", scale=scale, shift=shift)[1])  # noqa: E731
    streams = [x[r].float() for r in rows]  # 32-bit: norms leave unrounded
    for m, block in zip(mods, stack.blocks):
        q, k, v = [], [], []
        for s, w in enumerate(block):
            shift1, scale1 = m[s][0], m[s][1]
            qkv = w.qkv(norm(streams[s], scale1, shift1)).view(-1, 3, cfg.heads, cfg.head_dim)
            a, b = qib.qk_norm_rotary(qkv[:, 0].contiguous(), qkv[:, 1].contiguous(), pos[rows[s]], stack.axes, q_weight=w.q_norm, k_weight=w.k_norm)
            q.append(a), k.append(b), v.append(qkv[:, 2])
        q, k, v = (torch.cat(u).transpose(0, 1)[None] for u in (q, k, v))
        a = F.scaled_dot_product_attention(q, k, v)[0].transpose(0, 1).reshape(cfg.tokens, -1)
        for s, w in enumerate(block):
            gate1, shift2, scale2, gate2 = m[s][2], m[s][3], m[s][4], m[s][5]
            mid, _ = qib.gated_residual_norm(streams[s], w.out(a[rows[s]]), post="rms", post_weight=w.post_attn, gate=gate1, pre=None)
            h = w.up.forward_fused(norm(mid, scale2, shift2), activation="gelu_tanh")
            mid = mid.to(torch.bfloat16).float()  # the hidden state is bf16 between the sublayers
            end, _ = qib.gated_residual_norm(mid, w.down(h), post="rms", post_weight=w.post_ffn, gate=gate2, pre=None)
            streams[s] = end
        # (the next block's norm sees the unrounded state, its residual the rounded one)
        nxt = [e.to(torch.bfloat16).float() for e in streams]
        yield torch.cat(nxt).to(torch.bfloat16)
        streams = nxt


def test_one_block_equals_its_steps():
    cfg = MxStackConfig(**{**CFG.__dict__, "blocks": 1})
    stack = MxStack.random(cfg, seed=3)
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((cfg.tokens, cfg.hidden), generator=g, device="cuda").to(torch.bfloat16)
    temb = torch.randn((cfg.hidden,), generator=g, device="cuda").to(torch.bfloat16)
    want = next(apart(stack, x, temb))
    start, before = x.clone(), qib._lib.launch_count()
    got = stack.forward(x, temb)
    assert got is x and qib._lib.launch_count() > before and qib.device_error() == 0
    assert (want.float() - start.float()).norm() > 0.1 * start.float().norm()  # the block does something
    # Two orders of a 32-bit sum may turn a rounding, of a code or of bf16, in a few of a million places.
    assert (got != want).float().mean() < 0.01
    assert (got.float() - want.float()).norm() < 1e-3 * want.float().norm()


def test_each_stream_uses_its_own_weights_and_modulation():
    # Only the text stream's feed-forward differs: image rows of the last block are the same bits.
    cfg = MxStackConfig(**{**CFG.__dict__, "blocks": 1})
    stack = MxStack.random(cfg, seed=3)
    other = MxStack(cfg, [[stack.blocks[0][0], MxStack.random(cfg, seed=9).blocks[0][1]]])
    other.blocks[0][1].qkv, other.blocks[0][1].mod = stack.blocks[0][1].qkv, stack.blocks[0][1].mod
    other.blocks[0][1].q_norm, other.blocks[0][1].k_norm = stack.blocks[0][1].q_norm, stack.blocks[0][1].k_norm
    x = torch.randn((cfg.tokens, cfg.hidden), device="cuda").to(torch.bfloat16)
    temb = torch.randn((cfg.hidden,), device="cuda").to(torch.bfloat16)
    a, b = stack.forward(x.clone(), temb), other.forward(x.clone(), temb)
    assert torch.equal(a[:cfg.image], b[:cfg.image]) and not torch.equal(a[cfg.image:], b[cfg.image:])


def test_stack_repeats_and_runs_in_a_graph():
    stack = MxStack.random(CFG, seed=5)
    x0 = torch.randn((CFG.tokens, CFG.hidden), device="cuda").to(torch.bfloat16)
    temb = torch.randn((CFG.hidden,), device="cuda").to(torch.bfloat16)
    want = stack.forward(x0.clone(), temb)
    assert torch.equal(stack.forward(x0.clone(), temb), want)
    x = x0.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stack.forward(x, temb)
    x.copy_(x0)
    graph.replay()
    assert torch.equal(x, want)


def test_stack_refuses_other_shapes():
    stack = MxStack.random(MxStackConfig(height=2, width=2, text=1, blocks=1, hidden=256, heads=2, ffn=256))
    with pytest.raises(ValueError):
        stack.forward(torch.zeros((6, 256), device="cuda", dtype=torch.bfloat16), torch.zeros(256, device="cuda"))
    with pytest.raises(ValueError):
        MxStackConfig(height=2, width=2, text=1, axes=(8, 28, 29))


def test_state_itself_where_there_is_nothing_to_add():
    x = torch.randn((5, 512), device="cuda").to(torch.bfloat16)
    same, n = qib.gated_residual_norm(x, pre="rms")
    assert same is x or same.data_ptr() == x.data_ptr()
    copy, m = qib.gated_residual_norm(x, pre="rms", x_out=torch.empty_like(x))
    assert torch.equal(copy, x) and torch.equal(n, m) and copy.data_ptr() != x.data_ptr()
