"""The operators together, as a block of a served model uses them: LayerNorm, the adapted query / key / value projection, rotary positions in
place on the packed buffer, differential (or plain) attention, the adapted output projection on the residual stream. Every stage is
held against 64 bits on the stage's own inputs, with the tolerances of the operators' own tests; then the whole run is captured."""
import math

import pytest
import torch

import test_adapters
import test_diff_attention
import test_rotary
from fastbb_b200 import _lib, graphs
from fastbb_b200.adapters import Adapters, adapter_linear
from fastbb_b200.attention import attention
from fastbb_b200.diff_attention import diff_attention
from fastbb_b200.layernorm import layer_norm
from fastbb_b200.rotary import axial_plan, grid_positions, rotary

H = 4            # heads of the differential block: 2 H maps of 64 columns, H values of 128
C = 2 * H * 64


class Block:
    def __init__(self, differential, seed):
        g = torch.Generator("cuda").manual_seed(seed)
        rnd = lambda *s, std=1.0: (torch.randn(*s, generator=g, device="cuda") * std).half()  # noqa: E731
        self.differential = differential
        self.qkv_w, self.qkv_b = rnd(3 * C, C, std=C ** -0.5), rnd(3 * C, std=0.1)
        self.proj_w, self.proj_b, self.gamma = rnd(C, C, std=C ** -0.5), rnd(C, std=0.1), rnd(C, std=0.2)
        self.ln_w, self.ln_b = rnd(C, std=0.1) + 1, rnd(C, std=0.1)
        self.qkv_slots = Adapters(rnd(3, 16, C, std=C ** -0.5), rnd(3, 3 * C, 16, std=0.1), torch.tensor([1.0, 0.5, 2.0], device="cuda"))
        self.proj_slots = Adapters(rnd(3, 8, C, std=C ** -0.5), rnd(3, C, 8, std=0.1))
        self.lam, self.norm = torch.rand(H, generator=g, device="cuda") * 0.6 + 0.1, rnd(128, std=0.1) + 1
        self.plan = axial_plan(64, axes=2, theta=100.0, unit=2 * math.pi)

    def run(self, x, ids, where, lengths, keep=None):
        """x [B, N, C] -> the block's attention half, x + gamma * proj(...)."""
        B, N, _ = x.shape
        y = layer_norm(x, self.ln_w, self.ln_b)
        qkv = adapter_linear(y, self.qkv_w, self.qkv_slots, ids, b=self.qkv_b)
        before = qkv.clone() if keep is not None else None
        q, k, v = qkv.view(B, N, 3, 2 * H, 64).unbind(2)
        rotary(q, k, where, self.plan, n_prefix=N - where.shape[0], out=(q, k))
        if self.differential:
            o = diff_attention(q, k, v.reshape(B, N, H, 128), self.lam, weight=self.norm, out_scale=0.5, key_lengths=lengths)
        else:
            o = attention(q, k, v)
        out = adapter_linear(o.view(B, N, C), self.proj_w, self.proj_slots, ids, b=self.proj_b, res=x, gamma=self.gamma)
        if keep is not None:
            keep.update(y=y, before=before, q=q, k=k, v=v, o=o)
        return out


def make(B, h, w, registers, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(B, 1 + registers + h * w, C, generator=g, device="cuda").half()
    ids = torch.tensor([(i * 2 + 1) % 4 - 1 for i in range(B)], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([x.shape[1] - 7 * i for i in range(B)], dtype=torch.int32, device="cuda").clamp(min=0)
    return x, ids, grid_positions(h, w), lengths


@pytest.mark.gpu
@pytest.mark.parametrize("B,h,w,registers", [(1, 1, 1, 0), (3, 5, 7, 0), (5, 13, 11, 4), (2, 32, 40, 0)])
@pytest.mark.parametrize("differential", [True, False])
def test_a_block_stage_by_stage(B, h, w, registers, differential, oracle):
    block = Block(differential, B * h)
    x, ids, where, lengths = make(B, h, w, registers, w)
    N, kept, held = x.shape[1], {}, x.clone()
    out = block.run(x, ids, where, lengths, keep=kept)
    assert torch.equal(x, held)
    bounds = [i * N for i in range(B + 1)]
    # LayerNorm: fp32 arithmetic on fp16 rows, one rounding (2^-11), 2^-20 for a thousand fp32 roundings of the statistics
    y = torch.nn.functional.layer_norm(x.double(), (C,), block.ln_w.double(), block.ln_b.double(), 1e-6)
    assert bool(((kept["y"].double() - y).abs() <= y.abs() * 2.0 ** -11 + 2.0 ** -20 * (y.abs() + 10)).all())
    test_adapters.check(kept["before"], kept["y"], block.qkv_w, block.qkv_slots, ids.tolist(), bounds, b=block.qkv_b)
    parts = kept["before"].view(B, N, 3, 2 * H, 64)
    test_rotary.check(kept["q"], parts[:, :, 0], where, block.plan, n_prefix=1 + registers)
    test_rotary.check(kept["k"], parts[:, :, 1], where, block.plan, n_prefix=1 + registers)
    assert torch.equal(kept["v"], parts[:, :, 2])
    if differential:
        test_diff_attention.check(kept["o"], kept["q"], kept["k"], kept["v"].reshape(B, N, H, 128), block.lam, weight=block.norm, out_scale=0.5, lengths=lengths.tolist())
    else:
        want = oracle.attention(kept["q"].cpu(), kept["k"].cpu(), kept["v"].cpu())
        assert oracle.rel_l2(kept["o"].float().cpu(), want) < 1e-3
    test_adapters.check(out, kept["o"].reshape(B, N, C), block.proj_w, block.proj_slots, ids.tolist(), bounds, b=block.proj_b, res=x, gamma=block.gamma)
    assert _lib.device_status() == (0, 0, 0, 0)


@pytest.mark.gpu
def test_blocks_captured_and_on_two_streams():
    """Two blocks in one captured graph, replayed with other inputs, ids and lengths; the same blocks on another stream meanwhile."""
    first, second = Block(True, 1), Block(False, 2)
    x, ids, where, lengths = make(4, 9, 15, 1, 3)

    def run(x, ids, lengths):
        return second.run(first.run(x, ids, where, lengths), ids, where, lengths)

    captured = graphs.graphed(run)
    for seed in (3, 4, 5):
        x2, ids2, _, lengths2 = make(4, 9, 15, 1, seed)
        ids2, lengths2 = (ids2 + seed) % 4 - 1, (lengths2 - 10 * seed).clamp(min=0)
        want = run(x2, ids2, lengths2)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = run(x2, ids2, lengths2)
        got = captured(x2, ids2, lengths2)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want) and torch.equal(other, want)
    assert _lib.device_status() == (0, 0, 0, 0)
