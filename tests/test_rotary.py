"""rotary(): against the rotation in 64 bits over sizes, layouts, types and pairings; in place; refusals.

Tolerance. The angle's fraction of a turn is rounded to fp32 (half a step of 2^-25 at most: 2^-26 turns, 2^-23.3 radians), sine and
cosine are off by up to 2 steps (2^-23), the two products and their sum by one rounding each (2^-24 of |x| + |y| twice): together
less than (|x| + |y|) 2^-21. The result is rounded to its type once: half a step of it, eps / 2 relative, or half of the smallest
subnormal."""
import math
from fractions import Fraction

import pytest
import torch

from fastbb_b200 import _lib
from fastbb_b200.rotary import RotaryPlan, _checked, _side_by_side, axial_plan, grid_positions, rotary, rotary_plan


def reference(x, positions, plan, n_prefix, inverse):
    x = x.double().cpu()
    pos = positions.double().cpu()
    pos = pos if pos.dim() == 3 else pos.expand(x.shape[0], *pos.shape)
    angle = pos[..., plan.axes.cpu().long()] * plan.freqs.double().cpu()
    if inverse:
        angle = -angle
    c, s = angle.cos()[:, :, None], angle.sin()[:, :, None]
    p = plan.freqs.numel()
    out = x.clone()
    body = x[:, n_prefix:]
    a, b = (slice(0, p), slice(p, 2 * p)) if plan.pairing == "half" else (slice(0, 2 * p, 2), slice(1, 2 * p, 2))
    out[:, n_prefix:, :, a] = body[..., a] * c - body[..., b] * s
    out[:, n_prefix:, :, b] = body[..., b] * c + body[..., a] * s
    room = torch.zeros_like(x)
    room[:, n_prefix:, :, a] = room[:, n_prefix:, :, b] = body[..., a].abs() + body[..., b].abs()
    return out, room


def check(got, x, positions, plan, n_prefix=0, inverse=False):
    want, room = reference(x, positions, plan, n_prefix, inverse)
    info = torch.finfo(got.dtype)
    limit = room * 2.0 ** -21 + want.abs() * info.eps / 2 * (room > 0) + info.smallest_normal * info.eps / 2 * (room > 0)
    over = (got.double().cpu() - want).abs() - limit
    assert bool((over <= 0).all()), f"{int((over > 0).sum())} of {over.numel()} off, worst by {float(over.max()):.3g}"


def tensor(shape, dtype, layout, g):
    """A [B, N, H, D] view of the wanted layout."""
    B, N, H, D = shape
    if layout == "plain":
        return torch.randn(shape, generator=g).to(dtype).cuda()
    if layout == "heads":        # [B, H, N, D] in memory
        return torch.randn(B, H, N, D, generator=g).to(dtype).cuda().transpose(1, 2)
    if layout == "odd":          # rows of an odd number of elements, from an odd element on
        return torch.randn(B, N, H, D + 3, generator=g).to(dtype).cuda()[..., 1:D + 1]
    if layout == "wide":         # every other row and head of a larger buffer
        return torch.randn(B, 2 * N, 2 * H, D, generator=g).to(dtype).cuda()[:, ::2, 1::2]
    raise AssertionError(layout)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pairing", ["half", "pairs"])
@pytest.mark.parametrize("B,N,H,Hk,D,pairs,prefix,layout", [
    (1, 1, 1, 1, 64, 32, 0, "plain"), (1, 1, 3, 1, 64, 32, 1, "plain"), (2, 5, 6, 2, 64, 32, 1, "heads"), (3, 37, 12, 4, 80, 40, 0, "plain"),
    (1, 257, 6, 6, 64, 32, 1, "plain"), (2, 19, 4, 2, 128, 32, 5, "wide"), (1, 33, 5, 5, 64, 24, 0, "plain"), (2, 9, 3, 3, 20, 7, 2, "plain"),
    (1, 16, 2, 1, 64, 32, 0, "odd"), (1, 7, 2, 2, 2, 1, 0, "plain"), (1, 3, 2, 1, 1024, 512, 0, "plain"), (2, 40, 24, 24, 64, 32, 4, "plain"),
    (1, 700, 16, 16, 64, 32, 1, "plain")])
def test_matches_the_rotation_in_64_bits(B, N, H, Hk, D, pairs, prefix, layout, pairing, dtype):
    g = torch.Generator().manual_seed(N * 7 + D)
    q, k = tensor((B, N, H, D), dtype, layout, g), tensor((B, N, Hk, D), dtype, layout, g)
    axes = 1 + (N + D) % 3
    plan = rotary_plan([100.0 ** (-i / pairs) for i in range(pairs)], [i % axes for i in range(pairs - 1)] + [axes - 1] if pairs > 1 else [0], pairing=pairing)
    where = torch.randn(B, N - prefix, plan.n_axes, generator=g).mul_(30).cuda()
    if N % 2:
        where = where[0]
    for inverse in (False, True):
        q2, k2 = rotary(q, k, where, plan, n_prefix=prefix, inverse=inverse)
        check(q2, q, where, plan, prefix, inverse)
        check(k2, k, where, plan, prefix, inverse)
    only, none = rotary(q, None, where, plan, n_prefix=prefix, inverse=True)
    assert none is None and torch.equal(only, q2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.float32])
def test_far_positions_of_every_type(dtype):
    g = torch.Generator().manual_seed(3)
    q = torch.randn(1, 64, 2, 64, generator=g).cuda()
    plan = axial_plan(64, axes=2, theta=10000.0)
    far = 2 ** 31 - 129 if dtype != torch.float32 else 2 ** 24 - 64
    where = torch.stack((torch.arange(64), far + torch.arange(64)), -1)
    where = where.to(dtype).cuda()
    check(rotary(q, None, where, plan)[0], q, where, plan)
    check(rotary(q, None, -where, plan)[0], q, -where, plan)
    strided = torch.stack((where, torch.zeros_like(where)), 1).transpose(0, 1)[0]          # positions of strides of their own
    assert torch.equal(rotary(q, None, strided, plan)[0], rotary(q, None, where, plan)[0])
    columns = where.t().contiguous().t()
    assert torch.equal(rotary(q, None, columns, plan)[0], rotary(q, None, where, plan)[0])


def fractions_of_a_turn(positions, freqs):
    """position * freq / (2 pi) without its whole turns, from integers of 400 bits (pi by Machin's formula)."""
    def arctan_of_inverse(n, bits=400):
        term, total, k, sign = (1 << bits) // n, 0, 1, 1
        while term:
            total, term, k, sign = total + sign * (term // k), term // (n * n), k + 2, -sign
        return total
    turn = Fraction(2 * 4 * (4 * arctan_of_inverse(5) - arctan_of_inverse(239)), 1 << 400)
    turns = [[Fraction(p) * Fraction(f) / turn for f in freqs] for p in positions]
    return torch.tensor([[float(t - round(t)) for t in row] for row in turns], dtype=torch.float64)


def test_the_exact_fractions_are():
    got = fractions_of_a_turn([0, 1, -7, 3.5], [1.0, 0.25]) * 2 * math.pi
    for row, p in zip(got.tolist(), (0, 1, -7, 3.5)):
        for angle, f in zip(row, (1.0, 0.25)):
            assert math.isclose(math.cos(angle), math.cos(p * f), abs_tol=1e-14) and math.isclose(math.sin(angle), math.sin(p * f), abs_tol=1e-14)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,positions", [
    (torch.int64, [10 ** 12 + 7, 2 ** 40 + 1, 2 ** 50 + 3, -(2 ** 50) - 1, 2 ** 53 - 1, 2 ** 53 + 1, -(2 ** 53) - 1, 1733702400123456789, 2 ** 62 + 1, 2 ** 63 - 1,
                   2 ** 63 - 2 ** 9, -(2 ** 63), -(2 ** 63) + 1, 2 ** 32, 2 ** 32 - 1, -(2 ** 32), -1, 0]),
    (torch.int32, [2 ** 31 - 1, -(2 ** 31), 1234567891, -3, 0]), (torch.float32, [1.0e12, 2.0 ** 60 + 2.0 ** 37, -3.3e15, 0.1, -1e-30, 0.0])])
@pytest.mark.parametrize("unit", [1.0, 100.0])
def test_angles_of_positions_beyond_53_bits(dtype, positions, unit):
    """The tolerance is the module's: the fraction of a turn is rounded to fp32, whatever the position."""
    g = torch.Generator().manual_seed(4)
    plan = axial_plan(64, axes=1, theta=10000.0, unit=unit)
    where = torch.tensor(positions, dtype=dtype)[:, None]
    q = torch.randn(1, len(positions), 3, 64, generator=g)
    angle = 2 * math.pi * fractions_of_a_turn(where[:, 0].tolist(), plan.freqs.tolist())
    c, s = angle.cos()[None, :, None], angle.sin()[None, :, None]
    a, b = q.double().chunk(2, -1)
    for inverse in (False, True):
        got = rotary(q.cuda(), None, where.cuda(), plan, inverse=inverse)[0].cpu().double()
        turned = torch.cat((a * c - b * s, b * c + a * s) if not inverse else (a * c + b * s, b * c - a * s), -1)
        room = (a.abs() + b.abs()).repeat(1, 1, 1, 2) * 2.0 ** -21 + turned.abs() * 2.0 ** -24
        assert bool(((got - turned).abs() <= room).all()), float(((got - turned).abs() - room).max())


@pytest.mark.gpu
@pytest.mark.parametrize("pairing", ["half", "pairs"])
def test_in_place_on_the_packed_projection_leaves_the_rest(pairing):
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(2, 38, 3, 6, 64, generator=g).half().cuda()
    before = qkv.clone()
    plan, where = axial_plan(64, unit=2 * math.pi, pairing=pairing), grid_positions(4, 8)
    q, k, v = qkv.unbind(2)
    want = rotary(q, k, where, plan, n_prefix=6)
    got = rotary(q, k, where, plan, n_prefix=6, out=(q, k))
    assert got[0] is q and got[1] is k
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(v, before[:, :, 2]) and torch.equal(qkv[:, :6], before[:, :6])
    back = rotary(q, k, where, plan, n_prefix=6, inverse=True)
    assert float((back[0] - before[:, :, 0]).abs().max()) < 2 ** -8


@pytest.mark.gpu
def test_passing_rows_and_columns_keep_their_bits():
    g = torch.Generator().manual_seed(6)
    q = torch.randn(1, 12, 2, 64, generator=g).half().cuda()
    q[:, :3] = torch.tensor([float("inf"), float("nan"), -0.0, 65504.0]).half().cuda().repeat(16)
    q[..., 48:] = float("nan")
    plan = rotary_plan([0.5] * 24, [0] * 24)
    out = rotary(q, None, torch.arange(9, device="cuda").view(9, 1), plan, n_prefix=3)[0]
    assert torch.equal(out[:, :3].view(torch.int16), q[:, :3].view(torch.int16))
    assert torch.equal(out[..., 48:].view(torch.int16), q[..., 48:].view(torch.int16))
    check(out[:, 3:, :, :48], q[:, 3:, :, :48], torch.arange(9).view(9, 1), plan)


@pytest.mark.gpu
def test_gradients_against_the_formula_and_differences():
    """With loss = sum(w * rotary(x)) the gradient is the inverse rotation of w; the loss is linear in x, so a difference is exact up
    to the roundings: fp32 sums of 12 * 2 * 64 products of size about 1, 2^-24 each."""
    g = torch.Generator().manual_seed(7)
    x, w = torch.randn(1, 12, 2, 64, generator=g).cuda(), torch.randn(1, 12, 2, 64, generator=g).cuda()
    plan, where = axial_plan(64, unit=3.0), grid_positions(3, 4)
    grad = rotary(w, None, where, plan, inverse=True)[0]
    check(grad, w, where, plan, inverse=True)
    step = torch.randn(1, 12, 2, 64, generator=g).cuda()
    high, low = rotary(x + step, None, where, plan)[0], rotary(x - step, None, where, plan)[0]
    difference = float(((high.double() - low.double()) * w.double()).sum()) / 2
    along = float((grad.double() * step.double()).sum())
    assert abs(difference - along) < 12 * 2 * 64 * 4 * 2.0 ** -21


@pytest.mark.gpu
def test_other_stream_and_captured_graph():
    g = torch.Generator().manual_seed(8)
    q = torch.randn(1, 65, 6, 64, generator=g).half().cuda()
    plan, where = axial_plan(64), grid_positions(8, 8)
    want = rotary(q, q, where, plan, n_prefix=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = rotary(q, None, where, plan, n_prefix=1)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want[0])
    held = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = rotary(held, None, where, plan, n_prefix=1)[0]
    for scale in (1.0, -2.0):
        held.copy_(q * scale)
        graph.replay()
        assert torch.equal(captured, rotary(q * scale, None, where, plan, n_prefix=1)[0])


@pytest.mark.gpu
def test_empty_calls_and_no_rows_with_positions():
    plan = axial_plan(64)
    for shape in ((0, 5, 2, 64), (3, 0, 2, 64)):
        q = torch.zeros(shape, dtype=torch.float16, device="cuda")
        assert rotary(q, None, torch.zeros(shape[1], 2, device="cuda"), plan)[0].shape == shape
    q = torch.randn(2, 3, 2, 64, device="cuda")
    assert torch.equal(rotary(q, None, torch.zeros(0, 2, device="cuda"), plan, n_prefix=3)[0], q)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    plan, where = axial_plan(64), grid_positions(2, 4)
    qkv = torch.zeros(1, 8, 3, 2, 64, dtype=torch.float16, device="cuda")
    q, k, v = qkv.unbind(2)
    wide = torch.zeros(1, 8, 2, 64, dtype=torch.float16, device="cuda").expand(4, 8, 2, 64)
    for call in (
            lambda: rotary(q, k, where[:5], plan), lambda: rotary(q, k, where, plan, n_prefix=1), lambda: rotary(q, k, where, plan, n_prefix=9),
            lambda: rotary(q, k.float(), where, plan), lambda: rotary(q, k[:, :4], where, plan), lambda: rotary(q.double(), None, where, plan),
            lambda: rotary(q, k, where.half(), plan), lambda: rotary(q, k, where.cpu(), plan), lambda: rotary(q[..., ::2], None, where, plan),
            lambda: rotary(q, k, where, plan, out=(k, q)), lambda: rotary(q, k, where, plan, out=(q, q)), lambda: rotary(q, k, where, plan, out=(v, v)),
            lambda: rotary(q, None, where, plan, out=(qkv[:, :, 0:2].flatten(2, 3)[:, :, 1:3],)), lambda: rotary(q, k, where, plan, out=(q,)),
            lambda: rotary(wide, None, where, plan, out=(wide,)), lambda: rotary(q, k, where, axial_plan(128)),
            lambda: rotary(q, k, where, axial_plan(64, axes=3)), lambda: rotary(q, k, where, axial_plan(64, device="cpu")),
            lambda: rotary(q, k, where, RotaryPlan(plan.freqs, plan.axes, 2, "thirds"))):
        with pytest.raises(ValueError):
            call()
    assert torch.equal(rotary(q, k, where, plan, out=(v, torch.empty_like(k)))[0], q)  # another part of the buffer is fine


@pytest.mark.gpu
def test_outputs_over_the_positions_or_the_plan_are_refused():
    store = torch.zeros(4096, device="cuda")
    q, where = store[:1024].view(1, 8, 2, 64), store[1000:1016].view(8, 2)
    plan = axial_plan(64)
    held = store.clone()
    with pytest.raises(_lib.FastbbError, match="shares memory"):
        rotary(q, None, where, plan, out=(q, None))
    with pytest.raises(_lib.FastbbError, match="shares memory"):
        rotary(torch.zeros_like(q), q, where, plan, out=(torch.zeros_like(q), q))
    with pytest.raises(_lib.FastbbError, match="shares memory"):
        rotary(q, None, store[2000:2016].view(8, 2), RotaryPlan(store[64:96], plan.axes, 2, "half"), out=(q, None))
    assert torch.equal(store, held)
    rotary(q, None, store[1024:1040].view(8, 2), plan, out=(q, None))  # beside it is well


@pytest.mark.gpu
@pytest.mark.parametrize("B,N", [(1, 2 ** 31), (1, 2 ** 32 + 1), (2 ** 16, 2 ** 15), (2 ** 32 + 1, 1)])
def test_more_tokens_than_31_bits_count_are_refused(B, N):
    """(Views of a single row: nothing is allocated.)"""
    plan = axial_plan(64)
    row, where = torch.zeros(64, dtype=torch.float16, device="cuda"), torch.zeros(2, device="cuda")
    q = row.as_strided((B, N, 1, 64), (0, 0, 0, 1))
    with pytest.raises(ValueError, match="2\\^31 tokens"):
        rotary(q, None, where.as_strided((N, 2), (0, 1)), plan, out=(q, None))


# ------------------------------------------------------------------------------------------------------------------ CPU
def test_plans():
    plan = axial_plan(64, axes=3, theta=50.0, unit=2.0, shares=[8, 12, 12], device="cpu")
    assert plan.n_axes == 3 and plan.axes.tolist() == [0] * 8 + [1] * 12 + [2] * 12
    assert plan.freqs[0] == plan.freqs[8] == plan.freqs[20] == 2.0 and math.isclose(float(plan.freqs[9]), 2.0 * 50.0 ** (-1 / 12), rel_tol=1e-6)
    ladder = axial_plan(64, axes=3, theta=50.0, shared=True, device="cpu")
    assert ladder.axes.tolist() == [0] * 11 + [1] * 11 + [2] * 10 and math.isclose(float(ladder.freqs[31]), 50.0 ** (-31 / 32), rel_tol=1e-6)
    assert rotary_plan(torch.ones(4), torch.tensor([0, 1, 0, 1]), device="cpu").n_axes == 2
    where = grid_positions(2, 3, device="cpu")
    assert where.shape == (6, 2) and torch.allclose(where[1], torch.tensor([-0.5, 0.0])) and torch.allclose(where[5], torch.tensor([0.5, 2 / 3]))
    for bad in (lambda: rotary_plan([1.0], [0, 1], device="cpu"), lambda: rotary_plan([], [], device="cpu"), lambda: rotary_plan([1.0], [-1], device="cpu"),
                lambda: rotary_plan([1.0], [0.5], device="cpu"), lambda: rotary_plan([float("inf")], [0], device="cpu"),
                lambda: rotary_plan([1.0], [0], pairing="all", device="cpu"), lambda: axial_plan(63, device="cpu"),
                lambda: axial_plan(64, axes=2, shares=[10, 10], device="cpu"), lambda: axial_plan(4, axes=3, device="cpu")):
        with pytest.raises(ValueError):
            bad()


def test_cpu_tensors_are_refused():
    plan, q = axial_plan(64, device="cpu"), torch.zeros(1, 4, 2, 64)
    with pytest.raises(ValueError, match="no CPU path"):
        rotary(q, q, torch.zeros(4, 2), plan)


def test_views_that_share_memory():
    qkv = torch.zeros(2, 5, 3, 4, 8)
    q, k, v = qkv.unbind(2)
    assert _lib.disjoint(q, k) and _lib.disjoint(v, q) and not _lib.disjoint(q, q) and _lib.disjoint(q, torch.zeros_like(q))
    flat = torch.zeros(2, 5, 8, 8)
    assert _lib.disjoint(flat[:, :, :4], flat[:, :, 4:]) and not _lib.disjoint(flat[:, :, :5], flat[:, :, 4:]) and _lib.disjoint(flat[:, :, :6], flat[:, :, 6:])
    assert _lib.disjoint(flat[0], flat[1]) and not _lib.disjoint(flat[:, 1:], flat[:, :4]) and _lib.disjoint(flat[:, 3:], flat[:, :3])
    heads = torch.zeros(2, 3, 4, 5, 8)                       # [B, 3, H, N, D]
    assert _lib.disjoint(heads[:, 0].transpose(1, 2), heads[:, 2].transpose(1, 2))
    assert not _lib.disjoint(flat[:, ::2], flat[:, 0:3])
    assert _lib.writable(q) and _lib.writable(heads.transpose(1, 3)) and not _lib.writable(flat[:1].expand(2, 5, 8, 8))
    assert not _lib.writable(torch.zeros(20).as_strided((3, 8), (4, 1))) and _lib.same_view(q, qkv[:, :, 0]) and not _lib.same_view(q, k)


def test_views_called_disjoint_or_writable_are():
    """Against a count of every element's address; overlapping outer dimensions among them."""
    buf, said, quick = torch.zeros(4000), 0, 0
    for B, N, H, Hk, D in ((1, 2, 1, 1, 4), (2, 3, 2, 1, 4), (2, 1, 2, 2, 4), (3, 2, 1, 2, 6)):
        for sn in (4, 8, 12, 16, 24, 30):
            for sb in (4, 12, N * sn, N * sn + 4, 2 * sn, sn):
                for sh, th in ((4, 4), (6, 4), (3, 6), (12, 12)):
                    for q0, k0 in ((0, 4), (0, 8), (8, 0), (0, 12), (12, 0), (16, 4), (0, 500)):
                        q, k = buf.as_strided((B, N, H, D), (sb, sn, sh, 1), q0), buf.as_strided((B, N, Hk, D), (sb, sn, th, 1), k0)
                        at = [[t.storage_offset() + sum(i * s for i, s in zip(index, t.stride()))
                               for index in torch.cartesian_prod(*map(torch.arange, t.shape)).tolist()] for t in (q, k)]
                        for t, own in zip((q, k), at):
                            assert not _lib.writable(t) or len(set(own)) == len(own), (t.shape, t.stride())
                        assert not _lib.disjoint(q, k) or not set(at[0]) & set(at[1]), (q.shape, q.stride(), k.shape, k.stride(), q0, k0)
                        said += _lib.disjoint(q, k) and k0 != 500
                        if _side_by_side(q, k):
                            assert _lib.writable(q) and _lib.writable(k) and not set(at[0]) & set(at[1]), (q.shape, q.stride(), k.shape, k.stride(), q0, k0)
                            assert all(a is b for a, b in zip(_checked((q, k), q, k), (q, k)))
                            quick += 1
    assert said > quick > 20
    q, k, _ = torch.zeros(2, 5, 3, 4, 8).unbind(2)
    assert _side_by_side(q, k) and _side_by_side(k, q) and not _side_by_side(q, q)


def test_outputs_apart_from_inputs_of_any_type():
    store = torch.zeros(4096, dtype=torch.uint8)
    out = store[1024:2048].view(torch.float16).view(4, 2, 64)
    for dtype in (torch.float32, torch.int32, torch.int64, torch.float16):
        inside = lambda lo, hi: store[lo:hi].view(dtype)  # noqa: E731, B023
        assert _lib.apart(out, None, inside(0, 1024), inside(2048, 4096), inside(1024, 1024), torch.zeros(9, dtype=dtype))
        for lo, hi in ((1016, 1032), (1024, 1032), (2040, 2048), (2040, 4096), (0, 4096), (1500 // 8 * 8, 1600)):
            assert not _lib.apart(out, None, inside(0, 1024), inside(lo, hi))
        assert not _lib.apart(out, inside(0, 4096)[::4096 // dtype.itemsize - 1])                                  # the holes of another type's view count
        assert not _lib.apart(store[:2048].view(torch.float16).view(8, 128)[:, :8], store[20:24].view(torch.int32)) and _lib.apart(out[:0], inside(0, 4096))
    assert _lib.apart(out[..., :32], out[..., 32:]) and not _lib.apart(out[..., :32], out[..., 31:])             # views of its own type: the elements


def test_entry_point_refuses_outputs_over_the_positions_or_the_plan():
    lib, y = _lib.load(), 0x7F0000000000
    # y: [2, 5, 3, 64] fp32 in slots of 256, 2 x 5 x 4 of them but the last
    last = y + 4 * ((1 * 5 + 4) * 1024 + 2 * 256 + 64)

    def call(pos=y - 4096, freqs=y - 8192, ax=y - 16384, second=False, pd=2, p=(8, 2, 1), B=2):
        tensor, other = (y, y, 3, *(5120, 1024, 256) * 2), (y - (1 << 20), y - (1 << 20), 3, *(5120, 1024, 256) * 2)
        first, second = (other, tensor) if second else (tensor, other)
        status = lib.fbb_rotary_from(_lib.RotaryArgs.pack(*first, *second, pos, freqs, ax, 0, *p, 2, B, 5, 64, 32, 0, 1, pd, 2, 0, 2))
        return status, b"shares memory" in lib.fbb_last_error()

    for second in (False, True):
        for at in (y, last - 4, y + 4096, y + 300):
            assert call(pos=at, second=second) == call(freqs=at, second=second) == call(ax=at, second=second) == (-2, True)
        assert call(freqs=y - 4 * 31, second=second) == call(ax=y - 4 * 31, second=second) == (-2, True)
        assert call(pos=y - 4 * (8 + 3 * 2 + 1), second=second) == call(pos=y - 8 * (8 + 3 * 2 + 1), pd=1, second=second) == (-2, True)


def test_entry_point_refusals():
    import ctypes
    lib, A = _lib.load(), 0x7F0000000000

    def call(heads=2, x=A, y=A, n=1, B=1, N=4, D=64, pairs=32, pairing=0, prefix=0, pos=A, pd=2, axes=2, freqs=A, ax=A, dtype=0):
        t = (_lib.RotaryTensor * 2)()
        t[0].x, t[0].y, t[0].heads = x, y, heads
        return lib.fbb_rotary(ctypes.cast(t, ctypes.POINTER(_lib.RotaryTensor)), n, B, N, D, pairs, pairing, prefix, pos, pd, axes, 0, 2, 1, freqs, ax, 0, dtype, None)

    assert call(x=None) == call(y=None) == call(freqs=None) == call(ax=None) == call(pos=None) == -1
    assert call(heads=0) == call(n=3) == call(D=1026) == call(pairs=33) == call(pairs=0) == call(axes=0) == call(prefix=-1) == call(N=-1) == -2
    assert call(B=1 << 20, N=1 << 20) == -2
    assert call(x=A + 1) == call(y=A + 2, dtype=2) == call(pos=A + 4, pd=1) == -3
    assert call(pairing=2) == call(pd=3) == call(dtype=4) == -4
    assert call(B=0, x=None) == call(N=0, pos=None) == 0


def test_the_record_form_refuses_what_the_other_does():
    """Every field is where the entry point looks for it: broken alone, it is the one that is named."""
    lib, A = _lib.load(), 0x7F0000000000
    good = dict(x0=A, y0=A, h0=2, **{f"s{i}": 64 for i in range(6)}, x1=A, y1=A, h1=2, **{f"t{i}": 64 for i in range(6)}, pos=A, freqs=A, ax=A, stream=0,
                p0=0, p1=2, p2=1, n=2, B=1, N=4, D=64, pairs=32, pairing=0, prefix=0, pd=2, axes=2, inverse=0, dtype=0)

    def call(**kw):
        return lib.fbb_rotary_from(_lib.RotaryArgs.pack(*{**good, **kw}.values()))

    assert lib.fbb_rotary_from(None) == call(x0=0) == call(y0=0) == call(x1=0) == call(y1=0) == call(freqs=0) == call(ax=0) == call(pos=0) == -1
    assert call(h0=0) == call(h1=0) == call(n=3) == call(D=1026) == call(pairs=33) == call(axes=0) == call(prefix=-1) == call(N=-1) == call(B=-1) == -2
    assert call(y1=A + 1) == call(y0=A + 2, dtype=2) == call(pos=A + 4, pd=1) == -3 and call(pairing=2) == call(pd=3) == call(dtype=4) == -4
    assert call(B=0, x0=0) == call(N=0, x1=0) == call(n=1, B=0, h1=0) == 0
