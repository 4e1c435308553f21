"""Rotary positions on one or several axes (kernel: csrc/rotary.cu): queries and keys of tokens that lie on a patch grid or in a
video, turned in one launch between the qkv projection and the attention.

    plan = axial_plan(64, axes=2, theta=100.0, unit=2 * math.pi, device="cuda")      # once per model
    where = grid_positions(h, w, device="cuda")                                      # once per image size: [h * w, 2] in (-1, 1)
    q, k, v = linear(y, qkv.weight, qkv.bias).view(B, N, 3, H, 64).unbind(2)
    rotary(q, k, where, plan, n_prefix=1, out=(q, k))                                # in place; the cls row passes
    o = attention(q, k, v)

The reference has no counterpart: the models it speeds up add a learned position table to their tokens
(fastbb/vit.py FastViT.tokens).
"""
import collections
import ctypes

import torch

from . import _lib

_PAIRING = {"half": 0, "pairs": 1}
_POS_CODE = {torch.int32: 0, torch.int64: 1, torch.float32: 2}

RotaryPlan = collections.namedtuple("RotaryPlan", "freqs axes n_axes pairing")
RotaryPlan.__doc__ = """What a model's layers share: freqs [pairs] fp32 and axes [pairs] int32 on the GPU (pair i turns by the position on
axis axes[i] times freqs[i]), the number of axes, and how columns pair: "half" (i, i + pairs) or "pairs" (2i, 2i + 1)."""


def rotary_plan(freqs, axes, pairing="half", device="cuda"):
    """A RotaryPlan from any sequence (or CPU / GPU tensor) of frequencies in radians per unit of position and one of axis numbers, one
    of each per pair of columns: sections, interleaved axes and ladders of any kind are sequences. Reads GPU tensors back: make it once."""
    if pairing not in _PAIRING:
        raise ValueError(f"unsupported pairing: {pairing} (expected one of {tuple(_PAIRING)})")
    freqs = torch.as_tensor(freqs, dtype=torch.float64).flatten().cpu()
    axes = torch.as_tensor(axes).flatten().cpu()
    if axes.is_floating_point() or axes.dtype == torch.bool:
        raise ValueError("axes must be whole numbers")
    if freqs.numel() == 0 or freqs.numel() != axes.numel():
        raise ValueError("freqs and axes must hold one value per pair of columns")
    if int(axes.min()) < 0 or int(axes.max()) > 15:
        raise ValueError("axes must be numbers from 0 to 15")
    if not bool(torch.isfinite(freqs.float()).all()):
        raise ValueError("freqs must be finite")
    return RotaryPlan(freqs.to(torch.float32).to(device), axes.to(torch.int32).to(device), int(axes.max()) + 1, pairing)


def axial_plan(dim, axes=2, theta=100.0, unit=1.0, pairing="half", shares=None, shared=False, device="cuda"):
    """The usual plans over `dim` columns: the first pairs turn by axis 0, the next by axis 1, ... `shares` gives the pairs of each axis
    (default: as even as they go). shared=False: each axis has a ladder of its own, unit * theta^(-j / share); shared=True: one ladder
    over all pairs, unit * theta^(-i / pairs), of which each axis has its section."""
    if dim < 2 or dim % 2 or axes < 1:
        raise ValueError("dim must be even and at least 2, axes at least 1")
    pairs = dim // 2
    if shares is None:
        shares = [pairs // axes + (1 if a < pairs % axes else 0) for a in range(axes)]
    if len(shares) != axes or sum(shares) != pairs or min(shares) < 1:
        raise ValueError(f"shares must be {axes} positive numbers that add up to {pairs}")
    which = [a for a, n in enumerate(shares) for _ in range(n)]
    if shared:
        freqs = [unit * theta ** (-i / pairs) for i in range(pairs)]
    else:
        freqs = [unit * theta ** (-j / n) for n in shares for j in range(n)]
    return rotary_plan(freqs, which, pairing=pairing, device=device)


def grid_positions(*sizes, device="cuda"):
    """[prod(sizes), len(sizes)] fp32: the cells of a grid in row-major order, each axis from -1 to 1 (the cells' centres)."""
    axes = [(torch.arange(n, dtype=torch.float64) + 0.5) / n * 2.0 - 1.0 for n in sizes]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, len(sizes)).float().to(device)


def rotary(q, k, positions, plan, n_prefix=0, inverse=False, out=None):
    """(q', k'): q [B, N, H, D] and k [B, N, Hk, D] (fp16, bf16 or fp32, D contiguous, any other strides; k may be None) turned by the
    positions of their tokens. Columns from 2 * pairs on, and the first n_prefix rows of every sequence, pass unchanged.

    positions: [N - n_prefix, axes] for every sequence alike, or [B, N - n_prefix, axes]; int32, int64 or fp32.
    inverse: the transposed rotation, which undoes this one and takes gradients of (q', k') to gradients of (q, k).
    out: (q_out, k_out); each may be its own input (in place), otherwise it shares no memory with either input."""
    inputs = [q] if k is None else [q, k]
    for x in inputs:
        if not (x.is_cuda and x.dim() == 4 and x.dtype in _lib.DTYPE_CODE and (x.stride(3) == 1 or x.shape[3] == 1)):
            raise ValueError("rotary needs CUDA fp16, bf16 or fp32 [B, N, H, D] tensors with a contiguous last dim (there is no CPU path)")
    B, N, H, D = q.shape
    if k is not None and (k.device != q.device or k.dtype != q.dtype or k.shape[:2] != q.shape[:2] or k.shape[3] != D):
        raise ValueError("k must have q's batch, tokens, columns, dtype and device")
    if min(x.shape[2] for x in inputs) < 1 or D > 1024:
        raise ValueError("rotary needs at least one head and at most 1024 columns")
    pairs = plan.freqs.numel()
    if plan.freqs.device != q.device or plan.axes.device != q.device:
        raise ValueError(f"the plan is on {plan.freqs.device}, the tensors on {q.device}")
    if plan.freqs.dtype != torch.float32 or plan.axes.dtype != torch.int32 or plan.axes.numel() != pairs or plan.pairing not in _PAIRING:
        raise ValueError("plan must come from rotary_plan or axial_plan")
    if 2 * pairs > D:
        raise ValueError(f"the plan turns {2 * pairs} columns, a head has {D}")
    if n_prefix < 0 or n_prefix > N:
        raise ValueError(f"n_prefix must be from 0 to {N}")
    if positions.device != q.device or positions.dtype not in _POS_CODE:
        raise ValueError("positions must be int32, int64 or fp32 on the tensors' device")
    if positions.shape not in ((N - n_prefix, plan.n_axes), (B, N - n_prefix, plan.n_axes)):
        raise ValueError(f"positions must be [{N - n_prefix}, {plan.n_axes}] or [{B}, {N - n_prefix}, {plan.n_axes}], got {tuple(positions.shape)}")
    if out is None:
        outs = [torch.empty(x.shape, device=x.device, dtype=x.dtype) for x in inputs]
    else:
        outs = list(out)
        if len(outs) == 2 and k is None and outs[1] is None:
            outs.pop()
        if len(outs) != len(inputs):
            raise ValueError("out must be a pair (q_out, k_out)")
        for i, y in enumerate(outs):
            if y.shape != inputs[i].shape or y.dtype != q.dtype or y.device != q.device or (y.stride(3) != 1 and D > 1) or not _lib.writable(y):
                raise ValueError("out must match the inputs' shapes, dtype and device, with a contiguous last dim and no element twice")
            if not all(_lib.disjoint(y, x) or (i == j and _lib.same_view(y, x)) for j, x in enumerate(inputs)):
                raise ValueError("out must be its own input or share no memory with the inputs")
        if len(outs) == 2 and not _lib.disjoint(*outs):
            raise ValueError("the two outputs share memory")
    result = (outs[0], outs[1] if k is not None else None)
    if B == 0 or N == 0:
        return result
    tensors = (_lib.RotaryTensor * 2)()
    for t, x, y in zip(tensors, inputs, outs):
        t.x, t.y, t.heads = x.data_ptr(), y.data_ptr(), x.shape[2]
        t.x_sb, t.x_sn, t.x_sh = x.stride()[:3]
        t.y_sb, t.y_sn, t.y_sh = y.stride()[:3]
    sb, sn, sa = (0, *positions.stride()) if positions.dim() == 2 else positions.stride()
    with _lib.on(q.device):
        _lib.check(_lib.load().fbb_rotary(
            ctypes.cast(tensors, ctypes.POINTER(_lib.RotaryTensor)), len(inputs), B, N, D, pairs, _PAIRING[plan.pairing], n_prefix, positions.data_ptr(),
            _POS_CODE[positions.dtype], plan.n_axes, sb, sn, sa, plan.freqs.data_ptr(), plan.axes.data_ptr(), 1 if inverse else 0,
            _lib.DTYPE_CODE[q.dtype], _lib.stream_ptr(q.device)))
    _lib.launched()
    return result
