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
import torch

from . import _lib

_PAIRING = {"half": 0, "pairs": 1}
_POS_CODE = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
_ABSENT = (0,) * 9  # a second tensor's fields


class RotaryPlan:
    """What a model's layers share: freqs [pairs] fp32 and axes [pairs] int32 on the GPU (pair i turns by the position on axis axes[i]
    times freqs[i]), the number of axes, and how columns pair: "half" (i, i + pairs) or "pairs" (2i, 2i + 1). Made by rotary_plan."""
    __slots__ = ("freqs", "axes", "n_axes", "pairing", "pairs", "device")

    def __init__(self, freqs, axes, n_axes, pairing):
        if pairing not in _PAIRING:
            raise ValueError(f"unsupported pairing: {pairing} (expected one of {tuple(_PAIRING)})")
        if freqs.dtype != torch.float32 or axes.dtype != torch.int32 or freqs.device != axes.device or not (
                freqs.dim() == axes.dim() == 1 and freqs.numel() == axes.numel() > 0 and freqs.is_contiguous() and axes.is_contiguous()) or n_axes < 1:
            raise ValueError("freqs must be fp32 and axes int32 vectors of one length on one device, n_axes at least 1")
        self.freqs, self.axes, self.n_axes, self.pairing, self.pairs, self.device = freqs, axes, n_axes, pairing, freqs.numel(), freqs.device


def rotary_plan(freqs, axes, pairing="half", device="cuda"):
    """A RotaryPlan from any sequence (or CPU / GPU tensor) of frequencies in radians per unit of position and one of axis numbers, one
    of each per pair of columns: sections, interleaved axes and ladders of any kind are sequences. Reads GPU tensors back: make it once."""
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

    positions: [N - n_prefix, axes] for every sequence alike, or [B, N - n_prefix, axes]; int32, int64 or fp32. Angles keep fp32 accuracy
    up to position * frequency of 2^70.
    inverse: the transposed rotation, which undoes this one and takes gradients of (q', k') to gradients of (q, k).
    out: (q_out, k_out); each may be its own input (in place), otherwise it shares no memory with any input.
    Positions and plan lie outside it altogether, not in the gaps of a strided one."""
    shape, device, dtype = q.shape, q.device, q.dtype
    code = _lib.DTYPE_CODE.get(dtype)
    if not q.is_cuda or code is None or len(shape) != 4:
        raise ValueError("rotary needs CUDA fp16, bf16 or fp32 [B, N, H, D] tensors (there is no CPU path)")
    B, N, H, D = shape
    q_strides, heads = q.stride(), H
    if k is not None:
        k_shape, k_strides = k.shape, k.stride()
        if k.device != device or k.dtype != dtype or len(k_shape) != 4 or k_shape[0] != B or k_shape[1] != N or k_shape[3] != D:
            raise ValueError("k must have q's batch, tokens, columns, dtype and device")
        heads = min(H, k_shape[2])
    if D > 1 and (q_strides[3] != 1 or (k is not None and k_strides[3] != 1)):
        raise ValueError("rotary needs tensors with a contiguous last dim")
    if heads < 1 or D > 1024:
        raise ValueError("rotary needs at least one head and at most 1024 columns")
    if plan.device != device:
        raise ValueError(f"the plan is on {plan.device}, the tensors on {device}")
    pairs, n_axes = plan.pairs, plan.n_axes
    if B * N > 0x7FFFFFFF:
        raise ValueError("rotary takes fewer than 2^31 tokens")
    if 2 * pairs > D:
        raise ValueError(f"the plan turns {2 * pairs} columns, a head has {D}")
    if n_prefix < 0 or n_prefix > N:
        raise ValueError(f"n_prefix must be from 0 to {N}")
    pos_code, pos_shape, pos_strides = _POS_CODE.get(positions.dtype), positions.shape, positions.stride()
    if pos_code is None or positions.device != device:
        raise ValueError("positions must be int32, int64 or fp32 on the tensors' device")
    if pos_shape != (N - n_prefix, n_axes) and pos_shape != (B, N - n_prefix, n_axes):
        raise ValueError(f"positions must be [{N - n_prefix}, {n_axes}] or [{B}, {N - n_prefix}, {n_axes}], got {tuple(pos_shape)}")
    if len(pos_shape) == 2:
        pos_strides = (0, *pos_strides)
    if out is None:
        result = (torch.empty_like(q, memory_format=torch.contiguous_format),
                  torch.empty_like(k, memory_format=torch.contiguous_format) if k is not None else None)
    else:
        result = _checked(out, q, k)
    if B == 0 or N == 0:
        return result
    y, y_strides = result[0], result[0].stride()
    first = (q.data_ptr(), y.data_ptr(), H, *q_strides[:3], *y_strides[:3])
    second = _ABSENT
    if k is not None:
        y, y_strides = result[1], result[1].stride()
        second = (k.data_ptr(), y.data_ptr(), k_shape[2], *k_strides[:3], *y_strides[:3])
    with _lib.on(device):
        _lib.check(_lib.load().fbb_rotary_from(_lib.RotaryArgs.pack(
            *first, *second, positions.data_ptr(), plan.freqs.data_ptr(), plan.axes.data_ptr(), _lib.stream_ptr(device), *pos_strides,
            1 if k is None else 2, B, N, D, pairs, _PAIRING[plan.pairing], n_prefix, pos_code, n_axes, 1 if inverse else 0, code)))
    _lib.launched()
    return result


def _side_by_side(q, k):
    """Whether q and k surely are, as in a packed projection, parts of rows of one buffer that share no element with each other or
    among themselves (the general checks say the same of more views, and take 10 us for it)."""
    B, N, H, D = q.shape
    sb, sn, sh, _ = q.stride()
    tb, tn, th, _ = k.stride()
    if sn != tn or sb != tb or N < 2 or (B > 1 and sb < N * sn) or sh < D or th < D:
        return False
    gap, q_row, k_row = (k.data_ptr() - q.data_ptr()) // q.element_size(), (H - 1) * sh + D, (k.shape[2] - 1) * th + D
    return gap >= q_row and gap + k_row <= sn or -gap >= k_row and q_row - gap <= sn


def _checked(out, q, k):
    """The caller's pair of outputs, refused where two threads could meet on an element."""
    if k is not None and len(out) == 2 and out[0] is q and out[1] is k and _side_by_side(q, k):
        return q, k
    inputs, outs = [q] if k is None else [q, k], list(out)
    if len(outs) == 2 and k is None and outs[1] is None:
        outs.pop()
    if len(outs) != len(inputs):
        raise ValueError("out must be a pair (q_out, k_out)")
    for i, y in enumerate(outs):
        x = inputs[i]
        if y is not x and (y.shape != x.shape or y.dtype != q.dtype or y.device != q.device or (y.stride(3) != 1 and y.shape[3] > 1)) or not _lib.writable(y):
            raise ValueError("out must match the inputs' shapes, dtype and device, with a contiguous last dim and no element twice")
        if not (_lib.same_view(y, x) or _lib.disjoint(y, x)) or (k is not None and not _lib.disjoint(y, inputs[1 - i])):
            raise ValueError("out must be its own input or share no memory with the inputs")
    if len(outs) == 2 and (outs[0] is not q or outs[1] is not k) and not _lib.disjoint(*outs):
        raise ValueError("the two outputs share memory")
    return outs[0], outs[1] if k is not None else None
