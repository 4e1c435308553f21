"""Differential attention on the tcgen05 tensor cores (kernel: csrc/diff64.cu): the difference of two softmax maps over the same values.

    lam = (torch.exp((lq1 * lk1).sum(-1)) - torch.exp((lq2 * lk2).sum(-1)) + lam_init)       # fp32, a scalar or [H]
    o = diff_attention(q.view(B, N, 2 * H, 64), k.view(B, N, 2 * H, 64), v.view(B, N, H, 128), lam, weight=norm.weight, out_scale=1 - lam_init)

Beside attention(): the same conventions ([B, N, heads, columns] views, no copies, no fallback), head dimension 64 for the scores and
128 for the values. No counterpart in the reference.
"""
import torch

from . import _lib

_MOST = torch.finfo(torch.float32).max


def _usable(t, columns):
    """(shape, stride, address) of a view that the kernel takes, None of any other."""
    shape, stride, ptr = t.shape, t.stride(), t.data_ptr()
    if not t.is_cuda or t.dtype is not torch.float16 or len(shape) != 4 or shape[3] != columns or stride[3] != 1 or ptr & 15:
        return None
    a, b, c, _ = stride
    if ((a | b | c) & 7 or not (a and b and c)) and not all(n <= 1 or (s % 8 == 0 and s > 0) for n, s in zip(shape[:3], stride)):
        return None
    return shape, stride, ptr


def diff_attention(q, k, v, lam, weight=None, eps=1e-5, out_scale=1.0, scale=None, key_lengths=None, out=None):
    """o [B, Nq, H, 128] = softmax(scale q1 k1') v - lam softmax(scale q2 k2') v, of every head's maps 1 and 2.

    q: [B, Nq, 2H, 64], heads 2h and 2h + 1 are the two maps of head h; k: [B, Nk, 2Hk, 64] alike; v: [B, Nk, Hk, 128]; fp16 views (last
    dim contiguous, other strides multiples of 8 elements, no expanded dims). Hk divides H: query heads in a row share a key head.
    lam: fp32 tensor that broadcasts to [B, Nq, H] (a scalar, one per head, one per token and head).
    weight: [128] fp16 or fp32: each row of 128 is divided by its root mean square, sqrt(mean(o^2) + eps), and multiplied by it.
    out_scale: a factor of the result, with or without the norm. scale: of the scores, 64^-0.5 unless given, > 0. All of them finite.
    key_lengths: int32 [B] on the GPU: keys from key_lengths[b] on are not seen, whatever they hold; a row without keys is 0.
    out: fp16 [B, Nq, H, 128] that shares no memory with any input."""
    uq, uk, uv = _usable(q, 64), _usable(k, 64), _usable(v, 128)
    if uq is None or uk is None or uv is None:
        raise ValueError("diff_attention needs CUDA fp16 q, k [B, N, 2 * heads, 64] and v [B, N, heads, 128] with a contiguous last dim, other strides "
                         "that are multiples of 8 elements and 16-byte aligned storage (there is no fallback path)")
    (B, Nq, H2, _), qs, q_ptr = uq
    (Bk, Nk, Hk2, _), ks, k_ptr = uk
    (Bv, Nv, Hk, _), vs, v_ptr = uv
    H, device = H2 // 2, q.device
    if k.device != device or v.device != device or Bk != B or Bv != B or Nv != Nk or Hk2 != 2 * Hk or H2 % 2 or Hk == 0 or H == 0 or H % Hk:
        raise ValueError("q must be [B, Nq, 2H, 64], k [B, Nk, 2Hk, 64] and v [B, Nk, Hk, 128] on one device, Hk a divisor of H")
    if scale is None:
        scale = 0.125
    if not 0 < scale <= _MOST or not 0 <= eps <= _MOST or not abs(out_scale) <= _MOST:
        raise ValueError("scale must be > 0, eps >= 0, and both and out_scale finite in fp32")
    if not torch.is_tensor(lam) or lam.dtype != torch.float32 or lam.device != device:
        raise ValueError("lam must be an fp32 tensor on the inputs' device")
    if lam.dim() == 1 and lam.shape[0] == H:
        ls = (0, 0, lam.stride(0))
    else:
        try:
            ls = lam.expand(B, Nq, H).stride()
        except RuntimeError:
            raise ValueError(f"lam must broadcast to {(B, Nq, H)}, got {tuple(lam.shape)}") from None
    if weight is not None and (weight.device != device or weight.dtype not in (torch.float16, torch.float32) or weight.shape != (128,) or not weight.is_contiguous()):
        raise ValueError("weight must be a contiguous fp16 or fp32 vector of 128 on the inputs' device")
    if key_lengths is not None and (key_lengths.device != device or key_lengths.dtype != torch.int32 or key_lengths.shape != (B,)
                                    or not key_lengths.is_contiguous()):
        raise ValueError(f"key_lengths must be a contiguous int32 vector of {B} on the inputs' device")
    if out is None:
        out = q.new_empty((B, Nq, H, 128))
    elif not (_usable(out, 128) is not None and out.shape == (B, Nq, H, 128) and out.device == device and _lib.writable(out)):
        raise ValueError("out must be fp16 [B, Nq, H, 128] on the inputs' device, with a contiguous last dim, strides that are multiples of 8 elements, "
                         "16-byte aligned and no element twice")
    elif not _lib.apart(out, q, k, v, lam, weight, key_lengths):
        raise ValueError("out shares memory with an input")
    if B == 0 or Nq == 0:
        return out
    with _lib.on(device):
        lib = _lib.load()
        need = lib.fbb_diff64_workspace_bytes(B, Nq, Nk, H)
        ws = q.new_empty((need + 1) // 2) if need > 0 else None
        _lib.check(lib.fbb_diff64_f16_from(_lib.Diff64Args.pack(
            q_ptr, k_ptr, v_ptr, out.data_ptr(), lam.data_ptr(), _lib.address(weight), _lib.address(key_lengths), _lib.address(ws), _lib.stream_ptr(device),
            *qs[:3], *ks[:3], *vs[:3], *out.stride()[:3], *ls, need, B, Nq, Nk, H, Hk, _lib.DTYPE_CODE[weight.dtype] if weight is not None else 0,
            eps, out_scale, scale)))
        _lib.launched(2 if need > 0 else 1)
    return out
