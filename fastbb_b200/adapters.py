"""One shared projection and, beside it, the low-rank adapters of many requests (kernels: csrc/adapters.cu, csrc/gemm.cu): fine-tuned
variants of one backbone served in one batch.

    slots = Adapters(down, up, scale)                     # once per layer: [L, r, K], [L, N, r], [L]
    y = adapter_linear(x, qkv.weight, slots, ids, b=qkv.bias)                       # x [B, N, K], ids [B]: an image per request
    y = adapter_linear(x, fc1.weight, slots, ids, offsets, b=fc1.bias, act="gelu")  # x [M, K], images of any sizes one behind another

Beside linear(): the same layer, epilogues and conventions (gemm.py). No counterpart in the reference.
"""
import torch

from . import _lib
from .gemm import _ACT


class Adapters:
    """The adapters of one layer, stacked: row x of a request with adapter a gets scale[a] * (x down[a]^T) up[a]^T beside x w^T.

    down [L, r, K] and up [L, N, r] fp16, scale [L] fp32 (usually alpha / r; None: 1), contiguous and on one GPU; r a multiple of 8 up to 128.
    Adapters of a smaller rank are padded with rows (columns) of zeros; slots may be overwritten in place between calls."""
    __slots__ = ("down", "up", "scale", "count", "rank", "k", "n", "device")

    def __init__(self, down, up, scale=None):
        if not (down.is_cuda and down.dtype == up.dtype == torch.float16 and down.device == up.device and down.dim() == up.dim() == 3):
            raise ValueError("down [L, r, K] and up [L, N, r] must be fp16 tensors on one GPU (there is no CPU path)")
        count, rank, k = down.shape
        if up.shape[0] != count or up.shape[2] != rank or min(count, k, up.shape[1]) < 1:
            raise ValueError(f"down {tuple(down.shape)} and up {tuple(up.shape)} do not hold the same adapters")
        if rank < 8 or rank > 128 or rank % 8:
            raise ValueError(f"the rank must be a multiple of 8 up to 128, got {rank}: pad with zeros")
        if max(count * max(up.shape[1], rank), k) > 0x7FFFFFFF:
            raise ValueError("the adapters' rows, of either matrix, must number fewer than 2^31")
        if scale is None:
            scale = torch.ones(count, device=down.device)
        if scale.dtype != torch.float32 or scale.shape != (count,) or scale.device != down.device:
            raise ValueError("scale must be an fp32 vector with one number per adapter")
        if not (down.is_contiguous() and up.is_contiguous() and scale.is_contiguous() and down.data_ptr() % 16 == 0 and up.data_ptr() % 16 == 0):
            raise ValueError("down, up and scale must be contiguous, down and up 16-byte aligned")
        self.down, self.up, self.scale = down, up, scale
        self.count, self.rank, self.k, self.n, self.device = count, rank, k, up.shape[1], down.device


def adapter_linear(x, w, adapters, ids, offsets=None, b=None, act=None, res=None, gamma=None, out=None):
    """act(x w^T + b + scale_a (x down_a^T) up_a^T), a the adapter of the row's request; with res: res + gamma * that. As linear(): fp16 x [..., K],
    w [N, K], b and gamma vectors, res of the output's shape, act None | "gelu" | "swiglu"; fp32 accumulator. Each scale_a (x down_a^T) is rounded to
    fp16 on the way (but for few rows of many requests); a row of it with values beyond fp16's range is held times 2^-15, so up to 2^31.

    ids: int32 [S] on the GPU, the adapter of each request; a number out of [0, L) (say -1): none.
    offsets: int32 [S + 1] on the GPU, not decreasing: request s has rows offsets[s] .. offsets[s + 1] - 1 of x's rows taken in order; rows of
    no request have no adapter. Without offsets x's first dimension is the requests, [S, ..., K].
    out: fp16 and contiguous, may be res itself, shares no memory with any other input."""
    if act not in _ACT:
        raise ValueError(f"unsupported activation: {act}")
    device = x.device
    if not x.is_cuda or x.dtype != torch.float16 or w.dtype != torch.float16 or x.dim() < 1:
        raise ValueError("adapter_linear needs CUDA fp16 x and w (there is no CPU path)")
    shape, K, N = x.shape, x.shape[-1], w.shape[0]
    if w.dim() != 2 or w.shape[1] != K or w.device != device:
        raise ValueError("w must be [N, K] on the input's device")
    if adapters.device != device or adapters.k != K or adapters.n != N:
        raise ValueError(f"the adapters are for a layer of {adapters.k} inputs and {adapters.n} outputs on {adapters.device}, this one has {K} and {N} on {device}")
    n_out = N // 2 if act == "swiglu" else N
    oshape = (*shape[:-1], n_out)
    if ids.dtype != torch.int32 or ids.dim() != 1 or ids.device != device or not ids.is_contiguous() or ids.numel() < 1:
        raise ValueError("ids must be a contiguous int32 vector, one per request, on the input's device")
    S = ids.numel()
    if offsets is None:
        if len(shape) < 2 or shape[0] != S:
            raise ValueError(f"without offsets x must be [{S}, ..., K], a request in each part of the first dimension")
    elif offsets.dtype != torch.int32 or offsets.shape != (S + 1,) or offsets.device != device or not offsets.is_contiguous():
        raise ValueError(f"offsets must be a contiguous int32 vector of {S + 1} on the input's device")
    for t, n in ((b, N), (gamma, n_out)):
        if t is not None and (t.device != device or t.dtype != torch.float16 or not t.is_contiguous() or t.numel() != n):
            raise ValueError("bias / gamma must be contiguous fp16 vectors of the output width on the input's device")
    if res is not None and (res.device != device or res.dtype != torch.float16 or res.shape != oshape):
        raise ValueError("res must be fp16 with the output shape on the input's device")
    if gamma is not None and res is None:
        raise ValueError("gamma is the LayerScale of the residual epilogue: it needs res")
    if out is None:
        out = x.new_empty(oshape)
    else:
        if out.shape != oshape or out.device != device or out.dtype != torch.float16 or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError("out must be contiguous with the output shape, input dtype and device")
        if not (_lib.apart(out, x, w, b, gamma, adapters.down, adapters.up, adapters.scale, ids, offsets) and (
                res is None or _lib.same_view(out, res) or _lib.disjoint(out, res))):
            raise ValueError("out may be res itself and shares no memory with the other inputs")
    if x.is_contiguous():
        x2, lda = x, K
    else:
        x2 = x.reshape(-1, K)
        if x2.stride(-1) != 1:
            x2 = x2.contiguous()
        lda = x2.stride(0) if x2.shape[0] > 1 else K
    if w.stride(-1) != 1:
        w = w.contiguous()
    r2, ldr = res, n_out
    if res is not None and not res.is_contiguous():
        r2 = res.reshape(-1, n_out)
        if r2.stride(-1) != 1:
            r2 = r2.contiguous()
        ldr = r2.stride(0) if r2.shape[0] > 1 else n_out
    M = x.numel() // K if K else 0
    if M == 0:
        return out
    code = _ACT[act]
    with _lib.on(device):
        lib = _lib.load()
        need = lib.fbb_adapter_linear_workspace_bytes(M, N, K, code, adapters.rank, S)
        ws = x.new_empty((need + 1) // 2)
        _lib.check(lib.fbb_adapter_linear_f16_from(_lib.AdapterLinearArgs.pack(
            x2.data_ptr(), w.data_ptr(), out.data_ptr(), _lib.address(b), _lib.address(r2), _lib.address(gamma), adapters.down.data_ptr(), adapters.up.data_ptr(),
            adapters.scale.data_ptr(), ids.data_ptr(), _lib.address(offsets), ws.data_ptr(), _lib.stream_ptr(device), M, lda, w.stride(0) if N > 1 else K, n_out,
            ldr if res is not None else 0, need, N, K, code, adapters.count, adapters.rank, S)))
        _lib.launched(2)
    return out
