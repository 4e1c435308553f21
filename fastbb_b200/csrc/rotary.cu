// Rotary positions on several axes, for queries and keys in one launch: pair i of a head's columns at position p is turned by the
// angle t = p[axis_i] * freq_i,  (x, y) -> (x cos t - y sin t, y cos t + x sin t);  the transposed turn (t -> -t) is the gradient.
// Pairs are columns (i, i + P) ("half") or (2i, 2i + 1) ("pairs") for i < P; columns 2P .. D-1 and the first n_prefix rows of a
// sequence (cls and register tokens, which have no position) pass.
//
// Bound by memory: every element is read once and written once (50.4 MB at 6145 tokens x 16 + 16 heads x 64, fp16: 7.7 us at the
// measured copy rate). The angles of a token are the same for all its heads, so a CTA takes a few whole tokens, works their cos / sin
// out once into shared memory, and streams the tokens' heads through with 16-byte accesses, kUnroll vectors in flight per thread.
// The angle is a product in 64 bits (an integer position times an fp32 frequency, exact up to 2^29; far positions lose nothing),
// reduced to a fraction of a turn there; sincospif on |2 f| <= 1 then has fp32 accuracy at any position. The products and the
// sum are fp32, rounded once to the output type.
#include <cuda_bf16.h>

#include "common.cuh"
#include "internal.h"

namespace fbb {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryUnroll = 4;
constexpr int kRotaryTableEntries = 2048;  // (cos, sin) pairs of a CTA: 16 KB of shared memory

struct RotaryTensor {
    const char* x;
    char* y;
    int64_t x_sb, x_sn, x_sh, y_sb, y_sn, y_sh;  // bytes
};
struct RotaryArgs {
    RotaryTensor t[2];
    int heads0, heads;         // heads of tensor 0; of both
    int N, D, P, n_prefix;
    int64_t tokens;            // B * N
    int tokens_per_cta;
    int per_head;              // vectors (or, scalar form, columns) a head is worked on in
    const void* pos;
    int pos_dtype, n_axes;
    int64_t p_sb, p_sn, p_sa;  // elements
    const float* freqs;
    const int* axes;
    float sign;
};

__device__ __forceinline__ double rotary_position(const RotaryArgs& a, int64_t at) {
    if (a.pos_dtype == FBB_POS_I32) return (double)reinterpret_cast<const int*>(a.pos)[at];
    if (a.pos_dtype == FBB_POS_I64) return (double)reinterpret_cast<const int64_t*>(a.pos)[at];
    return (double)reinterpret_cast<const float*>(a.pos)[at];
}

template <typename T>
__device__ __forceinline__ void rotary_unpack(const uint4& v, float* f) {
    if constexpr (sizeof(T) == 4) {
        f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
    } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float2 p;
            if constexpr (std::is_same<T, __half>::value) p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            else p = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
            f[2 * i] = p.x, f[2 * i + 1] = p.y;
        }
    }
}
template <typename T>
__device__ __forceinline__ uint4 rotary_pack(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            w[i] = __float_as_uint(f[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
            w[i] = pack_h2(f[2 * i], f[2 * i + 1]);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ float rotary_value(T v) {
    if constexpr (std::is_same<T, __half>::value) return __half2float(v);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __bfloat162float(v);
    else return v;
}
template <typename T>
__device__ __forceinline__ T rotary_round(float v) {
    if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) return __float2bfloat16_rn(v);
    else return v;
}

// HALF: pairing. VEC: 16-byte accesses; the scalar form (columns one by one) takes every size and stride that is not a multiple of
// 16 bytes. A vector item of the half pairing is the two vectors at columns 8c and P + 8c, of the other pairing one vector; what is
// left of a head (columns from 2P on) are plain copies behind them.
template <typename T, bool HALF, bool VEC>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryArgs a) {
    __shared__ __align__(16) float2 s_turn[kRotaryTableEntries];
    grid_dependency_wait();
    grid_launch_dependents();
    const int64_t token0 = (int64_t)blockIdx.x * a.tokens_per_cta;
    const int count = (int)min((int64_t)a.tokens_per_cta, a.tokens - token0);
    for (int i = threadIdx.x; i < count * a.P; i += kRotaryThreads) {
        const int tok = i / a.P, p = i - tok * a.P;
        const int64_t b = (token0 + tok) / a.N;
        const int n = (int)(token0 + tok - b * a.N) - a.n_prefix;
        float2 turn = make_float2(1.f, 0.f);
        if (n >= 0) {
            const int axis = min(max(a.axes[p], 0), a.n_axes - 1);
            const double turns = rotary_position(a, b * a.p_sb + n * a.p_sn + axis * a.p_sa) * (double)a.freqs[p] * 0.15915494309189533577;
            sincospif(2.f * (float)(turns - rint(turns)), &turn.y, &turn.x);
            turn.y *= a.sign;
        }
        s_turn[i] = turn;
    }
    __syncthreads();

    constexpr int E = VEC ? 16 / (int)sizeof(T) : 1;
    const int per_token = a.heads * a.per_head;
    const int items = count * per_token;
    const int turned = VEC ? (HALF ? a.P / E : 2 * a.P / E) : a.P;  // items of a head that turn; the others copy
    for (int i0 = threadIdx.x; i0 < items; i0 += kRotaryThreads * kRotaryUnroll) {
        uint4 u[kRotaryUnroll], w[kRotaryUnroll];
        T su[kRotaryUnroll], sw[kRotaryUnroll];
        char* dst[kRotaryUnroll];
        int entry[kRotaryUnroll];  // first table entry; -1: one vector (column) to copy, -2: two
#pragma unroll
        for (int j = 0; j < kRotaryUnroll; ++j) {
            const int i = i0 + j * kRotaryThreads;
            if (i >= items) continue;
            const int tok = i / per_token, r = i - tok * per_token;
            int head = r / a.per_head;
            const int c = r - head * a.per_head;
            const int64_t b = (token0 + tok) / a.N;
            const int n = (int)(token0 + tok - b * a.N);
            const RotaryTensor& t = a.t[head >= a.heads0 ? 1 : 0];
            if (head >= a.heads0) head -= a.heads0;
            const bool turn = c < turned;
            const int col = HALF || !turn ? (turn ? c * E : 2 * a.P + (c - turned) * E) : c * (VEC ? E : 2);
            const char* src = t.x + b * t.x_sb + n * t.x_sn + head * t.x_sh + (int64_t)col * (int)sizeof(T);
            dst[j] = t.y + b * t.y_sb + n * t.y_sn + head * t.y_sh + (int64_t)col * (int)sizeof(T);
            const bool two = turn && (HALF || !VEC);
            entry[j] = (turn && n >= a.n_prefix) ? tok * a.P + (VEC && !HALF ? c * (E / 2) : c * E) : (two ? -2 : -1);
            const int64_t second = HALF ? (int64_t)a.P * (int)sizeof(T) : (int64_t)sizeof(T);
            if constexpr (VEC) {
                u[j] = *reinterpret_cast<const uint4*>(src);
                if (two) w[j] = *reinterpret_cast<const uint4*>(src + second);
            } else {
                su[j] = *reinterpret_cast<const T*>(src);
                if (two) sw[j] = *reinterpret_cast<const T*>(src + second);
            }
        }
#pragma unroll
        for (int j = 0; j < kRotaryUnroll; ++j) {
            if (i0 + j * kRotaryThreads >= items) continue;
            const int64_t second = HALF ? (int64_t)a.P * (int)sizeof(T) : (int64_t)sizeof(T);
            if constexpr (VEC) {
                if (entry[j] >= 0) {
                    float x[E], y[E];
                    rotary_unpack<T>(u[j], x);
                    if constexpr (HALF) {
                        rotary_unpack<T>(w[j], y);
#pragma unroll
                        for (int e = 0; e < E; e += 2) {
                            const float4 t = *reinterpret_cast<const float4*>(s_turn + entry[j] + e);
                            const float x0 = x[e], x1 = x[e + 1];
                            x[e] = fmaf(x0, t.x, -y[e] * t.y), y[e] = fmaf(y[e], t.x, x0 * t.y);
                            x[e + 1] = fmaf(x1, t.z, -y[e + 1] * t.w), y[e + 1] = fmaf(y[e + 1], t.z, x1 * t.w);
                        }
                        w[j] = rotary_pack<T>(y);
                    } else {
#pragma unroll
                        for (int e = 0; e < E; e += 2) {
                            const float2 t = s_turn[entry[j] + e / 2];
                            const float x0 = x[e];
                            x[e] = fmaf(x0, t.x, -x[e + 1] * t.y), x[e + 1] = fmaf(x[e + 1], t.x, x0 * t.y);
                        }
                    }
                    u[j] = rotary_pack<T>(x);
                }
                *reinterpret_cast<uint4*>(dst[j]) = u[j];
                if (HALF && entry[j] != -1) *reinterpret_cast<uint4*>(dst[j] + second) = w[j];
            } else {
                if (entry[j] >= 0) {
                    const float x = rotary_value<T>(su[j]), y = rotary_value<T>(sw[j]);
                    const float2 t = s_turn[entry[j]];
                    su[j] = rotary_round<T>(fmaf(x, t.x, -y * t.y));
                    sw[j] = rotary_round<T>(fmaf(y, t.x, x * t.y));
                }
                *reinterpret_cast<T*>(dst[j]) = su[j];
                if (entry[j] != -1) *reinterpret_cast<T*>(dst[j] + second) = sw[j];
            }
        }
    }
}

template <typename T>
static cudaError_t rotary_launch(RotaryArgs a, bool half, bool vec, cudaStream_t stream) {
    const int E = vec ? 16 / (int)sizeof(T) : 1;
    a.per_head = (vec ? (half ? a.P / E : 2 * a.P / E) : a.P) + (a.D - 2 * a.P) / E;
    // As many tokens a CTA as give each thread kRotaryUnroll items, fewer where that leaves SMs without two CTAs.
    const int per_token = a.heads * a.per_head;
    int64_t per_cta = (kRotaryThreads * kRotaryUnroll + per_token - 1) / per_token;
    per_cta = min(per_cta, (a.tokens + 2 * num_sms() - 1) / (2 * num_sms()));
    per_cta = min(per_cta, (int64_t)(kRotaryTableEntries / max(a.P, 1)));
    a.tokens_per_cta = (int)max(per_cta, (int64_t)1);
    const dim3 grid((unsigned)((a.tokens + a.tokens_per_cta - 1) / a.tokens_per_cta));
    auto kern = half ? (vec ? rotary_kernel<T, true, true> : rotary_kernel<T, true, false>) : (vec ? rotary_kernel<T, false, true> : rotary_kernel<T, false, false>);
    return launch_pdl(kern, grid, dim3(kRotaryThreads), 0, stream, a);
}

int launch_rotary(const fbb_rotary_tensor* t, int n_tensors, int B, int N, int D, int pairs, int pairing, int n_prefix, const void* pos, int pos_dtype,
                  int n_axes, int64_t p_sb, int64_t p_sn, int64_t p_sa, const float* freqs, const int* axes, int inverse, int dtype, cudaStream_t stream) {
    RotaryArgs a = {};
    const int size = dtype == FBB_DTYPE_F32 ? 4 : 2, per_vec = 16 / size;
    const bool half = pairing == FBB_ROTARY_HALF;
    bool vec = (half ? pairs : 2 * pairs) % per_vec == 0 && D % per_vec == 0;
    for (int i = 0; i < n_tensors; ++i) {
        RotaryTensor& r = a.t[i];
        r.x = (const char*)t[i].x, r.y = (char*)t[i].y;
        r.x_sb = t[i].x_sb * size, r.x_sn = t[i].x_sn * size, r.x_sh = t[i].x_sh * size;
        r.y_sb = t[i].y_sb * size, r.y_sn = t[i].y_sn * size, r.y_sh = t[i].y_sh * size;
        const int64_t bits = (int64_t)(uintptr_t)r.x | (int64_t)(uintptr_t)r.y | (B > 1 ? r.x_sb | r.y_sb : 0) | (N > 1 ? r.x_sn | r.y_sn : 0) |
                             (t[i].heads > 1 ? r.x_sh | r.y_sh : 0);
        vec = vec && (bits & 15) == 0;
    }
    a.heads0 = t[0].heads;
    a.heads = t[0].heads + (n_tensors > 1 ? t[1].heads : 0);
    a.N = N, a.D = D, a.P = pairs, a.n_prefix = n_prefix;
    a.tokens = (int64_t)B * N;
    a.pos = pos, a.pos_dtype = pos_dtype, a.n_axes = n_axes;
    a.p_sb = p_sb, a.p_sn = p_sn, a.p_sa = p_sa;
    a.freqs = freqs, a.axes = axes;
    a.sign = inverse ? -1.f : 1.f;
    const cudaError_t e = dtype == FBB_DTYPE_F16 ? rotary_launch<__half>(a, half, vec, stream)
                          : dtype == FBB_DTYPE_BF16 ? rotary_launch<__nv_bfloat16>(a, half, vec, stream)
                                                    : rotary_launch<float>(a, half, vec, stream);
    return e == cudaSuccess ? FBB_OK : fail((int)e, "rotary: %s", cudaGetErrorString(e));
}

}  // namespace fbb
