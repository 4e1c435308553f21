// Rotary positions on several axes, for queries and keys in one launch: pair i of a head's columns at position p is turned by the
// angle t = p[axis_i] * freq_i,  (x, y) -> (x cos t - y sin t, y cos t + x sin t);  the transposed turn (t -> -t) is the gradient.
// Pairs are columns (i, i + P) ("half") or (2i, 2i + 1) ("pairs") for i < P; columns 2P .. D-1 and the first n_prefix rows of a
// sequence (cls and register tokens, which have no position) pass.
//
// Bound by memory: every element is read once and written once (50.4 MB at 6145 tokens x 16 + 16 heads x 64, fp16: 7.7 us at the
// measured copy rate, 12.1 measured: 769 CTAs on 444 places are two waves, the second three quarters full; fp32 at 4 x 1374 tokens x 48 x 64:
// 20.6 and 24.4). The angles of a token are the same for all its
// heads, so a CTA takes a few whole tokens, works their cos / sin out once into shared memory, and streams the tokens' heads through with
// 16-byte accesses, kRotaryUnroll items in flight per thread (2 and 8 were slower: 54 - 66 and 53 us on 2 x 8184 x 20 x 128 bf16, now 37).
// The angle, position times fp32 frequency, and its number of turns are doubles up to 2^20 radians, off by 2^-31 radians at most. Beyond, each is
// a double and the remainder that its rounding left (Dekker's arithmetic: a product's remainder is one fma; 1 / (2 pi) is two doubles as
// well), off by 2^-105 of the number of turns: fp32 angles lose nothing up to position times frequency of 2^70, which every int64 position
// is within for frequencies up to 2^7. (All angles that way: 3 % more on the fp32 case above.) The turns' fraction is taken there;
// sincospif of twice that, at most 1, then has fp32 accuracy. The products and the sum are fp32, rounded once to the output type.
#include <cuda_bf16.h>

#include "common.cuh"
#include "internal.h"

namespace fbb {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryUnroll = 4;
constexpr int kRotaryTableEntries = 2048;  // (cos, sin) pairs of a CTA: 16 KB of shared memory
constexpr int kRotaryMaxTokens = 64;       // of a CTA

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
// The fraction of a turn, from -1/2 to 1/2, of the position at `at` times freq radians.
__device__ __forceinline__ double rotary_fraction(const RotaryArgs& a, int64_t at, double freq) {
    constexpr double kTurn = 0x1.45f306dc9c883p-3, kTurnRest = -0x1.6b01ec5417056p-57;  // their sum is 1 / (2 pi) to 2^-108 of it
    double position = rotary_position(a, at), angle = position * freq, turns = angle * kTurn, fraction = turns - rint(turns);
    if (fabs(angle) >= 1048576.0) {
        double angle_rest = 0.0;
        if (a.pos_dtype == FBB_POS_I64) {
            const int64_t p = reinterpret_cast<const int64_t*>(a.pos)[at];
            const double high = (double)(p >> 32) * 4294967296.0, low = (double)(uint32_t)p;  // (both exact)
            position = high + low;
            angle_rest = (low - (position - high)) * freq;
        }
        angle = position * freq;
        angle_rest += fma(position, freq, -angle);
        turns = angle * kTurn;
        fraction = (turns - rint(turns)) + (fma(angle, kTurn, -turns) + fma(angle, kTurnRest, angle_rest * kTurn));
        fraction -= rint(fraction);
    }
    return fraction;
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

// Where a token's heads begin in the two tensors; tensor 1's are heads heads0, heads0 + 1, ... of a row.
struct RotaryRow {
    const char* x[2];
    char* y[2];
};

// HALF: pairing. VEC: 16-byte accesses; the scalar form (columns one by one) takes every size and stride that is not a multiple of
// 16 bytes. A vector item of the half pairing is the two vectors at columns 8c and P + 8c, of the other pairing one vector; what is
// left of a head (columns from 2P on) are plain copies behind them.
// (Three or four CTAs an SM: left to itself the code for far angles takes 88 registers of the half pairing's vector form, 73 of the
// other's, and a CTA from each SM: 13.7 instead of 12.1 us on 6145 tokens, 42.7 instead of 37.3 on 2 x 8184 x 20 x 128.)
template <typename T, bool HALF, bool VEC>
__global__ void __launch_bounds__(kRotaryThreads, HALF && VEC ? 3 : 4) rotary_kernel(const RotaryArgs a) {
    __shared__ __align__(16) float2 s_turn[kRotaryTableEntries];
    __shared__ RotaryRow s_row[kRotaryMaxTokens];
    __shared__ int s_pass[kRotaryMaxTokens];  // a row without a position
    grid_dependency_wait();
    grid_launch_dependents();
    const int64_t token0 = (int64_t)blockIdx.x * a.tokens_per_cta;
    const int count = (int)min((int64_t)a.tokens_per_cta, a.tokens - token0);
    constexpr int E = VEC ? 16 / (int)sizeof(T) : 1;
    const int turned = VEC ? (HALF ? a.P / E : 2 * a.P / E) : a.P;  // items of a head that turn; the others copy
    const int64_t second = HALF ? (int64_t)a.P * (int)sizeof(T) : (int64_t)sizeof(T);
    // A thread keeps its item of a head and walks the CTA's (token, head) rows in steps of `step`: no divisions on the way.
    const int lanes = min(a.per_head, kRotaryThreads), step = kRotaryThreads / lanes;
    const int lane = (int)threadIdx.x % lanes, row0 = (int)threadIdx.x / lanes;
    for (int tok = threadIdx.x; tok < count; tok += kRotaryThreads) {
        const uint32_t at = (uint32_t)token0 + (uint32_t)tok, b = at / (uint32_t)a.N, n = at - b * (uint32_t)a.N;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const RotaryTensor& t = a.t[i];
            s_row[tok].x[i] = t.x + b * t.x_sb + n * t.x_sn - (i == 1 ? a.heads0 * t.x_sh : 0);
            s_row[tok].y[i] = t.y + b * t.y_sb + n * t.y_sn - (i == 1 ? a.heads0 * t.y_sh : 0);
        }
        s_pass[tok] = (int)n < a.n_prefix;
    }
    __syncthreads();

    struct Item {
        uint4 u, w;
        T su, sw;
        char* dst;
        int entry;  // first table entry, -1: copy, -2: beyond the CTA's rows
    };
    int c = lane, tok, head, first;
    bool turn, two;
    int64_t col;
    auto begin = [&]() {  // the rows of item c from the first on
        turn = c < turned;
        two = turn && (HALF || !VEC);
        col = (int64_t)(HALF || !turn ? (turn ? c * E : 2 * a.P + (c - turned) * E) : c * (VEC ? E : 2)) * (int)sizeof(T);
        first = VEC && !HALF ? c * (E / 2) : c * E;  // of the item's table entries
        tok = row0 / a.heads, head = row0 - tok * a.heads;
        if (row0 >= step || c >= a.per_head) tok = count;
    };
    const int64_t x_sh0 = a.t[0].x_sh, x_sh1 = a.t[1].x_sh, y_sh0 = a.t[0].y_sh, y_sh1 = a.t[1].y_sh;
    auto load = [&](Item& it) {
        it.entry = -2;
        if (tok >= count) return;
        const bool other = head >= a.heads0;
        const char* src = s_row[tok].x[other] + head * (other ? x_sh1 : x_sh0) + col;
        it.dst = s_row[tok].y[other] + head * (other ? y_sh1 : y_sh0) + col;
        it.entry = turn && !s_pass[tok] ? tok * a.P + first : -1;
        if constexpr (VEC) {
            it.u = *reinterpret_cast<const uint4*>(src);
            if (two) it.w = *reinterpret_cast<const uint4*>(src + second);
        } else {
            it.su = *reinterpret_cast<const T*>(src);
            if (two) it.sw = *reinterpret_cast<const T*>(src + second);
        }
        for (head += step; head >= a.heads; head -= a.heads) ++tok;
    };
    auto finish = [&](Item& it) {
        if (it.entry == -2) return;
        if constexpr (VEC) {
            if (it.entry >= 0) {
                float x[E], y[E];
                rotary_unpack<T>(it.u, x);
                if constexpr (HALF) {
                    rotary_unpack<T>(it.w, y);
#pragma unroll
                    for (int e = 0; e < E; e += 2) {
                        const float4 t = *reinterpret_cast<const float4*>(s_turn + it.entry + e);
                        const float x0 = x[e], x1 = x[e + 1];
                        x[e] = fmaf(x0, t.x, -y[e] * t.y), y[e] = fmaf(y[e], t.x, x0 * t.y);
                        x[e + 1] = fmaf(x1, t.z, -y[e + 1] * t.w), y[e + 1] = fmaf(y[e + 1], t.z, x1 * t.w);
                    }
                    it.w = rotary_pack<T>(y);
                } else {
#pragma unroll
                    for (int e = 0; e < E; e += 4) {
                        const float4 t = *reinterpret_cast<const float4*>(s_turn + it.entry + e / 2);
                        const float x0 = x[e], x2 = x[e + 2];
                        x[e] = fmaf(x0, t.x, -x[e + 1] * t.y), x[e + 1] = fmaf(x[e + 1], t.x, x0 * t.y);
                        x[e + 2] = fmaf(x2, t.z, -x[e + 3] * t.w), x[e + 3] = fmaf(x[e + 3], t.z, x2 * t.w);
                    }
                }
                it.u = rotary_pack<T>(x);
            }
            *reinterpret_cast<uint4*>(it.dst) = it.u;
            if (two) *reinterpret_cast<uint4*>(it.dst + second) = it.w;
        } else {
            if (it.entry >= 0) {
                const float x = rotary_value<T>(it.su), y = rotary_value<T>(it.sw);
                const float2 t = s_turn[it.entry];
                it.su = rotary_round<T>(fmaf(x, t.x, -y * t.y));
                it.sw = rotary_round<T>(fmaf(y, t.x, x * t.y));
            }
            *reinterpret_cast<T*>(it.dst) = it.su;
            if (two) *reinterpret_cast<T*>(it.dst + second) = it.sw;
        }
    };

    // The first rows are on their way while the table is worked out.
    Item items[kRotaryUnroll];
    begin();
#pragma unroll
    for (int j = 0; j < kRotaryUnroll; ++j) load(items[j]);
    for (int i = threadIdx.x; i < count * a.P; i += kRotaryThreads) {
        const int tok = i / a.P, p = i - tok * a.P;
        const uint32_t at = (uint32_t)token0 + (uint32_t)tok, b = at / (uint32_t)a.N;
        const int n = (int)(at - b * (uint32_t)a.N) - a.n_prefix;
        float2 turn = make_float2(1.f, 0.f);
        if (n >= 0) {
            const int axis = min(max(a.axes[p], 0), a.n_axes - 1);
            sincospif(2.f * (float)rotary_fraction(a, (int64_t)b * a.p_sb + n * a.p_sn + axis * a.p_sa, (double)a.freqs[p]), &turn.y, &turn.x);
            turn.y *= a.sign;
        }
        s_turn[i] = turn;
    }
    __syncthreads();
    for (;;) {
#pragma unroll
        for (int j = 0; j < kRotaryUnroll; ++j) finish(items[j]);
        if (tok >= count) {
            c += lanes;
            if (c >= a.per_head) break;
            begin();
        }
#pragma unroll
        for (int j = 0; j < kRotaryUnroll; ++j) load(items[j]);
    }
}

template <typename T>
static cudaError_t rotary_launch(RotaryArgs a, bool half, bool vec, cudaStream_t stream) {
    const int E = vec ? 16 / (int)sizeof(T) : 1;
    a.per_head = (vec ? (half ? a.P / E : 2 * a.P / E) : a.P) + (a.D - 2 * a.P) / E;
    // As many tokens a CTA as give each thread kRotaryUnroll items, fewer where that leaves SMs without two CTAs.
    const int per_token = a.heads * a.per_head;
    int64_t per_cta = kRotaryThreads * kRotaryUnroll / per_token;
    per_cta = min(per_cta, (a.tokens + 2 * num_sms() - 1) / (2 * num_sms()));
    per_cta = min(per_cta, (int64_t)min(kRotaryTableEntries / a.P, kRotaryMaxTokens));
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
