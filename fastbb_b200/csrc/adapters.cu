// One shared projection and the low-rank adapters of many requests beside it: rows [offsets[s], offsets[s + 1]) belong to request s, whose
// adapter a = ids[s] adds scale_a (x A_a^T) B_a^T to x W^T ahead of the bias and the activation (A_a [r, K], B_a [N, r]).
//
// Two launches: one makes h = scale (x A_a^T), rounded to fp16 because the tensor cores take it so (2^-11 of each value, as the
// projection's own output is rounded), and the linear kernel adds h B_a^T to the accumulator it holds anyway. The second launch starts
// under the first (its product with W needs nothing of it) and waits for it where it needs h. Two forms of the pair:
//  blocks  h is laid out per (row tile t, request s in it) as block t + s of a tile's rows with zeros outside the request's (the
//          requests of one tile follow one another, so t + s is a number of its own), and the linear kernel runs each as k-blocks behind
//          those of x and W: one k-block of 64 per request and tile for ranks up to 64.
//  rows    for requests of few rows, where that would be a k-block per row or so: h is [M, r], and the epilogue multiplies each
//          row with its adapter's rows of B on the CUDA cores.
// Rows of no request (ahead of offsets[0], behind offsets[S]) and of requests with an id out of [0, adapters) get x W^T alone.
#include "common.cuh"
#include "internal.h"

namespace fbb {

struct AdapterArgs {
    const __half* x;
    int64_t ldx;
    const __half* down;   // [L, r, K]
    const float* scale;   // [L]
    const int* ids;       // [S]
    const int* offsets;   // [S + 1] or null: `each` rows a request
    int M, K, L, r, S, each;
    int tile_rows;        // blocks form
    __half* h;
    int4* tiles;
    int* list;
};

__device__ __forceinline__ int adapter_begin(const AdapterArgs& a, int s) {
    return a.offsets != nullptr ? min(max(__ldcg(a.offsets + s), 0), a.M) : s * a.each;
}
__device__ __forceinline__ int adapter_id(const AdapterArgs& a, int s) {
    const int id = __ldcg(a.ids + s);
    return id >= 0 && id < a.L ? id : -1;
}
// First request whose end lies beyond `row` (S if none), by the whole warp: 32 probes a round.
__device__ __forceinline__ int adapter_request(const AdapterArgs& a, int row, int lane) {
    if (a.offsets == nullptr) return min(row / a.each, a.S);
    int lo = 0, hi = a.S;
    while (lo < hi) {
        const int step = (hi - lo + 31) / 32, probe = min(lo + (lane + 1) * step - 1, hi - 1);
        const uint32_t beyond = __ballot_sync(0xffffffffu, adapter_begin(a, probe + 1) > row);
        if (beyond == 0u) return hi;
        const int first = __ffs(beyond) - 1;
        hi = min(lo + (first + 1) * step - 1, hi - 1);  // its probe: the answer is there or before it, behind the probe ahead
        lo += first * step;
        if (step == 1) return hi;
    }
    return lo;
}

__device__ __forceinline__ void mma_m16n8k16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// h of the blocks form. A CTA takes 32 rows of x and, of every request among them, all r products: 4 warps share K, 16-byte loads
// straight into fragments (the order of K inside a fragment is free as long as both operands agree), partial sums joined in shared
// memory in a fixed order. The launch reads x once (bound by that and by latency): mma.sync with its operands in registers is the
// shortest way for products of 32 x r. The first CTA of a tile also writes the tables that the linear kernel goes by.
constexpr int kDownRows = 32, kDownWarps = 4;
template <int NT>  // r in chunks of 8 NT
__global__ void __launch_bounds__(kDownWarps * 32) adapter_down_blocks_kernel(const AdapterArgs a) {
    __shared__ float s_part[kDownWarps][kDownRows][8 * NT + 1];
    grid_dependency_wait();
    grid_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int m0 = (int)blockIdx.x * kDownRows, m1 = min(m0 + kDownRows, a.M);
    const int tile = m0 / a.tile_rows, t0 = tile * a.tile_rows, t1 = min(t0 + a.tile_rows, a.M);
    const int first = adapter_request(a, t0, lane), end = min(adapter_request(a, t1 - 1, lane) + 1, a.S);
    if (m0 == t0 && warp == 0) {
        int count = 0;
        for (int s0 = first; s0 < end; s0 += 32) {
            const int s = s0 + lane;
            int id = -1;
            if (s < end && max(adapter_begin(a, s), t0) < min(adapter_begin(a, s + 1), t1)) id = adapter_id(a, s);
            if (s < end) a.list[tile + s] = id;
            count += __popc(__ballot_sync(0xffffffffu, id >= 0));
        }
        if (lane == 0) a.tiles[tile] = make_int4(first, end, count, 0);
    }
    const int g = lane >> 2, q = lane & 3;
    for (int s = first; s < end; ++s) {
        const int b = adapter_begin(a, s), e = adapter_begin(a, s + 1), id = adapter_id(a, s);
        if (id < 0 || max(b, t0) >= min(e, t1)) continue;
        __half* dst = a.h + ((int64_t)(tile + s) * a.tile_rows + (m0 - t0)) * a.r;
        if (max(b, m0) >= min(e, m1)) {  // none of its rows are here
            for (int i = threadIdx.x; i < kDownRows * (a.r >> 3); i += kDownWarps * 32) reinterpret_cast<uint4*>(dst)[i] = make_uint4(0u, 0u, 0u, 0u);
            continue;
        }
        const float scale = __ldcg(a.scale + id);
        for (int n0 = 0; n0 < a.r; n0 += 8 * NT) {
            float acc[2][NT][4] = {};
            const __half* down = a.down + ((int64_t)id * a.r + n0 + g) * a.K;
            const __half* x[4];  // rows g, g + 8, g + 16, g + 24; beyond the last row the last one again
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = a.x + (int64_t)min(m0 + g + 8 * i, a.M - 1) * a.ldx;
#pragma unroll 2
            for (int k = (warp * 4 + q) * 8; k < (a.K + 31) / 32 * 32; k += kDownWarps * 32) {
                uint4 xv[4], dv[NT];
                const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (int i = 0; i < 4; ++i) xv[i] = k < a.K ? *reinterpret_cast<const uint4*>(x[i] + k) : zero;
#pragma unroll
                for (int n = 0; n < NT; ++n) dv[n] = (k < a.K && n0 + 8 * n < a.r) ? __ldg(reinterpret_cast<const uint4*>(down + (int64_t)(8 * n) * a.K + k)) : zero;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma_m16n8k16(acc[i][n], xv[2 * i].x, xv[2 * i + 1].x, xv[2 * i].y, xv[2 * i + 1].y, dv[n].x, dv[n].y);
                        mma_m16n8k16(acc[i][n], xv[2 * i].z, xv[2 * i + 1].z, xv[2 * i].w, xv[2 * i + 1].w, dv[n].z, dv[n].w);
                    }
            }
            __syncthreads();  // the previous sums have been read
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s_part[warp][16 * i + g + 8 * (j >> 1)][8 * n + 2 * q + (j & 1)] = acc[i][n][j];
            __syncthreads();
            const int cols = min(8 * NT, a.r - n0);
            for (int i = threadIdx.x; i < kDownRows * (cols >> 1); i += kDownWarps * 32) {
                const int row = i / (cols >> 1), c = 2 * (i - row * (cols >> 1));
                float v0 = 0.f, v1 = 0.f;
#pragma unroll
                for (int w = 0; w < kDownWarps; ++w) v0 += s_part[w][row][c], v1 += s_part[w][row][c + 1];
                const bool mine = m0 + row >= b && m0 + row < e;
                *reinterpret_cast<uint32_t*>(dst + (int64_t)row * a.r + n0 + c) = mine ? pack_h2(v0 * scale, v1 * scale) : 0u;
            }
        }
    }
}

// h of the rows form: one CTA per row, its warps take the r products in turn.
__global__ void __launch_bounds__(256) adapter_down_rows_kernel(const AdapterArgs a) {
    grid_dependency_wait();
    grid_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int m = (int)blockIdx.x;
    const int s = adapter_request(a, m, lane);
    const int id = s < a.S && adapter_begin(a, s) <= m ? adapter_id(a, s) : -1;
    if (threadIdx.x == 0) a.list[m] = id;
    if (id < 0) return;
    const uint4* x = reinterpret_cast<const uint4*>(a.x + (int64_t)m * a.ldx);
    const int vecs = a.K >> 3;
    const float scale = __ldcg(a.scale + id);
    for (int n = warp; n < a.r; n += 8) {
        const uint4* d = reinterpret_cast<const uint4*>(a.down + ((int64_t)id * a.r + n) * a.K);
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll 4
        for (int v = lane; v < vecs; v += 32) {
            const uint4 xv = x[v], dv = __ldg(d + v);
            const __half2 *xh = reinterpret_cast<const __half2*>(&xv), *dh = reinterpret_cast<const __half2*>(&dv);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = ffma2(__half22float2(xh[e]), __half22float2(dh[e]), acc);
        }
        float sum = acc.x + acc.y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) a.h[(int64_t)m * a.r + n] = __float2half_rn(sum * scale);
    }
}

template <int BN, bool SWIGLU, bool CTA2, AdaptMode ADAPT>
__global__ void __launch_bounds__(kGemmThreads, 1)
linear_adapter_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_h,
                      const __grid_constant__ CUtensorMap tmap_up, const __grid_constant__ CUtensorMap tmap_c, const GemmArgs g, AdaptArgs ad) {
    ad.map_h = &tmap_h;
    ad.map_up = &tmap_up;
    linear_umma_body<BN, SWIGLU, CTA2, false, ADAPT>(tmap_a, tmap_w, tmap_w, tmap_c, g, ad);
}

// The forms of a launch: which of the two pairs, and the linear kernel's tiles.
struct AdapterForm {
    bool rows;
    int bn;
    bool pairs;
};
static AdapterForm adapter_form(int64_t M, int N, int K, bool swiglu, int r, int S) {
    const int n_out = swiglu ? N / 2 : N, sms = num_sms();
    AdapterForm f = {};
    auto tiles = [&](int rows, int bn) { return ((M + rows - 1) / rows) * (int64_t)((n_out + (swiglu ? bn / 2 : bn) - 1) / (swiglu ? bn / 2 : bn)); };
    f.rows = M < 8 * (int64_t)S;
    const int pairs = gemm_pairs_enabled() ? (swiglu ? max_pairs<256, true>() : max_pairs<256, false>()) : 0;
    if (f.rows) {
        f.bn = !swiglu && tiles(BM, 128) <= sms / 2 ? 64 : 128;
    } else if (pairs > 0 && tiles(2 * BM, 256) > pairs / 2) {
        f.bn = 256;
        f.pairs = true;
    } else {
        f.bn = !swiglu && tiles(BM, 128) <= sms / 2 ? 64 : 128;
    }
    return f;
}

// Workspace: h, then the tile table, then the list, each on a 256-byte boundary.
struct AdapterSpace {
    int64_t tiles, list, bytes;
};
static AdapterSpace adapter_space(const AdapterForm& f, int64_t M, int r, int S) {
    AdapterSpace w;
    auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
    const int64_t tile_rows = f.pairs ? 2 * BM : BM, n_tiles = (M + tile_rows - 1) / tile_rows;
    w.tiles = up(f.rows ? M * r * 2 : (n_tiles + S) * tile_rows * r * 2);
    w.list = w.tiles + (f.rows ? 0 : up(n_tiles * (int64_t)sizeof(int4)));
    w.bytes = w.list + up((f.rows ? M : n_tiles + S) * (int64_t)sizeof(int));
    return w;
}

int64_t adapter_linear_workspace_bytes(int64_t M, int N, int K, int epilogue, int r, int S) {
    if (M <= 0 || S <= 0) return 0;
    return adapter_space(adapter_form(M, N, K, epilogue == FBB_EPI_SWIGLU, r, S), M, r, S).bytes;
}

template <int BN, bool SWIGLU, bool CTA2, AdaptMode ADAPT>
static int launch_adapter_variant(const CUtensorMap& ta, const CUtensorMap& tw, const CUtensorMap& th, const CUtensorMap& tu, const CUtensorMap& tc, GemmArgs g,
                                  const AdaptArgs& ad, cudaStream_t stream) {
    using S = GemmSmem<BN, CTA2>;
    auto kern = linear_adapter_kernel<BN, SWIGLU, CTA2, ADAPT>;
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kDynamic);
        if (e != cudaSuccess) return fail((int)e, "cudaFuncSetAttribute(linear_adapter_kernel): %s", cudaGetErrorString(e));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    constexpr int kOutCols = SWIGLU ? BN / 2 : BN, kTileRows = CTA2 ? 2 * BM : BM;
    g.tiles_n = (g.n_out + kOutCols - 1) / kOutCols;
    g.tiles_m = (g.M + kTileRows - 1) / kTileRows;
    const int64_t tiles = (int64_t)g.tiles_m * g.tiles_n;
    if (tiles > 0x7FFFFFFFll) return fail(FBB_ERR_SHAPE, "adapter_linear: too many tiles (%lld)", (long long)tiles);
    g.wide_tiles = (int)tiles;
    const int most = CTA2 ? max_pairs<BN, SWIGLU>() : num_sms(), workers = tiles < most ? (int)tiles : most;
    const cudaError_t e = launch_pdl_cluster(kern, dim3((unsigned)(CTA2 ? 2 * workers : workers)), dim3(kGemmThreads), S::kDynamic, stream, CTA2 ? 2u : 1u, ta, tw, th,
                                             tu, tc, g, ad);
    if (e != cudaSuccess) return fail((int)e, "linear_adapter_kernel launch: %s", cudaGetErrorString(e));
    return FBB_OK;
}

int launch_adapter_linear(const void* A, const void* W, void* C, const void* bias, const void* res, const void* gamma, int64_t M, int N, int K, int64_t lda,
                          int64_t ldw, int64_t ldc, int64_t ldr, int epilogue, const void* down, const void* up, const float* scale, int L, int r, const int* ids,
                          const int* offsets, int S, void* ws, int64_t ws_bytes, cudaStream_t stream) {
    const bool swiglu = epilogue == FBB_EPI_SWIGLU;
    const AdapterForm f = adapter_form(M, N, K, swiglu, r, S);
    const AdapterSpace space = adapter_space(f, M, r, S);
    if (ws == nullptr || ws_bytes < space.bytes)
        return fail(FBB_ERR_SHAPE, "adapter_linear: workspace of %lld bytes, %lld needed", (long long)(ws != nullptr ? ws_bytes : 0), (long long)space.bytes);
    uint8_t* w8 = reinterpret_cast<uint8_t*>(ws);
    const int tile_rows = f.pairs ? 2 * BM : BM;
    const int64_t h_rows = ((M + tile_rows - 1) / tile_rows + S) * tile_rows;
    if (h_rows > 0x7FFFFFFFll) return fail(FBB_ERR_SHAPE, "adapter_linear: too many requests (%d) for %lld rows", S, (long long)M);

    AdapterArgs d = {};
    d.x = reinterpret_cast<const __half*>(A);
    d.ldx = lda;
    d.down = reinterpret_cast<const __half*>(down);
    d.scale = scale, d.ids = ids, d.offsets = offsets;
    d.M = (int)M, d.K = K, d.L = L, d.r = r, d.S = S, d.each = offsets != nullptr ? 0 : (int)(M / S);
    d.tile_rows = tile_rows;
    d.h = reinterpret_cast<__half*>(ws);
    d.tiles = reinterpret_cast<int4*>(w8 + space.tiles);
    d.list = reinterpret_cast<int*>(w8 + space.list);
    cudaError_t e;
    if (f.rows) {
        e = launch_pdl(adapter_down_rows_kernel, dim3((unsigned)M), dim3(256), 0, stream, d);
    } else {
        const dim3 grid((unsigned)((M + kDownRows - 1) / kDownRows));
        auto kern = r <= 16 ? adapter_down_blocks_kernel<2> : (r <= 32 ? adapter_down_blocks_kernel<4> : adapter_down_blocks_kernel<8>);
        e = launch_pdl(kern, grid, dim3(kDownWarps * 32), 0, stream, d);
    }
    if (e != cudaSuccess) return fail((int)e, "adapter_down kernel launch: %s", cudaGetErrorString(e));

    GemmArgs g = {};
    g.C = reinterpret_cast<__half*>(C);
    g.bias = reinterpret_cast<const __half*>(bias);
    g.res = reinterpret_cast<const __half*>(res);
    g.gamma = res != nullptr ? reinterpret_cast<const __half*>(gamma) : nullptr;
    g.M = (int)M, g.N = N, g.K = K;
    g.n_out = swiglu ? N / 2 : N;
    g.ldc = ldc, g.ldr = ldr;
    g.act = epilogue == FBB_EPI_GELU ? 1 : 0;
    g.gemv_row0 = (int)M;
    AdaptArgs ad = {};
    ad.tiles = d.tiles;
    ad.list = d.list;
    ad.h = d.h;
    ad.up = reinterpret_cast<const __half*>(up);
    ad.r = r, ad.r_blocks = (r + BK - 1) / BK;

    // boxes: 128 rows of A and h; of W and the adapters' second matrices the rows that one CTA loads per k-block
    const uint32_t w_rows = swiglu ? (uint32_t)f.bn / 2 : (f.pairs ? (uint32_t)f.bn / 2 : (uint32_t)f.bn);
    struct { CUtensorMap map; const void* p; uint64_t cols, rows; int64_t stride; uint32_t box0, box1; CUtensorMapSwizzle swizzle; } t[5] = {
        {{}, A, (uint64_t)K, (uint64_t)M, lda, BK, BM, CU_TENSOR_MAP_SWIZZLE_128B},
        {{}, W, (uint64_t)K, (uint64_t)N, ldw, BK, w_rows, CU_TENSOR_MAP_SWIZZLE_128B},
        {{}, f.rows ? A : ws, (uint64_t)(f.rows ? K : r), (uint64_t)(f.rows ? M : h_rows), f.rows ? lda : r, BK, BM, CU_TENSOR_MAP_SWIZZLE_128B},
        {{}, up, (uint64_t)r, (uint64_t)L * (uint64_t)N, r, BK, w_rows, CU_TENSOR_MAP_SWIZZLE_128B},
        {{}, C, (uint64_t)g.n_out, (uint64_t)M, ldc, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B}};
    for (auto& m : t) {
        const uint64_t dims[2] = {m.cols, m.rows};
        const int64_t st[2] = {1, m.stride};
        const uint32_t box[2] = {m.box0, m.box1};
        const int rc = make_tmap_f16(&m.map, m.p, 2, dims, st, box, m.swizzle);
        if (rc != FBB_OK) return rc;
    }
#define FBB_ADAPTER_LAUNCH(BN, SWIGLU, CTA2, MODE) launch_adapter_variant<BN, SWIGLU, CTA2, MODE>(t[0].map, t[1].map, t[2].map, t[3].map, t[4].map, g, ad, stream)
    if (f.pairs) return swiglu ? FBB_ADAPTER_LAUNCH(256, true, true, kAdaptBlocks) : FBB_ADAPTER_LAUNCH(256, false, true, kAdaptBlocks);
    if (f.rows) {
        if (swiglu) return FBB_ADAPTER_LAUNCH(128, true, false, kAdaptRows);
        return f.bn == 64 ? FBB_ADAPTER_LAUNCH(64, false, false, kAdaptRows) : FBB_ADAPTER_LAUNCH(128, false, false, kAdaptRows);
    }
    if (swiglu) return FBB_ADAPTER_LAUNCH(128, true, false, kAdaptBlocks);
    return f.bn == 64 ? FBB_ADAPTER_LAUNCH(64, false, false, kAdaptBlocks) : FBB_ADAPTER_LAUNCH(128, false, false, kAdaptBlocks);
#undef FBB_ADAPTER_LAUNCH
}

}  // namespace fbb
