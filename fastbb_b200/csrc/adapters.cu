// One shared projection and the low-rank adapters of many requests beside it: rows [offsets[s], offsets[s + 1]) belong to request s, whose
// adapter a = ids[s] adds scale_a (x A_a^T) B_a^T to x W^T ahead of the bias and the activation (A_a [r, K], B_a [N, r]).
//
// Two launches: one makes h = scale (x A_a^T), rounded (in the blocks form) to fp16 because the tensor cores take it so (2^-11 of each value, as the
// projection's own output is rounded), and the linear kernel adds h B_a^T to the accumulator it holds anyway. The second launch starts
// under the first (its product with W needs nothing of it) and waits for it where it needs h. Two forms of the pair:
//  blocks  h is [M, r], and the linear kernel runs it as k-blocks behind those of x and W: of every request in a row tile one k-block of 64
//          (for ranks up to 64) against its adapter's second matrix, which adds to the request's rows of the accumulator alone (the
//          lanes of tensor memory that a product leaves as they are are an operand of the instruction). A row of h with values beyond fp16
//          is held times 2^-15 and marked: the row's first product multiplies what it has so far by that too (an operand of the
//          instruction as well), and the epilogue takes the whole sum back. So whether a request's output is finite does not
//          depend on the form, or on what else is in the batch. (The marks cost 0.3 us of 16 at 8 x 257, 768 -> 2304, rank 16, 0.8 of 53 at
//          6146 rows, 1024 -> 4096, rank 32, and 0.9 of 170 at 21920 rows, 4096 -> 1024, rank 64.)
//  rows    for few rows of many requests, where that would be a k-block per row or so: the first launch multiplies each row with both
//          of its adapter's matrices on the CUDA cores (bound by reading those), and the linear kernel's epilogue adds that in fp32.
// Rows of no request (ahead of offsets[0], behind offsets[S]) and of requests with an id out of [0, adapters) get x W^T alone.
#include "common.cuh"
#include "internal.h"

namespace fbb {

struct AdapterArgs {
    Requests requests;
    const float* scale;   // [L]
    int M, N, K, r;
    // blocks form
    int pass_cols, stages;  // columns of h in a pass, a multiple of 16 up to kDownCols; tiles of x on their way
    __half* h;
    uint32_t* lifted;       // [M / 32, up to whole 256 rows]: a bit per row whose h is held times 2^-15
    // rows form
    const __half* x;
    int64_t ldx;
    const __half* down;   // [L, r, K]
    const __half* up;     // [L, N, r]
    float* delta;
    int cols;
};

// h of the blocks form: a CTA takes 128 rows of x and multiplies them with the first matrices of their requests, up to 64 columns of
// h at a time, or 128 where tiles hold many requests (several requests side by side where the rank leaves room), as UMMAs fed by TMA: x is
// read once for most tiles. Many tiles: that read, 180 MB or 28 us at 21920 x 4096, rank 64, 16 requests, where the launch takes 50 under ncu:
// the 15 of its 172 tiles that hold rows of two requests make two passes, the second one alone at the end. Few tiles are bound by
// latency: x's tiles start ahead of the look-up of the requests, which is a chain of dependent loads, and as many are on their way as
// shared memory holds (49 tiles of K = 1024: 12 - 13 us under ncu).
//   warp 0   look-up of the requests, then TMA producer      warp 1   UMMA issuer      warps 2..5   rows of h out of tensor memory
constexpr int kDownCols = 128;
constexpr int kDownMaxStages = 12;
constexpr int kDownMaxRequests = 128;
constexpr int kDownThreads = 192;
struct DownSmem {  // ring of {x [128 x 64], first matrices [pass_cols x 64]} | barriers | table of requests
    static constexpr int kABytes = BM * BK * 2;
    static constexpr int kNumBars = 2 * kDownMaxStages + 4;  // full, empty, accumulator full[2], empty[2]
    static constexpr int kTailBytes = kNumBars * 8 + 16 + (int)(kDownMaxRequests * sizeof(int4)) + 16;
    static int stage_bytes(int pass_cols) { return kABytes + pass_cols * BK * 2; }
    static int dynamic_bytes(int pass_cols, int stages) { return 1024 + stages * stage_bytes(pass_cols) + kTailBytes; }
    static constexpr int kMaxDynamic = 227 * 1024;
};

__global__ void __launch_bounds__(kDownThreads) adapter_down_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_down,
                                                                    const AdapterArgs a) {
    using S = DownSmem;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    const uint32_t stage_bytes = (uint32_t)(S::kABytes + a.pass_cols * BK * 2), ring = (uint32_t)a.stages * stage_bytes;
    uint8_t* tail = smem_raw + (base - raw) + ring;
    const uint32_t bar0 = base + ring;
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (kDownMaxStages + s); };
    auto tfull_bar = [&](int i) { return bar0 + 8u * (2 * kDownMaxStages + i); };
    auto tempty_bar = [&](int i) { return bar0 + 8u * (2 * kDownMaxStages + 2 + i); };
    volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(tail + S::kNumBars * 8);
    volatile int* s_abort = reinterpret_cast<volatile int*>(tail + S::kNumBars * 8 + 4);
    int4* s_req = reinterpret_cast<int4*>(tail + S::kNumBars * 8 + 16);  // {first row, one behind its last, adapter, 0}
    volatile int* s_count = reinterpret_cast<volatile int*>(s_req + kDownMaxRequests);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int num_kb = (a.K + BK - 1) / BK;
    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(full_bar(s), 2);  // x's bytes, the adapters' bytes
            mbar_init(empty_bar(s), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(tfull_bar(i), 1);
            mbar_init(tempty_bar(i), 4);
        }
        *s_abort = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmap_x);
        tma_prefetch_desc(&tmap_down);
    }
    if (warp == 1) {
        __syncwarp();
        tmem_alloc<2 * kDownCols>(smem_u32(const_cast<uint32_t*>(s_tmem)));
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *s_tmem;
    grid_dependency_wait();
    grid_launch_dependents();

    const int m0 = (int)blockIdx.x * BM, m1 = min(m0 + BM, a.M);
    const int ahead = min(num_kb, a.stages);
    if (warp == 0) {
        if (lane == 0) {
            for (int s = 0; s < ahead; ++s) {
                mbar_arrive_expect_tx(full_bar(s), S::kABytes);
                tma_load_2d(base + s * stage_bytes, &tmap_x, full_bar(s), s * BK, m0);
            }
        }
        __syncwarp();
        int first, end, here = 0;
        a.requests.of_rows(m0, m1, lane, first, end);
        for (int s0 = first; s0 < end; s0 += 32) {
            const int s = s0 + lane, id = s < end ? a.requests.adapter_in(s, m0, m1) : -1;
            const uint32_t mine = __ballot_sync(0xffffffffu, id >= 0);
            const int at = here + __popc(mine & ((1u << lane) - 1u));
            if (id >= 0 && at < kDownMaxRequests) s_req[at] = make_int4(a.requests.begin(s), a.requests.begin(s + 1), id, 0);
            here += __popc(mine);
        }
        if (lane == 0) *s_count = min(here, kDownMaxRequests);
    }
    __syncthreads();
    const int requests = *s_count, per_pass = a.pass_cols / a.r, passes = (requests + per_pass - 1) / per_pass;  // per_pass requests side by side
    if (warp == 0) {
        // (the whole warp, one elected lane issues: see common.cuh)
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int p = 0; p < passes && ok; ++p) {
            const int req0 = p * per_pass, n = min(per_pass, requests - req0);
            const int row = s_req[req0 + min(lane, n - 1)].z * a.r;  // lane i: of request req0 + i (per_pass is 16 at most)
            for (int kb = 0; kb < num_kb; ++kb) {
                const uint32_t st = base + s * stage_bytes;
                if (p > 0 || kb >= ahead) {
                    if (__all_sync(0xffffffffu, mbar_wait(empty_bar(s), ph ^ 1u, s_abort, DEV_TIMEOUT_SMEM_EMPTY, s)) == 0) { ok = false; break; }
                    if (lane == 0) mbar_arrive_expect_tx(full_bar(s), S::kABytes);
                    __syncwarp();
                    tma_load_2d_warp(st, &tmap_x, full_bar(s), kb * BK, m0);
                }
                if (lane == 0) mbar_arrive_expect_tx(full_bar(s), (uint32_t)(n * a.r * BK * 2));
                __syncwarp();
                for (int i = 0; i < n; ++i)
                    tma_load_2d_warp(st + S::kABytes + (uint32_t)(i * a.r * BK * 2), &tmap_down, full_bar(s), kb * BK, __shfl_sync(0xffffffffu, row, i));
                if (++s == a.stages) { s = 0; ph ^= 1u; }
            }
        }
        if (passes == 0)  // nobody waits for what was sent ahead, but it must land before the CTA leaves
            for (int i = 0; i < ahead; ++i) {
                if (lane == 0) mbar_arrive(full_bar(i));
                __syncwarp();
                ok = ok && mbar_wait(full_bar(i), 0, s_abort, DEV_TIMEOUT_TMA_FULL, i);
            }
        if (!ok) __nanosleep(20000);
    } else if (warp == 1) {
        constexpr uint64_t desc_hi = make_smem_desc_hi(16, 1024);
        auto all_ok = [&](bool mine) { return __all_sync(0xffffffffu, mine) != 0; };
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int p = 0; p < passes && ok; ++p) {
            const int n = min(per_pass, requests - p * per_pass), acc = p & 1;
            ok = all_ok(mbar_wait(tempty_bar(acc), (((uint32_t)p >> 1) & 1u) ^ 1u, s_abort, DEV_TIMEOUT_TMEM_EMPTY, acc));
            if (!ok) break;
            tc_fence_after();
            const uint32_t idesc = make_idesc_f16(BM, (n * a.r + 15) / 16 * 16, true, false, false);
            for (int kb = 0; kb < num_kb; ++kb) {
                if (!all_ok(mbar_wait(full_bar(s), ph, s_abort, DEV_TIMEOUT_TMA_FULL, s))) { ok = false; break; }
                tc_fence_after();
                const uint64_t adesc = smem_desc(base + s * stage_bytes, desc_hi);
                umma_kblock_commit_warp(tmem_base + (uint32_t)(acc * kDownCols), adesc, adesc + (uint64_t)(S::kABytes >> 4), idesc, kb != 0 ? 1u : 0u, empty_bar(s));
                if (++s == a.stages) { s = 0; ph ^= 1u; }
            }
            if (ok) umma_commit_warp(tfull_bar(acc));
        }
    } else {
        const int quad = warp & 3, row = m0 + quad * 32 + lane;
        uint32_t lifted = 0;
        for (int p = 0; p < passes; ++p) {
            const int req0 = p * per_pass, n = min(per_pass, requests - req0), acc = p & 1;
            const float scales = __ldcg(a.scale + s_req[req0 + min(lane, n - 1)].z);  // lane i: of request req0 + i (per_pass is 16 at most)
            if (!mbar_wait(tfull_bar(acc), ((uint32_t)p >> 1) & 1u, s_abort, DEV_TIMEOUT_TMEM_FULL, acc)) break;
            tc_fence_after();
            for (int i = 0; i < n; ++i) {
                const int4 req = s_req[req0 + i];
                const float scale = __shfl_sync(0xffffffffu, scales, i);
                const bool mine = row >= req.x && row < req.y;
                uint4* dst = reinterpret_cast<uint4*>(a.h + (int64_t)row * a.r);
                const uint32_t src = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * kDownCols + i * a.r);
                // once, and a second time for rows with a value beyond fp16, times 2^-15
                bool on = mine;
                float f = scale;
#pragma unroll 1
                for (int once = 0; once < 2; ++once) {
                    __half2 most = __float2half2_rn(0.f);
                    for (int c = 0; c < a.r; c += 8) {
                        uint32_t v[8];
                        tmem_ld8(src + (uint32_t)c, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            v[j] = pack_h2(__uint_as_float(v[2 * j]) * f, __uint_as_float(v[2 * j + 1]) * f);
                            most = __hmax2(most, __habs2(*reinterpret_cast<const __half2*>(&v[j])));
                        }
                        if (on) dst[c >> 3] = make_uint4(v[0], v[1], v[2], v[3]);
                    }
                    on = on && __hisinf(__hmax(__low2half(most), __high2half(most)));
                    const uint32_t beyond = __ballot_sync(0xffffffffu, on);
                    if (beyond == 0u || once == 1) break;
                    lifted |= beyond;
                    f = scale * 0x1p-15f;
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty_bar(acc));
        }
        if (lane == 0) {
            a.lifted[(m0 >> 5) + quad] = lifted;
            if (blockIdx.x + 1 == gridDim.x && (blockIdx.x & 1u) == 0u) a.lifted[(m0 >> 5) + 4 + quad] = 0;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc<2 * kDownCols>(tmem_base);
    }
}

// The rows form's adapters: delta[m, n] = scale (x[m] A_a^T) B_a^T in fp32, which the linear kernel's epilogue adds. One CTA per row and
// `cols` of its columns (a few CTAs share a row where there are few rows): the r products in turn by its warps, then a column per thread.
__global__ void __launch_bounds__(256) adapter_rows_kernel(const AdapterArgs a) {
    __shared__ __align__(16) float s_h[128];
    grid_dependency_wait();
    grid_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int m = (int)blockIdx.x, n0 = (int)blockIdx.y * a.cols, n1 = min(n0 + a.cols, a.N);
    const int s = a.requests.at_row(m, lane);
    const int id = s < a.requests.S && a.requests.begin(s) <= m ? a.requests.adapter(s) : -1;
    float* delta = a.delta + (int64_t)m * a.N;
    if (id < 0) {
        for (int n = n0 + threadIdx.x; n < n1; n += 256) delta[n] = 0.f;
        return;
    }
    const uint4* x = reinterpret_cast<const uint4*>(a.x + (int64_t)m * a.ldx);
    const int vecs = a.K >> 3;
    const float scale = __ldcg(a.scale + id);
    // two products at a time: their loads wait for memory together
    for (int n = 2 * warp; n < a.r; n += 16) {
        const uint4* d = reinterpret_cast<const uint4*>(a.down + ((int64_t)id * a.r + n) * a.K);
        float2 acc0 = make_float2(0.f, 0.f), acc1 = acc0;
#pragma unroll 4
        for (int v = lane; v < vecs; v += 32) {
            const uint4 xv = x[v], d0 = __ldg(d + v), d1 = __ldg(d + vecs + v);
            const __half2 *xh = reinterpret_cast<const __half2*>(&xv), *h0 = reinterpret_cast<const __half2*>(&d0), *h1 = reinterpret_cast<const __half2*>(&d1);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 xf = __half22float2(xh[e]);
                acc0 = ffma2(xf, __half22float2(h0[e]), acc0);
                acc1 = ffma2(xf, __half22float2(h1[e]), acc1);
            }
        }
        float sum0 = acc0.x + acc0.y, sum1 = acc1.x + acc1.y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            sum0 += __shfl_xor_sync(0xffffffffu, sum0, o);
            sum1 += __shfl_xor_sync(0xffffffffu, sum1, o);
        }
        if (lane == 0) s_h[n] = sum0 * scale, s_h[n + 1] = sum1 * scale;
    }
    __syncthreads();
    for (int n = n0 + threadIdx.x; n < n1; n += 256) {
        const uint4* u = reinterpret_cast<const uint4*>(a.up + ((int64_t)id * a.N + n) * a.r);
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll 2
        for (int v = 0; v < (a.r >> 3); ++v) {
            const uint4 uv = __ldg(u + v);
            const __half2* uh = reinterpret_cast<const __half2*>(&uv);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = ffma2(*reinterpret_cast<const float2*>(s_h + 8 * v + 2 * e), __half22float2(uh[e]), acc);
        }
        delta[n] = acc.x + acc.y;
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
    // What the forms add to the layer itself, us, fitted to measurements on B200 (rows / blocks, K = N = 1024, rank 16): 512 rows of 64
    // requests 8.2 / 19, of 32 8.2 / 10, of 16 8.0 / 6.7; 2000 of 1000 19 / 82; K = 768, N = 2304: 1200 of 150 22 / 21, of 75 22 / 11. Rows: both
    // matrices of every row's adapter are read once per row. Blocks: a product with either matrix per request and row tile. Beyond 2^26
    // outputs the rows form's workspace would pass 256 MB: blocks, also where single rows make them slow.
    const double rows_us = 4.3 + (double)M * r * ((double)K + N) * 2.0 / 6e6, per_tile = 1.0 + 128.0 * S / (double)M;
    f.rows = M * (int64_t)N <= (1 << 26) && rows_us < 3.2 + per_tile * (0.4 + 0.03 * r);
    const int pairs = gemm_pairs_enabled() ? (swiglu ? max_pairs<256, true>() : max_pairs<256, false>()) : 0;
    f.pairs = !f.rows && pairs > 0 && tiles(2 * BM, 256) > pairs / 2;
    f.bn = f.pairs ? 256 : (!swiglu && tiles(BM, 128) <= sms / 2 ? 64 : 128);
    if (const char* e = getenv("FBB_ADAPTER_FORM")) {  // r | s64 | s128 | p256: tuning and test aid
        f.rows = e[0] == 'r';
        f.pairs = e[0] == 'p' && pairs > 0;
        f.bn = f.pairs ? 256 : (e[0] == 's' && e[1] == '6' && !swiglu ? 64 : 128);
    }
    return f;
}

// Workspace: h and the bits of lifted rows, or the rows form's delta.
static int64_t adapter_space(const AdapterForm& f, int64_t M, int N, int r) { return f.rows ? M * N * (int64_t)sizeof(float) : M * r * 2 + (M + 255) / 256 * 32; }

int64_t adapter_linear_workspace_bytes(int64_t M, int N, int K, int epilogue, int r, int S) {
    if (M <= 0 || S <= 0) return 0;
    return adapter_space(adapter_form(M, N, K, epilogue == FBB_EPI_SWIGLU, r, S), M, N, r);
}

template <int BN, bool SWIGLU, bool CTA2, AdaptMode ADAPT>
static int launch_adapter_variant(const CUtensorMap& ta, const CUtensorMap& tw, const CUtensorMap& th, const CUtensorMap& tu, const CUtensorMap& tc, GemmArgs g,
                                  const AdaptArgs& ad, cudaStream_t stream) {
    using S = GemmSmem<BN, CTA2>;
    constexpr int kDynamic = S::kDynamic + 12 * S::kStages;  // and three numbers per stage
    auto kern = linear_adapter_kernel<BN, SWIGLU, CTA2, ADAPT>;
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kDynamic);
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
    const cudaError_t e = launch_pdl_cluster(kern, dim3((unsigned)(CTA2 ? 2 * workers : workers)), dim3(kGemmThreads), kDynamic, stream, CTA2 ? 2u : 1u, ta, tw, th,
                                             tu, tc, g, ad);
    if (e != cudaSuccess) return fail((int)e, "linear_adapter_kernel launch: %s", cudaGetErrorString(e));
    return FBB_OK;
}

int launch_adapter_linear(const void* A, const void* W, void* C, const void* bias, const void* res, const void* gamma, int64_t M, int N, int K, int64_t lda,
                          int64_t ldw, int64_t ldc, int64_t ldr, int epilogue, const void* down, const void* up, const float* scale, int L, int r, const int* ids,
                          const int* offsets, int S, void* ws, int64_t ws_bytes, cudaStream_t stream) {
    const bool swiglu = epilogue == FBB_EPI_SWIGLU;
    const AdapterForm f = adapter_form(M, N, K, swiglu, r, S);
    const int64_t need = adapter_space(f, M, N, r);
    if (ws == nullptr || ws_bytes < need)
        return fail(FBB_ERR_SHAPE, "adapter_linear: workspace of %lld bytes, %lld needed", (long long)(ws != nullptr ? ws_bytes : 0), (long long)need);

    AdapterArgs d = {};
    d.requests.ids = ids, d.requests.offsets = offsets;
    d.requests.S = S, d.requests.each = offsets != nullptr ? 0 : (int)(M / S), d.requests.M = (int)M, d.requests.L = L;
    d.scale = scale;
    d.M = (int)M, d.N = N, d.K = K, d.r = r;
    d.h = reinterpret_cast<__half*>(ws);
    d.lifted = reinterpret_cast<uint32_t*>(d.h + M * r);  // (r is a multiple of 8)
    d.x = reinterpret_cast<const __half*>(A);
    d.ldx = lda;
    d.down = reinterpret_cast<const __half*>(down);
    d.up = reinterpret_cast<const __half*>(up);
    d.delta = reinterpret_cast<float*>(ws);
    // Columns of h in a pass: room for several requests where a tile has more than a couple. One CTA with all of shared memory where that
    // gives every tile an SM, else two on each.
    const int down_tiles = (int)((M + BM - 1) / BM);
    d.pass_cols = M < 64 * (int64_t)S || r > 64 ? kDownCols : 64;
    const int room = (down_tiles <= num_sms() ? DownSmem::kMaxDynamic : DownSmem::kMaxDynamic / 2 - 1024) - 1024 - DownSmem::kTailBytes;
    d.stages = room / DownSmem::stage_bytes(d.pass_cols);
    if (d.stages > kDownMaxStages) d.stages = kDownMaxStages;

    // boxes: 128 rows of A and h, 64 columns of h in the first launch; of W and the adapters' second matrices the rows that one CTA loads
    // per k-block
    const uint32_t w_rows = swiglu || f.pairs ? (uint32_t)f.bn / 2 : (uint32_t)f.bn;
    CUtensorMap ta, tw, th, tu, td, tc;
    struct { CUtensorMap* map; const void* p; uint64_t cols, rows; int64_t stride; uint32_t box0, box1; CUtensorMapSwizzle swizzle; } maps[6] = {
        {&ta, A, (uint64_t)K, (uint64_t)M, lda, BK, BM, CU_TENSOR_MAP_SWIZZLE_128B},
        {&tw, W, (uint64_t)K, (uint64_t)N, ldw, BK, w_rows, CU_TENSOR_MAP_SWIZZLE_128B},
        {&tc, C, (uint64_t)(swiglu ? N / 2 : N), (uint64_t)M, ldc, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B},
        {&th, ws, (uint64_t)r, (uint64_t)M, r, BK, BM, CU_TENSOR_MAP_SWIZZLE_128B},
        {&tu, up, (uint64_t)r, (uint64_t)L * (uint64_t)N, r, BK, w_rows, CU_TENSOR_MAP_SWIZZLE_128B},
        {&td, down, (uint64_t)K, (uint64_t)L * (uint64_t)r, K, BK, (uint32_t)r, CU_TENSOR_MAP_SWIZZLE_128B}};
    for (int i = 0; i < (f.rows ? 3 : 6); ++i) {
        const uint64_t dims[2] = {maps[i].cols, maps[i].rows};
        const int64_t st[2] = {1, maps[i].stride};
        const uint32_t box[2] = {maps[i].box0, maps[i].box1};
        const int rc = make_tmap_f16(maps[i].map, maps[i].p, 2, dims, st, box, maps[i].swizzle);
        if (rc != FBB_OK) return rc;
    }
    cudaError_t e;
    if (f.rows) {
        // enough CTAs to give every SM one, none with fewer columns than threads
        int64_t parts = (num_sms() + M - 1) / M;
        parts = parts > (N + 255) / 256 ? (N + 255) / 256 : parts;
        d.cols = (int)((N + parts - 1) / parts);
        th = tu = ta;
        e = launch_pdl(adapter_rows_kernel, dim3((unsigned)M, (unsigned)parts), dim3(256), 0, stream, d);
    } else {
        static bool configured[64] = {};
        int dev = 0;
        cudaGetDevice(&dev);
        if (dev < 0 || dev >= 64 || !configured[dev]) {
            e = cudaFuncSetAttribute(adapter_down_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, DownSmem::kMaxDynamic);
            if (e != cudaSuccess) return fail((int)e, "cudaFuncSetAttribute(adapter_down_kernel): %s", cudaGetErrorString(e));
            if (dev >= 0 && dev < 64) configured[dev] = true;
        }
        e = launch_pdl(adapter_down_kernel, dim3((unsigned)down_tiles), dim3(kDownThreads), (size_t)DownSmem::dynamic_bytes(d.pass_cols, d.stages), stream, ta, td, d);
    }
    if (e != cudaSuccess) return fail((int)e, "adapter kernel launch: %s", cudaGetErrorString(e));

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
    ad.requests = d.requests;
    ad.delta = d.delta;
    ad.lifted = d.lifted;
    ad.r_blocks = (r + BK - 1) / BK;

#define FBB_ADAPTER_LAUNCH(BN, SWIGLU, CTA2, MODE) launch_adapter_variant<BN, SWIGLU, CTA2, MODE>(ta, tw, th, tu, tc, g, ad, stream)
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
