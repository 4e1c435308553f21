// Differential attention: o = softmax(scale q1 k1') v - lam softmax(scale q2 k2') v, two maps of head dimension 64 over the same
// values of 128 columns, and the root-mean-square norm of every head's row behind it. No mask but a number of keys per batch entry.
//
// One CTA takes 128 queries of one (batch, head) and walks its keys in blocks of 128, both maps at once, so that v is read once and
// no map or half of an output ever leaves the chip (as four calls of the flash64 kernel, one per map and half of v, every score is
// computed twice and three passes over the outputs follow).
//   warp 0          TMA producer: the two Q tiles, then K1, K2 and V of each block into a ring of stages (128-byte swizzle)
//   warps 1, 2      UMMA issuers, one per map: S_t = Q_t K_t^T of half a block (64 keys) into one of two halves of the map's tensor memory;
//                   once the softmax warps have put P_t (fp16) over it, O_t += P_t V (A from tensor memory, V as the MN-major B
//                   operand, N = 128), then S_t of the half after the next in the same place. UMMAs of one thread execute in the
//                   order of their issue, so S_t may be overwritten right behind the P.V that reads P_t.
//   warp 3          the norm's weight into shared memory
//   warps 4..11/12..19 softmax of map 0 / 1, 16 query rows per warp in the fragment layout of flash64.cu, whose pieces they use: the
//                   running maximum is raised only where a half exceeds it by more than 2^8, P is at most 2^8 and as accurate
//                   in fp16 as relative to the maximum itself; sums and outputs are fp32
// Tensor memory is what decides the layout: O_1 and O_2 take 2 x 128 columns, S_1 and S_2 the other 256, so P lies over S. With one
// S of a whole block per map, its exponentials and its products took turns (3700 clocks per block and both maps); in halves, one half's
// P.V and the scores after it run under the other half's exponentials.
//
// Few queries over many keys (fewer tiles than SMs): the keys are split over `splits` CTAs, each of which leaves its unnormalised rows,
// maxima and sums in the workspace for diff64_join_kernel. Keys beyond a batch entry's number are masked by selection, never by
// adding, and their rows of V are zeroed in shared memory ahead of the product, so that no infinity or NaN in them is seen.
#include <type_traits>

#include "common.cuh"
#include "internal.h"

namespace fbb {

constexpr int kDiffStages = 3;
constexpr int kDiffPart = 16 * 128 + 16 * 2;  // floats of 16 rows of a share and map: the outputs, then {maximum, sum} of each row

struct DiffSmem {
    static constexpr int kQOff = 0;                       // Q_1 | Q_2
    static constexpr int kStageOff = 2 * kTileBytes;      // stages of K_1 | K_2 | V columns 0..63 | V columns 64..127
    static constexpr int kStageBytes = 4 * kTileBytes;
    static constexpr int kBarOff = kStageOff + kDiffStages * kStageBytes;
    // q_full, w_ready, k_full[2][S], k_empty[2][S], v_full[S], v_empty[S], then of each map and half s_full, p_ready, pv_done
    static constexpr int kNumBars = 2 + 6 * kDiffStages + 12;
    static constexpr int kWeightOff = kBarOff + kNumBars * 8 + 16;  // [128] fp32
    static constexpr int kBytes = kWeightOff + 128 * 4;
};
static_assert(DiffSmem::kBytes <= 232448, "more shared memory than a CTA can have");

struct DiffArgs {
    __half* o;
    int64_t o_sb, o_sn, o_sh;
    const float* lam;
    int64_t l_sb, l_sn, l_sh;
    const void* weight;      // [128] fp16 or fp32, null: no norm
    int weight_f32;
    float eps, out_scale, scale_log2;
    const int* lengths;      // keys of each batch entry, null: Nk
    int B, H, group;         // group = query heads per key head
    int Nq, Nk, q_tiles, splits;
    float* part;             // [tile][split][map][16-row group][kDiffPart], null when splits == 1
    int row_groups;          // of a tile that hold rows: min(8, ceil(Nq / 16))
};

// Keys of batch entry b, and the blocks of them that split `split` takes.
__device__ __forceinline__ int diff_keys(const DiffArgs& a, int b) { return a.lengths != nullptr ? min(max(__ldcg(a.lengths + b), 0), a.Nk) : a.Nk; }
__device__ __forceinline__ void diff_share(int keys, int split, int splits, int& kb0, int& kb1) {
    const int blocks = (int)(((unsigned)keys + FK - 1) / FK);
    kb0 = 0;
    kb1 = blocks;
    if (splits > 1) {  // (at most 2^24 blocks, kDiffMaxSplits splits)
        kb0 = (int)((unsigned)blocks * (unsigned)split / (unsigned)splits);
        kb1 = (int)((unsigned)blocks * (unsigned)(split + 1) / (unsigned)splits);
    }
}
__device__ __forceinline__ float diff_weight(const DiffArgs& a, int col) {
    return a.weight_f32 ? reinterpret_cast<const float*>(a.weight)[col] : __half2float(reinterpret_cast<const __half*>(a.weight)[col]);
}

// A from tensor memory (8 columns per K16 step), B MN-major (2048 bytes per step): the four steps of 64 keys, and a commit.
__device__ __forceinline__ void umma_ts4_commit_warp(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate, uint32_t bar) {
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        ".reg .b32 a1, a2, a3;\n\t"
        ".reg .b64 b1, b2, b3;\n\t"
        "add.u32 a1, %1, 8;\n\t"
        "add.s64 b1, %2, 128;\n\t"
        "add.u32 a2, %1, 16;\n\t"
        "add.s64 b2, %2, 256;\n\t"
        "add.u32 a3, %1, 24;\n\t"
        "add.s64 b3, %2, 384;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|q, 0xFFFFFFFF;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, 1;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, 1;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, 1;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t"
        "}\n"
        ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void st_shared_16(uint32_t addr, float x, float y, float z, float w) {
    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(x), "f"(y), "f"(z), "f"(w) : "memory");
}
__device__ __forceinline__ float4 ld_shared_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

constexpr int kDiffEarly = 2;  // key groups of eight exponentiated ahead of the vote on the running maximum (see kEarly in flash64.cu)

__global__ void __launch_bounds__(640, 1)
diff64_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
              const DiffArgs a) {
    using S = DiffSmem;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t base = smem_u32(smem_raw);
    const uint32_t bar0 = base + S::kBarOff;
    const uint32_t q_full = bar0, w_ready = bar0 + 8u;
    auto k_full = [&](int t, int s) { return bar0 + 8u * (2 + t * kDiffStages + s); };
    auto k_empty = [&](int t, int s) { return bar0 + 8u * (2 + (2 + t) * kDiffStages + s); };
    auto v_full = [&](int s) { return bar0 + 8u * (2 + 4 * kDiffStages + s); };
    auto v_empty = [&](int s) { return bar0 + 8u * (2 + 5 * kDiffStages + s); };
    auto s_full = [&](int t, int half) { return bar0 + 8u * (2 + 6 * kDiffStages + 2 * t + half); };
    auto p_ready = [&](int t, int half) { return bar0 + 8u * (2 + 6 * kDiffStages + 4 + 2 * t + half); };
    auto pv_done = [&](int t, int half) { return bar0 + 8u * (2 + 6 * kDiffStages + 8 + 2 * t + half); };
    volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(smem_raw + S::kBarOff + S::kNumBars * 8);
    volatile int* s_abort = reinterpret_cast<volatile int*>(smem_raw + S::kBarOff + S::kNumBars * 8 + 4);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kNumBars; ++i) {
            // v_empty: both maps' issuers; p_ready: the eight softmax warps of a map
            const int v0 = 2 + 5 * kDiffStages, p0 = 2 + 6 * kDiffStages + 4;
            mbar_init(bar0 + 8u * i, i >= v0 && i < v0 + kDiffStages ? 2 : (i >= p0 && i < p0 + 4 ? 8 : 1));
        }
        *s_abort = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmap_q);
        tma_prefetch_desc(&tmap_k);
        tma_prefetch_desc(&tmap_v);
    }
    if (warp == 1) {
        __syncwarp();
        tmem_alloc<512>(smem_u32(const_cast<uint32_t*>(s_tmem)));
        tmem_relinquish();
    }
    const unsigned tile = a.splits > 1 ? blockIdx.x / (unsigned)a.splits : blockIdx.x;
    const int split = (int)(blockIdx.x - tile * (unsigned)a.splits);
    const int bh = (int)(tile / (unsigned)a.q_tiles), q0 = (int)(tile - (unsigned)bh * (unsigned)a.q_tiles) * FQ;
    const int b = (int)((unsigned)bh / (unsigned)a.H), h = bh - b * a.H;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *s_tmem;
    grid_dependency_wait();
    grid_launch_dependents();

    const int keys = diff_keys(a, b);
    int kb0, kb1;
    diff_share(keys, split, a.splits, kb0, kb1);
    const int here = min(keys - kb0 * FK, (kb1 - kb0) * FK);  // keys of this share, the last ones' block may be ragged
    const int halves = (here + 63) / 64;                     // half-blocks that hold a key

    if (warp == 0) {
        if (lane == 0 && halves > 0) {
            const int hk = a.group > 1 ? (int)((unsigned)h / (unsigned)a.group) : h;
            mbar_arrive_expect_tx(q_full, 2 * kTileBytes);
            for (int t = 0; t < 2; ++t) tma_load_4d(base + S::kQOff + t * kTileBytes, &tmap_q, q_full, 0, 2 * h + t, q0, b);
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
#pragma unroll 1
            for (int kb = kb0; kb < kb1 && ok; ++kb) {
                const uint32_t st = base + S::kStageOff + s * S::kStageBytes;
#pragma unroll 1
                for (int t = 0; t < 2; ++t) {
                    ok = ok && mbar_wait(k_empty(t, s), ph ^ 1u, s_abort, DEV_TIMEOUT_SMEM_EMPTY, 2 * s + t);
                    if (!ok) break;
                    mbar_arrive_expect_tx(k_full(t, s), kTileBytes);
                    tma_load_4d(st + t * kTileBytes, &tmap_k, k_full(t, s), 0, 2 * hk + t, kb * FK, b);
                }
                ok = ok && mbar_wait(v_empty(s), ph ^ 1u, s_abort, DEV_TIMEOUT_SMEM_EMPTY, 16 + s);
                if (!ok) break;
                mbar_arrive_expect_tx(v_full(s), 2 * kTileBytes);
                for (int t = 0; t < 2; ++t) tma_load_4d(st + (2 + t) * kTileBytes, &tmap_v, v_full(s), 64 * t, hk, kb * FK, b);
                if (++s == kDiffStages) { s = 0; ph ^= 1u; }
            }
            if (!ok) __nanosleep(20000);
        }
    } else if (warp < 3) {
        const int t = warp - 1;
        const uint32_t idesc_qk = make_idesc_f16(FQ, 64, true, false, false);
        const uint32_t idesc_pv = make_idesc_f16(FQ, 128, true, false, true);
        const uint64_t qd = smem_desc(base + S::kQOff + t * kTileBytes, make_smem_desc_hi(16, 1024));
        const uint64_t kd0 = smem_desc(base + S::kStageOff + t * kTileBytes, make_smem_desc_hi(16, 1024));
        const uint64_t vd0 = smem_desc(base + S::kStageOff + 2 * kTileBytes, make_smem_desc_hi(kTileBytes, 1024));  // column halves a tile apart
        const uint32_t dS = tmem_base + t * 128, dO = tmem_base + 256 + t * 128;
        auto all_ok = [&](bool mine) { return __all_sync(0xffffffffu, mine) != 0; };
        // unit g: half g & 1 of block g / 2; 64 keys are 8 KB further in a tile of K or V
        int ks = 0, vs = 0;  // stages of the next unit's K and V
        uint32_t kph = 0, vph = 0;
        auto scores = [&](int g) -> bool {
            const int half = g & 1;
            if (half == 0 && !all_ok(mbar_wait(k_full(t, ks), kph, s_abort, DEV_TIMEOUT_TMA_FULL, 2 * ks + t))) return false;
            tc_fence_after();
            const uint64_t kd = kd0 + (uint64_t)((ks * S::kStageBytes + half * (kTileBytes / 2)) >> 4);
            umma_kblock_commit_warp(dS + 64u * half, qd, kd, idesc_qk, 0u, s_full(t, half));
            if (half == 1) {
                umma_commit_warp(k_empty(t, ks));
                if (++ks == kDiffStages) { ks = 0; kph ^= 1u; }
            }
            return true;
        };
        bool ok = halves > 0 && all_ok(mbar_wait(q_full, 0, s_abort, DEV_TIMEOUT_TMA_FULL, 100));
        ok = ok && scores(0);
        if (ok && halves > 1) ok = scores(1);
#pragma unroll 1
        for (int g = 0; g < halves && ok; ++g) {
            const int half = g & 1;
            if (half == 0 && !all_ok(mbar_wait(v_full(vs), vph, s_abort, DEV_TIMEOUT_TMA_FULL, 16 + vs))) break;
            const uint32_t vt = S::kStageOff + vs * S::kStageBytes + 2 * kTileBytes + half * (kTileBytes / 2);
            if (g + 1 == halves && here < 64 * halves && kb0 * FK + here < a.Nk) {
                // rows of V beyond the entry's keys hold whatever the tensor holds there (beyond the tensor the copy wrote zeros); both
                // issuers write the same zeros
                for (int i = (here - 64 * g) * 8 + lane; i < 64 * 8; i += 32)
                    for (int c = 0; c < 2; ++c) st_shared_16(base + vt + c * kTileBytes + 16u * i, 0.f, 0.f, 0.f, 0.f);
                fence_proxy_async_smem();
                __syncwarp();
            }
            if (!all_ok(mbar_wait(p_ready(t, half), (g >> 1) & 1u, s_abort, DEV_TIMEOUT_OTHER, 200 + 2 * t + half))) break;
            tc_fence_after();
            umma_ts4_commit_warp(dO, dS + 64u * half, vd0 + (uint64_t)((vt - S::kStageOff - 2 * kTileBytes) >> 4), idesc_pv, g > 0 ? 1u : 0u, pv_done(t, half));
            if (half == 1) {
                umma_commit_warp(v_empty(vs));
                if (++vs == kDiffStages) { vs = 0; vph ^= 1u; }
            }
            if (g + 2 < halves) ok = scores(g + 2);
        }
    } else if (warp == 3) {
        if (a.weight != nullptr) {
            float* s_w = reinterpret_cast<float*>(smem_raw + S::kWeightOff);
#pragma unroll
            for (int i = 0; i < 4; ++i) s_w[lane + 32 * i] = diff_weight(a, lane + 32 * i) * a.out_scale;
            __syncwarp();
            if (lane == 0) mbar_arrive(w_ready);
        }
    } else {
        const int u = (warp - 4) & 7;
        const int t = (warp - 4) >> 3;
        const int lane_base = (u & 3) * 32 + (u >> 2) * 16;
        const int cq = lane & 3;
        const uint32_t tS = tmem_base + ((uint32_t)lane_base << 16) + t * 128;
        const uint32_t tO = tmem_base + ((uint32_t)lane_base << 16) + 256 + t * 128;
        const float sl = a.scale_log2;
        const float lazy = kLazyMax / sl;
        const int rowA = q0 + lane_base + (lane >> 2), rowB = rowA + 8;
        if (q0 + lane_base >= a.Nq) {
            // a warp of rows beyond Nq only keeps the barriers moving: S_t of unit g exists only after the issuer has taken P_t of unit g - 2
#pragma unroll 1
            for (int g = 0; g < halves; ++g) {
                if (!mbar_wait(s_full(t, g & 1), (g >> 1) & 1u, s_abort, DEV_TIMEOUT_TMEM_FULL, 2 * t + (g & 1))) break;
                tc_fence_after();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready(t, g & 1));
            }
        } else {
            float fA = 1.f, fB = 1.f;  // factors of the map's rows in the result
            if (t == 1 && a.splits == 1) {
                fA = rowA < a.Nq ? a.lam[b * a.l_sb + rowA * a.l_sn + h * a.l_sh] : 0.f;
                fB = rowB < a.Nq ? a.lam[b * a.l_sb + rowB * a.l_sn + h * a.l_sh] : 0.f;
            }
            float tA = 0.f, tB = 0.f;
            float mA = -INFINITY, mB = -INFINITY, lA = 0.f, lB = 0.f;
            bool ok = true;
            // one half-block; `last`: the one that may have keys beyond the entry's
            auto unit = [&](int g, auto last) -> bool {
                const int half = g & 1;
                const uint32_t tSh = tS + 64u * half;
                if (!mbar_wait(s_full(t, half), (g >> 1) & 1u, s_abort, DEV_TIMEOUT_TMEM_FULL, 2 * t + half)) return false;
                tc_fence_after();
                uint32_t sc[32], pk[16];
                float mxA, mxB;
                tmem_ld_16x256b_x8(tSh, sc);
                tmem_wait_ld();
                tmem_tie32(sc);
                if constexpr (decltype(last)::value) mask_frag(sc, 64 * g + 2 * cq, here);
                max_frag<8>(sc, mxA, mxB);
                float2 accA = make_float2(0.f, 0.f), accB = make_float2(0.f, 0.f);
                exp_frag<kDiffEarly>(sc, sl, mA, mB, accA, accB, pk);
                if (g == 0 || __any_sync(0xffffffffu, mxA > tA || mxB > tB)) {
                    mxA = fmaxf(mxA, __shfl_xor_sync(0xffffffffu, mxA, 1));
                    mxB = fmaxf(mxB, __shfl_xor_sync(0xffffffffu, mxB, 1));
                    mxA = fmaxf(mxA, __shfl_xor_sync(0xffffffffu, mxA, 2));
                    mxB = fmaxf(mxB, __shfl_xor_sync(0xffffffffu, mxB, 2));
                    const float nA = fmaxf(mA, mxA * sl), nB = fmaxf(mB, mxB * sl);
                    if (g > 0) {
                        // the unit before this one may still be adding to O_t
                        if (!mbar_wait(pv_done(t, half ^ 1), ((g - 1) >> 1) & 1u, s_abort, DEV_TIMEOUT_TMEM_FULL, 8 + 2 * t + half)) return false;
                        tc_fence_after();
                        const float cA = ex2_approx(mA - nA), cB = ex2_approx(mB - nB);
#pragma unroll 1
                        for (int c = 0; c < 8; ++c) {
                            uint32_t o[8];
                            tmem_ld_16x256b_x2(tO + 16u * c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                o[4 * k] = __float_as_uint(__uint_as_float(o[4 * k]) * cA);
                                o[4 * k + 1] = __float_as_uint(__uint_as_float(o[4 * k + 1]) * cA);
                                o[4 * k + 2] = __float_as_uint(__uint_as_float(o[4 * k + 2]) * cB);
                                o[4 * k + 3] = __float_as_uint(__uint_as_float(o[4 * k + 3]) * cB);
                            }
                            tmem_st_16x256b_x2(tO + 16u * c, o);
                        }
                        lA *= cA;
                        lB *= cB;
                    }
                    mA = nA;
                    mB = nB;
                    tA = g == 0 ? mxA + lazy : fmaxf(tA, mxA + lazy);
                    tB = g == 0 ? mxB + lazy : fmaxf(tB, mxB + lazy);
                    accA = accB = make_float2(0.f, 0.f);
                    exp_frag<kDiffEarly>(sc, sl, mA, mB, accA, accB, pk);
                }
                exp_frag<8 - kDiffEarly>(sc + 4 * kDiffEarly, sl, mA, mB, accA, accB, pk + 2 * kDiffEarly);
                tmem_st_16x128b_x8(tSh, pk);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready(t, half));
                lA += accA.x + accA.y;
                lB += accB.x + accB.y;
                return true;
            };
            const int plain = here / 64;  // halves full of keys
#pragma unroll 1
            for (int g = 0; g < plain && ok; ++g) ok = unit(g, std::false_type());
            if (ok && plain < halves) ok = unit(plain, std::true_type());
            if (ok && halves > 0) {
                const int g = halves - 1;
                ok = mbar_wait(pv_done(t, g & 1), (g >> 1) & 1u, s_abort, DEV_TIMEOUT_TMEM_FULL, 12 + t);
            }
            tc_fence_after();
            // a row's sum is spread over the four threads that share it
            lA += __shfl_xor_sync(0xffffffffu, lA, 1);
            lB += __shfl_xor_sync(0xffffffffu, lB, 1);
            lA += __shfl_xor_sync(0xffffffffu, lA, 2);
            lB += __shfl_xor_sync(0xffffffffu, lB, 2);
            // What follows runs once: rolled loops over 16 columns at a time, because instructions that run once cost their fetch.
            if (a.splits > 1) {
                // the rows of this share for diff64_join_kernel (which asks for no share without keys)
                if (halves > 0) {
                    float* dst = a.part + (((int64_t)blockIdx.x * 2 + t) * a.row_groups + (lane_base >> 4)) * kDiffPart;
                    float2* outA = reinterpret_cast<float2*>(dst + (lane >> 2) * 128 + 2 * cq);
#pragma unroll 1
                    for (int c = 0; c < 8; ++c) {
                        uint32_t o[8];
                        tmem_ld_16x256b_x2(tO + 16u * c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            outA[8 * c + 4 * i] = make_float2(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]));
                            outA[8 * c + 4 * i + 8 * 64] = make_float2(__uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));  // row B
                        }
                    }
                    float2* stat = reinterpret_cast<float2*>(dst + 16 * 128);
                    if (cq == 0) stat[lane >> 2] = make_float2(mA, lA);
                    if (cq == 1) stat[(lane >> 2) + 8] = make_float2(mB, lB);
                }
            } else {
                // Map 1's warps leave lam O_2 / l_2 in shared memory, where their twins of map 0, which hold the same elements of O_1, take it:
                // 16 values of every thread in Q_2 and in each stage's K_2, which only map 1's products read (they have completed).
                fA = halves > 0 ? fA / lA : 0.f;
                fB = halves > 0 ? fB / lB : 0.f;
                auto twin = [&](int c) {  // two 16-byte vectors, 4 KB apart, of columns 16 c ..
                    const int quarter = c >> 1;
                    return (quarter == 0 ? base + S::kQOff + kTileBytes : base + S::kStageOff + (quarter - 1) * S::kStageBytes + kTileBytes) +
                           (uint32_t)((c & 1) * 8192 + (u * 32 + lane) * 16);
                };
                float sA = 0.f, sB = 0.f;
                if (t == 0) named_bar_sync(1 + u, 64);
#pragma unroll 1
                for (int c = 0; c < 8; ++c) {
                    uint32_t r[8];
                    float o[8];
                    tmem_ld_16x256b_x2(tO + 16u * c, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = halves > 0 ? __uint_as_float(r[i]) * ((i & 2) ? fB : fA) : 0.f;
                    const uint32_t at = twin(c);
                    if (t == 0) {
                        const float4 x = ld_shared_f4(at), y = ld_shared_f4(at + 4096u);
                        o[0] -= x.x, o[1] -= x.y, o[2] -= x.z, o[3] -= x.w, o[4] -= y.x, o[5] -= y.y, o[6] -= y.z, o[7] -= y.w;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            if (i & 2) sB = fmaf(o[i], o[i], sB);
                            else sA = fmaf(o[i], o[i], sA);
                        }
                    }
                    st_shared_16(at, o[0], o[1], o[2], o[3]);
                    st_shared_16(at + 4096u, o[4], o[5], o[6], o[7]);
                }
                if (t == 1) named_bar_sync(1 + u, 64);
                if (t == 0) {
                    float rA = a.out_scale, rB = a.out_scale;
                    const bool norm = a.weight != nullptr;
                    if (norm) {
                        sA += __shfl_xor_sync(0xffffffffu, sA, 1);
                        sB += __shfl_xor_sync(0xffffffffu, sB, 1);
                        sA += __shfl_xor_sync(0xffffffffu, sA, 2);
                        sB += __shfl_xor_sync(0xffffffffu, sB, 2);
                        rA = rsqrtf(sA * (1.f / 128.f) + a.eps);  // (the weight in shared memory holds out_scale)
                        rB = rsqrtf(sB * (1.f / 128.f) + a.eps);
                        ok = mbar_wait(w_ready, 0, s_abort, DEV_TIMEOUT_OTHER, 220) && ok;
                    }
                    // The warp's 16 rows of 256 bytes go through 4 KB of shared memory that only map 0's products read (Q_1, the first
                    // stage's K_1), 16-byte units swizzled by the row, and leave by 16-byte stores, a row's by 16 lanes.
                    const uint32_t st = (u < 4 ? base + S::kQOff : base + S::kStageOff) + (uint32_t)(u & 3) * 4096u;
                    const uint32_t strow = (uint32_t)(lane & 15);
                    const float* s_w = reinterpret_cast<const float*>(smem_raw + S::kWeightOff) + 2 * cq;
#pragma unroll 1
                    for (int c = 0; c < 8; ++c) {
                        const float4 x = ld_shared_f4(twin(c)), y = ld_shared_f4(twin(c) + 4096u);
                        const float2 one = make_float2(1.f, 1.f);
                        const float2 w0 = norm ? *reinterpret_cast<const float2*>(s_w + 16 * c) : one, w1 = norm ? *reinterpret_cast<const float2*>(s_w + 16 * c + 8) : one;
                        const uint32_t unit = (uint32_t)(2 * c + (lane >> 4)) ^ (strow & 7u);
                        stmatrix_x4(st + strow * 256u + unit * 16u, pack_h2(x.x * rA * w0.x, x.y * rA * w0.y), pack_h2(x.z * rB * w0.x, x.w * rB * w0.y),
                                    pack_h2(y.x * rA * w1.x, y.y * rA * w1.y), pack_h2(y.z * rB * w1.x, y.w * rB * w1.y));
                    }
                    __syncwarp();
                    __half* dst = a.o + (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + 8 * (lane & 15);
#pragma unroll 2
                    for (int i = 0; i < 8; ++i) {
                        const int r = 2 * i + (lane >> 4), row = q0 + lane_base + r;
                        const uint4 v = ld_shared_16(st + (uint32_t)r * 256u + (uint32_t)(((lane & 15) ^ (r & 7)) * 16));
                        if (ok && row < a.Nq) *reinterpret_cast<uint4*>(dst + (int64_t)row * a.o_sn) = v;
                    }
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc<512>(tmem_base);
    }
}

// Joins the shares of a 16-row group's keys: a share's weight is 2^(its maximum - the row's) over the row's sum. A chain of latencies (the
// partial rows are a few hundred KB in L2): what does not depend on anything is loaded at once, every share's maxima and sums by one
// thread each and the first shares' outputs ahead of the weights. Thread = (map, row, eight columns); those of rows beyond Nq rest.
constexpr int kDiffMaxSplits = 160;
constexpr int kJoinBatch = 8;
__global__ void __launch_bounds__(512) diff64_join_kernel(const DiffArgs a) {
    __shared__ float2 s_stat[kDiffMaxSplits][2][16];  // [share][map][row]: {maximum, sum}, then {weight, -}
    __shared__ __align__(16) float s_o[16][128];      // map 1's rows
    const unsigned tile = blockIdx.x / (unsigned)a.row_groups, rg = blockIdx.x - tile * (unsigned)a.row_groups;
    const unsigned bh = tile / (unsigned)a.q_tiles;
    const int row0 = (int)(tile - bh * (unsigned)a.q_tiles) * FQ + (int)rg * 16;
    const int b = (int)(bh / (unsigned)a.H), h = (int)bh - b * a.H;
    const int t = threadIdx.x >> 8, r = (threadIdx.x >> 4) & 15, c = (threadIdx.x & 15) * 8, strand = threadIdx.x & 15;
    grid_dependency_wait();
    grid_launch_dependents();
    if (row0 >= a.Nq) return;
    const bool used = row0 + r < a.Nq;
    const int keys = diff_keys(a, b);
    const int step = 2 * a.row_groups * kDiffPart;  // floats from share to share, from map to map half of it
    const float* part = a.part + (int64_t)tile * a.splits * step + (int64_t)rg * kDiffPart;
    // the shares that hold keys: all of them, or as many as there are blocks
    const int blocks = (int)(((unsigned)keys + FK - 1) / FK), live = min(blocks, a.splits);
    auto share = [&](int j) { return blocks >= a.splits ? j : (int)(((unsigned)(j + 1) * (unsigned)a.splits + (unsigned)blocks - 1u) / (unsigned)blocks) - 1; };

    const float* src = part + t * (step / 2) + r * 128 + c;
    float4 x[kJoinBatch][2];
    auto load = [&](int j0) {
#pragma unroll
        for (int j = 0; j < kJoinBatch; ++j) {
            if (j0 + j >= live) break;
            const float4* at = reinterpret_cast<const float4*>(src + (int64_t)share(j0 + j) * step);
            x[j][0] = __ldcg(at);
            x[j][1] = __ldcg(at + 1);
        }
    };
    if (used) load(0);
    float lam = 1.f;
    if (t == 1 && used) lam = a.lam[b * a.l_sb + (row0 + r) * a.l_sn + h * a.l_sh];
    for (int i = threadIdx.x; i < live * 32; i += 512) {
        const int j = i >> 5, mr = i & 31;
        s_stat[j][mr >> 4][mr & 15] = __ldcg(reinterpret_cast<const float2*>(part + (int64_t)share(j) * step + (mr >> 4) * (step / 2) + 16 * 128) + (mr & 15));
    }
    __syncthreads();
    if (used) {  // (whole rows of 16 threads, whose shuffles stay among themselves)
        const unsigned mask = 0xffffu << (threadIdx.x & 16);
        float m = -INFINITY, l = 0.f;
        for (int j = strand; j < live; j += 16) m = fmaxf(m, s_stat[j][t][r].x);
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) m = fmaxf(m, __shfl_xor_sync(mask, m, d));
        for (int j = strand; j < live; j += 16) {
            const float w = ex2_approx(s_stat[j][t][r].x - m);
            l = fmaf(w, s_stat[j][t][r].y, l);
            s_stat[j][t][r].x = w;
        }
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) l += __shfl_xor_sync(mask, l, d);
        const float f = lam / l;
        __syncwarp(mask);
        float acc[8] = {};
        for (int j0 = 0; j0 < live; j0 += kJoinBatch) {
            if (j0 > 0) load(j0);
#pragma unroll
            for (int j = 0; j < kJoinBatch; ++j) {
                if (j0 + j >= live) break;
                const float w = s_stat[j0 + j][t][r].x;
                acc[0] = fmaf(x[j][0].x, w, acc[0]), acc[1] = fmaf(x[j][0].y, w, acc[1]), acc[2] = fmaf(x[j][0].z, w, acc[2]), acc[3] = fmaf(x[j][0].w, w, acc[3]);
                acc[4] = fmaf(x[j][1].x, w, acc[4]), acc[5] = fmaf(x[j][1].y, w, acc[5]), acc[6] = fmaf(x[j][1].z, w, acc[6]), acc[7] = fmaf(x[j][1].w, w, acc[7]);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = live > 0 ? acc[i] * f : 0.f;
        if (t == 1) {
            *reinterpret_cast<float4*>(&s_o[r][c]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
            *reinterpret_cast<float4*>(&s_o[r][c + 4]) = make_float4(acc[4], acc[5], acc[6], acc[7]);
        }
        x[0][0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
        x[0][1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
    }
    __syncthreads();
    if (t == 1 || !used) return;
    const float4 y0 = *reinterpret_cast<const float4*>(&s_o[r][c]), y1 = *reinterpret_cast<const float4*>(&s_o[r][c + 4]);
    float o[8] = {x[0][0].x - y0.x, x[0][0].y - y0.y, x[0][0].z - y0.z, x[0][0].w - y0.w, x[0][1].x - y1.x, x[0][1].y - y1.y, x[0][1].z - y1.z, x[0][1].w - y1.w};
    float scale = a.out_scale;
    if (a.weight != nullptr) {
        const unsigned mask = 0xffffu << (threadIdx.x & 16);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(o[i], o[i], sum);
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) sum += __shfl_xor_sync(mask, sum, d);
        scale *= rsqrtf(sum * (1.f / 128.f) + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] *= diff_weight(a, c + i);
    }
    *reinterpret_cast<uint4*>(a.o + b * a.o_sb + (int64_t)(row0 + r) * a.o_sn + h * a.o_sh + c) =
        make_uint4(pack_h2(o[0] * scale, o[1] * scale), pack_h2(o[2] * scale, o[3] * scale), pack_h2(o[4] * scale, o[5] * scale), pack_h2(o[6] * scale, o[7] * scale));
}

// Shares of the keys: as many as fill the SMs once, none of less than two blocks.
static int diff64_splits(int B, int Nq, int Nk, int H) {
    const int64_t tiles = (int64_t)B * H * ((Nq + FQ - 1) / FQ), blocks = (Nk + FK - 1) / FK;
    int64_t s = num_sms() / (tiles > 0 ? tiles : 1);
    s = s > blocks / 2 ? blocks / 2 : s;
    s = s > kDiffMaxSplits ? kDiffMaxSplits : s;
    return s < 1 ? 1 : (int)s;
}
static int diff64_row_groups(int Nq) { return Nq >= FQ ? FQ / 16 : (Nq + 15) / 16; }

int64_t diff64_workspace_bytes(int B, int Nq, int Nk, int H) {
    if (B <= 0 || Nq <= 0 || H <= 0) return 0;
    const int splits = diff64_splits(B, Nq, Nk, H);
    if (splits == 1) return 0;
    return (int64_t)B * H * ((Nq + FQ - 1) / FQ) * splits * 2 * diff64_row_groups(Nq) * kDiffPart * (int64_t)sizeof(float);
}
int diff64_launches(int B, int Nq, int Nk, int H) { return B > 0 && Nq > 0 && H > 0 ? (diff64_splits(B, Nq, Nk, H) > 1 ? 2 : 1) : 0; }

int launch_diff64(const void* q, const void* k, const void* v, void* o, int B, int Nq, int Nk, int H, int Hk, const int64_t* qs, const int64_t* ks,
                  const int64_t* vs, const int64_t* os, const float* lam, const int64_t* ls, const void* weight, int weight_dtype, float eps,
                  float out_scale, float scale, const int* lengths, void* ws, int64_t ws_bytes, cudaStream_t stream) {
    DiffArgs a = {};
    a.o = reinterpret_cast<__half*>(o);
    a.o_sb = os[0], a.o_sn = os[1], a.o_sh = os[2];
    a.lam = lam;
    a.l_sb = ls[0], a.l_sn = ls[1], a.l_sh = ls[2];
    a.weight = weight, a.weight_f32 = weight_dtype == FBB_DTYPE_F32;
    a.eps = eps, a.out_scale = out_scale, a.scale_log2 = scale * 1.4426950408889634f;
    a.lengths = lengths;
    a.B = B, a.H = H, a.group = H / Hk;
    a.Nq = Nq, a.Nk = Nk, a.q_tiles = (Nq + FQ - 1) / FQ;
    a.splits = diff64_splits(B, Nq, Nk, H);
    a.row_groups = diff64_row_groups(Nq);
    const int64_t need = diff64_workspace_bytes(B, Nq, Nk, H);
    if (need > 0 && (ws == nullptr || ws_bytes < need))
        return fail(FBB_ERR_SHAPE, "diff64: workspace of %lld bytes, %lld needed", (long long)(ws != nullptr ? ws_bytes : 0), (long long)need);
    a.part = need > 0 ? reinterpret_cast<float*>(ws) : nullptr;
    const int64_t ctas = (int64_t)B * H * a.q_tiles * a.splits;
    if (ctas > 0x7FFFFFFFll) return fail(FBB_ERR_SHAPE, "diff64: too many query tiles (%lld)", (long long)ctas);

    CUtensorMap tq, tk, tv;
    struct { CUtensorMap* map; const void* p; const int64_t* st; uint64_t cols, heads, rows; } t[3] = {
        {&tq, q, qs, 64, 2 * (uint64_t)H, (uint64_t)Nq}, {&tk, k, ks, 64, 2 * (uint64_t)Hk, (uint64_t)Nk}, {&tv, v, vs, 128, (uint64_t)Hk, (uint64_t)Nk}};
    for (auto& m : t) {
        if (m.rows == 0) m.p = q, m.rows = 1;  // no keys: nothing is loaded through this map
        // innermost first; a dimension of one element may carry any stride, it gets a valid one
        const uint64_t dims[4] = {m.cols, m.heads, m.rows, (uint64_t)B};
        const int64_t st[4] = {1, m.heads > 1 ? m.st[2] : 128, m.rows > 1 ? m.st[1] : 128, B > 1 ? m.st[0] : 128};
        const uint32_t box[4] = {64, 1, 128, 1};
        const int rc = make_tmap_f16(m.map, m.p, 4, dims, st, box);
        if (rc != FBB_OK) return rc;
    }
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(diff64_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, DiffSmem::kBytes);
        if (e != cudaSuccess) return fail((int)e, "cudaFuncSetAttribute(diff64_kernel): %s", cudaGetErrorString(e));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    cudaError_t e = launch_pdl(diff64_kernel, dim3((unsigned)ctas), dim3(640), DiffSmem::kBytes, stream, tq, tk, tv, a);
    if (e != cudaSuccess) return fail((int)e, "diff64_kernel launch: %s", cudaGetErrorString(e));
    if (a.splits > 1) {
        e = launch_pdl(diff64_join_kernel, dim3((unsigned)(B * (int64_t)H * a.q_tiles * a.row_groups)), dim3(512), 0, stream, a);
        if (e != cudaSuccess) return fail((int)e, "diff64_join_kernel launch: %s", cudaGetErrorString(e));
    }
    return FBB_OK;
}

}  // namespace fbb
