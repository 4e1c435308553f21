// Differential attention: o = softmax(scale q1 k1') v - lam softmax(scale q2 k2') v, two maps of head dimension 64 over the same
// values of 128 columns, and the root-mean-square norm of every head's row behind it. No mask but a number of keys per batch entry.
//
// One CTA takes 128 queries of one (batch, head) and walks its keys in blocks of 128, both maps at once, so that v is read once and
// no map or half of an output ever leaves the chip (as four calls of the flash64 kernel, one per map and half of v, every score is
// computed twice and three passes over the outputs follow).
//   warp 0          TMA producer: the two Q tiles, then K1, K2 and V of each block into a ring of stages (128-byte swizzle)
//   warps 1, 2      UMMA issuers, one per map: S_t = Q_t K_t^T into tensor memory; once the softmax warps have put P_t (fp16) over
//                   S_t, O_t += P_t V (A from tensor memory, V as the MN-major B operand, N = 128), then S_t of the next block.
//                   UMMAs of one thread execute in the order of their issue, so S_t may be overwritten right behind the P.V that
//                   reads P_t, and a commit behind S_t also tells that this P.V has completed.
//   warps 4..11/12..19 softmax of map 0 / 1, 16 query rows per warp in the fragment layout of flash64.cu, whose pieces they use: the
//                   running maximum is raised only where a block exceeds it by more than 2^8, P is at most 2^8 and as accurate
//                   in fp16 as relative to the maximum itself; sums and outputs are fp32
// Tensor memory is what decides the layout: O_1 and O_2 take 2 x 128 columns, S_1 and S_2 the other 256, so P lies over S and a map's
// next scores wait for its P.V. The other map's exponentials cover that: per block both maps need 2048 clocks of the transcendental
// unit and 1536 of the tensor core.
//
// Few queries over many keys (fewer tiles than SMs): the keys are split over `splits` CTAs, each of which leaves its unnormalised rows,
// maxima and sums in the workspace for diff64_join_kernel. Keys beyond a batch entry's number are masked by selection, never by
// adding, and their rows of V are zeroed in shared memory ahead of the product, so that no infinity or NaN in them is seen.
#include "common.cuh"
#include "internal.h"

namespace fbb {

constexpr int kDiffStages = 3;
constexpr int kDiffRowValues = 68;  // of a lane in a 16-row group of one map: 64 outputs, two maxima, two sums

struct DiffSmem {
    static constexpr int kQOff = 0;                       // Q_1 | Q_2
    static constexpr int kStageOff = 2 * kTileBytes;      // stages of K_1 | K_2 | V columns 0..63 | V columns 64..127
    static constexpr int kStageBytes = 4 * kTileBytes;
    static constexpr int kBarOff = kStageOff + kDiffStages * kStageBytes;
    // q_full, k_full[2][S], k_empty[2][S], v_full[S], v_empty[S], s_full[2], p_ready[2], pv_done[2]
    static constexpr int kNumBars = 1 + 6 * kDiffStages + 6;
    static constexpr int kBytes = kBarOff + kNumBars * 8 + 16;
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
    float* part;             // [tile][split][map][16-row group][kDiffRowValues][32], null when splits == 1
    int row_groups;          // of a tile that hold rows: min(8, ceil(Nq / 16))
};

// Keys of batch entry b, and the blocks of them that split `split` takes.
__device__ __forceinline__ int diff_keys(const DiffArgs& a, int b) { return a.lengths != nullptr ? min(max(__ldcg(a.lengths + b), 0), a.Nk) : a.Nk; }
__device__ __forceinline__ void diff_share(int keys, int split, int splits, int& kb0, int& kb1) {
    const int blocks = (keys + FK - 1) / FK;
    kb0 = (int)((int64_t)blocks * split / splits);
    kb1 = (int)((int64_t)blocks * (split + 1) / splits);
}
__device__ __forceinline__ float diff_weight(const DiffArgs& a, int col) {
    return a.weight_f32 ? reinterpret_cast<const float*>(a.weight)[col] : __half2float(reinterpret_cast<const __half*>(a.weight)[col]);
}

// A from tensor memory (8 columns per K16 step), B MN-major (2048 bytes per step): eight steps, one commit.
__device__ __forceinline__ void umma_ts8_commit_warp(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate, uint32_t bar) {
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        ".reg .b32 a1, a2, a3, a4, a5, a6, a7;\n\t"
        ".reg .b64 b1, b2, b3, b4, b5, b6, b7;\n\t"
        "add.u32 a1, %1, 8;\n\t"
        "add.s64 b1, %2, 128;\n\t"
        "add.u32 a2, %1, 16;\n\t"
        "add.s64 b2, %2, 256;\n\t"
        "add.u32 a3, %1, 24;\n\t"
        "add.s64 b3, %2, 384;\n\t"
        "add.u32 a4, %1, 32;\n\t"
        "add.s64 b4, %2, 512;\n\t"
        "add.u32 a5, %1, 40;\n\t"
        "add.s64 b5, %2, 640;\n\t"
        "add.u32 a6, %1, 48;\n\t"
        "add.s64 b6, %2, 768;\n\t"
        "add.u32 a7, %1, 56;\n\t"
        "add.s64 b7, %2, 896;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|q, 0xFFFFFFFF;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, 1;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, 1;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, 1;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a4], b4, %3, 1;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a5], b5, %3, 1;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a6], b6, %3, 1;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a7], b7, %3, 1;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%5];\n\t"
        "}\n"
        ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(bar)
        : "memory");
}

__global__ void __launch_bounds__(640, 1)
diff64_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
              const DiffArgs a) {
    using S = DiffSmem;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t base = smem_u32(smem_raw);
    const uint32_t bar0 = base + S::kBarOff;
    const uint32_t q_full = bar0;
    auto k_full = [&](int t, int s) { return bar0 + 8u * (1 + t * kDiffStages + s); };
    auto k_empty = [&](int t, int s) { return bar0 + 8u * (1 + (2 + t) * kDiffStages + s); };
    auto v_full = [&](int s) { return bar0 + 8u * (1 + 4 * kDiffStages + s); };
    auto v_empty = [&](int s) { return bar0 + 8u * (1 + 5 * kDiffStages + s); };
    auto s_full = [&](int t) { return bar0 + 8u * (1 + 6 * kDiffStages + t); };
    auto p_ready = [&](int t) { return bar0 + 8u * (1 + 6 * kDiffStages + 2 + t); };
    auto pv_done = [&](int t) { return bar0 + 8u * (1 + 6 * kDiffStages + 4 + t); };
    volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(smem_raw + S::kBarOff + S::kNumBars * 8);
    volatile int* s_abort = reinterpret_cast<volatile int*>(smem_raw + S::kBarOff + S::kNumBars * 8 + 4);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int s = 0; s < kDiffStages; ++s) {
            for (int t = 0; t < 2; ++t) {
                mbar_init(k_full(t, s), 1);
                mbar_init(k_empty(t, s), 1);
            }
            mbar_init(v_full(s), 1);
            mbar_init(v_empty(s), 2);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(s_full(t), 1);
            mbar_init(p_ready(t), 8);
            mbar_init(pv_done(t), 1);
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
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *s_tmem;
    grid_dependency_wait();
    grid_launch_dependents();

    const int tile = (int)blockIdx.x / a.splits, split = (int)blockIdx.x - tile * a.splits;
    const int bh = tile / a.q_tiles, q0 = (tile - bh * a.q_tiles) * FQ;
    const int b = bh / a.H, h = bh - b * a.H;
    const int keys = diff_keys(a, b);
    int kb0, kb1;
    diff_share(keys, split, a.splits, kb0, kb1);
    const int n_blocks = kb1 - kb0;
    const bool ragged = kb1 * FK > keys;  // the last block of this share has keys beyond the entry's

    if (warp < 4) {
        setmaxnreg_dec<kRegsCtl>();
        if (warp == 0) {
            if (lane == 0 && n_blocks > 0) {
                const int hk = h / a.group;
                mbar_arrive_expect_tx(q_full, 2 * kTileBytes);
                for (int t = 0; t < 2; ++t) tma_load_4d(base + S::kQOff + t * kTileBytes, &tmap_q, q_full, 0, 2 * h + t, q0, b);
                int s = 0;
                uint32_t ph = 0;
                bool ok = true;
#pragma unroll 1
                for (int kb = kb0; kb < kb1 && ok; ++kb) {
                    const uint32_t st = base + S::kStageOff + s * S::kStageBytes;
                    for (int t = 0; t < 2 && ok; ++t) {
                        ok = mbar_wait(k_empty(t, s), ph ^ 1u, s_abort, DEV_TIMEOUT_SMEM_EMPTY, 2 * s + t);
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
            const uint32_t idesc_qk = make_idesc_f16(FQ, FK, true, false, false);
            const uint32_t idesc_pv = make_idesc_f16(FQ, 128, true, false, true);
            const uint64_t qd = smem_desc(base + S::kQOff + t * kTileBytes, make_smem_desc_hi(16, 1024));
            const uint64_t kd0 = smem_desc(base + S::kStageOff + t * kTileBytes, make_smem_desc_hi(16, 1024));
            const uint64_t vd0 = smem_desc(base + S::kStageOff + 2 * kTileBytes, make_smem_desc_hi(kTileBytes, 1024));  // column halves a tile apart
            const uint32_t dS = tmem_base + t * 128, dO = tmem_base + 256 + t * 128;
            auto all_ok = [&](bool mine) { return __all_sync(0xffffffffu, mine) != 0; };
            bool ok = n_blocks > 0 && all_ok(mbar_wait(q_full, 0, s_abort, DEV_TIMEOUT_TMA_FULL, 100));
            if (ok) ok = all_ok(mbar_wait(k_full(t, 0), 0, s_abort, DEV_TIMEOUT_TMA_FULL, t));
            if (ok) {
                tc_fence_after();
                umma_kblock_commit2_warp(dS, qd, kd0, idesc_qk, s_full(t), k_empty(t, 0));
            }
            int s = 0;
            uint32_t ph = 0;
#pragma unroll 1
            for (int g = 0; g < n_blocks && ok; ++g) {
                const bool last = g + 1 == n_blocks;
                ok = all_ok(mbar_wait(v_full(s), ph, s_abort, DEV_TIMEOUT_TMA_FULL, 16 + s));
                if (!ok) break;
                if (last && ragged && keys < a.Nk) {
                    // rows of V beyond the entry's keys hold whatever the tensor holds there (beyond the tensor the copy wrote zeros); both
                    // issuers write the same zeros
                    const uint32_t vt = base + S::kStageOff + s * S::kStageBytes + 2 * kTileBytes;
                    for (int i = (keys - (kb1 - 1) * FK) * 8 + lane; i < FK * 8; i += 32)
                        for (int half = 0; half < 2; ++half)
                            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vt + half * kTileBytes + 16u * i), "r"(0) : "memory");
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                ok = all_ok(mbar_wait(p_ready(t), g & 1u, s_abort, DEV_TIMEOUT_OTHER, 200 + t));
                if (!ok) break;
                tc_fence_after();
                umma_ts8_commit_warp(dO, dS, vd0 + (uint64_t)(s * (S::kStageBytes >> 4)), idesc_pv, g > 0 ? 1u : 0u, v_empty(s));
                if (last) {
                    umma_commit_warp(pv_done(t));
                    break;
                }
                if (++s == kDiffStages) { s = 0; ph ^= 1u; }
                ok = all_ok(mbar_wait(k_full(t, s), ph, s_abort, DEV_TIMEOUT_TMA_FULL, 2 * s + t));
                if (!ok) break;
                tc_fence_after();
                umma_kblock_commit2_warp(dS, qd, kd0 + (uint64_t)(s * (S::kStageBytes >> 4)), idesc_qk, s_full(t), k_empty(t, s));
            }
        }
    } else {
        setmaxnreg_inc<kRegsSoftmax>();
        const int u = (warp - 4) & 7;
        const int t = (warp - 4) >> 3;
        const int lane_base = (u & 3) * 32 + (u >> 2) * 16;
        const int cq = lane & 3;
        const uint32_t tS = tmem_base + ((uint32_t)lane_base << 16) + t * 128;
        const uint32_t tO = tmem_base + ((uint32_t)lane_base << 16) + 256 + t * 128;
        const float sl = a.scale_log2;
        const float lazy = kLazyMax / sl;
        const bool has_rows = q0 + lane_base < a.Nq;
        const int rowA = q0 + lane_base + (lane >> 2), rowB = rowA + 8;
        const int key0 = (kb1 - 1) * FK + 2 * cq;  // of the last block
        float tA = 0.f, tB = 0.f;
        float mA = -INFINITY, mB = -INFINITY, lA = 0.f, lB = 0.f;
        bool ok = true;
        if (!has_rows) {
            // a warp of rows beyond Nq only keeps the barriers moving: S_t of unit g exists only after the issuer has taken unit g - 1's P_t
#pragma unroll 1
            for (int g = 0; g < n_blocks; ++g) {
                if (!mbar_wait(s_full(t), g & 1u, s_abort, DEV_TIMEOUT_TMEM_FULL, t)) break;
                tc_fence_after();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready(t));
            }
        } else {
#pragma unroll 1
            for (int g = 0; g < n_blocks; ++g) {
                if (!mbar_wait(s_full(t), g & 1u, s_abort, DEV_TIMEOUT_TMEM_FULL, t)) { ok = false; break; }
                tc_fence_after();
                const bool masked = ragged && g + 1 == n_blocks;
                uint32_t sc[64], pk[32];
                float mxA, mxB;
                tmem_ld_16x256b_x16(tS, sc);
                tmem_wait_ld();
                tmem_tie32(sc);
                tmem_tie32(sc + 32);
                if (masked) {
                    mask_frag(sc, key0, keys);
                    mask_frag(sc + 32, key0 + 64, keys);
                }
                max_frag<16>(sc, mxA, mxB);
                if (g == 0 || __any_sync(0xffffffffu, mxA > tA || mxB > tB)) {
                    mxA = fmaxf(mxA, __shfl_xor_sync(0xffffffffu, mxA, 1));
                    mxB = fmaxf(mxB, __shfl_xor_sync(0xffffffffu, mxB, 1));
                    mxA = fmaxf(mxA, __shfl_xor_sync(0xffffffffu, mxA, 2));
                    mxB = fmaxf(mxB, __shfl_xor_sync(0xffffffffu, mxB, 2));
                    const float nA = fmaxf(mA, mxA * sl), nB = fmaxf(mB, mxB * sl);
                    if (g > 0) {
                        // S_t is complete, and with it every P.V before it: O_t may be rescaled in place
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
                }
                float2 accA = make_float2(0.f, 0.f), accB = make_float2(0.f, 0.f);
                exp_frag<16>(sc, sl, mA, mB, accA, accB, pk);
                tmem_st_16x128b_x16(tS, pk);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready(t));
                lA += accA.x + accA.y;
                lB += accB.x + accB.y;
            }
            if (ok && n_blocks > 0) ok = mbar_wait(pv_done(t), 0, s_abort, DEV_TIMEOUT_TMEM_FULL, 8 + t);
            tc_fence_after();
            // a row's sum is spread over the four threads that share it
            lA += __shfl_xor_sync(0xffffffffu, lA, 1);
            lB += __shfl_xor_sync(0xffffffffu, lB, 1);
            lA += __shfl_xor_sync(0xffffffffu, lA, 2);
            lB += __shfl_xor_sync(0xffffffffu, lB, 2);
            if (a.splits > 1) {
                // the rows of this share for diff64_join_kernel (which asks for no share without keys)
                if (n_blocks > 0) {
                    float* dst = a.part + ((((int64_t)blockIdx.x * 2 + t) * a.row_groups + (lane_base >> 4)) * kDiffRowValues) * 32 + lane;
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
                        uint32_t o[32];
                        tmem_ld_16x256b_x8(tO + 64u * half, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) dst[(32 * half + i) * 32] = __uint_as_float(o[i]);
                    }
                    dst[64 * 32] = mA;
                    dst[65 * 32] = mB;
                    dst[66 * 32] = lA;
                    dst[67 * 32] = lB;
                }
            } else {
                // Map 1's warps leave lam O_2 / l_2 in shared memory, where their twins of map 0, which hold the same elements of O_1, take it:
                // 16 values of every thread in Q_2 and in each stage's K_2, which only map 1's products read (they have completed).
                const float fA = t == 0 ? 1.f / lA : (rowA < a.Nq ? a.lam[b * a.l_sb + rowA * a.l_sn + h * a.l_sh] / lA : 0.f);
                const float fB = t == 0 ? 1.f / lB : (rowB < a.Nq ? a.lam[b * a.l_sb + rowB * a.l_sn + h * a.l_sh] / lB : 0.f);
                auto twin = [&](int v) {
                    const int quarter = v >> 4;
                    return (quarter == 0 ? base + S::kQOff + kTileBytes : base + S::kStageOff + (quarter - 1) * S::kStageBytes + kTileBytes) +
                           (uint32_t)((v & 15) * 1024 + (u * 32 + lane) * 4);
                };
                uint32_t o[64];
                if (n_blocks > 0) {
                    tmem_ld_16x256b_x16(tO, o);
                    tmem_wait_ld();
                    tmem_tie32(o);
                    tmem_tie32(o + 32);
#pragma unroll
                    for (int i = 0; i < 64; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * ((i & 2) ? fB : fA));
                } else {
#pragma unroll
                    for (int i = 0; i < 64; ++i) o[i] = 0u;
                }
                if (t == 1) {
#pragma unroll
                    for (int i = 0; i < 64; ++i) asm volatile("st.shared.u32 [%0], %1;" ::"r"(twin(i)), "r"(o[i]) : "memory");
                }
                named_bar_sync(1 + u, 64);
                if (t == 0) {
                    float sA = 0.f, sB = 0.f;
#pragma unroll
                    for (int i = 0; i < 64; ++i) {
                        float x;
                        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(twin(i)) : "memory");
                        x = __uint_as_float(o[i]) - x;
                        o[i] = __float_as_uint(x);
                        if (i & 2) sB = fmaf(x, x, sB);
                        else sA = fmaf(x, x, sA);
                    }
                    float rA = a.out_scale, rB = a.out_scale;
                    if (a.weight != nullptr) {
                        sA += __shfl_xor_sync(0xffffffffu, sA, 1);
                        sB += __shfl_xor_sync(0xffffffffu, sB, 1);
                        sA += __shfl_xor_sync(0xffffffffu, sA, 2);
                        sB += __shfl_xor_sync(0xffffffffu, sB, 2);
                        rA *= rsqrtf(sA * (1.f / 128.f) + a.eps);
                        rB *= rsqrtf(sB * (1.f / 128.f) + a.eps);
                    }
                    // The warp's 16 rows of 256 bytes go through 4 KB of shared memory that only map 0's products read (Q_1, the first
                    // stage's K_1), 16-byte units swizzled by the row, and leave by 16-byte stores, a row's by 16 lanes.
                    const uint32_t st = (u < 4 ? base + S::kQOff : base + S::kStageOff) + (uint32_t)(u & 3) * 4096u;
                    const uint32_t strow = (uint32_t)(lane & 15);
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        float w[4] = {1.f, 1.f, 1.f, 1.f};
                        if (a.weight != nullptr) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) w[j] = diff_weight(a, 8 * (k + (j >> 1)) + 2 * cq + (j & 1));
                        }
                        const uint32_t unit = (uint32_t)(k + (lane >> 4)) ^ (strow & 7u);
                        stmatrix_x4(st + strow * 256u + unit * 16u,
                                    pack_h2(__uint_as_float(o[4 * k]) * rA * w[0], __uint_as_float(o[4 * k + 1]) * rA * w[1]),
                                    pack_h2(__uint_as_float(o[4 * k + 2]) * rB * w[0], __uint_as_float(o[4 * k + 3]) * rB * w[1]),
                                    pack_h2(__uint_as_float(o[4 * k + 4]) * rA * w[2], __uint_as_float(o[4 * k + 5]) * rA * w[3]),
                                    pack_h2(__uint_as_float(o[4 * k + 6]) * rB * w[2], __uint_as_float(o[4 * k + 7]) * rB * w[3]));
                    }
                    __syncwarp();
                    __half* dst = a.o + (int64_t)b * a.o_sb + (int64_t)h * a.o_sh + 8 * (lane & 15);
#pragma unroll
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

// Joins the shares of a 16-row group's keys. Eight warps: four quarters of the 64 values of each map; a share's weight is
// 2^(its maximum - the row's). Then 16 threads per row take the difference, the norm and the store.
constexpr int kDiffMaxSplits = 160;
__global__ void __launch_bounds__(256) diff64_join_kernel(const DiffArgs a) {
    __shared__ float s_weight[kDiffMaxSplits][2][16];  // [share][map][row], then divided by the row's sum (and times lam)
    __shared__ __align__(16) float s_o[2][16][132];    // [map][row][column]; rows 4 banks apart
    grid_dependency_wait();
    grid_launch_dependents();
    const int tile = (int)blockIdx.x / a.row_groups, rg = (int)blockIdx.x - tile * a.row_groups;
    const int bh = tile / a.q_tiles, row0 = (tile - bh * a.q_tiles) * FQ + rg * 16;
    const int b = bh / a.H, h = bh - b * a.H;
    if (row0 >= a.Nq) return;
    const int keys = diff_keys(a, b);
    const int64_t step = (int64_t)2 * a.row_groups * kDiffRowValues * 32;  // floats from share to share
    const float* part = a.part + (int64_t)tile * a.splits * step + (int64_t)rg * kDiffRowValues * 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto empty = [&](int s) {
        int kb0, kb1;
        diff_share(keys, s, a.splits, kb0, kb1);
        return kb0 == kb1;
    };
    // weights: thread = (map, row, one of 8 strands of the shares)
    {
        const int pair = threadIdx.x >> 3, strand = threadIdx.x & 7, t = pair >> 4, r = pair & 15;
        const float* stat = part + ((int64_t)t * a.row_groups * kDiffRowValues + 64 + (r >> 3)) * 32 + (r & 7) * 4;  // the row's maximum; its sum 64 floats on
        float m = -INFINITY;
        for (int s = strand; s < a.splits; s += 8)
            if (!empty(s)) m = fmaxf(m, __ldcg(stat + s * step));
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        float l = 0.f;
        for (int s = strand; s < a.splits; s += 8) {
            float w = 0.f;
            if (!empty(s)) {
                w = ex2_approx(__ldcg(stat + s * step) - m);
                l = fmaf(w, __ldcg(stat + s * step + 64), l);
            }
            s_weight[s][t][r] = w;
        }
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        float f = keys > 0 ? 1.f / l : 0.f;
        if (t == 1) f *= row0 + r < a.Nq ? a.lam[b * a.l_sb + (row0 + r) * a.l_sn + h * a.l_sh] : 0.f;
        for (int s = strand; s < a.splits; s += 8) s_weight[s][t][r] *= f;
    }
    __syncthreads();
    {
        const int t = warp >> 2, v0 = (warp & 3) * 16;
        const float* src = part + ((int64_t)t * a.row_groups * kDiffRowValues + v0) * 32 + lane;
        const int rA = lane >> 2, rB = rA + 8;
        const bool useA = row0 + rA < a.Nq, useB = row0 + rB < a.Nq;
        float acc[16] = {};
#pragma unroll 2
        for (int s = 0; s < a.splits; ++s) {
            if (empty(s)) continue;
            const float wA = s_weight[s][t][rA], wB = s_weight[s][t][rB];
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = ((i & 2) ? useB : useA) ? __ldcg(src + s * step + i * 32) : 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[i] = fmaf(x[i], (i & 2) ? wB : wA, acc[i]);
        }
#pragma unroll
        for (int i = 0; i < 16; i += 2)
            *reinterpret_cast<float2*>(&s_o[t][(i & 2) ? rB : rA][8 * ((v0 + i) >> 2) + 2 * (lane & 3)]) = make_float2(acc[i], acc[i + 1]);
    }
    __syncthreads();
    const int r = threadIdx.x >> 4, c = (threadIdx.x & 15) * 8;
    float o[8], sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        o[i] = s_o[0][r][c + i] - s_o[1][r][c + i];
        sum = fmaf(o[i], o[i], sum);
    }
    float scale = a.out_scale;
    if (a.weight != nullptr) {
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        scale *= rsqrtf(sum * (1.f / 128.f) + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] *= diff_weight(a, c + i);
    }
    if (row0 + r < a.Nq)
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
    return (int64_t)B * H * ((Nq + FQ - 1) / FQ) * splits * 2 * diff64_row_groups(Nq) * kDiffRowValues * 32 * (int64_t)sizeof(float);
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
        e = launch_pdl(diff64_join_kernel, dim3((unsigned)(B * (int64_t)H * a.q_tiles * a.row_groups)), dim3(256), 0, stream, a);
        if (e != cudaSuccess) return fail((int)e, "diff64_join_kernel launch: %s", cudaGetErrorString(e));
    }
    return FBB_OK;
}

}  // namespace fbb
