// Differential attention: o = softmax(scale q1 k1') v - lam softmax(scale q2 k2') v, two maps of head dimension 64 over the same
// values of 128 columns, and the root-mean-square norm of every head's row behind it. No mask but a number of keys per batch entry.
//
// A tile is 128 queries of one (batch, head); it walks its keys in blocks of 128, both maps at once, so that v is read once and no map
// or half of an output ever leaves the chip (as four calls of the flash64 kernel, one per map and half of v, every score is computed
// twice and three passes over the outputs follow). One persistent CTA per SM takes every so-manieth tile. Where the SMs are twice the
// tiles or more (few queries over many keys), each is split over the keys instead, and the splits' unnormalised rows, maxima and sums go
// through the workspace to diff64_join_kernel. (From 75 to 147 tiles on 148 SMs there is one CTA a tile, and the other SMs rest.)
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
// The next item's Q, K and first scores are on their way while the softmax warps finish the last one; only its first P.V waits for them
// to have read O. Map 0's and map 1's warps of the same rows finish a tile together, half of the columns each: both read O_1 and O_2.
//
// Keys beyond a batch entry's number are masked by selection, never by adding, and their rows of V are zeroed in shared memory ahead
// of the product, so that no infinity or NaN in them is seen.
//
// Bound by the exponentials where tiles are many: 6145 queries x 8 heads take 237 us in a row of launches (979 TFLOP/s; a launch's first tiles
// run on SMs that the one ahead has left) and 272 by itself, with the transcendental unit busy for 70 % of the clocks an SM is active and
// the tensor pipe for 53 %. Few queries are bound by the chain of half-blocks, of whose 16 softmax warps two have a row: 1 x 16385 x 8
// takes 23.8 us, 14 half-blocks of 1.6 k clocks after one another 12 of them (the read of K and V, 10, runs beside), the merge about
// 5, set-up and the tile's end the rest. Short tiles pay for their ends: 6.6 k clocks behind 2.8 k a block.
#include <cfloat>

#include "common.cuh"
#include "internal.h"

namespace fbb {

constexpr int kDiffStages = 3;
constexpr int kDiffPart = 16 * 128 + 16 * 2;  // floats of 16 rows of a part and map: the outputs, then {maximum, sum (-sum: of far rows)} of each row

struct DiffSmem {
    static constexpr int kQOff = 0;                       // Q_1 | Q_2
    static constexpr int kStageOff = 2 * kTileBytes;      // stages of K_1 | K_2 | V columns 0..63 | V columns 64..127
    static constexpr int kStageBytes = 4 * kTileBytes;
    static constexpr int kRowOff = kStageOff + kDiffStages * kStageBytes;  // [2][128] row sums of the maps, [2][128] sums of squares of the halves
    static constexpr int kWeightOff = kRowOff + 4 * 128 * 4;               // [128] fp32
    static constexpr int kBarOff = kWeightOff + 128 * 4;
    // q_full, q_empty, w_ready, o_free, k_full[2][S], k_empty[2][S], v_full[S], v_empty[S], then of each map and half s_full, p_ready, pv_done,
    // then where the two maps' softmax warps of the same rows meet
    static constexpr int kNumBars = 4 + 6 * kDiffStages + 12 + 8;
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
    int Nq, Nk, q_tiles;
    int splits, items;       // items = tiles x splits
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
// A CTA's items: one of every gridDim.x, from the front and from the back of each such row in turn, so that the sums come out even
// where the tiles' lengths fall along the row: batch entries are taken by falling number of keys (up to 32 of them, whose numbers the
// lanes of a warp hold; more are taken in their order). All lanes of a warp go through the items together.
struct DiffItems {
    int w, round;         // item, and the row of gridDim.x items it is in
    int b, h, qt;         // (b: the place until the lengths are known)
    int keys, kb0, here;  // keys of the batch entry; first block and number of keys of the item
    int order;            // the batch entry that is `lane`-th, and its keys times 32
    __device__ __forceinline__ explicit DiffItems(const DiffArgs& a) {
        w = (int)blockIdx.x;
        round = 0;
        decode(a);
    }
    __device__ __forceinline__ static bool sorted(const DiffArgs& a) { return a.lengths != nullptr && a.B <= 32 && a.Nk < (1 << 26); }
    __device__ __forceinline__ void decode(const DiffArgs& a) {
        const unsigned tile = a.splits > 1 ? (unsigned)w / (unsigned)a.splits : (unsigned)w;
        const unsigned bh = tile / (unsigned)a.q_tiles;
        qt = (int)(tile - bh * (unsigned)a.q_tiles);
        b = a.B > 1 ? (int)(bh / (unsigned)a.H) : 0;
        h = (int)bh - b * a.H;
    }
    // The rest of the set-up, which reads the lengths.
    __device__ __forceinline__ void begin(const DiffArgs& a, int lane) {
        if (sorted(a)) {
            const int mine = lane < a.B ? diff_keys(a, lane) : 0;
            int place = 0;
            for (int j = 0; j < a.B; ++j) {
                const int other = __shfl_sync(0xffffffffu, mine, j);
                place += other > mine || (other == mine && j < lane);
            }
            for (int j = 0; j < a.B; ++j) {
                const int entry = __shfl_sync(0xffffffffu, mine, j) * 32 + j;
                if (__shfl_sync(0xffffffffu, place, j) == lane) order = entry;
            }
        }
        item(a);
    }
    __device__ __forceinline__ void item(const DiffArgs& a) {
        if (a.lengths == nullptr) {
            keys = a.Nk;
        } else if (sorted(a)) {
            const int entry = __shfl_sync(0xffffffffu, order, b);
            b = entry & 31;
            keys = entry >> 5;
        } else {
            keys = w < a.items ? diff_keys(a, b) : 0;
        }
        int kb1;
        diff_share(keys, a.splits > 1 ? (int)((unsigned)w % (unsigned)a.splits) : 0, a.splits, kb0, kb1);
        here = min(keys, kb1 * FK) - kb0 * FK;
    }
    // Where the rows of a split go in the workspace: by the tile itself, not by its place.
    __device__ __forceinline__ int64_t part(const DiffArgs& a) const {
        return (((int64_t)b * a.H + h) * a.q_tiles + qt) * a.splits + (int)((unsigned)w % (unsigned)a.splits);
    }
    __device__ __forceinline__ bool more(const DiffArgs& a) const { return w < a.items; }
    __device__ __forceinline__ void next(const DiffArgs& a) {
        const int in_row = (int)((++round & 1) ? gridDim.x - 1u - blockIdx.x : blockIdx.x);
        w = round * (int)gridDim.x + in_row;
        if (w >= a.items) return;
        decode(a);
        item(a);
    }
};
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

// A row's exponents are s sl - m, m its running maximum times sl, rounded: the same m for all of them, so its rounding drops out with the sum.
// From 2^22 on that rounding would be an exponent's worth and more. Rows of such scores are far: theirs are (s - r) sl, r the maximum itself,
// whose difference is exact for the scores that matter.
constexpr float kDiffFar = 4194304.f;

constexpr int kDiffEarly = 2;  // key groups of eight exponentiated ahead of the vote on the running maximum (see kEarly in flash64.cu)

// Four 32-bit values of each of the four lanes of a quad, [lane][k] -> [k][lane].
__device__ __forceinline__ void quad_transpose(uint32_t* m, int cq) {
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, (cq & 1) ? m[k] : m[k + 1], 1);
        if (cq & 1) m[k] = got;
        else m[k + 1] = got;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, (cq & 2) ? m[k] : m[k + 2], 2);
        if (cq & 2) m[k] = got;
        else m[k + 2] = got;
    }
}

__global__ void __launch_bounds__(640, 1)
diff64_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
              const DiffArgs a) {
    using S = DiffSmem;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t base = smem_u32(smem_raw);
    const uint32_t bar0 = base + S::kBarOff;
    const uint32_t q_full = bar0, q_empty = bar0 + 8u, w_ready = bar0 + 16u, o_free = bar0 + 24u;
    constexpr int kK = 4, kV = kK + 4 * kDiffStages, kS = kV + 2 * kDiffStages;
    auto k_full = [&](int t, int s) { return bar0 + 8u * (kK + t * kDiffStages + s); };
    auto k_empty = [&](int t, int s) { return bar0 + 8u * (kK + (2 + t) * kDiffStages + s); };
    auto v_full = [&](int s) { return bar0 + 8u * (kV + s); };
    auto v_empty = [&](int s) { return bar0 + 8u * (kV + kDiffStages + s); };
    auto s_full = [&](int t, int half) { return bar0 + 8u * (kS + 2 * t + half); };
    auto p_ready = [&](int t, int half) { return bar0 + 8u * (kS + 4 + 2 * t + half); };
    auto pv_done = [&](int t, int half) { return bar0 + 8u * (kS + 8 + 2 * t + half); };
    auto meeting = [&](int u) { return bar0 + 8u * (kS + 12 + u); };
    volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(smem_raw + S::kBarOff + S::kNumBars * 8);
    volatile int* s_abort = reinterpret_cast<volatile int*>(smem_raw + S::kBarOff + S::kNumBars * 8 + 4);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kNumBars; ++i) {
            int count = 1;
            if (i == 1 || (i >= kV + kDiffStages && i < kS)) count = 2;  // q_empty, v_empty: both maps' issuers
            if (i >= kS + 12) count = 2;
            if (i == 3) count = 16;                                    // o_free: the softmax warps
            if (i >= kS + 4 && i < kS + 8) count = 8;                  // p_ready: a map's softmax warps
            mbar_init(bar0 + 8u * i, count);
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
    DiffItems it(a);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *s_tmem;
    grid_dependency_wait();
    grid_launch_dependents();
    it.begin(a, lane);

    if (warp < 4) {
        setmaxnreg_dec<kRegsCtl>();
        if (warp == 0) {
            int s = 0, nq = 0;
            uint32_t ph = 0;
            bool ok = true;
#pragma unroll 1
            for (; it.more(a) && ok; it.next(a)) {
                if (it.here <= 0) continue;
                if (lane == 0) {
                    const int b = it.b, h = it.h, hk = a.group > 1 ? (int)((unsigned)h / (unsigned)a.group) : h;
                    ok = nq == 0 || mbar_wait(q_empty, (uint32_t)(nq - 1) & 1u, s_abort, DEV_TIMEOUT_SMEM_EMPTY, 32);
                    if (ok) {
                        mbar_arrive_expect_tx(q_full, 2 * kTileBytes);
                        for (int t = 0; t < 2; ++t) tma_load_4d(base + S::kQOff + t * kTileBytes, &tmap_q, q_full, 0, 2 * h + t, it.qt * FQ, b);
                    }
                    const int kb1 = it.kb0 + (it.here + FK - 1) / FK;
#pragma unroll 1
                    for (int kb = it.kb0; kb < kb1 && ok; ++kb) {
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
                }
                ++nq;
                ok = __all_sync(0xffffffffu, ok) != 0;
            }
            if (!ok) __nanosleep(20000);
        } else if (warp < 3) {
            const int t = warp - 1;
            const uint32_t idesc_qk = make_idesc_f16(FQ, 64, true, false, false);
            const uint32_t idesc_pv = make_idesc_f16(FQ, 128, true, false, true);
            const uint64_t qd = smem_desc(base + S::kQOff + t * kTileBytes, make_smem_desc_hi(16, 1024));
            const uint64_t kd0 = smem_desc(base + S::kStageOff + t * kTileBytes, make_smem_desc_hi(16, 1024));
            const uint64_t vd0 = smem_desc(base + S::kStageOff + 2 * kTileBytes, make_smem_desc_hi(kTileBytes, 1024));  // column halves a tile apart
            const uint32_t dS = tmem_base + t * 128, dO = tmem_base + 256 + t * 128;
            auto all_ok = [&](bool mine) { return __all_sync(0xffffffffu, mine) != 0; };
            // Units (half-blocks) are counted over all items, g, which gives the half of tensor memory and the barriers' phases, and inside
            // an item, i: half i & 1 of a block, whose 64 keys are 8 KB further in a tile of K or V.
            int ks = 0, vs = 0;  // stages of the next unit's K and V
            uint32_t kph = 0, vph = 0;
            auto scores = [&](uint32_t g, int i, bool last) -> bool {
                if ((i & 1) == 0 && !all_ok(mbar_wait(k_full(t, ks), kph, s_abort, DEV_TIMEOUT_TMA_FULL, 2 * ks + t))) return false;
                tc_fence_after();
                const uint64_t kd = kd0 + (uint64_t)((ks * S::kStageBytes + (i & 1) * (kTileBytes / 2)) >> 4);
                umma_kblock_commit_warp(dS + 64u * (g & 1u), qd, kd, idesc_qk, 0u, s_full(t, g & 1u));
                if ((i & 1) == 1 || last) {
                    umma_commit_warp(k_empty(t, ks));
                    if (++ks == kDiffStages) { ks = 0; kph ^= 1u; }
                }
                if (last) umma_commit_warp(q_empty);
                return true;
            };
            uint32_t g = 0;
            int n = 0;  // items with keys; of others no barrier hears anything
            bool ok = true;
#pragma unroll 1
            for (; it.more(a) && ok; it.next(a)) {
                const int here = it.here, halves = (here + 63) / 64;
                if (here <= 0) continue;
                ok = all_ok(mbar_wait(q_full, (uint32_t)n & 1u, s_abort, DEV_TIMEOUT_TMA_FULL, 100));
                ok = ok && scores(g, 0, halves == 1);
                if (ok && halves > 1) ok = scores(g + 1u, 1, halves == 2);
                // the softmax warps have read the last such item's O. No phase of theirs is missed here: the next one needs this item's
                // products of both maps, which come behind this wait.
                if (ok && n > 0) ok = all_ok(mbar_wait(o_free, (uint32_t)(n - 1) & 1u, s_abort, DEV_TIMEOUT_TMEM_EMPTY, 40 + t));
                ++n;
#pragma unroll 1
                for (int i = 0; i < halves && ok; ++i, ++g) {
                    if ((i & 1) == 0 && !all_ok(mbar_wait(v_full(vs), vph, s_abort, DEV_TIMEOUT_TMA_FULL, 16 + vs))) { ok = false; break; }
                    const uint32_t vt = vs * S::kStageBytes + (i & 1) * (kTileBytes / 2);
                    if (i + 1 == halves && here < 64 * halves && it.keys < a.Nk) {
                        // rows of V beyond the entry's keys hold whatever the tensor holds there (beyond the tensor the copy wrote zeros);
                        // both issuers write the same zeros
                        const uint32_t at = base + S::kStageOff + 2 * kTileBytes + vt;
                        for (int j = (here - 64 * i) * 8 + lane; j < 64 * 8; j += 32)
                            for (int c = 0; c < 2; ++c) st_shared_16(at + c * kTileBytes + 16u * j, 0.f, 0.f, 0.f, 0.f);
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                    if (!all_ok(mbar_wait(p_ready(t, g & 1u), (g >> 1) & 1u, s_abort, DEV_TIMEOUT_OTHER, 200 + 2 * t + (g & 1u)))) { ok = false; break; }
                    tc_fence_after();
                    umma_ts4_commit_warp(dO, dS + 64u * (g & 1u), vd0 + (uint64_t)(vt >> 4), idesc_pv, i > 0 ? 1u : 0u, pv_done(t, g & 1u));
                    if ((i & 1) == 1 || i + 1 == halves) {
                        umma_commit_warp(v_empty(vs));
                        if (++vs == kDiffStages) { vs = 0; vph ^= 1u; }
                    }
                    if (i + 2 < halves) ok = scores(g + 2u, i + 2, i + 3 == halves);
                }
            }
        } else if (a.weight != nullptr) {
            float* s_w = reinterpret_cast<float*>(smem_raw + S::kWeightOff);
#pragma unroll
            for (int i = 0; i < 4; ++i) s_w[lane + 32 * i] = diff_weight(a, lane + 32 * i) * a.out_scale;
            __syncwarp();
            if (lane == 0) mbar_arrive(w_ready);
        }
    } else {
        setmaxnreg_inc<kRegsSoftmax>();
        const int u = (warp - 4) & 7;
        const int t = (warp - 4) >> 3;
        const int lane_base = (u & 3) * 32 + (u >> 2) * 16;
        const int cq = lane & 3;
        const uint32_t tl = tmem_base + ((uint32_t)lane_base << 16);  // this warp's lanes
        const uint32_t tS = tl + t * 128, tO = tl + 256 + t * 128;
        const float sl = a.scale_log2;
        const float lazy = fminf(kLazyMax / sl, FLT_MAX);
        bool ok = true;
        uint32_t g = 0;
        int n = 0;
        // Both maps' warps of these rows have got here (a barrier with a limit: a warp that gave up does not come).
        uint32_t met = 0;
        auto meet = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(meeting(u));
            ok = mbar_wait(meeting(u), met & 1u, s_abort, DEV_TIMEOUT_OTHER, 230 + u) && ok;
            ++met;
        };
        // the end of an item with keys: O has been read (an earlier one's phase must be complete before this one's arrivals begin). Items
        // without keys have no part in it: nothing would hold these warps back there, and a phase that completes before an issuer has
        // looked for the one ahead of it takes that one from its sight.
        auto release = [&]() {
            tc_fence_before();
            ok = (n == 0 || mbar_wait(o_free, (uint32_t)(n - 1) & 1u, s_abort, DEV_TIMEOUT_OTHER, 44)) && ok;
            __syncwarp();
            if (lane == 0) mbar_arrive(o_free);
            ++n;
        };
#pragma unroll 1
        for (; it.more(a) && ok; it.next(a)) {
            const int here = it.here, halves = (here + 63) / 64;
            const int row0 = it.qt * FQ + lane_base, rowA = row0 + (lane >> 2), rowB = rowA + 8;
            if (row0 >= a.Nq) {
                // a warp of rows beyond Nq only keeps the barriers moving: S_t of unit g exists only after the issuer has taken P_t of unit g - 2
#pragma unroll 1
                for (int i = 0; i < halves && ok; ++i, ++g) {
                    ok = mbar_wait(s_full(t, g & 1u), (g >> 1) & 1u, s_abort, DEV_TIMEOUT_TMEM_FULL, 2 * t + (g & 1u));
                    tc_fence_after();
                    tc_fence_before();
                    __syncwarp();
                    if (ok && lane == 0) mbar_arrive(p_ready(t, g & 1u));
                }
                if (halves > 0) release();
                continue;
            }
            const bool whole = a.splits == 1;
            float lamA = 0.f, lamB = 0.f;
            if (whole) {
                const float* lam = a.lam + it.b * a.l_sb + it.h * a.l_sh;
                if (rowA < a.Nq) lamA = lam[rowA * a.l_sn];
                if (rowB < a.Nq) lamB = lam[rowB * a.l_sn];
            }
            float tA = 0.f, tB = 0.f;
            // (no lower: the maximum of keys that are all at minus infinity is subtracted from it)
            float mA = -FLT_MAX, mB = -FLT_MAX, lA = 0.f, lB = 0.f;
            bool far = false;  // this warp's rows are far, from the first half-block that has one on: mA and mB are the maxima themselves
            // One half-block; false: a wait ran out, or (far is set, nothing else is changed) rows turned out far.
            auto unit = [&](auto far_rows, int i) -> bool {
                constexpr bool kFar = decltype(far_rows)::value;
                const uint32_t half = g & 1u, tSh = tS + 64u * half;
                if (!mbar_wait(s_full(t, half), (g >> 1) & 1u, s_abort, DEV_TIMEOUT_TMEM_FULL, 2 * t + half)) return false;
                tc_fence_after();
                uint32_t sc[32], pk[16];
                float mxA, mxB;
                tmem_ld_16x256b_x8(tSh, sc);
                tmem_wait_ld();
                tmem_tie32(sc);
                if (64 * (i + 1) > here) mask_frag(sc, 64 * i + 2 * cq, here);  // (the last one may have keys beyond the entry's)
                max_frag<8>(sc, mxA, mxB);
                float2 accA = make_float2(0.f, 0.f), accB = make_float2(0.f, 0.f);
                if constexpr (!kFar) exp_frag<kDiffEarly>(sc, sl, mA, mB, accA, accB, pk);
                if (i == 0 || __any_sync(0xffffffffu, kFar ? mxA - mA > lazy || mxB - mB > lazy || tA != 0.f || tB != 0.f : mxA > tA || mxB > tB)) {
                    mxA = fmaxf(mxA, __shfl_xor_sync(0xffffffffu, mxA, 1));
                    mxB = fmaxf(mxB, __shfl_xor_sync(0xffffffffu, mxB, 1));
                    mxA = fmaxf(mxA, __shfl_xor_sync(0xffffffffu, mxA, 2));
                    mxB = fmaxf(mxB, __shfl_xor_sync(0xffffffffu, mxB, 2));
                    if constexpr (!kFar) {
                        if (__any_sync(0xffffffffu, fmaxf(fabsf(mxA), fabsf(mxB)) * sl >= kDiffFar)) {  // (infinities too)
                            far = true;
                            return false;
                        }
                    }
                    const float nA = fmaxf(mA, kFar ? mxA : mxA * sl), nB = fmaxf(mB, kFar ? mxB : mxB * sl);
                    if (i > 0) {
                        // the unit before this one may still be adding to O_t
                        if (!mbar_wait(pv_done(t, half ^ 1u), ((g - 1u) >> 1) & 1u, s_abort, DEV_TIMEOUT_TMEM_FULL, 8 + 2 * t + half)) return false;
                        tc_fence_after();
                        const float cA = ex2_approx(kFar ? (mA - nA) * sl + tA : mA - nA), cB = ex2_approx(kFar ? (mB - nB) * sl + tB : mB - nB);
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
                    if constexpr (kFar) {
                        tA = tB = 0.f;
                    } else {
                        tA = i == 0 ? mxA + lazy : fmaxf(tA, mxA + lazy);
                        tB = i == 0 ? mxB + lazy : fmaxf(tB, mxB + lazy);
                        accA = accB = make_float2(0.f, 0.f);
                        exp_frag<kDiffEarly>(sc, sl, mA, mB, accA, accB, pk);
                    }
                }
                if constexpr (kFar) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) sc[j] = __float_as_uint(__uint_as_float(sc[j]) - ((j & 2) ? mB : mA));
                    exp_frag<8>(sc, sl, 0.f, 0.f, accA, accB, pk);
                } else {
                    exp_frag<8 - kDiffEarly>(sc + 4 * kDiffEarly, sl, mA, mB, accA, accB, pk + 2 * kDiffEarly);
                }
                tmem_st_16x128b_x8(tSh, pk);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready(t, half));
                lA += accA.x + accA.y;
                lB += accB.x + accB.y;
                return true;
            };
            int i = 0;
#pragma unroll 1
            for (; i < halves; ++i, ++g)
                if (!(ok = unit(std::false_type{}, i))) break;
            if (far) {
                // The maxima so far become scores again (a maximum of no score yet stays the lowest number). The exponent by which that
                // changes them goes into what O and the sums are raised by right after.
                ok = true;
                const float rA = mA == -FLT_MAX ? mA : mA / sl, rB = mB == -FLT_MAX ? mB : mB / sl;
                tA = mA == -FLT_MAX ? 0.f : fmaf(-rA, sl, mA);
                tB = mB == -FLT_MAX ? 0.f : fmaf(-rB, sl, mB);
                mA = rA;
                mB = rB;
#pragma unroll 1
                for (; i < halves && ok; ++i, ++g) ok = unit(std::true_type{}, i);
            }
            if (ok && halves > 0) ok = mbar_wait(pv_done(t, (g - 1u) & 1u), ((g - 1u) >> 1) & 1u, s_abort, DEV_TIMEOUT_TMEM_FULL, 12 + t);
            // a row's sum is spread over the four threads that share it
            lA += __shfl_xor_sync(0xffffffffu, lA, 1);
            lB += __shfl_xor_sync(0xffffffffu, lB, 1);
            lA += __shfl_xor_sync(0xffffffffu, lA, 2);
            lB += __shfl_xor_sync(0xffffffffu, lB, 2);
            tc_fence_after();
            if (!whole) {
                // a split's rows, for diff64_join_kernel (which asks for no split without keys)
                if (halves > 0) {
                    float* dst = a.part + ((it.part(a) * 2 + t) * a.row_groups + (lane_base >> 4)) * kDiffPart;
                    float2* outA = reinterpret_cast<float2*>(dst + (lane >> 2) * 128 + 2 * cq);
#pragma unroll 1
                    for (int c = 0; c < 8; ++c) {
                        uint32_t o[8];
                        tmem_ld_16x256b_x2(tO + 16u * c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            outA[8 * c + 4 * i] = make_float2(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]));
                            if (rowB < a.Nq) outA[8 * c + 4 * i + 8 * 64] = make_float2(__uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
                        }
                    }
                    float2* stat = reinterpret_cast<float2*>(dst + 16 * 128);
                    if (cq == 0) stat[lane >> 2] = make_float2(mA, far ? -lA : lA);
                    if (cq == 1) stat[(lane >> 2) + 8] = make_float2(mB, far ? -lB : lB);
                    release();
                }
                continue;
            }
            // Columns 64 t .. 64 t + 63 of the tile's rows: o = O_1 / l_1 - lam O_2 / l_2. The other map's warp of these rows has waited for
            // its last product when it arrives with its sums.
            float* s_l = reinterpret_cast<float*>(smem_raw + S::kRowOff);
            float* s_q = s_l + 256;
            const int rA = lane_base + (lane >> 2);
            float o[32];
            if (halves > 0) {
                if (cq == 0) {
                    s_l[t * 128 + rA] = lA;
                    s_l[t * 128 + rA + 8] = lB;
                }
                tc_fence_before();
                meet();
                tc_fence_after();
                const float f1A = 1.f / s_l[rA], f1B = 1.f / s_l[rA + 8], f2A = lamA / s_l[128 + rA], f2B = lamB / s_l[128 + rA + 8];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t x[8], y[8];
                    tmem_ld_16x256b_x2(tl + 256 + 64 * t + 16 * c, x);
                    tmem_ld_16x256b_x2(tl + 384 + 64 * t + 16 * c, y);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[8 * c + i] = __uint_as_float(x[i]) * ((i & 2) ? f1B : f1A) - __uint_as_float(y[i]) * ((i & 2) ? f2B : f2A);
                }
                release();
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0.f;
            }
            float scA = a.out_scale, scB = a.out_scale;
            const bool norm = a.weight != nullptr && halves > 0;
            if (norm) {
                float sA = 0.f, sB = 0.f;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    if (i & 2) sB = fmaf(o[i], o[i], sB);
                    else sA = fmaf(o[i], o[i], sA);
                }
                sA += __shfl_xor_sync(0xffffffffu, sA, 1);
                sB += __shfl_xor_sync(0xffffffffu, sB, 1);
                sA += __shfl_xor_sync(0xffffffffu, sA, 2);
                sB += __shfl_xor_sync(0xffffffffu, sB, 2);
                if (cq == 0) {
                    s_q[t * 128 + rA] = sA;
                    s_q[t * 128 + rA + 8] = sB;
                }
                ok = mbar_wait(w_ready, 0, s_abort, DEV_TIMEOUT_OTHER, 220) && ok;
                meet();
                scA = rsqrtf((s_q[rA] + s_q[128 + rA]) * (1.f / 128.f) + a.eps);  // (the weight in shared memory holds out_scale)
                scB = rsqrtf((s_q[rA + 8] + s_q[128 + rA + 8]) * (1.f / 128.f) + a.eps);
            }
            const float* s_w = reinterpret_cast<const float*>(smem_raw + S::kWeightOff) + 64 * t + 2 * cq;
            __half* out = a.o + (int64_t)it.b * a.o_sb + (int64_t)it.h * a.o_sh + 64 * t + 8 * cq;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                // a quad's lanes hold two columns each of four groups of eight: afterwards each holds the eight of one
                uint32_t hA[4], hB[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float* v = o + 16 * j + 4 * k;
                    const float2 w = norm ? *reinterpret_cast<const float2*>(s_w + 32 * j + 8 * k) : make_float2(1.f, 1.f);
                    hA[k] = pack_h2(v[0] * scA * w.x, v[1] * scA * w.y);
                    hB[k] = pack_h2(v[2] * scB * w.x, v[3] * scB * w.y);
                }
                quad_transpose(hA, cq);
                quad_transpose(hB, cq);
                if (ok && rowA < a.Nq) *reinterpret_cast<uint4*>(out + (int64_t)rowA * a.o_sn + 32 * j) = make_uint4(hA[0], hA[1], hA[2], hA[3]);
                if (ok && rowB < a.Nq) *reinterpret_cast<uint4*>(out + (int64_t)rowB * a.o_sn + 32 * j) = make_uint4(hB[0], hB[1], hB[2], hB[3]);
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
    int far = 0;  // some of these rows are, in some share
    for (int i = threadIdx.x; i < live * 32; i += 512) {
        const int j = i >> 5, mr = i & 31;
        const float2 stat = __ldcg(reinterpret_cast<const float2*>(part + (int64_t)share(j) * step + (mr >> 4) * (step / 2) + 16 * 128) + (mr & 15));
        s_stat[j][mr >> 4][mr & 15] = stat;
        far |= signbit(stat.y);
    }
    far = __syncthreads_or(far);
    if (used) {  // (whole rows of 16 threads, whose shuffles stay among themselves)
        const unsigned mask = 0xffffu << (threadIdx.x & 16);
        float m = -INFINITY, l = 0.f;
        if (far) {  // maxima become exponents relative to the greatest, a far share's or another's
            float top = -INFINITY, near = -FLT_MAX;
            for (int j = strand; j < live; j += 16) {
                const float2 stat = s_stat[j][t][r];
                if (signbit(stat.y)) top = fmaxf(top, stat.x);
                else near = fmaxf(near, stat.x);
            }
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) {
                top = fmaxf(top, __shfl_xor_sync(mask, top, d));
                near = fmaxf(near, __shfl_xor_sync(mask, near, d));
            }
            const bool from_top = fmaf(top, a.scale_log2, -near) > 0.f;
            for (int j = strand; j < live; j += 16) {
                const float2 stat = s_stat[j][t][r];
                const float x = signbit(stat.y) ? (from_top ? (stat.x - top) * a.scale_log2 : fmaf(stat.x, a.scale_log2, -near))
                                                : (from_top ? fmaf(-top, a.scale_log2, stat.x) : stat.x - near);
                s_stat[j][t][r] = make_float2(x, fabsf(stat.y));
            }
        }
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
    if (a.weight != nullptr && live > 0) {  // (a row without keys is 0, with an eps of 0 too)
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
    const int64_t items = (int64_t)B * H * a.q_tiles * a.splits;
    if (items > 0x3FFFFFFFll) return fail(FBB_ERR_SHAPE, "diff64: too many query tiles (%lld)", (long long)items);
    a.items = (int)items;
    a.row_groups = diff64_row_groups(Nq);
    const int64_t need = diff64_workspace_bytes(B, Nq, Nk, H);
    if (need > 0 && (ws == nullptr || ws_bytes < need))
        return fail(FBB_ERR_SHAPE, "diff64: workspace of %lld bytes, %lld needed", (long long)(ws != nullptr ? ws_bytes : 0), (long long)need);
    a.part = need > 0 ? reinterpret_cast<float*>(ws) : nullptr;
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
    cudaError_t e = launch_pdl(diff64_kernel, dim3((unsigned)(a.items < num_sms() ? a.items : num_sms())), dim3(640), DiffSmem::kBytes, stream, tq, tk, tv, a);
    if (e != cudaSuccess) return fail((int)e, "diff64_kernel launch: %s", cudaGetErrorString(e));
    if (a.splits > 1) {
        e = launch_pdl(diff64_join_kernel, dim3((unsigned)(B * (int64_t)H * a.q_tiles * a.row_groups)), dim3(512), 0, stream, a);
        if (e != cudaSuccess) return fail((int)e, "diff64_join_kernel launch: %s", cudaGetErrorString(e));
    }
    return FBB_OK;
}

}  // namespace fbb
