// Product of two microscaled matrices, out[m, n] = sum_k A[m, k] B[n, k] + bias[n], on the block-scaled tensor core.
//
// Both operands are K-major with one E8M0 byte for every 32 elements of a row, which is what the instruction multiplies
// into the product itself: the codes go from global to shared memory by TMA and are never widened.  A tile is 128 rows of
// one operand (P) by TN rows of the other (Q), 128 bytes of K (256 E2M1 or 128 E4M3 / E5M2 elements) at a time.
//
// The tensor core takes such a step of a 256 x 256 tile in 0.287 us (4.3 PFLOP/s 8-bit, 8.6 4-bit over 148 SMs), so a
// kernel of this kind lives by handing it operands without a pause.  Measured: 8192^3 4-bit 189 to 196 us in a short run (5.6 to
// 5.8 PFLOP/s, tensor pipe active in 81 % of the cycles), 219 to 229 us in a long one, where the card's power limit lowers the
// clock; 8192 x 4096 x 4096 E4M3 103 and 120 to 125 us (76 %).  Few tokens are bound by reading the weights: 24 x 16384 x 8192
// E4M3 28 us (5.0 TB/s); one token x 4096 x 4096 4-bit by latency, 5.8 us with the weights in L2, 6.2 from memory.
#include <algorithm>

#include "mx_kernels.cuh"
#include "tcgen05.cuh"

namespace morb {
namespace {

struct MmArgs {
    const uint8_t *sp, *sq;   // scale bytes of P and Q
    const uint16_t* bias;
    uint16_t* out;
    int64_t p_rows, q_rows;
    int64_t groups;           // scale bytes a row (K / 32)
    int64_t ldo;              // row pitch of out (= n)
    int64_t p_tiles;
    uint32_t idesc;
    int ktiles, splits, vec_out;
};

constexpr int kPRows = 128;
constexpr int kPairsBelow = 14;   // steps that splitting the sum would save

template <bool FP4, int TN>
struct MmShape {
    static constexpr int kBlk = FP4 ? 2 : 1;                       // 512-byte scale blocks (128 rows x 4 groups) of P per step
    static constexpr int kQBlk = kBlk;
    static constexpr int kPBytes = kPRows * 128, kQBytes = TN * 128;
    static constexpr int kSfOff = kPBytes + kQBytes;
    static constexpr int kStage = (kSfOff + (kBlk + kQBlk) * 512 + 1023) & ~1023;
    static constexpr int kStages = (200 * 1024) / kStage < 8 ? (200 * 1024) / kStage : 8;
    static constexpr int kSmem = kStages * kStage + 1024;          // more than half of an SM: one CTA each, so the columns of tensor memory suffice
    static constexpr int kSfCols = 4 * (kBlk + kQBlk);
    static constexpr int kNeed = TN + 2 * kSfCols;
    static constexpr int kCols = kNeed <= 64 ? 64 : (kNeed <= 128 ? 128 : (kNeed <= 256 ? 256 : 512));
    static_assert(kSmem > 114 * 1024, "one CTA per SM");
};

// Scale bytes of a row for the next kBatch steps, W words of four, wherever they lie: 16-byte loads that cover them (no
// byte outside the tensor is read), moved into place when they are used, so that a batch can be in flight while the one
// before is stored.  A step's words go to the places the tensor core's copy takes them from (512 bytes for four groups of 128
// rows: 16 for each row mod 32, four for each row / 32); rows and groups outside read as zero, a finite scale.
constexpr int kBatch = 4;
template <int W>
struct ScaleWords {
    static constexpr int kChunks = W / 4 + 1;
    uint32_t x[4 * kChunks];
    int offset, valid;   // of the first byte in the first chunk; groups left in the row
    __device__ __forceinline__ void load(const uint8_t* s, int64_t rows, int64_t groups, int64_t row, int64_t g0) {
        const int64_t o = row * groups + g0, total = rows * groups, left = groups - g0;
        valid = row < rows && left > 0 ? (int)(left < 4 * W ? left : 4 * W) : 0;
        offset = (int)(o & 15);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t at = o - offset + 16 * c;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (offset + valid > 16 * c && valid > 0) {
                if (at + 16 <= total) {
                    v = __ldg(reinterpret_cast<const uint4*>(s + at));
                } else {   // the tensor's last bytes
                    uint32_t w[4] = {};
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (at + e < total) w[e >> 2] |= (uint32_t)__ldg(s + at + e) << (8 * (e & 3));
                    v = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            x[4 * c] = v.x; x[4 * c + 1] = v.y; x[4 * c + 2] = v.z; x[4 * c + 3] = v.w;
        }
    }
    __device__ __forceinline__ void place(uint32_t (&w)[W]) {
        constexpr int n = 4 * kChunks;
#pragma unroll
        for (int j = 0; j < n - 2; ++j) x[j] = offset & 8 ? x[j + 2] : x[j];
#pragma unroll
        for (int j = 0; j < n - 3; ++j) x[j] = offset & 4 ? x[j + 1] : x[j];
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const int left = valid - 4 * j;
            w[j] = __funnelshift_r(x[j], x[j + 1], 8 * (offset & 3));
            w[j] = left >= 4 ? w[j] : (left <= 0 ? 0u : w[j] & ((1u << (8 * left)) - 1u));
        }
    }
};
__device__ __forceinline__ void store_word(uint32_t dst, uint32_t w) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst), "r"(w) : "memory"); }

// SWAP: P is B (rows of out's columns) and Q is A, so that few tokens fill a narrow tile of many weight rows.
// Warps 0-3 fetch scale bytes and then write the result, warp 4 loads codes, warp 5 issues.
template <bool FP4, int TN, bool SWAP>
__global__ void __launch_bounds__(192, 1) mx_matmul_kernel(const __grid_constant__ CUtensorMap map_p, const __grid_constant__ CUtensorMap map_q,
                                                           const MmArgs a) {
    using S = MmShape<FP4, TN>;
    constexpr int kGroupsPerStep = FP4 ? 8 : 4;
    extern __shared__ uint8_t s_raw[];
    __shared__ __align__(8) uint64_t full[S::kStages], empty[S::kStages], acc_done, drained;
    __shared__ uint32_t s_tmem;
    __shared__ int s_late;   // a wait ran out: copies may still land where the result would pass through
    uint8_t* smem = s_raw + ((1024 - (smem_u32(s_raw) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int split = (int)(blockIdx.x % (unsigned)a.splits);
    const int64_t tile = blockIdx.x / (unsigned)a.splits, tp = tile % a.p_tiles, tq = tile / a.p_tiles;
    const int64_t p0 = tp * kPRows, q0 = tq * TN;
    const int k_first = (int)((int64_t)a.ktiles * split / a.splits), k_last = (int)((int64_t)a.ktiles * (split + 1) / a.splits);
    const int n = k_last - k_first;

    if (warp == 4 && lane == 0) {
        for (int s = 0; s < S::kStages; ++s) { mbar_init(&full[s], 1 + 4); mbar_init(&empty[s], 1); }
        mbar_init(&acc_done, 1);
        mbar_init(&drained, 1);
        s_late = 0;
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_p));
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q));
    }
    if (warp == 5) tmem_alloc<1>(&s_tmem, S::kCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    pdl_launch_dependents();
    pdl_wait();

    bool ok = true;   // a wait that ran out ends the role's loop; the tile is then written as NaN
    if (warp == 4) {
        Slot<S::kStages> sl;
        for (int i = 0; i < n; ++i) {
            ok = mbar_wait_warp(&empty[sl.s], sl.phase ^ 1);
            if (!ok) break;
            if (elect_one()) {
                uint8_t* st = smem + sl.s * S::kStage;
                uint64_t* bar = &full[sl.s];
                const int x = (k_first + i) * 128;
                mbar_expect_tx(bar, S::kPBytes + S::kQBytes);
                tma_load_2d(st, &map_p, x, (int)p0, bar);
                tma_load_2d(st + S::kPBytes, &map_q, x, (int)q0, bar);
            }
            __syncwarp();
            sl.advance();
        }
        if (!ok)   // copies in flight land before the shared memory is handed on: every slot's last round
            for (int s = 0; s < S::kStages; ++s) mbar_wait_bounded(&full[s], s < sl.s ? sl.phase : sl.phase ^ 1);
    } else if (warp == 5) {
        Slot<S::kStages> sl;
        const uint64_t d0 = umma_desc_kmajor(smem_u32(smem));
        for (int i = 0; i < n; ++i) {
            ok = mbar_wait_warp(&full[sl.s], sl.phase);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
                const uint32_t sf = smem_u32(smem) + sl.s * S::kStage + S::kSfOff;
                const uint32_t sfp = tmem + TN + (i & 1) * S::kSfCols, sfq = sfp + 4 * S::kBlk;
#pragma unroll
                for (int b = 0; b < S::kBlk + S::kQBlk; ++b) tc_copy_scales<1>(sfp + 4 * b, sf + 512 * b);
                const uint64_t dp = d0 + sl.s * (S::kStage / 16), dq = dp + S::kPBytes / 16;
#pragma unroll
                for (int k = 0; k < 4; ++k) {   // 32 bytes of K each
                    const uint32_t blk = FP4 ? k >> 1 : 0, id = FP4 ? (k & 1) * 2 : k;
                    tc_mma_scaled<1, FP4>(tmem, dp + 2 * k, dq + 2 * k, idesc_with_scale_id(a.idesc, id), sfp + 4 * blk, sfq + 4 * blk, (i | k) != 0);
                }
                tc_commit(&empty[sl.s]);
                if (i == n - 1) tc_commit(&acc_done);
            }
            __syncwarp();
            sl.advance();
        }
        if (!ok) {   // products in flight end before the tensor memory is handed on
            if (elect_one()) tc_commit(&drained);
            __syncwarp();
            mbar_wait_bounded(&drained, 0);
        }
    } else {
        const int t = threadIdx.x;   // 0..127
        const uint32_t sf = smem_u32(smem) + S::kSfOff + (t & 31) * 16 + (t >> 5) * 4;
        constexpr int W = kBatch * S::kBlk;
        Slot<S::kStages> sl;
        ScaleWords<W> p, q, next_p, next_q;
        const int64_t g0 = (int64_t)k_first * kGroupsPerStep;
        const bool has_q = warp < (TN + 31) / 32;
        p.load(a.sp, a.p_rows, a.groups, p0 + t, g0);
        if (has_q) q.load(a.sq, a.q_rows, a.groups, q0 + t, g0);
        for (int i = 0; i < n && ok; i += kBatch) {
            if (i + kBatch < n) {
                next_p.load(a.sp, a.p_rows, a.groups, p0 + t, g0 + (int64_t)(i + kBatch) * kGroupsPerStep);
                if (has_q) next_q.load(a.sq, a.q_rows, a.groups, q0 + t, g0 + (int64_t)(i + kBatch) * kGroupsPerStep);
            }
            uint32_t wp[W], wq[W];
            p.place(wp);
            if (has_q) q.place(wq);
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                if (i + u >= n) break;
                ok = mbar_wait_warp(&empty[sl.s], sl.phase ^ 1);
                if (!ok) break;
                const uint32_t to = sf + sl.s * S::kStage;
#pragma unroll
                for (int b = 0; b < S::kBlk; ++b) {
                    store_word(to + 512 * b, wp[u * S::kBlk + b]);
                    if (has_q) store_word(to + 512 * (S::kBlk + b), wq[u * S::kBlk + b]);
                }
                fence_async_shared();
                __syncwarp();
                if (elect_one()) mbar_arrive(&full[sl.s]);
                sl.advance();
            }
            p = next_p;
            q = next_q;
        }
        ok = ok && mbar_wait_warp(&acc_done, 0);
        if (!ok) s_late = 1;
        tc_fence_after();
    }

    // The result leaves through shared memory (the operands are no longer needed), where the partial sums of a cluster
    // meet and neighbouring lanes get neighbouring elements of a row of out.
    __syncwarp();
    if (a.splits > 1) cluster_sync();   // no CTA is still reading operands
    const ClusterSum<TN> sums{smem_u32(smem), a.splits, split};
    static_assert(ClusterSum<TN>::kBytes <= S::kStages * S::kStage, "partial sums");
    if (warp < 4) {
        const uint32_t lanes = tmem + ((uint32_t)warp << 21);   // lane field of the address: 32 per warp
        constexpr int C = TN < 32 ? 16 : 32;
        const uint32_t to = sums.place(threadIdx.x);
#pragma unroll 1
        for (int c0 = 0; c0 < TN && q0 + c0 < a.q_rows; c0 += C) {
            uint32_t r[C];
            if constexpr (C == 32) tmem_load32(lanes + c0, r); else tmem_load16(lanes + c0, r);
            tmem_wait_loads();
            if (!ok) {
#pragma unroll
                for (int c = 0; c < C; ++c) r[c] = 0x7FFFFFFFu;
            }
#pragma unroll
            for (int c = 0; c < C; c += 4)
                if (q0 + c0 + c < a.q_rows) sums.push(to + 4 * (c0 + c), r[c], r[c + 1], r[c + 2], r[c + 3]);
        }
    }
    __syncwarp();
    if (a.splits > 1) cluster_sync();
    else if (warp < 4) named_barrier(1, 128);
    if (warp < 4) {
        const int rows = sums.rows(), first_row = split * rows;
        const float late = s_late ? u2f(0x7FFFFFFFu) : 0.0f;
        if constexpr (SWAP) {
            // out's rows run along P: a lane takes one P row, a warp four tokens at a time
            for (int i = threadIdx.x; i < rows * (TN / 4); i += 128) {
                const int r = i % rows, c = i / rows * 4;
                const int64_t p = p0 + first_row + r;
                if (p >= a.p_rows || q0 + c >= a.q_rows) continue;
                const float4 v = sums.sum4(r, c);
                const float bias = (a.bias ? u2f((uint32_t)__ldg(a.bias + p) << 16) : 0.0f) + late;
                const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (q0 + c + j < a.q_rows) a.out[(q0 + c + j) * a.ldo + p] = (uint16_t)pack_bf16_rne(0.0f, e[j] + bias);
            }
        } else {
            constexpr int kLanes = TN / 4;   // a lane takes four columns
            const int c = (threadIdx.x % kLanes) * 4;
            const int64_t q = q0 + c;
            float bias[4] = {late, late, late, late};
            if (a.bias)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (q + j < a.q_rows) bias[j] += u2f((uint32_t)__ldg(a.bias + q + j) << 16);
#pragma unroll 4
            for (int r = threadIdx.x / kLanes; r < rows; r += 128 / kLanes) {
                const int64_t p = p0 + first_row + r;
                if (p >= a.p_rows) break;
                const float4 v = sums.sum4(r, c);
                uint16_t* o = a.out + p * a.ldo + q;
                const uint2 w = make_uint2(pack_bf16_rne(v.y + bias[1], v.x + bias[0]), pack_bf16_rne(v.w + bias[3], v.z + bias[2]));
                if (a.vec_out && q + 4 <= a.q_rows) {
                    *reinterpret_cast<uint2*>(o) = w;
                } else {
                    if (q < a.q_rows) o[0] = (uint16_t)w.x;
                    if (q + 1 < a.q_rows) o[1] = (uint16_t)(w.x >> 16);
                    if (q + 2 < a.q_rows) o[2] = (uint16_t)w.y;
                    if (q + 3 < a.q_rows) o[3] = (uint16_t)(w.y >> 16);
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 5) { tc_fence_after(); tmem_free<1>(tmem, S::kCols); }
}

// ---------------------------------------------------------------------------------
// large products: pairs of CTAs on 256 x 256
// ---------------------------------------------------------------------------------
// Scale bytes [rows, groups] in the order the tensor core's copy wants them: for every 128 rows and four groups 512 bytes,
// 16 for each r mod 32, four for each r / 32, zeros where there is no row or group.  One thread takes 16 groups of a row.
__global__ void __launch_bounds__(128) order_scales_kernel(const uint8_t* __restrict__ sa, int64_t rows_a, uint32_t* __restrict__ oa, int blocks_a,
                                                          const uint8_t* __restrict__ sb, int64_t rows_b, uint32_t* __restrict__ ob, int64_t groups,
                                                          int kblocks, int fast) {
    pdl_launch_dependents();
    pdl_wait();
    const bool first = (int)blockIdx.x < blocks_a;
    const int64_t rb = first ? blockIdx.x : blockIdx.x - blocks_a;
    const uint8_t* s = first ? sa : sb;
    const int64_t row = rb * 128 + (threadIdx.x & 3) * 32 + (threadIdx.x >> 2);
    const bool in = row < (first ? rows_a : rows_b);
    uint32_t* o = (first ? oa : ob) + rb * kblocks * 128 + threadIdx.x;
    for (int b = blockIdx.y * 4; b < kblocks; b += gridDim.y * 4) {
        uint32_t w[4] = {};
        const uint8_t* src = s + row * groups + b * 4;
        if (in && fast) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(src));   // groups is a multiple of 16
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else if (in) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (b * 4 + i < groups) w[i >> 2] |= (uint32_t)__ldg(src + i) << (8 * (i & 3));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (b + i < kblocks) o[(int64_t)(b + i) * 128] = w[i];
    }
}

struct PairArgs {
    const uint8_t *sa, *sb;   // scale bytes of A and B
    const uint16_t* bias;
    uint16_t* out;
    int64_t m, n;
    uint32_t idesc;
    int64_t groups;
    int m_tiles, n_tiles, ksteps, tma_out;
    PairWork work;
    uint32_t idesc_half;
    int ordered;              // the scale bytes have been put in order ahead
};

template <bool FP4>
struct PairShape {
    static constexpr int kBlk = FP4 ? 2 : 1;
    static constexpr int kTile = 128 * 128;                                  // bytes of 128 rows of an operand, one step
    static constexpr int kSfP = kBlk * 512, kSfQ = 2 * kSfP;
    static constexpr int kSfOff = 2 * kTile, kStage = kSfOff + ((kSfP + kSfQ + 1023) & ~1023);
    static constexpr int kStages = 5;
    static constexpr int kOutOff = kStages * kStage, kOutBytes = 128 * 128;  // 128 x 64 results on their way out, one for each half of the columns
    static constexpr int kSmem = kOutOff + 2 * kOutBytes + 1024;
    static constexpr int kSfCols = 12 * kBlk;                                // columns of tensor memory for a step's scales
    static_assert(kSmem <= 227 * 1024 - 2048, "shared memory");
};

// Each operand byte crosses from L2 once for 256 rows of the other operand (11 to 13 TB/s for the whole card at the rates
// above; single CTAs on 128 x 128 need twice that and take 290 us where pairs take 103).
// Warps 0-7 write the results, warp 8 loads, warp 9 issues (in the first CTA) or says that this CTA's operands are there
// (in the second).  Each CTA loads 128 rows of either operand, A's scales for its rows and B's for all 256 columns.  The
// accumulator fills half of tensor memory and the scales need some of the rest, so there is one: between two tiles the
// issuer waits until it is in registers, packed to bf16 (64 of them a thread); the stores go on under the next tile.
template <bool FP4>
__global__ void __launch_bounds__(320, 1) mx_matmul_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                                const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
                                                                const __grid_constant__ CUtensorMap map_out, const PairArgs a) {
    using S = PairShape<FP4>;
    extern __shared__ uint8_t s_raw[];
    __shared__ __align__(8) uint64_t full[S::kStages], empty[S::kStages], acc_full, acc_empty, drained;
    __shared__ uint32_t s_tmem;
    __shared__ __align__(16) float s_bias[256];
    __shared__ int s_late[2];   // a wait ran out: copies may still land in the operands' memory
    uint8_t* smem = s_raw + ((1024 - (smem_u32(s_raw) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank();
    const int pair = (int)(blockIdx.x >> 1);
    if (warp == 8 && lane == 0) {
        for (int s = 0; s < S::kStages; ++s) { mbar_init(&full[s], (rank == 0 ? 2 : 1) + (a.ordered ? 0 : 8)); mbar_init(&empty[s], 1); }
        mbar_init(&acc_full, 1);
        mbar_init(&acc_empty, 16);
        mbar_init(&drained, 1);
        s_late[0] = s_late[1] = 0;
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a));
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b));
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_sa));
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_sb));
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_out));
    }
    if (warp == 9) tmem_alloc<2>(&s_tmem, 512);
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    pdl_launch_dependents();
    pdl_wait();

    bool ok = true;   // a wait that ran out ends the role; what it would have computed is written as NaN
    if (warp == 8) {
        Slot<S::kStages> sl;
        for (int i = 0, t, part; ok && a.work.piece(i, pair, t, part); ++i) {
            int tm, tn;
            tile_place(t, a.m_tiles, a.n_tiles, tm, tn);
            // of a half tile each CTA brings 64 rows of B; the copy takes 64 more, which nobody reads
            const int row_b = tn * 256 + (part < 0 ? rank * 128 : part * 128 + rank * 64), block_b = tn * 2 + (part > 0 ? 1 : 0);
            for (int j = 0; j < a.ksteps; ++j) {
                ok = mbar_wait_warp(&empty[sl.s], sl.phase ^ 1);
                if (!ok) break;
                if (elect_one()) {
                    uint8_t* st = smem + sl.s * S::kStage;
                    uint64_t* bar = &full[sl.s];
                    mbar_expect_tx(bar, 2 * S::kTile + (a.ordered ? S::kSfP + S::kSfQ : 0));
                    tma_load_2d(st, &map_a, j * 128, tm * 256 + rank * 128, bar);
                    tma_load_2d(st + S::kTile, &map_b, j * 128, row_b, bar);
                    if (a.ordered) {
                        tma_load_2d(st + S::kSfOff, &map_sa, j * (S::kBlk * 128), tm * 2 + rank, bar);
                        tma_load_2d(st + S::kSfOff + S::kSfP, &map_sb, j * (S::kBlk * 128), block_b, bar);
                    }
                }
                __syncwarp();
                sl.advance();
            }
        }
        if (!ok)   // copies in flight land before the shared memory is handed on: every slot's last round
            for (int s = 0; s < S::kStages; ++s) mbar_wait_bounded(&full[s], s < sl.s ? sl.phase : sl.phase ^ 1);
    } else if (warp == 9) {
        Slot<S::kStages> sl;
        if (rank == 1) {
            const uint32_t full0 = map_to_rank(smem_u32(&full[0]), 0);
            const int64_t total = (int64_t)a.work.pieces(pair) * a.ksteps;
            for (int64_t i = 0; i < total; ++i) {
                if (!mbar_wait_warp(&full[sl.s], sl.phase)) break;
                if (elect_one()) mbar_arrive_peer(full0 + 8 * sl.s);
                __syncwarp();
                sl.advance();
            }
        } else {
            const uint64_t d0 = umma_desc_kmajor(smem_u32(smem));
            for (int it = 0, t, part; ok && a.work.piece(it, pair, t, part); ++it) {
                const uint32_t idesc = part < 0 ? a.idesc : a.idesc_half;
                if (it > 0) ok = mbar_wait_warp(&acc_empty, (it - 1) & 1);
                if (!ok) break;
                for (int j = 0; j < a.ksteps; ++j) {
                    ok = mbar_wait_warp(&full[sl.s], sl.phase);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t sf = smem_u32(smem) + sl.s * S::kStage + S::kSfOff;
                        const uint32_t tp = tmem + 256 + (j & 1) * S::kSfCols, tq = tp + 4 * S::kBlk;
#pragma unroll
                        for (int b = 0; b < S::kBlk; ++b) {   // a block is four groups of K: four columns for A's 128 rows, eight for B's 256
                            tc_copy_scales<2>(tp + 4 * b, sf + 512 * b);
                            tc_copy_scales<2>(tq + 8 * b, sf + S::kSfP + 512 * b);
                            if (part < 0) tc_copy_scales<2>(tq + 8 * b + 4, sf + 2 * S::kSfP + 512 * b);
                        }
                        const uint64_t da = d0 + sl.s * (S::kStage / 16), db = da + S::kTile / 16;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {   // 32 bytes of K each
                            const uint32_t blk = FP4 ? k >> 1 : 0, id = FP4 ? (k & 1) * 2 : k;
                            tc_mma_scaled<2, FP4>(tmem, da + 2 * k, db + 2 * k, idesc_with_scale_id(idesc, id), tp + 4 * blk, tq + 8 * blk, (j | k) != 0);
                        }
                        tc_commit_pair(&empty[sl.s]);
                        if (j == a.ksteps - 1) tc_commit_pair(&acc_full);
                    }
                    __syncwarp();
                    sl.advance();
                }
            }
            if (!ok) {   // products in flight end before the tensor memory is handed on
                if (elect_one()) tc_commit_pair(&drained);
                __syncwarp();
                mbar_wait_bounded(&drained, 0);
            }
        }
    } else {
        const int half = warp >> 2, t128 = threadIdx.x & 127;   // columns 128 half ..., accumulator row
        const uint32_t empty0 = map_to_rank(smem_u32(&acc_empty), 0);
        uint8_t* os = smem + S::kOutOff + half * S::kOutBytes;
        if (!a.ordered) {   // the pair's only tile: these warps have nothing to write yet
            int t, part, tm, tn;
            a.work.piece(0, pair, t, part);
            tile_place(t, a.m_tiles, a.n_tiles, tm, tn);
            constexpr int W = kBatch * S::kBlk;
            const bool has_q = part < 0 || half == 0;
            const int64_t row_p = (int64_t)tm * 256 + rank * 128 + t128, row_q = (int64_t)tn * 256 + (part > 0 ? 128 : 0) + threadIdx.x;
            const uint32_t sf = smem_u32(smem) + S::kSfOff + (t128 & 31) * 16 + (t128 >> 5) * 4, sfq = sf + S::kSfP * (1 + half);
            Slot<S::kStages> sl;
            ScaleWords<W> p, q, next_p, next_q;
            if (half == 0) p.load(a.sa, a.m, a.groups, row_p, 0);
            if (has_q) q.load(a.sb, a.n, a.groups, row_q, 0);
            for (int i = 0; i < a.ksteps && ok; i += kBatch) {
                if (i + kBatch < a.ksteps) {
                    const int64_t g = (int64_t)(i + kBatch) * (4 * S::kBlk);
                    if (half == 0) next_p.load(a.sa, a.m, a.groups, row_p, g);
                    if (has_q) next_q.load(a.sb, a.n, a.groups, row_q, g);
                }
                uint32_t wp[W], wq[W];
                if (half == 0) p.place(wp);
                if (has_q) q.place(wq);
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    if (i + u >= a.ksteps) break;
                    ok = mbar_wait_warp(&empty[sl.s], sl.phase ^ 1);
                    if (!ok) break;
#pragma unroll
                    for (int b = 0; b < S::kBlk; ++b) {
                        if (half == 0) store_word(sf + sl.s * S::kStage + 512 * b, wp[u * S::kBlk + b]);
                        if (has_q) store_word(sfq + sl.s * S::kStage + 512 * b, wq[u * S::kBlk + b]);
                    }
                    fence_async_shared();
                    __syncwarp();
                    if (elect_one()) mbar_arrive(&full[sl.s]);
                    sl.advance();
                }
                p = next_p;
                q = next_q;
            }
        }
        for (int it = 0, t, part; a.work.piece(it, pair, t, part); ++it) {
            int tm, tn;
            tile_place(t, a.m_tiles, a.n_tiles, tm, tn);
            const int columns = part < 0 ? 128 : 64;   // of these four warps
            const uint32_t acc = tmem + half * columns + ((uint32_t)(warp & 3) << 21);
            const int64_t m0 = (int64_t)tm * 256 + rank * 128, n0 = (int64_t)tn * 256 + (part > 0 ? 128 : 0) + half * columns;
            if (a.bias) {
                named_barrier(1 + half, 128);   // the tile before is through with these
                s_bias[half * 128 + t128] = n0 + t128 < a.n ? u2f((uint32_t)__ldg(a.bias + n0 + t128) << 16) : 0.0f;
                named_barrier(1 + half, 128);
            }
            ok = ok && mbar_wait_warp(&acc_full, it & 1);
            tc_fence_after();
            uint32_t w[64];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (32 * c >= columns) break;
                uint32_t r[32];
                tmem_load32(acc + 32 * c, r);
                tmem_wait_loads();
                if (a.bias) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4 v = *reinterpret_cast<const float4*>(&s_bias[half * 128 + 32 * c + e]);
                        r[e] = f2u(u2f(r[e]) + v.x);
                        r[e + 1] = f2u(u2f(r[e + 1]) + v.y);
                        r[e + 2] = f2u(u2f(r[e + 2]) + v.z);
                        r[e + 3] = f2u(u2f(r[e + 3]) + v.w);
                    }
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) w[16 * c + e] = pack_bf16_rne(u2f(r[2 * e + 1]), u2f(r[2 * e]));
            }
            tc_fence_before();
            __syncwarp();
            if (elect_one()) mbar_arrive_peer(empty0);
            if (!ok) s_late[half] = 1;
            bool at_once = false;   // after the last tile the operands' shared memory is free: both 64 columns go out at once
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if (64 * c >= columns) break;
                uint8_t* to = c == 1 && at_once ? smem + half * S::kOutBytes : os;
                if (c == 0 || !at_once) {
                    if (t128 == 0) bulk_wait_reads();
                    named_barrier(1 + half, 128);
                }
                const bool late = s_late[half] != 0;
                if (c == 0) at_once = !late && it + 1 == a.work.pieces(pair);
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const uint32_t* v = w + 32 * c + 4 * q;
                    *reinterpret_cast<uint4*>(to + t128 * 128 + ((q ^ (t128 & 7)) << 4)) =
                        late ? make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu) : make_uint4(v[0], v[1], v[2], v[3]);
                }
                fence_async_shared();
                named_barrier(1 + half, 128);
                const int64_t nc = n0 + 64 * c;
                if (a.tma_out) {
                    if (t128 == 0) {
                        if (m0 < a.m && nc < a.n) tma_store_2d(&map_out, to, (int)nc, (int)m0);
                        bulk_commit();
                    }
                } else {   // rows that do not start on 16 bytes: a warp writes one row at a time
                    for (int r = (warp & 3) * 32; r < (warp & 3) * 32 + 32 && m0 + r < a.m; ++r) {
                        const uint32_t v = *reinterpret_cast<const uint32_t*>(to + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
                        uint16_t* o = a.out + (m0 + r) * a.n + nc + 2 * lane;
                        if (nc + 2 * lane < a.n) o[0] = (uint16_t)v;
                        if (nc + 2 * lane + 1 < a.n) o[1] = (uint16_t)(v >> 16);
                    }
                }
            }
        }
        if (t128 == 0) bulk_wait_reads();
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();
    if (warp == 9) { tc_fence_after(); tmem_free<2>(tmem, 512); }
}

// columns of scale blocks of a row of tiles, padded to whole steps of either format
inline int64_t scale_blocks(int64_t k) { return ((k / 32 + 3) / 4 + 1) & ~int64_t(1); }

// Pairs that take one tile each have warps to spare for fetching scale bytes; those that go on to further tiles have not,
// and the kernel that puts the bytes in order first costs them little.  It costs the others a launch and about a microsecond:
// 1024 x 4096 x 4096 E4M3 17.6 us with it, 17.0 without.
inline bool orders_scales(int64_t m, int64_t n) { return ((m + 255) / 256) * ((n + 255) / 256) > sm_count() / 2; }

// The scale bytes of both operands in tensor-core order, in the workspace, and the maps that load them: blk blocks of 128
// rows for A, of 256 for B
bool order_scales(const MxMatmulArgs& x, int blk, CUtensorMap* map_a, CUtensorMap* map_b, cudaStream_t st) {
    const int64_t kb = scale_blocks(x.k), rb_a = (x.m + 127) / 128, rb_b = (x.n + 127) / 128, groups = x.k / 32;
    auto* sa = static_cast<uint32_t*>(x.workspace);
    uint32_t* sb = sa + rb_a * kb * 128;
    if (!make_word_map(map_a, sa, rb_a, kb * 128, blk * 128, 1) || !make_word_map(map_b, sb, rb_b, kb * 128, blk * 128, 2)) return false;
    const int fast = groups % 16 == 0 && ((reinterpret_cast<uintptr_t>(x.a_scales) | reinterpret_cast<uintptr_t>(x.b_scales)) & 15) == 0;
    const dim3 grid((unsigned)(rb_a + rb_b), (unsigned)std::min<int64_t>((kb + 3) / 4, 64));
    return launch_pdl(order_scales_kernel, grid, dim3(128), 0, st, x.a_scales, x.m, sa, (int)rb_a, x.b_scales, x.n, sb, groups, (int)kb, fast) == cudaSuccess;
}

template <bool FP4>
int go_pair(const MxMatmulArgs& x, cudaStream_t st) {
    using S = PairShape<FP4>;
    auto kern = mx_matmul_pair_kernel<FP4>;
    static SmemOptIn opt;
    if (!opt(kern, S::kSmem)) return kErrLaunch;
    PairArgs a = {};
    a.bias = static_cast<const uint16_t*>(x.bias);
    a.out = static_cast<uint16_t*>(x.out);
    a.m = x.m; a.n = x.n;
    a.m_tiles = (int)((x.m + 255) / 256); a.n_tiles = (int)((x.n + 255) / 256);
    if ((int64_t)a.m_tiles * a.n_tiles > (1 << 30)) return kErrTooLarge;
    a.work = pair_work((int64_t)a.m_tiles * a.n_tiles, sm_count());
    const int64_t row_bytes = FP4 ? x.k / 2 : x.k;
    a.ksteps = (int)((row_bytes + 127) / 128);
    a.idesc = idesc_scaled(256, 256, FP4 ? 1u : (uint32_t)x.a_fmt, FP4 ? 1u : (uint32_t)x.b_fmt);
    a.idesc_half = idesc_scaled(256, 128, FP4 ? 1u : (uint32_t)x.a_fmt, FP4 ? 1u : (uint32_t)x.b_fmt);
    a.tma_out = x.n % 8 == 0 && (reinterpret_cast<uintptr_t>(x.out) & 15) == 0;
    CUtensorMap ma, mb, msa, msb, mo;
    if (!make_swizzled_map(&ma, x.a, x.m, row_bytes, row_bytes, 1, 128) || !make_swizzled_map(&mb, x.b, x.n, row_bytes, row_bytes, 1, 128)) return kErrLaunch;
    if (!a.tma_out) mo = ma;
    else if (!make_swizzled_map(&mo, x.out, x.m, x.n, x.n * 2, 2, 128)) return kErrLaunch;
    a.sa = x.a_scales; a.sb = x.b_scales;
    a.groups = x.k / 32;
    a.ordered = orders_scales(x.m, x.n);
    if (!a.ordered) msa = msb = ma;   // not used
    else if (!order_scales(x, S::kBlk, &msa, &msb, st)) return kErrLaunch;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * a.work.launched()));
    cfg.blockDim = dim3(320);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {2, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, ma, mb, msa, msb, mo, a) == cudaSuccess ? check_launch() : kErrLaunch;
}

template <bool FP4, int TN, bool SWAP>
int go(const CUtensorMap& mp, const CUtensorMap& mq, const MmArgs& a, int64_t tiles, cudaStream_t st) {
    using S = MmShape<FP4, TN>;
    auto k = mx_matmul_kernel<FP4, TN, SWAP>;
    static SmemOptIn opt;
    if (!opt(k, S::kSmem)) return kErrLaunch;
    if (tiles * a.splits > 0x7FFFFFFF) return kErrTooLarge;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * a.splits));
    cfg.blockDim = dim3(192);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {(unsigned)a.splits, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = a.splits > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, mp, mq, a) == cudaSuccess ? check_launch() : kErrLaunch;
}

template <bool FP4>
int dispatch(const MxMatmulArgs& x, cudaStream_t st) {
    if (!bind_context()) return kErrLaunch;
    const int64_t row_bytes = FP4 ? x.k / 2 : x.k;
    const bool swap = x.m <= 64;
    if (!swap && takes_pairs(x.m, x.n, (row_bytes + 127) / 128, sm_count(), kPairsBelow)) return go_pair<FP4>(x, st);
    const int tn = !swap ? 128 : (x.m <= 16 ? 16 : (x.m <= 32 ? 32 : 64));
    MmArgs a = {};
    const void *p = swap ? x.b : x.a, *q = swap ? x.a : x.b;
    a.sp = swap ? x.b_scales : x.a_scales;
    a.sq = swap ? x.a_scales : x.b_scales;
    a.p_rows = swap ? x.n : x.m;
    a.q_rows = swap ? x.m : x.n;
    a.bias = static_cast<const uint16_t*>(x.bias);
    a.out = static_cast<uint16_t*>(x.out);
    a.groups = x.k / 32;
    a.ldo = x.n;
    a.p_tiles = (a.p_rows + kPRows - 1) / kPRows;
    a.ktiles = (int)((row_bytes + 127) / 128);
    const int pf = swap ? x.b_fmt : x.a_fmt, qf = swap ? x.a_fmt : x.b_fmt;
    a.idesc = idesc_scaled(128, tn, FP4 ? 1u : (uint32_t)pf, FP4 ? 1u : (uint32_t)qf);
    a.vec_out = x.n % 4 == 0 && (reinterpret_cast<uintptr_t>(x.out) & 7) == 0;   // eight bytes hold four columns
    const int64_t tiles = a.p_tiles * ((a.q_rows + tn - 1) / tn);
    a.splits = k_splits(tiles, a.ktiles, sm_count());
    CUtensorMap mp, mq;
    if (!make_swizzled_map(&mp, p, a.p_rows, row_bytes, row_bytes, 1, kPRows)) return kErrLaunch;
    if (!make_swizzled_map(&mq, q, a.q_rows, row_bytes, row_bytes, 1, tn)) return kErrLaunch;
    if (!swap) return go<FP4, 128, false>(mp, mq, a, tiles, st);
    if (tn == 16) return go<FP4, 16, true>(mp, mq, a, tiles, st);
    if (tn == 32) return go<FP4, 32, true>(mp, mq, a, tiles, st);
    return go<FP4, 64, true>(mp, mq, a, tiles, st);
}

}  // namespace

size_t mx_matmul_workspace(int64_t m, int64_t n, int64_t k, int fp4) {
    const int64_t steps = ((fp4 ? k / 2 : k) + 127) / 128;
    if (m <= 64 || !takes_pairs(m, n, steps, sm_count(), kPairsBelow) || !orders_scales(m, n)) return 0;
    return (size_t)(((m + 127) / 128 + (n + 127) / 128) * scale_blocks(k) * 512);
}

int launch_mx_matmul(const MxMatmulArgs& x, cudaStream_t st) {
    return x.a_fmt == kE2M1 ? dispatch<true>(x, st) : dispatch<false>(x, st);
}

}  // namespace morb
