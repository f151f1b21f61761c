// Fifth-generation tensor core: descriptors and instruction wrappers shared by the matrix-product kernels.
//
// Shared-memory operands are tiles whose rows are 128 bytes long under the 128-byte swizzle that TMA writes; a
// descriptor names the tile's first byte, and the next slice along the contraction starts 32 bytes further (K-major)
// or a few 8-row groups further (MN-major).  Accumulators and block scales live in tensor memory.
#pragma once

#include "tma.cuh"

namespace morb {

// shared-memory operand descriptor: 14-bit fields in units of 16 bytes, version 1, layout 2 = 128-byte swizzle, 0 = none
__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, uint32_t lbo_bytes, uint32_t sbo_bytes, uint32_t layout) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo_bytes >> 4) << 16) | ((uint64_t)(sbo_bytes >> 4) << 32) |
           (1ull << 46) | ((uint64_t)layout << 61);
}
constexpr uint32_t kLayoutNone = 0, kLayoutSwizzle128 = 2;

// K-major tile, rows of 128 bytes, groups of eight rows 1024 bytes apart
__device__ __forceinline__ uint64_t umma_desc_kmajor(uint32_t addr) { return umma_desc(addr, 16, 1024, kLayoutSwizzle128); }

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t columns) {   // one whole warp
    if constexpr (CG == 1)
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(columns) : "memory");
    else
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(columns) : "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {     // the warp that allocated
    if constexpr (CG == 1) {
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
    } else {
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
    }
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// arrives on the barrier when every tensor-core operation issued so far by this thread is done
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// the same on the barrier at this offset in both CTAs of a pair
__device__ __forceinline__ void tc_commit_pair(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}

// 512 bytes of scales, 16 bytes a row for 32 rows, to four columns of tensor memory (repeated in every quarter of the lanes)
template <int CG>
__device__ __forceinline__ void tc_copy_scales(uint32_t taddr, uint32_t saddr) {
    const uint64_t d = umma_desc(saddr, 128, 128, kLayoutNone);
    if constexpr (CG == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
    else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}

// D (+)= A * B with block scales: 4-bit elements (64 of K, two scales a row) or 8-bit ones (32 of K, one scale)
template <int CG, bool FP4>
__device__ __forceinline__ void tc_mma_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (CG == 1 && FP4)
        asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %6, 0;\n"
                     "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
    else if constexpr (CG == 1)
        asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %6, 0;\n"
                     "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
    else if constexpr (FP4)
        asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %6, 0;\n"
                     "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
    else
        asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %6, 0;\n"
                     "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// bf16 elements (16 of K)
template <int CG>
__device__ __forceinline__ void tc_mma_bf16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
                     "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\n"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// instruction descriptors
// bf16 operands, binary32 accumulator; a major-ness bit is 1 where the operand's rows run along M (or N) instead of K
__host__ __device__ constexpr uint32_t idesc_bf16(int m, int n, bool a_mn, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}
// block-scaled operands, E8M0 scales; fields for the scale bytes to use: B in bits 4-5, A in bits 29-30
__host__ __device__ constexpr uint32_t idesc_scaled(int m, int n, uint32_t a_fmt, uint32_t b_fmt) {
    return (a_fmt << 7) | (b_fmt << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27);
}
__device__ __forceinline__ uint32_t idesc_with_scale_id(uint32_t idesc, uint32_t id) { return idesc | (id << 4) | (id << 29); }

// 32 consecutive columns of this warp's quarter of the lanes: one accumulator row per lane
__device__ __forceinline__ void tmem_load32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_load16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// a tile of shared memory to global memory under the map's swizzle; what lies outside the tensor is not written
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(smem_u32(src)) : "memory");
}
template <int N>
__device__ __forceinline__ void bulk_wait_reads_but() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
// a barrier of some warps of the CTA
__device__ __forceinline__ void named_barrier(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// clusters
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}

// arrival on a barrier of another CTA of the cluster (its shared::cluster address), and the wait that pairs with it
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t remote) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
}
// The same without a fence to the cluster's scope, which takes about 0.9 us: for a CTA that vouches for what lies in its
// own shared memory and is read there, by its own SM's tensor core, after the writers' proxy fences.
__device__ __forceinline__ void mbar_arrive_peer(uint32_t remote) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
}
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity) {   // bounded, by a whole warp
    bool done = false;
    for (uint32_t spin = 0; spin < kSpinLimit; ++spin) {
        uint32_t ok;
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                     : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
        if (ok) { done = true; break; }
    }
    return __all_sync(0xFFFFFFFFu, done) != 0;
}

// One lane of a converged warp.  The roles of a product kernel run as whole warps, every lane waiting on the barriers, and
// only what is issued once is issued by the elected lane: a wait in a branch of one lane takes 190 cycles even when it is
// over before it begins, one of a whole warp 90.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}
// a whole warp waits, and all its lanes learn alike whether the wait ran out
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity) {
    return __all_sync(0xFFFFFFFFu, mbar_wait_bounded(bar, parity)) != 0;
}

// Sums over the CTAs of a cluster that each hold partial sums of one tile of 128 rows: the CTA of rank z adds up rows
// [z, z + 1) 128 / splits.  Every CTA pushes its rows to their owners in 16-byte stores (remote loads would wait some 200
// cycles each) once all are done with the shared memory they land in, then each owner adds in rank order, so results do
// not depend on timing.  N columns, rows of N + 4 words: neighbouring rows start four banks apart.
template <int N>
struct ClusterSum {
    static constexpr int kPitch = N + 4, kBytes = 128 * kPitch * 4;
    uint32_t base;      // the same place in every CTA
    int splits, rank;
    __device__ __forceinline__ int rows() const { return 128 / splits; }
    __device__ __forceinline__ uint32_t place(int row) const {   // where this CTA's part of a row goes
        const int owner = row / rows();
        return map_to_rank(base, owner) + (uint32_t)((rank * rows() + row - owner * rows()) * kPitch) * 4;
    }
    __device__ __forceinline__ static void push(uint32_t to, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
        asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
    }
    __device__ __forceinline__ float4 sum4(int local_row, int col) const {   // after the cluster has met again
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int z = 0; z < splits; ++z) {
            float4 v;
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                         : "r"(base + (uint32_t)((z * rows() + local_row) * kPitch + col) * 4) : "memory");
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        return s;
    }
};

// four-byte asynchronous copies, zero-filled where `valid` is 0
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, int valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
}
// one arrival on the barrier when all such copies of this thread so far have landed
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// two binary32 values to a packed bf16 word, round to nearest even (lo = the element at the lower address)
__device__ __forceinline__ uint32_t pack_bf16_rne(float hi, float lo) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// 2 ** (byte - 127), NaN for 255
__device__ __forceinline__ float e8m0_to_f32(uint32_t byte) {
    return u2f(byte == 0 ? 0x00400000u : (byte == 255u ? 0x7FFFFFFFu : byte << 23));
}

// The encoder of tensor maps is a driver call and wants a context on the calling thread; a thread whose first CUDA call
// this is (an autograd worker) has none until the runtime is told its device.
inline bool bind_context() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
}

// a place in a ring of N slots and the parity of the round
template <int N>
struct Slot {
    int s = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void advance(int by = 1) {
        if ((s += by) >= N) { s -= N; phase ^= 1; }
    }
};

// Output tile number -> its place: bands of eight rows of tiles, down a band's columns, so that the CTAs at work at one
// time share rows of one operand and columns of the other in L2.
__device__ __forceinline__ void tile_place(int t, int m_tiles, int n_tiles, int& tm, int& tn) {
    constexpr int kBand = 8;
    const int band = t / (kBand * n_tiles), in = t - band * (kBand * n_tiles);
    const int rows = min(kBand, m_tiles - band * kBand);
    tn = in / rows;
    tm = band * kBand + in - tn * rows;
}

// The work of the pairs of CTAs on 256 x 256 tiles: `rounds` whole tiles each, then the tiles that are left, as halves of 128
// columns where there are pairs for them: 1024^3 E4M3 (16 tiles) 7.9 us in whole tiles, 6.8 in halves; gradient 512 x 4096 x
// 4096 27.3 and 23.9; 2560 x 2560 x 8192 4-bit (100 tiles) 28.4 and 26.4.
struct PairWork {
    int pairs, rounds, rest, halves;
    __host__ __device__ int launched() const { return rounds ? pairs : (halves ? 2 * rest : rest); }
    // the i-th piece of a pair: a tile, and which half of its columns (-1: all)
    __device__ __forceinline__ bool piece(int i, int pair, int& tile, int& half) const {
        half = -1;
        tile = i * pairs + pair;
        if (i < rounds) return true;
        if (i > rounds || pair >= (halves ? 2 * rest : rest)) return false;
        if (halves) {
            half = pair & 1;
            tile = rounds * pairs + (pair >> 1);
        }
        return true;
    }
    __device__ __forceinline__ int pieces(int pair) const { return rounds + (pair < (halves ? 2 * rest : rest) ? 1 : 0); }
};
inline PairWork pair_work(int64_t tiles, int sms) {
    PairWork w = {};
    w.pairs = sms / 2;
    w.rounds = (int)(tiles / w.pairs);
    w.rest = (int)(tiles % w.pairs);
    w.halves = w.rest > 0 && 2 * w.rest <= w.pairs;
    return w;
}

// How many CTAs of a cluster share the sum over k of a tile, when single CTAs take tiles of 128 x (n per tile): as many as leave each
// an SM of its own and four steps.  A cluster lies within one group of the card's SMs, so of those with one CTA an SM 74 of two are
// resident at a time, but 32 of four (34 are not) and 15 of eight (16 are not), and the ones that wait take a second round:
// one token x 2048 x 4096 E4M3 (16 tiles) in eighths 9.5 us, in quarters 6.2; x 4352 (34) in quarters 11.8, in halves 8.4;
// gradients 128 x 2048 x 4096 24.8 and 15.7, 128 x 4352 x 4096 30.9 and 21.4.
inline int k_splits(int64_t tiles, int64_t steps, int sms) {
    int s = 1;
    while (s < 8 && tiles <= (s == 1 ? sms / 2 : (s == 2 ? 32 : 15)) && steps >= s * 4) s *= 2;
    return s;
}
// Pairs of CTAs on 256 x 256 or single ones on 128 x 128?  A pair takes a step in about the time of a single CTA with four
// times the result, so pairs win unless few tiles let single CTAs split the sum: each step saved is worth about 0.3 us,
// meeting in the cluster costs about 4 in a product, 7 in a gradient, whose CTAs have more to set up; `limit` is what has to be
// saved.  Measured on both sides, pairs and single, in us (steps saved).  Products, 14: 128 x 4096 x 4096 E4M3 14.5 and 12.2
// (24), 4-bit 10.7 and 10.9 (12); 256 x 4096 x 4096 E4M3 14.5 and 13.9 (16), 4-bit 10.7 and 11.7 (8); 128 x 1024 x 2048 E4M3
// 9.1 and 9.0 (14), 512 x 1024 x 2048 9.1 and 10.5 (12), x 8192 24.3 and 14.8 (48); 100 x 8192 x 8192 4-bit 18.0 and 15.2 (16);
// 1111 x 1003 x 2080 4-bit 10.5 and 12.6 (5); 1536 x 1536 x 4096 E4M3 15.5 and 20.2 (0).  Gradients, 24: 128 x 4096 x 1024 9.5
// and 12.4 (12), x 1536 11.8 and 13.2 (18), x 2048 14.1 and 14.0 (24), x 4096 22.7 and 17.2 (48); 256 x 4096 x 2560 16.4 and 17.4
// (20), x 4096 22.9 and 22.0 (32); 512 x 1024 x 2048 13.5 and 13.8 (24); 128 x 1024 x 1024 8.9 and 10.7 (14).  Gradients whose scale
// bytes a pair's two warps fetch one by one, 14: 128 x 4000 x 1536 16.0 and 13.6 (18), 256 x 4000 x 1536 16.2 and 15.5 (12),
// 300 x 992 x 1000 11.4 and 11.8 (12), 1000 x 992 x 1024 11.6 and 13.1 (8).
inline bool takes_pairs(int64_t m, int64_t n, int64_t steps, int sms, int limit) {
    const int s = k_splits(((m + 127) / 128) * ((n + 127) / 128), steps, sms);
    return steps - steps / s < limit;
}

// row-major matrix of bytes (or bf16) with a row pitch, boxes of 128 bytes x box_rows under the 128-byte swizzle; what lies outside reads as zero
inline bool make_swizzled_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t pitch_bytes, int elem_bytes,
                              int box_rows) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return false;
    const cuuint64_t gdim[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t gstride[1] = {(cuuint64_t)pitch_bytes};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / elem_bytes), (cuuint32_t)box_rows};
    const cuuint32_t estride[2] = {1, 1};
    return fn(map, elem_bytes == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), gdim,
              gstride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// row-major matrix of 32-bit words, boxes of box_cols x box_rows without swizzle
inline bool make_word_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int box_cols, int box_rows) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return false;
    const cuuint64_t gdim[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t gstride[1] = {(cuuint64_t)cols * 4};
    const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
    const cuuint32_t estride[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), gdim, gstride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace morb
