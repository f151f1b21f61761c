// Product of a bf16 gradient with a microscaled matrix kept in 8 or 4 bits, out[m, n] = sum_k op(g)[m, k] W[k, n], W =
// decode(codes) * 2^(scale - 127): a linear layer's input gradient from its quantised weights (op(g) = g) and its weight
// gradient from the quantised activations (op(g) = g transposed).  The scales of W lie along n, so they cannot be
// multiplied into a product over k by the tensor core; the codes are widened to bf16 (exact: four significant bits at
// most) on the way from the staged codes to the operand tile, which costs no global traffic beyond the codes.
//
// One kernel, persistent over output tiles.  Per step of 64 k warp 4 requests the gradient's tile by TMA, warp 6 the
// codes, warps 7-8 their scale bytes, the widening warps turn the codes into the operand tile, warp 5 issues the products, and
// warps 0-3 write one tile by TMA while the next accumulates (two accumulators).  The gradient's tiles, the codes and the widened tiles pass through rings of their own: codes are let go as soon as they are
// in registers, and a widened tile is needed only briefly, so most of the shared memory covers the latency of loads.
// In its large form two CTAs work as a pair on 256 x 256: each loads 128 rows of the gradient and widens 128 columns of W,
// so every widened element meets 256 rows.
//
// A step of a pair is 0.287 us of the tensor core.  8192 x 4096 x 4096 E4M3: 188 to 195 us in a short run (1.41 to 1.46
// PFLOP/s), 213 to 227 us in a long one (power limit).  Of its cycles the tensor pipe is active in 76 %, the integer pipe, which
// widens, in 50 %, the shared-memory pipe in 69 %.  Two widening groups of four warps took 207 us, three
// 187, four 188 (4096^3 4-bit: 139, 121, 116): what counts is that a group's waits hide behind the others' work.
#include <algorithm>
#include <type_traits>

#include "mx_kernels.cuh"
#include "tcgen05.cuh"

namespace morb {
namespace {

struct GrArgs {
    const uint8_t* scales;
    uint16_t* out;
    int64_t m, n, k, groups;
    int m_tiles, n_tiles, tiles;
    int ksteps, across, splits, fast_scales;
    PairWork work;              // pairs
};

constexpr int kTK = 64;                 // k a step: 128 bytes of bf16
constexpr int kABytes = 128 * kTK * 2;  // a CTA's rows of the gradient
constexpr int kConvWarps = 4, kConvGroups = 4;   // warps that widen a step together; the groups take the steps in turn
constexpr int kFirstConv = 9;                    // warps 0-3 write, 4 gradient, 5 products, 6 codes, 7-8 scales
constexpr int kThreads = 32 * (kFirstConv + kConvWarps * kConvGroups);

template <int FMT, int CG, int NB>      // CTAs to a tile; columns of W that one CTA widens
struct GrShape {
    static constexpr int kTM = 128 * CG, kTN = NB * CG;
    static constexpr int kRowBytes = FMT == kE2M1 ? NB / 2 : NB;   // codes of one k
    static constexpr int kBBytes = NB * kTK * 2;
    static constexpr int kCodeBytes = kRowBytes * kTK, kCStage = kCodeBytes + kTK * 4;   // and their scale bytes
    static constexpr int kSA = 4, kSB = 4, kSC = 4;                // depths of the rings
    static constexpr int kBOff = kSA * kABytes, kCOff = kBOff + kSB * kBBytes;
    static constexpr int kOutOff = kCOff + ((kSC * kCStage + 1023) & ~1023), kOutBytes = 128 * 128;   // two tiles of 128 x 64 on their way out
    static constexpr int kSmem = kOutOff + 2 * kOutBytes + 1024;
    static constexpr int kCols = 2 * kTN;
    static_assert(kSmem > 114 * 1024, "one CTA per SM, so the columns of tensor memory suffice");
    static_assert(kSmem <= 227 * 1024 - 512 && (kCols == 256 || kCols == 512), "shape");
};

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Eight codes to eight bf16 values times the scale.  The exponent and mantissa of a code are the low bits of a bf16
// pattern's: moved there, the pattern stands for the value times 2^-120 (E4M3; 2^-112, 2^-126 for the others), subnormal
// codes included, since both formats count subnormals alike.  One multiplication by 2^(scale - 127 + 120) undoes that and
// applies the scale, with the only rounding there is.  It serves every scale whose product with 2^120 a bf16 holds and
// every code that is a number; `odd` gets a bit of kOdd for the rest, which widen8_any takes.  A byte permutation that repeats
// each code's sign up to the top of its half word leaves one shift and one mask for two codes: the widening warps fill
// the integer pipe, so each instruction here shows in the kernel's time.
constexpr uint32_t kOdd = 0x80808180u;
template <uint32_t SEL>
__device__ __forceinline__ uint32_t permute(uint32_t a, uint32_t b) {   // with the sign-repeating selectors 8-15, which __byte_perm drops
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "n"(SEL));
    return r;
}
template <int FMT>
__device__ __forceinline__ uint4 widen8(uint2 c, uint32_t scale, uint32_t& odd) {
    constexpr uint32_t lift = FMT == kE4M3 ? 120u : (FMT == kE5M2 ? 112u : 126u);
    uint32_t o[4];
    if constexpr (FMT == kE2M1) {
        const uint32_t lo = (c.x << 4) & 0xF0F0F0F0u, hi = c.x & 0xF0F0F0F0u;   // even and odd columns' codes on top of their bytes
        o[0] = (permute<0xC480u>(lo, hi) << 2) & 0x81C081C0u;
        o[1] = (permute<0xD591u>(lo, hi) << 2) & 0x81C081C0u;
        o[2] = (permute<0xE6A2u>(lo, hi) << 2) & 0x81C081C0u;
        o[3] = (permute<0xF7B3u>(lo, hi) << 2) & 0x81C081C0u;
    } else if constexpr (FMT == kE2M3) {
        const uint32_t w[2] = {c.x << 2, c.y << 2};                             // six bits: sign to the top of the byte
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            o[2 * i] = (permute<0x9180u>(w[i], 0) << 2) & 0x81F081F0u;
            o[2 * i + 1] = (permute<0xB3A2u>(w[i], 0) << 2) & 0x81F081F0u;
        }
    } else {
        constexpr int sh = FMT == kE4M3 ? 4 : 5;
        constexpr uint32_t mask = FMT == kE4M3 ? 0x87F087F0u : 0x8FE08FE0u;
        const uint32_t w[2] = {c.x, c.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            o[2 * i] = (permute<0x9180u>(w[i], 0) << sh) & mask;
            o[2 * i + 1] = (permute<0xB3A2u>(w[i], 0) << sh) & mask;
        }
        constexpr uint32_t past = FMT == kE4M3 ? 0x01010101u : 0x04040404u;     // carries into bit 7 from 0x7F, from 0x7C up
        odd |= (((c.x & 0x7F7F7F7Fu) + past) | ((c.y & 0x7F7F7F7Fu) + past)) & 0x80808080u;
    }
    const uint32_t up = scale * 0x00800080u + lift * 0x00800080u;               // both halves; right while scale + lift < 255
    odd |= (scale + lift + 1u) & 0x100u;
    return make_uint4(mul_bf16x2(o[0], up), mul_bf16x2(o[1], up), mul_bf16x2(o[2], up), mul_bf16x2(o[3], up));
}
template <int FMT>
__device__ __forceinline__ uint4 widen8_any(uint2 c, uint32_t scale) {
    const float k = e8m0_to_f32(scale);
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t h2;
        if constexpr (FMT == kE2M1) {
            const uint32_t b = (c.x >> (8 * i)) & 0xFFu;
            asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %1;\ncvt.rn.f16x2.e2m1x2 %0, a;\n}" : "=r"(h2) : "r"(b));
        } else {
            h2 = codes_to_h2<FMT>(((i < 2 ? c.x : c.y) >> (16 * (i & 1))) & 0xFFFFu);
        }
        o[i] = pack_bf16_rne(__fmul_rn(h_hi_to_f32(h2), k), __fmul_rn(h_lo_to_f32(h2), k));
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

template <int FMT, int CG, int NB>
__global__ void __launch_bounds__(kThreads, 1) mx_grad_kernel(const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_c,
                                                              const __grid_constant__ CUtensorMap map_out, const GrArgs a) {
    using S = GrShape<FMT, CG, NB>;
    extern __shared__ uint8_t s_raw[];
    __shared__ __align__(8) uint64_t full_a[S::kSA], empty_a[S::kSA], full_c[S::kSC], empty_c[S::kSC], wide[S::kSB], empty_b[S::kSB],
        acc_full[2], acc_empty[2], drained;
    __shared__ uint32_t s_tmem;
    __shared__ int s_late;   // a wait ran out: copies may still land where partial sums meet
    uint8_t* smem = s_raw + ((1024 - (smem_u32(s_raw) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CG == 2 ? (int)cluster_rank() : 0;
    // work of this CTA (pair): tiles first, first + step, ... over steps [k_first, k_first + ks) of each
    const int split = CG == 2 ? 0 : (int)(blockIdx.x % (unsigned)a.splits);
    const int first = CG == 2 ? (int)(blockIdx.x >> 1) : (int)(blockIdx.x / (unsigned)a.splits);
    const int step = CG == 2 ? (int)(gridDim.x >> 1) : (int)(gridDim.x / (unsigned)a.splits);
    const int k_first = (int)((int64_t)a.ksteps * split / a.splits), k_last = (int)((int64_t)a.ksteps * (split + 1) / a.splits);
    const int ks = k_last - k_first;
    // piece by piece: a tile, and which half of its columns
    auto piece = [&](int i, int& tile, int& half) {
        if constexpr (CG == 2) return a.work.piece(i, first, tile, half);
        tile = first + i * step;
        half = -1;
        return tile < a.tiles;
    };
    const int64_t whole = CG == 2 ? (a.work.halves ? (int64_t)a.work.rounds * ks : INT64_MAX) : INT64_MAX;   // steps before those of a half tile

    if (warp == 4 && lane == 0) {
        for (int s = 0; s < S::kSA; ++s) { mbar_init(&full_a[s], 1); mbar_init(&empty_a[s], 1); }
        for (int s = 0; s < S::kSB; ++s) { mbar_init(&wide[s], kConvWarps * CG); mbar_init(&empty_b[s], 1); }
        for (int s = 0; s < S::kSC; ++s) { mbar_init(&full_c[s], 1 + kTK); mbar_init(&empty_c[s], kConvWarps); }
        for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 4 * CG); }
        mbar_init(&drained, 1);
        s_late = 0;
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_g));
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_c));
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_out));
    }
    if (warp == 5) tmem_alloc<CG>(&s_tmem, S::kCols);
    tc_fence_before();
    if constexpr (CG == 2) cluster_sync(); else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    pdl_launch_dependents();
    pdl_wait();

    // A wait that ran out ends the role; what it would have computed is written as NaN.  A slot's first use finds its
    // `empty` barrier in the phase before the first: waiting for the parity opposite to the round's passes at once.
    bool ok = true;
    const ClusterSum<S::kTN> sums{smem_u32(smem), a.splits, split};
    if (warp == 4) {
        Slot<S::kSA> sa;
        for (int i = 0, t, half; ok && piece(i, t, half); ++i) {
            int tm, tn;
            tile_place(t, a.m_tiles, a.n_tiles, tm, tn);
            const int m0 = tm * S::kTM + rank * 128;
            for (int j = 0; j < ks; ++j) {
                ok = mbar_wait_warp(&empty_a[sa.s], sa.phase ^ 1);
                if (!ok) break;
                if (elect_one()) {
                    const int k0 = (k_first + j) * kTK;
                    uint8_t* as = smem + sa.s * kABytes;
                    mbar_expect_tx(&full_a[sa.s], kABytes);
                    if (a.across) {   // g is [k, m]: two boxes of 64 m x 64 k
                        tma_load_2d(as, &map_g, m0, k0, &full_a[sa.s]);
                        tma_load_2d(as + kABytes / 2, &map_g, m0 + 64, k0, &full_a[sa.s]);
                    } else {
                        tma_load_2d(as, &map_g, k0, m0, &full_a[sa.s]);
                    }
                }
                __syncwarp();
                sa.advance();
            }
        }
        if (!ok)   // copies in flight land before the shared memory is handed on: every slot's last round
            for (int s = 0; s < S::kSA; ++s) mbar_wait_bounded(&full_a[s], s < sa.s ? sa.phase : sa.phase ^ 1);
    } else if (warp == 5) {
        if (rank == 0) {
            const uint32_t idesc_whole = idesc_bf16(S::kTM, S::kTN, a.across != 0, true), idesc_half = idesc_bf16(S::kTM, S::kTN / 2, a.across != 0, true);
            const uint32_t step_a = a.across ? 2048 / 16 : 32 / 16;
            // operands whose rows run along m (n): 64 of them to a 128-byte row, such columns of tiles 8 KiB apart, eight k 1 KiB
            const uint64_t da0 = a.across ? umma_desc(smem_u32(smem), 8192, 1024, kLayoutSwizzle128) : umma_desc_kmajor(smem_u32(smem));
            const uint64_t db0 = umma_desc(smem_u32(smem + S::kBOff), 8192, 1024, kLayoutSwizzle128);
            Slot<S::kSA> sa;
            Slot<S::kSB> sb;
            for (int it = 0, t, half; ok && piece(it, t, half); ++it) {
                const int b = it & 1;
                const uint32_t idesc = half < 0 ? idesc_whole : idesc_half;
                if (it >= 2) ok = mbar_wait_cluster(&acc_empty[b], (it / 2 - 1) & 1);
                if (!ok) break;
                for (int j = 0; j < ks; ++j) {
                    ok = mbar_wait_warp(&wide[sb.s], sb.phase);   // says that the gradient's tile is there too
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t da = da0 + sa.s * (kABytes / 16), db = db0 + sb.s * (S::kBBytes / 16);
#pragma unroll
                        for (int k = 0; k < kTK / 16; ++k)
                            tc_mma_bf16<CG>(tmem + b * S::kTN, da + k * step_a, db + k * (2048 / 16), idesc, (j | k) != 0);
                        if constexpr (CG == 2) { tc_commit_pair(&empty_b[sb.s]); tc_commit_pair(&empty_a[sa.s]); }
                        else { tc_commit(&empty_b[sb.s]); tc_commit(&empty_a[sa.s]); }
                        if (j == ks - 1) { if constexpr (CG == 2) tc_commit_pair(&acc_full[b]); else tc_commit(&acc_full[b]); }
                    }
                    __syncwarp();
                    sa.advance();
                    sb.advance();
                }
            }
            if (!ok) {   // products in flight end before the tensor memory is handed on
                if (elect_one()) { if constexpr (CG == 2) tc_commit_pair(&drained); else tc_commit(&drained); }
                __syncwarp();
                mbar_wait_bounded(&drained, 0);
            }
        }
    } else if (warp == 6) {
        Slot<S::kSC> sc;
        for (int i = 0, t, half; ok && piece(i, t, half); ++i) {
            int tm, tn;
            tile_place(t, a.m_tiles, a.n_tiles, tm, tn);
            // of a half tile each CTA widens 64 columns; the copy brings 64 more, which nobody reads
            const int n0 = tn * S::kTN + (half < 0 ? rank * NB : half * NB + rank * (NB / 2));
            for (int j = 0; j < ks; ++j) {
                ok = mbar_wait_warp(&empty_c[sc.s], sc.phase ^ 1);
                if (!ok) break;
                if (elect_one()) {
                    mbar_expect_tx(&full_c[sc.s], S::kCodeBytes);
                    tma_load_2d(smem + S::kCOff + sc.s * S::kCStage, &map_c, FMT == kE2M1 ? n0 / 2 : n0, (k_first + j) * kTK, &full_c[sc.s]);
                }
                __syncwarp();
                sc.advance();
            }
        }
        if (!ok)
            for (int s = 0; s < S::kSC; ++s) mbar_wait_bounded(&full_c[s], s < sc.s ? sc.phase : sc.phase ^ 1);
    } else if (warp == 7 || warp == 8) {
        // scale bytes of one k to a lane: four neighbouring groups
        const int r = threadIdx.x - 7 * 32;
        const uint32_t dst0 = smem_u32(smem + S::kCOff + S::kCodeBytes) + 4 * r;
        const int64_t stride = (int64_t)kTK * a.groups;
        Slot<S::kSC> sc;
        for (int i = 0, t, half; ok && piece(i, t, half); ++i) {
            int tm, tn;
            tile_place(t, a.m_tiles, a.n_tiles, tm, tn);
            const int grp = (tn * S::kTN + (half < 0 ? rank : half) * NB) / 32;   // both CTAs of a half tile share four groups
            int64_t left = grp < a.groups ? a.k - (int64_t)k_first * kTK - r : 0;   // this lane's k is inside while positive
            const uint8_t* src = a.scales + ((int64_t)k_first * kTK + r) * a.groups + grp;
            for (int j = 0; j < ks; ++j) {
                ok = mbar_wait_warp(&empty_c[sc.s], sc.phase ^ 1);
                if (!ok) break;
                const uint32_t dst = dst0 + sc.s * S::kCStage;
                if (a.fast_scales) {
                    cp_async4(dst, left > 0 ? src : a.scales, left > 0 ? 4 : 0);
                } else {
                    uint32_t w = 0;
                    if (left > 0) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (grp + e < a.groups) w |= (uint32_t)__ldg(src + e) << (8 * e);
                    }
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst), "r"(w) : "memory");
                }
                if (a.fast_scales) cp_async_arrive(&full_c[sc.s]); else mbar_arrive(&full_c[sc.s]);
                sc.advance();
                src += stride;
                left -= kTK;
            }
        }
        cp_async_wait_all();
    } else if (warp >= kFirstConv) {
        // a lane owns eight neighbouring n of a row; eight lanes one 128-byte row of the operand tile
        constexpr int kLanesPerRow = NB / 8, kRowsPerPass = 32 * kConvWarps / kLanesPerRow, kPasses = kTK / kRowsPerPass;
        const int ct = (threadIdx.x - 32 * kFirstConv) % (32 * kConvWarps), group = (warp - kFirstConv) / kConvWarps, u = ct & 7, nc = (ct / 8) % (NB / 64), r0 = ct / kLanesPerRow;
        const uint32_t wide0 = CG == 2 ? map_to_rank(smem_u32(&wide[0]), 0) : smem_u32(&wide[0]);   // the pair's issuer waits for both halves
        const int sbyte = nc * 2 + (u >> 2);
        const int64_t total = CG == 2 ? (int64_t)a.work.pieces(first) * ks : (first < a.tiles ? (int64_t)((a.tiles - 1 - first) / step + 1) * ks : 0);
        Slot<S::kSA> sa;
        Slot<S::kSB> sb;
        Slot<S::kSC> sc;
        sa.s = sb.s = sc.s = group;
        for (int64_t i = group; i < total; i += kConvGroups) {
            ok = mbar_wait_warp(&full_c[sc.s], sc.phase);
            if (!ok) break;
            const uint8_t* cs = smem + S::kCOff + sc.s * S::kCStage;
            uint8_t* bs = smem + S::kBOff + sb.s * S::kBBytes;
            // rows r, r + ROWS, ... of eight columns each; passes are a multiple of eight rows apart: the same swizzle
            auto widen = [&](auto passes, int rows, int r, int col, int scale_byte, uint8_t* to) {
                constexpr int P = decltype(passes)::value;
                uint2 c[P];
                uint32_t k8[P], odd = 0;
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const int row = r + p * rows;
                    if constexpr (FMT == kE2M1) c[p] = make_uint2(*reinterpret_cast<const uint32_t*>(cs + row * S::kRowBytes + col / 2), 0u);
                    else c[p] = *reinterpret_cast<const uint2*>(cs + row * S::kRowBytes + col);
                    k8[p] = cs[S::kCodeBytes + 4 * row + scale_byte];
                }
                __syncwarp();
                if (elect_one()) mbar_arrive(&empty_c[sc.s]);
                if (!mbar_wait_warp(&empty_b[sb.s], sb.phase ^ 1)) return false;
#pragma unroll
                for (int p = 0; p < P; ++p) *reinterpret_cast<uint4*>(to + p * rows * 128) = widen8<FMT>(c[p], k8[p], odd);
                if (odd & kOdd) {
#pragma unroll
                    for (int p = 0; p < P; ++p) *reinterpret_cast<uint4*>(to + p * rows * 128) = widen8_any<FMT>(c[p], k8[p]);
                }
                return true;
            };
            if (i < whole) {
                ok = widen(std::integral_constant<int, kPasses>{}, kRowsPerPass, r0, nc * 64 + u * 8, sbyte, bs + nc * 8192 + r0 * 128 + ((u ^ (r0 & 7)) << 4));
            } else {   // 64 columns: all lanes on them
                const int r = ct >> 3;
                ok = widen(std::integral_constant<int, kPasses / 2>{}, 2 * kRowsPerPass, r, u * 8, rank * 2 + (u >> 2), bs + r * 128 + ((u ^ (r & 7)) << 4));
            }
            if (!ok) break;
            fence_async_shared();
            if (ct < 32) ok = mbar_wait_warp(&full_a[sa.s], sa.phase);   // one warp's arrival vouches for the gradient's tile
            if (!ok) break;
            __syncwarp();
            if (elect_one()) mbar_arrive_peer(wide0 + 8 * sb.s);
            sa.advance(kConvGroups);
            sb.advance(kConvGroups);
            sc.advance(kConvGroups);
        }
        // A wait by parity passes when the barrier is a whole round behind.  A slot of codes belongs to one group, which has
        // seen its round before; the other two rings are safe because a group that found its widened tile's slot free
        // knows that the products of kSB steps ago, and all before them, are done.
        static_assert(S::kSC % kConvGroups == 0 && S::kSA <= S::kSB && kConvGroups <= S::kSA, "parities");
        static_assert(kRowsPerPass % 8 == 0, "swizzle");
    } else {
        const uint32_t sums_to = sums.place(threadIdx.x);
        const uint32_t empty0 = CG == 2 ? map_to_rank(smem_u32(&acc_empty[0]), 0) : smem_u32(&acc_empty[0]);
        int ob = 0;
        for (int it = 0, t, half; piece(it, t, half); ++it) {
            int tm, tn;
            tile_place(t, a.m_tiles, a.n_tiles, tm, tn);
            const int m0 = tm * S::kTM + rank * 128, n0 = tn * S::kTN + (half > 0 ? NB : 0), columns = half < 0 ? S::kTN : S::kTN / 2;
            const int b = it & 1;
            ok = ok && mbar_wait_warp(&acc_full[b], (it / 2) & 1);
            if (!ok) s_late = 1;
            tc_fence_after();
            const uint32_t acc = tmem + b * S::kTN + ((uint32_t)warp << 21);
            if (CG == 1 && a.splits > 1) cluster_sync();   // no CTA is still reading operands; the other warps meet this below
#pragma unroll 1
            for (int c0 = 0; c0 < columns; c0 += 64) {
                uint32_t r[2][32];
                tmem_load32(acc + c0, r[0]);
                tmem_load32(acc + c0 + 32, r[1]);
                tmem_wait_loads();
                if (!ok) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) r[0][c] = r[1][c] = 0x7FFFFFFFu;
                }
                if (CG == 1 && a.splits > 1) {
#pragma unroll
                    for (int c = 0; c < 64; c += 4) {
                        const uint32_t* q = &r[c >> 5][c & 31];
                        ClusterSum<S::kTN>::push(sums_to + 4 * (c0 + c), q[0], q[1], q[2], q[3]);
                    }
                } else {
                    uint8_t* os = smem + S::kOutOff + ob * S::kOutBytes;
                    if (threadIdx.x == 0) bulk_wait_reads_but<1>();   // the store from this buffer before last has read it
                    named_barrier(1, 128);
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const uint32_t* q = &r[c >> 2][(c & 3) * 8];
                        *reinterpret_cast<uint4*>(os + threadIdx.x * 128 + ((c ^ (threadIdx.x & 7)) << 4)) =
                            make_uint4(pack_bf16_rne(u2f(q[1]), u2f(q[0])), pack_bf16_rne(u2f(q[3]), u2f(q[2])), pack_bf16_rne(u2f(q[5]), u2f(q[4])),
                                       pack_bf16_rne(u2f(q[7]), u2f(q[6])));
                    }
                    fence_async_shared();
                    named_barrier(1, 128);
                    if (threadIdx.x == 0) {
                        if (m0 < a.m && n0 + c0 < a.n) tma_store_2d(&map_out, os, n0 + c0, m0);
                        bulk_commit();
                    }
                    ob ^= 1;
                }
            }
            tc_fence_before();
            __syncwarp();
            if (elect_one()) mbar_arrive_cluster(empty0 + 8 * b);
        }
        if (threadIdx.x == 0) bulk_wait_reads();
    }

    if (CG == 1 && a.splits > 1) {   // one tile to a CTA: its partial sums meet those of the cluster's other CTAs
        __syncwarp();
        if (warp >= 4) cluster_sync();
        cluster_sync();
        if (warp < 4) {
            static_assert(ClusterSum<S::kTN>::kBytes <= S::kOutOff, "partial sums");
            int tm, tn;
            tile_place(first, a.m_tiles, a.n_tiles, tm, tn);
            constexpr int kLanes = S::kTN / 4;   // a lane takes four columns
            const int c = (threadIdx.x % kLanes) * 4;
            const int64_t m0 = (int64_t)tm * 128 + split * sums.rows(), n = (int64_t)tn * S::kTN + c;
#pragma unroll 4
            for (int r = threadIdx.x / kLanes; r < sums.rows(); r += 128 / kLanes) {
                if (m0 + r >= a.m || n >= a.n) break;
                const float4 v = sums.sum4(r, c);
                *reinterpret_cast<uint2*>(a.out + (m0 + r) * a.n + n) =
                    s_late ? make_uint2(0x7FFF7FFFu, 0x7FFF7FFFu) : make_uint2(pack_bf16_rne(v.y, v.x), pack_bf16_rne(v.w, v.z));
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    if constexpr (CG == 2) cluster_sync(); else __syncthreads();
    if (warp == 5) { tc_fence_after(); tmem_free<CG>(tmem, S::kCols); }
}

// codes as a matrix of bytes, boxes of one tile without swizzle
bool make_code_map(CUtensorMap* map, const void* base, int64_t rows, int64_t row_bytes, int box_bytes, int box_rows) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return false;
    const cuuint64_t gdim[2] = {(cuuint64_t)row_bytes, (cuuint64_t)rows};
    const cuuint64_t gstride[1] = {(cuuint64_t)row_bytes};
    const cuuint32_t box[2] = {(cuuint32_t)box_bytes, (cuuint32_t)box_rows};
    const cuuint32_t estride[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), gdim, gstride, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// rows of scales that lie on four bytes are fetched by asynchronous copies, others byte by byte
inline bool fast_scales(const MxGradArgs& x) { return x.n % 128 == 0 && (reinterpret_cast<uintptr_t>(x.scales) & 3) == 0; }

template <int FMT, int CG, int NB>
int go(const MxGradArgs& x, cudaStream_t st) {
    using S = GrShape<FMT, CG, NB>;
    auto kern = mx_grad_kernel<FMT, CG, NB>;
    static SmemOptIn opt;
    if (!bind_context() || !opt(kern, S::kSmem)) return kErrLaunch;
    GrArgs a = {};
    a.scales = x.scales;
    a.out = static_cast<uint16_t*>(x.out);
    a.m = x.m; a.n = x.n; a.k = x.k;
    a.groups = x.n / 32;
    const int64_t mt = (x.m + S::kTM - 1) / S::kTM, nt = (x.n + S::kTN - 1) / S::kTN;
    if (mt * nt > (1 << 30)) return kErrTooLarge;
    a.m_tiles = (int)mt; a.n_tiles = (int)nt; a.tiles = (int)(mt * nt);
    a.ksteps = (int)((x.k + kTK - 1) / kTK);
    a.across = x.across;
    a.fast_scales = fast_scales(x);
    a.splits = 1;
    int grid;
    if constexpr (CG == 2) {
        a.work = pair_work(a.tiles, sm_count());
        grid = 2 * a.work.launched();
    } else {
        a.splits = k_splits(a.tiles, a.ksteps, sm_count());
        grid = a.splits > 1 ? a.tiles * a.splits : std::min(a.tiles, sm_count());
    }
    CUtensorMap mg, mc, mo;
    const bool made = x.across ? make_swizzled_map(&mg, x.g, x.k, x.m, x.g_pitch * 2, 2, kTK) : make_swizzled_map(&mg, x.g, x.m, x.k, x.g_pitch * 2, 2, 128);
    if (!made || !make_code_map(&mc, x.payload, x.k, FMT == kE2M1 ? x.n / 2 : x.n, S::kRowBytes, kTK)) return kErrLaunch;
    if (!make_swizzled_map(&mo, x.out, x.m, x.n, x.n * 2, 2, 128)) return kErrLaunch;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {(unsigned)(CG == 2 ? 2 : a.splits), 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = CG == 2 || a.splits > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, mg, mc, mo, a) == cudaSuccess ? check_launch() : kErrLaunch;
}

template <int FMT>
int pick(const MxGradArgs& x, cudaStream_t st) {
    return takes_pairs(x.m, x.n, (x.k + kTK - 1) / kTK, sm_count(), fast_scales(x) ? 24 : 14) ? go<FMT, 2, 128>(x, st) : go<FMT, 1, 128>(x, st);
}

}  // namespace

int launch_mx_grad(const MxGradArgs& x, cudaStream_t st) {
    if (x.fmt == kE4M3) return pick<kE4M3>(x, st);
    if (x.fmt == kE5M2) return pick<kE5M2>(x, st);
    if (x.fmt == kE2M3) return pick<kE2M3>(x, st);
    return pick<kE2M1>(x, st);
}

}  // namespace morb
