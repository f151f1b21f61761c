// Product of a bf16 gradient with a microscaled matrix kept in 8 or 4 bits, out[m, n] = sum_k op(g)[m, k] W[k, n], W =
// decode(codes) * 2^(scale - 127): a linear layer's input gradient from its quantised weights (op(g) = g) and its weight
// gradient from the quantised activations (op(g) = g transposed).  The scales of W lie along n, so they cannot be
// multiplied into a product over k by the tensor core; the codes are widened to bf16 (exact: four significant bits at
// most) on the way from the staged codes to the operand tile, which costs no global traffic beyond the codes.
//
// One kernel, persistent over output tiles.  Per step of 64 k a thread of warp 4 requests the gradient's tile and the
// codes by TMA, warps 6-7 fetch the scale bytes, warps 8-15 widen the codes into the operand tile, a thread of warp 5
// issues the products, and warps 0-3 write the tile before last while the next one accumulates (two accumulators).
// In its large form two CTAs work as a pair on 256 x 256: each loads 128 rows of the gradient and widens 128 columns of W,
// so every widened element meets 256 rows.
#include <algorithm>

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
};

constexpr int kTK = 64;                 // k a step: 128 bytes of bf16
constexpr int kABytes = 128 * kTK * 2;  // a CTA's rows of the gradient
constexpr int kConvWarps = 8;
constexpr int kThreads = 32 * (8 + kConvWarps);

template <int FMT, int CG, int NB>      // CTAs to a tile; columns of W that one CTA widens
struct GrShape {
    static constexpr int kTM = 128 * CG, kTN = NB * CG;
    static constexpr int kRowBytes = FMT == kE2M1 ? NB / 2 : NB;   // codes of one k
    static constexpr int kBBytes = NB * kTK * 2;
    static constexpr int kCodeBytes = kRowBytes * kTK;
    static constexpr int kCodeOff = kABytes + kBBytes, kScaleOff = kCodeOff + kCodeBytes;
    static constexpr int kStage = (kScaleOff + kTK * 4 + 1023) & ~1023;
    static constexpr int kStages = (212 * 1024) / kStage;
    static constexpr int kSmem = kStages * kStage + 1024;
    static constexpr int kCols = 2 * kTN;
    static_assert(kSmem > 114 * 1024, "one CTA per SM, so the columns of tensor memory suffice");
    static_assert(kStages >= 4 && (kCols == 256 || kCols == 512), "shape");
};

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// 2^(byte - 127) in both halves of a word, as bf16; NaN for 255
__device__ __forceinline__ uint32_t e8m0_to_bf16x2(uint32_t byte) {
    uint32_t b = byte << 7;
    b = byte == 0 ? 0x0040u : b;
    b = byte == 255u ? 0x7FFFu : b;
    return b | (b << 16);
}

// Eight codes to eight bf16 values times the scale.  The exponent and mantissa of a code are the low bits of a bf16
// pattern's: moved there, the pattern stands for the value times 2^-120 (E4M3; 2^-112, 2^-126 for the others), subnormal
// codes included, since both formats count subnormals alike.  One multiplication undoes that exactly, a second
// applies the scale with the only rounding there is.  Codes that are no finite number take the conversion instruction.
template <int FMT>
__device__ __forceinline__ uint4 widen8(uint2 c, uint32_t scale2) {
    uint32_t o[4];
    if constexpr (FMT == kE2M1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // nibbles 2i, 2i + 1
            const uint32_t x = (c.x >> (8 * i)) & 0xFu;
            const uint32_t y = (c.x >> (8 * i + 4)) & 0xFu;
            const uint32_t p = x | (y << 16);
            o[i] = ((p << 12) & 0x80008000u) | ((p << 6) & 0x01C001C0u);
        }
    } else {
        const uint32_t w[2] = {c.x, c.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (FMT == kE2M3) {
                const uint32_t lo = __byte_perm(w[i], 0, 0x4140), hi = __byte_perm(w[i], 0, 0x4342);
                o[2 * i] = ((lo << 10) & 0x80008000u) | ((lo << 4) & 0x01F001F0u);
                o[2 * i + 1] = ((hi << 10) & 0x80008000u) | ((hi << 4) & 0x01F001F0u);
            } else {
                constexpr int sh = FMT == kE4M3 ? 4 : 3;
                constexpr uint32_t mask = FMT == kE4M3 ? 0x07F007F0u : 0x0FE00FE0u;
                const uint32_t lo = __byte_perm(w[i], 0, 0x1404), hi = __byte_perm(w[i], 0, 0x3424);
                o[2 * i] = (lo & 0x80008000u) | ((lo >> sh) & mask);
                o[2 * i + 1] = (hi & 0x80008000u) | ((hi >> sh) & mask);
            }
        }
    }
    constexpr uint32_t up = FMT == kE4M3 ? 0x7B807B80u : (FMT == kE5M2 ? 0x77807780u : 0x7E807E80u);   // 2^120, 2^112, 2^126
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = mul_bf16x2(o[i], up);
    if constexpr (FMT == kE4M3 || FMT == kE5M2) {
        constexpr uint32_t past = FMT == kE4M3 ? 0x01010101u : 0x04040404u;   // carries into bit 7 from 0x7F, from 0x7C up
        if ((((c.x & 0x7F7F7F7Fu) + past) | ((c.y & 0x7F7F7F7Fu) + past)) & 0x80808080u) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t h2 = codes_to_h2<FMT>(((i < 2 ? c.x : c.y) >> (16 * (i & 1))) & 0xFFFFu);
                o[i] = pack_bf16_rne(h_hi_to_f32(h2), h_lo_to_f32(h2));
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = mul_bf16x2(o[i], scale2);
    return make_uint4(o[0], o[1], o[2], o[3]);
}

// Output tile number -> its place: bands of eight rows of tiles, down a band's columns, so that the CTAs at work at one
// time share rows of the gradient and columns of W in L2.
__device__ __forceinline__ void tile_place(int t, int m_tiles, int n_tiles, int& tm, int& tn) {
    constexpr int kBand = 8;
    const int band = t / (kBand * n_tiles), in = t - band * (kBand * n_tiles);
    const int rows = min(kBand, m_tiles - band * kBand);
    tn = in / rows;
    tm = band * kBand + in - tn * rows;
}

template <int FMT, int CG, int NB>
__global__ void __launch_bounds__(kThreads, 1) mx_grad_kernel(const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_c,
                                                              const GrArgs a) {
    using S = GrShape<FMT, CG, NB>;
    constexpr int kLag = 3;
    extern __shared__ uint8_t s_raw[];
    __shared__ __align__(8) uint64_t full[S::kStages], wide[S::kStages], empty[S::kStages], acc_full[2], acc_empty[2], drained;
    __shared__ uint32_t s_tmem;
    uint8_t* smem = s_raw + ((1024 - (smem_u32(s_raw) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CG == 2 ? (int)cluster_rank() : 0;
    // work of this CTA (pair): tiles first, first + step, ... over steps [k_first, k_first + ksteps) of each
    const int split = CG == 2 ? 0 : (int)(blockIdx.x % (unsigned)a.splits);
    const int first = CG == 2 ? (int)(blockIdx.x >> 1) : (int)(blockIdx.x / (unsigned)a.splits);
    const int step = CG == 2 ? (int)(gridDim.x >> 1) : (int)(gridDim.x / (unsigned)a.splits);
    const int k_first = (int)((int64_t)a.ksteps * split / a.splits), k_last = (int)((int64_t)a.ksteps * (split + 1) / a.splits);
    const int ks = k_last - k_first;

    if (warp == 4 && lane == 0) {
        for (int s = 0; s < S::kStages; ++s) { mbar_init(&full[s], 1 + 2); mbar_init(&wide[s], kConvWarps * CG); mbar_init(&empty[s], 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 4 * CG); }
        mbar_init(&drained, 1);
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_g));
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_c));
    }
    if (warp == 5) tmem_alloc<CG>(&s_tmem, S::kCols);
    tc_fence_before();
    if constexpr (CG == 2) cluster_sync(); else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    pdl_launch_dependents();
    pdl_wait();

    bool ok = true;   // a wait that ran out ends the role; what it would have computed is written as NaN
    if (warp == 4) {
        if (lane == 0) {
            int i = 0;
            for (int t = first; t < a.tiles && ok; t += step) {
                int tm, tn;
                tile_place(t, a.m_tiles, a.n_tiles, tm, tn);
                const int m0 = tm * S::kTM + rank * 128, n0 = tn * S::kTN + rank * NB;
                for (int j = 0; j < ks; ++j, ++i) {
                    const int s = i % S::kStages;
                    if (i >= S::kStages) ok = mbar_wait_bounded(&empty[s], (i / S::kStages - 1) & 1);
                    if (!ok) break;
                    uint8_t* st = smem + s * S::kStage;
                    const int k0 = (k_first + j) * kTK;
                    mbar_expect_tx(&full[s], kABytes + S::kCodeBytes);
                    if (a.across) {   // g is [k, m]: two boxes of 64 m x 64 k
                        tma_load_2d(st, &map_g, m0, k0, &full[s]);
                        tma_load_2d(st + kABytes / 2, &map_g, m0 + 64, k0, &full[s]);
                    } else {
                        tma_load_2d(st, &map_g, k0, m0, &full[s]);
                    }
                    tma_load_2d(st + S::kCodeOff, &map_c, FMT == kE2M1 ? n0 / 2 : n0, k0, &full[s]);
                }
            }
            if (!ok)   // copies in flight land before the shared memory is handed on
                for (int j = i > S::kStages ? i - S::kStages : 0; j < i; ++j) mbar_wait_bounded(&full[j % S::kStages], (j / S::kStages) & 1);
        }
        __syncwarp();
    } else if (warp == 5) {
        if (lane == 0 && rank == 0) {
            const uint32_t idesc = idesc_bf16(S::kTM, S::kTN, a.across != 0, true);
            const uint32_t step_a = a.across ? 2048 / 16 : 32 / 16;
            int i = 0, it = 0;
            for (int t = first; t < a.tiles && ok; t += step, ++it) {
                const int b = it & 1;
                if (it >= 2) ok = mbar_wait_cluster(&acc_empty[b], (it / 2 - 1) & 1);
                if (!ok) break;
                tc_fence_after();
                for (int j = 0; j < ks; ++j, ++i) {
                    const int s = i % S::kStages;
                    ok = mbar_wait_cluster(&wide[s], (i / S::kStages) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t st = smem_u32(smem + s * S::kStage);
                    // operands whose rows run along m (n): 64 of them to a 128-byte row, such columns of tiles 8 KiB apart, eight k 1 KiB
                    const uint64_t da = a.across ? umma_desc(st, 8192, 1024, kLayoutSwizzle128) : umma_desc_kmajor(st);
                    const uint64_t db = umma_desc(st + kABytes, 8192, 1024, kLayoutSwizzle128);
#pragma unroll
                    for (int k = 0; k < kTK / 16; ++k)
                        tc_mma_bf16<CG>(tmem + b * S::kTN, da + k * step_a, db + k * (2048 / 16), idesc, (j | k) != 0);
                    if constexpr (CG == 2) tc_commit_pair(&empty[s]); else tc_commit(&empty[s]);
                }
                if (!ok) break;
                if constexpr (CG == 2) tc_commit_pair(&acc_full[b]); else tc_commit(&acc_full[b]);
            }
            if (!ok) {   // products in flight end before the tensor memory is handed on
                if constexpr (CG == 2) tc_commit_pair(&drained); else tc_commit(&drained);
                mbar_wait_bounded(&drained, 0);
            }
        }
        __syncwarp();
    } else if (warp == 6 || warp == 7) {
        // scale bytes of one k each: four neighbouring groups
        const int r = threadIdx.x - 192;
        int i = 0, j = ks, t = first - step, grp = 0;
        int64_t total = t < a.tiles && first < a.tiles ? (int64_t)((a.tiles - 1 - first) / step + 1) * ks : 0;
        for (; i < total + kLag; ++i) {
            if (i < total) {
                if (j == ks) {
                    j = 0;
                    t += step;
                    int tm, tn;
                    tile_place(t, a.m_tiles, a.n_tiles, tm, tn);
                    grp = tn * (S::kTN / 32) + (NB == 128 ? rank * 4 : 0);
                }
                const int s = i % S::kStages;
                if (i >= S::kStages) ok = mbar_wait_bounded(&empty[s], (i / S::kStages - 1) & 1);
                ok = __all_sync(0xFFFFFFFFu, ok);
                if (!ok) break;
                const int64_t k = (int64_t)(k_first + j) * kTK + r;
                const bool in = k < a.k && grp < a.groups;
                const uint8_t* src = a.scales + (in ? k * a.groups + grp : 0);
                const uint32_t dst = smem_u32(smem + s * S::kStage + S::kScaleOff) + 4 * r;
                if (a.fast_scales) {
                    cp_async4(dst, src, in ? 4 : 0);
                } else {
                    uint32_t w = 0;
                    if (in) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (grp + e < a.groups) w |= (uint32_t)__ldg(src + e) << (8 * e);
                    }
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst), "r"(w) : "memory");
                }
                ++j;
            }
            cp_async_commit();
            if (i >= kLag) {
                cp_async_wait<kLag>();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[(i - kLag) % S::kStages]);
            }
        }
        cp_async_wait<0>();
    } else if (warp >= 8) {
        // a lane owns eight neighbouring n of a row; eight lanes one 128-byte row of the operand tile
        constexpr int kLanesPerRow = NB / 8, kRowsPerPass = 32 * kConvWarps / kLanesPerRow, kPasses = kTK / kRowsPerPass;
        const int ct = threadIdx.x - 256, u = ct & 7, nc = (ct / 8) % (NB / 64), r0 = ct / kLanesPerRow;
        const uint32_t wide0 = CG == 2 ? map_to_rank(smem_u32(&wide[0]), 0) : smem_u32(&wide[0]);
        const int sbyte = nc * 2 + (u >> 2) + (NB == 64 ? rank * 2 : 0);
        const int64_t total = first < a.tiles ? (int64_t)((a.tiles - 1 - first) / step + 1) * ks : 0;
        for (int64_t i = 0; i < total; ++i) {
            const int s = (int)(i % S::kStages);
            ok = mbar_wait_bounded(&full[s], (uint32_t)(i / S::kStages) & 1);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            uint8_t* st = smem + s * S::kStage;
            uint2 c[kPasses];
            uint32_t sb[kPasses];
#pragma unroll
            for (int p = 0; p < kPasses; ++p) {
                const int row = r0 + p * kRowsPerPass;
                const uint8_t* codes = st + S::kCodeOff + row * S::kRowBytes;
                if constexpr (FMT == kE2M1) c[p] = make_uint2(*reinterpret_cast<const uint32_t*>(codes + nc * 32 + u * 4), 0u);
                else c[p] = *reinterpret_cast<const uint2*>(codes + nc * 64 + u * 8);
                sb[p] = st[S::kScaleOff + 4 * row + sbyte];
            }
#pragma unroll
            for (int p = 0; p < kPasses; ++p) {
                const int row = r0 + p * kRowsPerPass;
                *reinterpret_cast<uint4*>(st + kABytes + nc * 8192 + row * 128 + ((u ^ (row & 7)) << 4)) = widen8<FMT>(c[p], e8m0_to_bf16x2(sb[p]));
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(wide0 + 8 * s);
        }
    } else {
        int it = 0;
        const uint32_t empty0 = CG == 2 ? map_to_rank(smem_u32(&acc_empty[0]), 0) : smem_u32(&acc_empty[0]);
        for (int t = first; t < a.tiles; t += step, ++it) {
            int tm, tn;
            tile_place(t, a.m_tiles, a.n_tiles, tm, tn);
            const int64_t m = (int64_t)tm * S::kTM + rank * 128 + threadIdx.x, n0 = (int64_t)tn * S::kTN;
            const int b = it & 1;
            ok = ok && mbar_wait_bounded(&acc_full[b], (it / 2) & 1);
            ok = __all_sync(0xFFFFFFFFu, ok);
            tc_fence_after();
            const uint32_t acc = tmem + b * S::kTN + ((uint32_t)warp << 21);
#pragma unroll 1
            for (int c0 = 0; c0 < S::kTN; c0 += 32) {
                uint32_t r[32];
                tmem_load32(acc + c0, r);
                tmem_wait_loads();
                if (!ok) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) r[c] = 0x7FFFFFFFu;
                }
                if (a.splits > 1) {
                    float* part = reinterpret_cast<float*>(smem);   // [column][128 rows]; the operands are no longer needed
#pragma unroll
                    for (int c = 0; c < 32; ++c) part[(c0 + c) * 128 + threadIdx.x] = u2f(r[c]);
                } else if (m < a.m && n0 + c0 < a.n) {   // n is a multiple of 32
                    uint16_t* o = a.out + m * a.n + n0 + c0;
#pragma unroll
                    for (int c = 0; c < 32; c += 8)
                        *reinterpret_cast<uint4*>(o + c) = make_uint4(
                            pack_bf16_rne(u2f(r[c + 1]), u2f(r[c])), pack_bf16_rne(u2f(r[c + 3]), u2f(r[c + 2])),
                            pack_bf16_rne(u2f(r[c + 5]), u2f(r[c + 4])), pack_bf16_rne(u2f(r[c + 7]), u2f(r[c + 6])));
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(empty0 + 8 * b);
        }
    }

    if (CG == 1 && a.splits > 1) {   // partial sums of one tile in the CTAs of a cluster: each adds up some of the columns, in rank order
        __syncwarp();
        cluster_sync();
        if (warp < 4) {
            int tm, tn;
            tile_place(first, a.m_tiles, a.n_tiles, tm, tn);
            const int64_t m = (int64_t)tm * 128 + threadIdx.x, n0 = (int64_t)tn * S::kTN;
            const uint32_t mine = smem_u32(smem) + 4 * threadIdx.x;
            for (int c = 8 * split; c < S::kTN && n0 + c < a.n; c += 8 * a.splits) {
                float sum[8] = {};
                for (int z = 0; z < a.splits; ++z)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float v;
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_rank(mine + (c + e) * 512, z)) : "memory");
                        sum[e] += v;
                    }
                if (m < a.m)
                    *reinterpret_cast<uint4*>(a.out + m * a.n + n0 + c) = make_uint4(pack_bf16_rne(sum[1], sum[0]), pack_bf16_rne(sum[3], sum[2]),
                                                                                      pack_bf16_rne(sum[5], sum[4]), pack_bf16_rne(sum[7], sum[6]));
            }
        }
        __syncwarp();
        cluster_sync();
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
    a.fast_scales = a.groups % 4 == 0 && (reinterpret_cast<uintptr_t>(x.scales) & 3) == 0;
    a.splits = 1;
    int grid;
    if constexpr (CG == 2) {
        grid = 2 * std::min(a.tiles, sm_count() / 2);
    } else {
        while (a.splits < 8 && a.tiles * a.splits * 2 <= sm_count() && a.ksteps >= a.splits * 4) a.splits *= 2;
        grid = a.splits > 1 ? a.tiles * a.splits : std::min(a.tiles, sm_count());
    }
    CUtensorMap mg, mc;
    const bool made = x.across ? make_swizzled_map(&mg, x.g, x.k, x.m, x.g_pitch * 2, 2, kTK) : make_swizzled_map(&mg, x.g, x.m, x.k, x.g_pitch * 2, 2, 128);
    if (!made || !make_code_map(&mc, x.payload, x.k, FMT == kE2M1 ? x.n / 2 : x.n, S::kRowBytes, kTK)) return kErrLaunch;
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
    return cudaLaunchKernelEx(&cfg, kern, mg, mc, a) == cudaSuccess ? check_launch() : kErrLaunch;
}

// Pairs where the 256 x 256 tiles fill at least half of the pairs' slots in the last round; single CTAs on 128 x 128, with the sum over
// k split within a cluster where even those are few, otherwise.
template <int FMT>
int pick(const MxGradArgs& x, cudaStream_t st) {
    const int64_t big = ((x.m + 255) / 256) * ((x.n + 255) / 256);
    if (big * 2 >= sm_count() / 2) return go<FMT, 2, 128>(x, st);
    return go<FMT, 1, 128>(x, st);
}

}  // namespace

int launch_mx_grad(const MxGradArgs& x, cudaStream_t st) {
    if (x.fmt == kE4M3) return pick<kE4M3>(x, st);
    if (x.fmt == kE5M2) return pick<kE5M2>(x, st);
    if (x.fmt == kE2M3) return pick<kE2M3>(x, st);
    return pick<kE2M1>(x, st);
}

}  // namespace morb
