// Product of a bf16 gradient with a microscaled matrix kept in 8 or 4 bits, out[m, n] = sum_k op(g)[m, k] W[k, n], W =
// decode(codes) * 2^(scale - 127): a linear layer's input gradient from its quantised weights (op(g) = g) and its weight
// gradient from the quantised activations (op(g) = g transposed).  The scales of W lie along n, so they cannot be
// multiplied into a product over k by the tensor core; the codes are widened to bf16 (exact: four significant bits at
// most) on the way from the staged codes to the operand tile, which costs no global traffic beyond the codes.
#include "mx_kernels.cuh"
#include "tcgen05.cuh"

namespace morb {
namespace {

struct GrArgs {
    const uint8_t* scales;
    uint16_t* out;
    int64_t m, n, k, groups;
    int64_t m_tiles;
    int ksteps, across, splits;
};

constexpr int kTM = 128, kTN = 128, kTK = 64;
constexpr int kABytes = kTM * kTK * 2, kBBytes = kTN * kTK * 2;

template <int FMT>
struct GrShape {
    static constexpr int kRowBytes = FMT == kE2M1 ? kTN / 2 : kTN;   // codes of one k in a tile
    static constexpr int kCodeBytes = kRowBytes * kTK;
    static constexpr int kStage = kABytes + kBBytes + kCodeBytes;
    static constexpr int kStages = (200 * 1024) / kStage;
    static constexpr int kSmem = kStages * kStage + 1024;
    static_assert(kSmem > 114 * 1024, "one CTA per SM");
};

// Eight codes to eight bf16 (16 bytes); k is the scale
template <int FMT>
__device__ __forceinline__ uint4 widen8(uint2 c, float k) {
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

template <int FMT>
__global__ void __launch_bounds__(192, 1) mx_grad_kernel(const __grid_constant__ CUtensorMap map_g, const __grid_constant__ CUtensorMap map_c,
                                                         const GrArgs a) {
    using S = GrShape<FMT>;
    extern __shared__ uint8_t s_raw[];
    __shared__ __align__(8) uint64_t full[S::kStages], wide[S::kStages], empty[S::kStages], acc_done, drained;
    __shared__ uint32_t s_tmem;
    uint8_t* smem = s_raw + ((1024 - (smem_u32(s_raw) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = (int)(blockIdx.x % (unsigned)a.splits);
    const int64_t tile = blockIdx.x / (unsigned)a.splits;
    const int64_t m0 = (tile % a.m_tiles) * kTM, n0 = (tile / a.m_tiles) * kTN;
    const int k_first = (int)((int64_t)a.ksteps * split / a.splits), k_last = (int)((int64_t)a.ksteps * (split + 1) / a.splits);
    const int n = k_last - k_first;

    if (warp == 4 && lane == 0) {
        for (int s = 0; s < S::kStages; ++s) { mbar_init(&full[s], 1); mbar_init(&wide[s], 4); mbar_init(&empty[s], 1); }
        mbar_init(&acc_done, 1);
        mbar_init(&drained, 1);
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_g));
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_c));
    }
    if (warp == 5) tmem_alloc<1>(&s_tmem, kTN);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    pdl_launch_dependents();
    pdl_wait();

    bool ok = true;   // a wait that ran out ends the role's loop; the tile is then written as NaN
    if (warp == 4) {
        if (lane == 0) {
            int i = 0;
            for (; i < n; ++i) {
                const int s = i % S::kStages;
                if (i >= S::kStages) ok = mbar_wait_bounded(&empty[s], (i / S::kStages - 1) & 1);
                if (!ok) break;
                uint8_t* st = smem + s * S::kStage;
                const int k0 = (k_first + i) * kTK;
                mbar_expect_tx(&full[s], kABytes + S::kCodeBytes);
                if (a.across) {   // g is [k, m]: two boxes of 64 m x 64 k
                    tma_load_2d(st, &map_g, (int)m0, k0, &full[s]);
                    tma_load_2d(st + kABytes / 2, &map_g, (int)m0 + 64, k0, &full[s]);
                } else {
                    tma_load_2d(st, &map_g, k0, (int)m0, &full[s]);
                }
                tma_load_2d(st + kABytes + kBBytes, &map_c, (int)(FMT == kE2M1 ? n0 / 2 : n0), k0, &full[s]);
            }
            if (!ok)   // copies in flight land before the shared memory is handed on
                for (int j = i > S::kStages ? i - S::kStages : 0; j < i; ++j) mbar_wait_bounded(&full[j % S::kStages], (j / S::kStages) & 1);
        }
        __syncwarp();
    } else if (warp == 5) {
        if (lane == 0) {
            const uint32_t idesc = idesc_bf16(kTM, kTN, a.across != 0, true);
            for (int i = 0; i < n; ++i) {
                const int s = i % S::kStages;
                ok = mbar_wait_bounded(&full[s], (i / S::kStages) & 1) && mbar_wait_bounded(&wide[s], (i / S::kStages) & 1);
                if (!ok) break;
                tc_fence_after();
                const uint32_t st = smem_u32(smem + s * S::kStage);
                // operands whose rows run along m (n): 64 of them to a 128-byte row, such columns of tiles 8 KiB apart, eight k 1 KiB
                const uint64_t da = a.across ? umma_desc(st, 8192, 1024, kLayoutSwizzle128) : umma_desc_kmajor(st);
                const uint64_t db = umma_desc(st + kABytes, 8192, 1024, kLayoutSwizzle128);
                const uint32_t step_a = a.across ? 2048 / 16 : 32 / 16;
#pragma unroll
                for (int k = 0; k < kTK / 16; ++k) tc_mma_bf16<1>(tmem, da + k * step_a, db + k * (2048 / 16), idesc, (i | k) != 0);
                tc_commit(&empty[s]);
            }
            tc_commit(ok ? &acc_done : &drained);
            if (!ok) mbar_wait_bounded(&drained, 0);
        }
        __syncwarp();
    } else {
        // a lane owns eight neighbouring n; eight lanes one 128-byte row of the operand tile
        const int u = threadIdx.x & 7, r0 = threadIdx.x >> 3;
        for (int i = 0; i < n; ++i) {
            const int s = i % S::kStages;
            const int64_t k0 = (int64_t)(k_first + i) * kTK;
            uint32_t sb[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int idx = r0 + 16 * j, row = idx & 63, nc = idx >> 6;
                const int64_t grp = n0 / 32 + nc * 2 + (u >> 2);
                sb[j] = (k0 + row < a.k && grp < a.groups) ? __ldg(a.scales + (k0 + row) * a.groups + grp) : 127u;
            }
            ok = mbar_wait_bounded(&full[s], (i / S::kStages) & 1);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            uint8_t* st = smem + s * S::kStage;
            const uint8_t* codes = st + kABytes + kBBytes;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int idx = r0 + 16 * j, row = idx & 63, nc = idx >> 6;
                uint2 c;
                if constexpr (FMT == kE2M1) c = make_uint2(*reinterpret_cast<const uint32_t*>(codes + row * S::kRowBytes + nc * 32 + u * 4), 0u);
                else c = *reinterpret_cast<const uint2*>(codes + row * S::kRowBytes + nc * 64 + u * 8);
                *reinterpret_cast<uint4*>(st + kABytes + nc * 8192 + row * 128 + ((u ^ (row & 7)) << 4)) = widen8<FMT>(c, e8m0_to_f32(sb[j]));
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(&wide[s]);
        }
        ok = ok && mbar_wait_bounded(&acc_done, 0);
        ok = __all_sync(0xFFFFFFFFu, ok);
        tc_fence_after();
    }

    if (warp < 4) {
        const uint32_t lanes = tmem + ((uint32_t)warp << 21);
        const float bad = u2f(0x7FFFFFFFu);
        const int64_t m = m0 + threadIdx.x;
#pragma unroll 1
        for (int c0 = 0; c0 < kTN; c0 += 32) {
            uint32_t r[32];
            tmem_load32(lanes + c0, r);
            tmem_wait_loads();
            if (!ok) {
#pragma unroll
                for (int c = 0; c < 32; ++c) r[c] = f2u(bad);
            }
            if (a.splits > 1) {
                float* part = reinterpret_cast<float*>(smem);
#pragma unroll
                for (int c = 0; c < 32; ++c) part[(c0 + c) * kTM + threadIdx.x] = u2f(r[c]);
            } else if (m < a.m && n0 + c0 < a.n) {   // n is a multiple of 32
                uint16_t* o = a.out + m * a.n + n0 + c0;
#pragma unroll
                for (int c = 0; c < 32; c += 8)
                    *reinterpret_cast<uint4*>(o + c) = make_uint4(
                        pack_bf16_rne(u2f(r[c + 1]), u2f(r[c])), pack_bf16_rne(u2f(r[c + 3]), u2f(r[c + 2])),
                        pack_bf16_rne(u2f(r[c + 5]), u2f(r[c + 4])), pack_bf16_rne(u2f(r[c + 7]), u2f(r[c + 6])));
            }
        }
    }
    if (a.splits > 1) {   // partial sums of one tile in the CTAs of a cluster: each adds up some of the columns, in rank order
        cluster_sync();
        if (warp < 4) {
            const int64_t m = m0 + threadIdx.x;
            const uint32_t mine = smem_u32(smem) + 4 * threadIdx.x;
            for (int c = 8 * split; c < kTN && n0 + c < a.n; c += 8 * a.splits) {
                float sum[8] = {};
                for (int z = 0; z < a.splits; ++z)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float v;
                        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(map_to_rank(mine + (c + e) * (kTM * 4), z)) : "memory");
                        sum[e] += v;
                    }
                if (m < a.m)
                    *reinterpret_cast<uint4*>(a.out + m * a.n + n0 + c) = make_uint4(pack_bf16_rne(sum[1], sum[0]), pack_bf16_rne(sum[3], sum[2]),
                                                                                      pack_bf16_rne(sum[5], sum[4]), pack_bf16_rne(sum[7], sum[6]));
            }
        }
        cluster_sync();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 5) { tc_fence_after(); tmem_free<1>(tmem, kTN); }
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

template <int FMT>
int go(const MxGradArgs& x, cudaStream_t st) {
    using S = GrShape<FMT>;
    auto kern = mx_grad_kernel<FMT>;
    static SmemOptIn opt;
    if (!opt(kern, S::kSmem)) return kErrLaunch;
    GrArgs a = {};
    a.scales = x.scales;
    a.out = static_cast<uint16_t*>(x.out);
    a.m = x.m; a.n = x.n; a.k = x.k;
    a.groups = x.n / 32;
    a.m_tiles = (x.m + kTM - 1) / kTM;
    a.ksteps = (int)((x.k + kTK - 1) / kTK);
    a.across = x.across;
    const int64_t tiles = a.m_tiles * ((x.n + kTN - 1) / kTN);
    a.splits = 1;
    while (a.splits < 8 && tiles * a.splits * 2 <= sm_count() && a.ksteps >= a.splits * 4) a.splits *= 2;
    if (tiles * a.splits > 0x7FFFFFFF) return kErrTooLarge;
    CUtensorMap mg, mc;
    const bool made = x.across ? make_swizzled_map(&mg, x.g, x.k, x.m, x.g_pitch * 2, 2, kTK) : make_swizzled_map(&mg, x.g, x.m, x.k, x.g_pitch * 2, 2, kTM);
    if (!made || !make_code_map(&mc, x.payload, x.k, FMT == kE2M1 ? x.n / 2 : x.n, S::kRowBytes, kTK)) return kErrLaunch;
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
    return cudaLaunchKernelEx(&cfg, kern, mg, mc, a) == cudaSuccess ? check_launch() : kErrLaunch;
}

}  // namespace

int launch_mx_grad(const MxGradArgs& x, cudaStream_t st) {
    if (x.fmt == kE4M3) return go<kE4M3>(x, st);
    if (x.fmt == kE5M2) return go<kE5M2>(x, st);
    if (x.fmt == kE2M3) return go<kE2M3>(x, st);
    return go<kE2M1>(x, st);
}

}  // namespace morb
