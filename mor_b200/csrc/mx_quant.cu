// 4-bit microscaled quantisation (E2M1 codes, one E8M0 scale byte for every 32 columns) and the way back from codes to
// values for every format of the framework's real quantised outputs.
#include <cuda_bf16.h>

#include "mx_kernels.cuh"
#include "tcgen05.cuh"

namespace morb {

int sm_count() {
    static int cached[64] = {0};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) dev = 0;
    if (cached[dev] == 0) {
        int n = 0;
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        cached[dev] = n > 0 ? n : 148;
    }
    return cached[dev];
}
int check_launch() { return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch; }

namespace {

constexpr int kQThreads = 256;

// Eight binary32 values to eight E2M1 codes, round to nearest even, element i in bits [4 i, 4 i + 4).
__device__ __forceinline__ uint32_t e2m1_codes8(const float (&f)[8]) {
    uint32_t r;
    asm("{\n.reg .b8 a, b, c, d;\n"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        "mov.b32 %0, {a, b, c, d};\n}"
        : "=r"(r)
        : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
    return r;
}

// The scale byte s of a group from the largest magnitude's bit pattern (binary32 with the sign cleared): the largest
// power of two 2^(127 - s) that keeps amax at or below 6 = 1.5 * 2^2.  With amax = 1.m * 2^(f - 127) that is s = f - 2,
// one more where 1.m > 1.5; magnitudes below 2^-124 get 0, a group of zeros 127, one with an infinity or NaN 255.
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t amax_bits) {
    const int s = (int)(amax_bits >> 23) - 2 + ((amax_bits & 0x7FFFFFu) > 0x400000u ? 1 : 0);
    uint32_t byte = (uint32_t)max(s, 0);
    byte = amax_bits == 0u ? 127u : byte;
    return amax_bits >= 0x7F800000u ? 255u : byte;
}

// A lane owns eight consecutive elements, four lanes a group, a warp U times 256 elements in a row.  blockIdx.y walks the
// rows (one row where the matrix is contiguous, whose groups then follow each other without a gap), blockIdx.x slices of
// a row.  Bound by memory, with the integer pipe close behind (72 %): all loads of a thread stand before their first use,
// four of 16 (32) bytes in flight each (8192^2 bf16: two take 34.0 us, four 30.4, eight 30.2), and a warp's scale bytes
// leave in one store (29.1 us = 5.8 TB/s; 1003 x 4128 float32 out of wider rows 5.0 us).
constexpr int kQU = 4;
template <bool FP32>
__global__ void __launch_bounds__(kQThreads) quantize_fp4_kernel(const void* __restrict__ in, uint32_t* __restrict__ payload,
                                                                 uint8_t* __restrict__ scales, int64_t rows, int64_t vec_per_row,
                                                                 int64_t pitch) {
    const int lane = threadIdx.x & 31;
    const int64_t first = (int64_t)blockIdx.x * (kQThreads * kQU) + (threadIdx.x >> 5) * (32 * kQU);
    pdl_wait();
    pdl_launch_dependents();
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const char* row = static_cast<const char*>(in) + r * pitch * (FP32 ? 4 : 2);
        for (int64_t v0 = first; v0 < vec_per_row; v0 += (int64_t)gridDim.x * (kQThreads * kQU)) {
            uint4 w[kQU][FP32 ? 2 : 1];
            uint32_t bytes = 0;   // of the group 8 u + lane % 8, for u = lane / 8
#pragma unroll
            for (int u = 0; u < kQU; ++u) {
                const int64_t v = v0 + u * 32 + lane;
                const uint4* p = reinterpret_cast<const uint4*>(row + v * (FP32 ? 32 : 16));
                w[u][0] = v < vec_per_row ? ld_stream(p) : make_uint4(0, 0, 0, 0);
                if constexpr (FP32) w[u][1] = v < vec_per_row ? ld_stream(p + 1) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int u = 0; u < kQU; ++u) {
                const int64_t v = v0 + u * 32 + lane;
                uint32_t amax;
                float f[8];
                if constexpr (FP32) {
                    const uint32_t a[8] = {w[u][0].x, w[u][0].y, w[u][0].z, w[u][0].w, w[u][1].x, w[u][1].y, w[u][1].z, w[u][1].w};
                    amax = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) { f[i] = u2f(a[i]); amax = max(amax, a[i] & 0x7FFFFFFFu); }
                } else {
                    const uint32_t a[4] = {w[u][0].x, w[u][0].y, w[u][0].z, w[u][0].w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) { f[2 * i] = bf16_lo(a[i]); f[2 * i + 1] = bf16_hi(a[i]); }
                    amax = hmax_halves(umax16x2_vec(mag2(a[0]), mag2(a[1]), mag2(a[2]), mag2(a[3]))) << 16;
                }
                amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
                amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
                const uint32_t byte = fp4_scale_byte(amax);
                const float up = u2f((254u - min(byte, 253u)) << 23);   // 2^(127 - byte), never subnormal: byte <= 253
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = __fmul_rn(f[i], up);   // exact but for values far below the smallest code
                if (v < vec_per_row) payload[r * vec_per_row + v] = byte == 255u ? 0u : e2m1_codes8(f);
                const uint32_t mine = __shfl_sync(0xFFFFFFFFu, byte, (lane & 7) * 4);
                bytes = (lane >> 3) == u ? mine : bytes;
            }
            if (v0 + 4 * lane < vec_per_row) scales[((r * vec_per_row + v0) >> 2) + lane] = (uint8_t)bytes;
        }
    }
}
static_assert(kQU == 4, "a warp's 32 scale bytes, one a lane");

// Two codes to two binary32 values: `c` holds two bytes (8-bit formats), or two nibbles (E2M1), the lower element low.
template <int FMT>
__device__ __forceinline__ void decode2(uint32_t c, float& lo, float& hi) {
    uint32_t h2;
    if constexpr (FMT == kE2M1) asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %1;\ncvt.rn.f16x2.e2m1x2 %0, a;\n}" : "=r"(h2) : "r"(c));
    else h2 = codes_to_h2<FMT>(c);
    lo = h_lo_to_f32(h2);
    hi = h_hi_to_f32(h2);
}

// A lane writes 16 bytes: eight bf16 or four binary32 values.  value = decode(code) * 2^(scale - 127) is exact in
// binary32 (at most four significant bits, nothing below 2^-143), so the one rounding is the one to bf16, to nearest
// even, and only subnormal results meet it.  Bound by memory: 16384 x 8192 E4M3 to bf16 61.5 us = 6.6 TB/s, 8192^2 E2M1
// 27.0 us = 6.3 TB/s (two loads of codes in flight a thread 30.2, four 27.0, eight 27.9).
template <int FMT, bool FP32, int U>
__global__ void __launch_bounds__(kQThreads) dequantize_kernel(const uint8_t* __restrict__ payload, const uint8_t* __restrict__ scales,
                                                               uint4* __restrict__ out, int64_t nvec, int log2_group) {
    constexpr int E = FP32 ? 4 : 8;                       // elements a lane and step
    constexpr int B = FMT == kE2M1 ? E / 2 : E;           // bytes of codes
    pdl_wait();
    pdl_launch_dependents();
    for (int64_t v0 = (int64_t)blockIdx.x * (kQThreads * U); v0 < nvec; v0 += (int64_t)gridDim.x * (kQThreads * U)) {
        uint2 c[U];
        uint32_t s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t v = v0 + u * kQThreads + threadIdx.x;
            c[u] = make_uint2(0, 0);
            s[u] = 0;
            if (v < nvec) {
                if constexpr (B == 8) c[u] = __ldcs(reinterpret_cast<const uint2*>(payload) + v);
                else if constexpr (B == 4) c[u].x = __ldcs(reinterpret_cast<const uint32_t*>(payload) + v);
                else c[u].x = __ldcs(reinterpret_cast<const uint16_t*>(payload) + v);
                s[u] = __ldg(scales + ((v * E) >> log2_group));
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t v = v0 + u * kQThreads + threadIdx.x;
            if (v >= nvec) continue;
            const float k = e8m0_to_f32(s[u]);
            float f[E];
#pragma unroll
            for (int i = 0; i < E / 2; ++i) {
                uint32_t two;
                if constexpr (FMT == kE2M1) two = (c[u].x >> (8 * i)) & 0xFFu;
                else two = ((i < 2 ? c[u].x : c[u].y) >> (16 * (i & 1))) & 0xFFFFu;
                decode2<FMT>(two, f[2 * i], f[2 * i + 1]);
            }
            uint4 o;
            if constexpr (FP32) {
                o = make_uint4(f2u(__fmul_rn(f[0], k)), f2u(__fmul_rn(f[1], k)), f2u(__fmul_rn(f[2], k)), f2u(__fmul_rn(f[3], k)));
            } else {
                o = make_uint4(pack_bf16_rne(__fmul_rn(f[1], k), __fmul_rn(f[0], k)), pack_bf16_rne(__fmul_rn(f[3], k), __fmul_rn(f[2], k)),
                               pack_bf16_rne(__fmul_rn(f[5], k), __fmul_rn(f[4], k)), pack_bf16_rne(__fmul_rn(f[7], k), __fmul_rn(f[6], k)));
            }
            st_stream(out + v, o);
        }
    }
}

// out[c] = sum_r g[r, c], the gradient of a bias.  A CTA takes kSumCols columns, lanes of 16 bytes along a row and kSumLanes rows
// at a time; the CTAs of a cluster share the rows.  Every sum is formed in one order -- a lane's rows, then the lanes, then
// the CTAs by rank -- so results repeat bit for bit.  Bound by memory and, at these sizes, by starting: 4096 x
// 4096 9.1 us from memory (3.7 TB/s), 6.5 where the L2 holds the gradient, 8192 x 4096 14.0 (4.8 TB/s) and 9.1; other shapes
// on an earlier form, 9.3 and 14.5 for this one: 256 columns and 512 threads 16.0 and 29.2, 64 and 512 13.4 and 21.8.
constexpr int kSumCols = 128, kSumVecs = kSumCols / 8, kSumThreads = 1024, kSumLanes = kSumThreads / kSumVecs;
__global__ void __launch_bounds__(kSumThreads) column_sums_kernel(const uint16_t* __restrict__ g, int64_t pitch, int64_t rows, int64_t cols,
                                                                    uint16_t* __restrict__ out, int splits) {
    __shared__ float part[kSumLanes][kSumCols + 1];
    __shared__ float sums[8][kSumCols];   // of the cluster's CTAs, in rank 0
    const int rank = (int)(blockIdx.x % (unsigned)splits), t = threadIdx.x, lane = t / kSumVecs;
    const int64_t c0 = (int64_t)(blockIdx.x / (unsigned)splits) * kSumCols, c = c0 + (t % kSumVecs) * 8;
    pdl_launch_dependents();
    pdl_wait();
    float s[8] = {};
    if (c + 8 <= cols) {
        const int64_t step = (int64_t)splits * kSumLanes;
        int64_t r = (int64_t)rank * kSumLanes + lane;
        for (; r + 3 * step < rows; r += 4 * step) {   // four loads in flight a lane
            uint4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = __ldg(reinterpret_cast<const uint4*>(g + (r + u * step) * pitch + c));
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) { s[2 * i] += bf16_lo(w[i]); s[2 * i + 1] += bf16_hi(w[i]); }
            }
        }
        for (; r < rows; r += step) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(g + r * pitch + c));
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) { s[2 * i] += bf16_lo(w[i]); s[2 * i + 1] += bf16_hi(w[i]); }
        }
    } else {
        for (int64_t r = (int64_t)rank * kSumLanes + lane; r < rows; r += (int64_t)splits * kSumLanes)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < cols) s[i] += u2f((uint32_t)__ldg(g + r * pitch + c + i) << 16);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) part[lane][(t % kSumVecs) * 8 + i] = s[i];
    if (splits > 1) cluster_sync(); else __syncthreads();   // the other CTAs have started, too
    if (t < kSumCols) {
        float sum = 0.0f;
        for (int l = 0; l < kSumLanes; ++l) sum += part[l][t];
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(map_to_rank(smem_u32(&sums[rank][t]), 0)), "f"(sum) : "memory");
    }
    if (splits > 1) cluster_sync(); else __syncthreads();
    if (rank == 0 && t < kSumCols && c0 + t < cols) {
        float sum = 0.0f;
        for (int z = 0; z < splits; ++z) sum += sums[z][t];
        out[c0 + t] = (uint16_t)pack_bf16_rne(0.0f, sum);
    }
}

inline unsigned grid_x(int64_t nvec, int per_cta) {
    const int64_t g = (nvec + per_cta - 1) / per_cta;
    return (unsigned)(g < (1 << 30) ? g : (1 << 30));
}

}  // namespace

int launch_quantize_fp4(const void* in, int is_fp32, int64_t rows, int64_t cols, int64_t pitch, void* payload, uint8_t* scales, cudaStream_t st) {
    int64_t r = rows, vpr = cols / 8;
    if (pitch == cols) { vpr *= r; r = 1; }
    const dim3 grid(grid_x(vpr, kQThreads * kQU), (unsigned)(r < 65535 ? r : 65535));
    auto* p = static_cast<uint32_t*>(payload);
    const cudaError_t e = is_fp32 ? launch_pdl(quantize_fp4_kernel<true>, grid, dim3(kQThreads), 0, st, in, p, scales, r, vpr, pitch)
                                  : launch_pdl(quantize_fp4_kernel<false>, grid, dim3(kQThreads), 0, st, in, p, scales, r, vpr, pitch);
    return e == cudaSuccess ? check_launch() : kErrLaunch;
}

int launch_column_sums(const void* g, int64_t pitch, int64_t rows, int64_t cols, void* out, cudaStream_t st) {
    const int64_t strips = (cols + kSumCols - 1) / kSumCols;
    int splits = 1;
    while (splits < 8 && strips * splits < 4 * sm_count() && rows >= (int64_t)splits * 4 * kSumLanes) splits *= 2;
    if (strips * splits > 0x7FFFFFFF) return kErrTooLarge;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(strips * splits));
    cfg.blockDim = dim3(kSumThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {(unsigned)splits, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = splits > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, column_sums_kernel, static_cast<const uint16_t*>(g), pitch, rows, cols, static_cast<uint16_t*>(out), splits);
    return e == cudaSuccess ? check_launch() : kErrLaunch;
}

int launch_dequantize(const void* payload, const uint8_t* scales, void* out, int out_fp32, int64_t rows, int64_t cols, int bcols, int fmt,
                      cudaStream_t st) {
    const int64_t nvec = rows * cols / (out_fp32 ? 4 : 8);
    constexpr int U = 4;
    int lg = 0;
    while ((1 << lg) < bcols) ++lg;
    const dim3 grid(grid_x(nvec, kQThreads * U));
    auto* p = static_cast<const uint8_t*>(payload);
    auto* o = static_cast<uint4*>(out);
    cudaError_t e = cudaErrorInvalidValue;
#define MORB_GO(F)                                                                                                    \
    e = out_fp32 ? launch_pdl(dequantize_kernel<F, true, U>, grid, dim3(kQThreads), 0, st, p, scales, o, nvec, lg)    \
                 : launch_pdl(dequantize_kernel<F, false, U>, grid, dim3(kQThreads), 0, st, p, scales, o, nvec, lg)
    if (fmt == kE4M3) MORB_GO(kE4M3);
    else if (fmt == kE5M2) MORB_GO(kE5M2);
    else if (fmt == kE2M3) MORB_GO(kE2M3);
    else if (fmt == kE2M1) MORB_GO(kE2M1);
#undef MORB_GO
    return e == cudaSuccess ? check_launch() : kErrLaunch;
}

}  // namespace morb
