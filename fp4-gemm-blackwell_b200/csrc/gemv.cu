// gemv.cu -- few rows of BF16 activations times a cached NVFP4 weight.
//
//   y[m, n] = w_alpha * sum_k x[m, k] * W[n, k] (+ bias[n]),
//   W[n, k] = e2m1[n, k] * ue4m3[n, k / 16]
//
// with the activations as they are: at one to a few rows the time is that of
// the weight's N * K * 9 / 16 bytes, so nothing is gained by quantizing x.
//
// Products.  mma.sync m16n8k16 in FP16 with fp32 sums: 16 weight rows times 8
// activation rows (tcgen05 would need the weight unpacked to shared memory in
// its own layout first, as much work as the products).  A decoded weight has
// at most 6 significant bits and lies in FP16's range, so it enters exactly;
// its scale enters as 2^-8 of its value, a shift of its byte.  The activations
// of one row's chunk of K are multiplied by the power of two that puts their
// largest into [2^14, 2^15): exact, down to 2^-32 of that largest (below, they
// lose bits that fp32 sums lose too); the chunk's sums are multiplied back.
//
// Reads.  A warp takes 32 weight rows, the four rows r, r + 32, r + 64, r + 96
// of eight r: their scales for 64 elements of K are 16 neighbouring bytes of
// the scale layout, so the cache is read as it lies, each byte once.  Per 128
// elements of K a lane copies the 16 code bytes of its four rows and its 16
// scale bytes to shared memory with cp.async, several steps ahead, and reads
// back only what it copied itself: no barrier for the weights.  The order of K
// inside a step is free; a lane's 32 elements are the ones that it holds.
//
// Split.  A CTA's W warps are RG groups of 32 rows times W / RG slices of K (its
// steps in turn), joined in shared memory: more rows in a CTA read x less
// often, fewer rows give more CTAs.
//
// x.  Few elements of x (up to kWholeBytes in FP16) are converted by every CTA
// for itself, whole, before its first step.  More of them would cost each CTA
// more than its weights: a kernel of its own converts them first, into the
// image of shared memory that the CTAs then copy chunk by chunk; the weights'
// stream starts while it runs.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>
#include <mutex>

#include "decode_core.cuh"
#include "fp4b_internal.h"
#include "ptx_sm100.cuh"

#define FP4B_EXPORT extern "C" __attribute__((visibility("default")))

namespace fp4b {
namespace {

using namespace decode;

constexpr int kStep = 128;                     // elements of K of one step
constexpr int kStageBytes = 5 * 512;           // a warp's step: four code pieces and the scales, 16 bytes a lane
constexpr int kStages = 3;
constexpr int kWholeBytes = 49152;             // of x in FP16 that every CTA converts for itself
constexpr int kChunkBytes = 32768;             // a chunk of x in FP16

struct GemvParams {
    const uint16_t* x;
    const uint8_t* w;
    const uint8_t* sf;
    uint16_t* y;
    const uint16_t* bias;
    long ldx, ldy;
    int m, n, k, k_pad;
    int x_vec;  // rows of x are 16-byte aligned
    float alpha;
    uint8_t* image;  // x in FP16, chunk by chunk as in shared memory, and the rows' factors; null: converted by each CTA
    float* factors;
};

// Chunk c (8 elements) of row g of a chunk of x: where it lies, so that the
// eight lanes of one phase of the reads meet distinct banks.
__device__ __forceinline__ int x_offset(int row_bytes, int g, int c) { return g * row_bytes + 16 * (c ^ ((c >> 3) & 1) ^ ((g & 1) << 1)); }

// Elements of a chunk of x with 8 NT rows.
template <int NT>
constexpr int chunk_elements() { return kChunkBytes / (16 * NT); }

// Elements k .. k+7 of a row of x, zeros past its end.
__device__ __forceinline__ uint4 x_eight(const GemvParams& p, const uint16_t* row, int k) {
    if (p.x_vec && k + 8 <= p.k) return __ldg(reinterpret_cast<const uint4*>(row + k));
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (k + e < p.k) w[e / 2] |= (uint32_t)row[k + e] << (16 * (e & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint32_t max_magnitudes(uint32_t top, uint4 v) {
    return max_abs_bf16x2(max_abs_bf16x2(max_abs_bf16x2(max_abs_bf16x2(top, v.x), v.y), v.z), v.w);
}

// From a row's largest magnitude (fp32 bits): the power of two that its elements
// are multiplied by, as an exponent.
__device__ __forceinline__ int scale_exponent(uint32_t top) { return min(max(141 - (int)(top >> 23), -126), 126); }
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((127 + e) << 23); }

__device__ __forceinline__ uint4 eight_to_f16(uint4 v, float f) {
    return make_uint4(pack_f16(bf16_lo(v.x) * f, bf16_hi(v.x) * f), pack_f16(bf16_lo(v.y) * f, bf16_hi(v.y) * f),
                      pack_f16(bf16_lo(v.z) * f, bf16_hi(v.z) * f), pack_f16(bf16_lo(v.w) * f, bf16_hi(v.w) * f));
}

// x into its image: a CTA a row.
template <int NT>
__global__ void __launch_bounds__(256) gemv_image_kernel(const __grid_constant__ GemvParams p) {
    constexpr int KC = chunk_elements<NT>();
    __shared__ uint32_t s_top[8];
    chain();
    const int row = blockIdx.x, tile = row / (8 * NT), in_tile = row % (8 * NT);
    const int chunks = (p.k + KC - 1) / KC;
    const uint16_t* src = p.x + (size_t)row * p.ldx;
    uint32_t top = 0;
    for (int k = 8 * threadIdx.x; k < p.k; k += 8 * 256) top = max_magnitudes(top, x_eight(p, src, k));
    top = group_umax<32>(max((top << 16) & 0x7FFF0000u, top & 0x7FFF0000u));
    if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, s_top[i]);
    const int e = scale_exponent(top);
    const float f = power_of_two(e);
    if (threadIdx.x == 0) p.factors[row] = power_of_two(-e);
    uint8_t* image = p.image + (size_t)tile * chunks * kChunkBytes;
    for (int k = 8 * threadIdx.x; k < chunks * KC; k += 8 * 256)
        *reinterpret_cast<uint4*>(image + (size_t)(k / KC) * kChunkBytes + x_offset(2 * KC, in_tile, (k % KC) / 8)) =
            eight_to_f16(k < p.k ? x_eight(p, src, k) : make_uint4(0u, 0u, 0u, 0u), f);
}

template <int NT, int RG, int W, bool IMAGE>
__global__ void __launch_bounds__(32 * W) gemv_kernel(const __grid_constant__ GemvParams p) {
    constexpr int kThreads = 32 * W;
    constexpr int KS = W / RG;                        // slices of K
    constexpr int KC = chunk_elements<NT>();          // elements of a chunk
    constexpr int kChunkSteps = KC / kStep;
    static_assert(kChunkSteps % KS == 0, "every warp has the same steps of a whole chunk");
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_factor[8 * NT];
    [[maybe_unused]] __shared__ uint32_t s_top[8 * NT];
    uint8_t* sx = smem + W * kStages * kStageBytes;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int rg = warp % RG, ks = warp / RG;
    const int part = blockIdx.x % (4 / RG), block = blockIdx.x / (4 / RG);  // which of the 128 rows' r
    const int r0 = 8 * (part * RG + rg);                                    // the warp's first r
    const int m0 = blockIdx.y * 8 * NT, rows = min(8 * NT, p.m - m0);
    const int steps = p.k_pad / kStep;
    const int nsb = p.k_pad / 16;

    // ---- the stream of the warp's weights: steps ks, ks + KS, ...
    const uint8_t* w_src = p.w + ((size_t)(block * 128 + r0 + g) * p.k_pad >> 1) + 16 * t;
    const size_t w_row32 = (size_t)16 * p.k_pad;  // 32 rows further
    const uint8_t* s_src = p.sf + (size_t)block * 128 * nsb + (r0 + g) * 16 + (t >> 1) * 512;
    uint8_t* ring = smem + warp * kStages * kStageBytes + 16 * lane;
    const uint32_t ring_addr = ptx::smem_u32(ring);
    const int used = min(steps, (p.k + kStep - 1) / kStep);  // x is zero past p.k
    const int mine = (used - ks + KS - 1) / KS;
    auto issue = [&](int i, int slot) {
        if (i < mine) {
            const int step = ks + i * KS;
            const uint32_t dst = ring_addr + slot * kStageBytes;
#pragma unroll
            for (int q = 0; q < 4; ++q) copy_async<16>(dst + 512 * q, w_src + q * w_row32 + (size_t)step * (kStep / 2), true);
            copy_async<16>(dst + 2048, s_src + (size_t)step * 1024, true);
        }
        copy_commit();
    };

    // ---- x, whole or by chunks
    const int chunks = IMAGE ? (p.k + KC - 1) / KC : 1;
    const int row_bytes = IMAGE ? 2 * KC : 2 * used * kStep;
    const uint8_t* image = IMAGE ? p.image + (size_t)blockIdx.y * chunks * kChunkBytes + 16 * tid : nullptr;
    auto fetch = [&](int c) {
        const uint32_t dst = ptx::smem_u32(sx) + (c & 1) * kChunkBytes + 16 * tid;
#pragma unroll
        for (int i = 0; i < kChunkBytes / (16 * kThreads); ++i)
            copy_async<16>(dst + i * 16 * kThreads, image + (size_t)c * kChunkBytes + i * 16 * kThreads, true);
    };
    if constexpr (IMAGE) {
        // The image's kernel lets this one start once all that came before it is
        // complete, the weights among it: only x is waited for.
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) issue(i, i);
        chain();
        fetch(0);
        copy_commit();
        if (tid < rows) s_factor[tid] = p.factors[m0 + tid];
        copy_wait<0>();
    } else {
        chain();
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) issue(i, i);
        // A row to kThreads / 2^q threads, 2^q rows or more.
        const int q = rows > 1 ? 32 - __clz(rows - 1) : 0, team = kThreads >> q, row = tid / team, at = tid % team;
        const uint16_t* src = p.x + (size_t)(m0 + row) * p.ldx;
        if (tid < 8 * NT) s_top[tid] = 0;
        __syncthreads();
        uint32_t top = 0;
        if (row < rows) {
#pragma unroll 4
            for (int k = 8 * at; k < p.k; k += 8 * team) top = max_magnitudes(top, x_eight(p, src, k));
        }
        top = max((top << 16) & 0x7FFF0000u, top & 0x7FFF0000u);
        top = team >= 32 ? group_umax<32>(top) : group_umax<16>(top);
        if (row < rows && (at & 15) == 0) atomicMax(&s_top[row], top);
        __syncthreads();
        if (row < rows) {
            const int e = scale_exponent(s_top[row]);
            const float f = power_of_two(e);
            if (at == 0) s_factor[row] = power_of_two(-e);
#pragma unroll 4
            for (int k = 8 * at; k < used * kStep; k += 8 * team)
                *reinterpret_cast<uint4*>(sx + x_offset(row_bytes, row, k / 8)) =
                    eight_to_f16(k < p.k ? x_eight(p, src, k) : make_uint4(0u, 0u, 0u, 0u), f);
        }
    }
    __syncthreads();

    float acc[2][NT][4];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[a][nt][e] = 0.0f;

    const uint32_t pick0 = t & 1 ? 0x4242u : 0x4040u, pick1 = t & 1 ? 0x4343u : 0x4141u;  // the lane's two scale bytes
    // x_offset of chunk 4 t + u of the lane's row: the permutation moves u alone.
    // Lanes whose row does not exist read row 0; their columns are never stored.
    const uint8_t* x_lane[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) x_lane[nt] = sx + (8 * nt + g < rows ? 8 * nt + g : (g & 1) < rows ? (g & 1) : 0) * row_bytes + 64 * t;
    const int x_swap = 16 * ((t >> 1) ^ ((rows > 1 ? g & 1 : 0) << 1));
    int i = 0, slot = 0;
    for (int c = 0; c < chunks; ++c) {
        if (IMAGE && c + 1 < chunks) fetch(c + 1);  // completes with the weights' next groups
        const int end = IMAGE ? min(used, (c + 1) * kChunkSteps) : used;
        const int x_base = (IMAGE ? (c & 1) * kChunkBytes - c * kChunkSteps * 256 : 0);
        for (int step = ks + i * KS; step < end; step += KS, ++i) {
            copy_wait<kStages - 2>();
            const uint8_t* st = ring + slot * kStageBytes;
            uint32_t w[4][4], s0[4], s1[4];
            const uint4 sc = lds128(st + 2048);
            const uint32_t sw[4] = {sc.x, sc.y, sc.z, sc.w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint4 v = lds128(st + 512 * q);
                w[q][0] = v.x, w[q][1] = v.y, w[q][2] = v.z, w[q][3] = v.w;
                s0[q] = ue4m3x2_to_f16(__byte_perm(sw[q], 0u, pick0));
                s1[q] = ue4m3x2_to_f16(__byte_perm(sw[q], 0u, pick1));
            }
            issue(i + kStages - 1, slot == 0 ? kStages - 1 : slot - 1);
            slot = slot == kStages - 1 ? 0 : slot + 1;
            const int at = x_base + step * 256;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                uint4 xv[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) xv[nt] = lds128(x_lane[nt] + at + ((16 * u) ^ x_swap));
                uint32_t a[4][4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    e2m1x8_to_f16(w[q][u], a[q]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[q][e] = mul_f16x2(a[q][e], u < 2 ? s0[q] : s1[q]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma<false>(acc[0][nt], a[0][0], a[1][0], a[0][1], a[1][1], xv[nt].x, xv[nt].y);
                    mma<false>(acc[1][nt], a[2][0], a[3][0], a[2][1], a[3][1], xv[nt].x, xv[nt].y);
                    mma<false>(acc[0][nt], a[0][2], a[1][2], a[0][3], a[1][3], xv[nt].z, xv[nt].w);
                    mma<false>(acc[1][nt], a[2][2], a[3][2], a[2][3], a[3][3], xv[nt].z, xv[nt].w);
                }
            }
        }
        if (IMAGE && c + 1 < chunks) {
            // The next chunk's copies are in the group of this chunk's first step.
            copy_wait<(kChunkSteps / KS > 1 ? kStages - 2 : 0)>();
            __syncthreads();
        }
    }

    // ---- the slices of K joined in their order; row 8 RG q + 8 rg + g of the CTA is weight row
    // 128 block + 32 q + 8 (part RG + rg) + g
    copy_wait<0>();
    __syncthreads();  // the rings are idle
    float* red = reinterpret_cast<float*>(smem);
    constexpr int kRows = 32 * RG;
    static_assert(KS * 8 * NT * kRows * 4 <= W * kStages * kStageBytes, "the rings hold the slices' sums");
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 8 * RG * (2 * a + (e >> 1)) + 8 * rg + g, col = 8 * nt + 2 * t + (e & 1);
                red[(ks * 8 * NT + col) * kRows + row] = acc[a][nt][e];
            }
    __syncthreads();
    for (int j = tid; j < rows * kRows; j += kThreads) {
        const int col = j / kRows, row = j - col * kRows;
        const int n = 128 * block + 32 * (row / (8 * RG)) + 8 * part * RG + row % (8 * RG);
        if (n >= p.n) continue;
        float y = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) y += red[(s * 8 * NT + col) * kRows + row];
        y *= s_factor[col] * p.alpha;
        if (p.bias) y += bf16_lo(p.bias[n]);
        p.y[(size_t)(m0 + col) * p.ldy + n] = (uint16_t)(pack_bf16(y, 0.0f) & 0xFFFFu);
    }
}

constexpr int kMaxDevices = 64;

template <int NT, int RG, int W, bool IMAGE>
cudaError_t launch(const GemvParams& p, cudaStream_t st) {
    constexpr int kRing = W * kStages * kStageBytes;
    static std::mutex mu;
    static bool ready[kMaxDevices];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= kMaxDevices) return cudaErrorInvalidDevice;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (!ready[dev]) {
            e = cudaFuncSetAttribute(gemv_kernel<NT, RG, W, IMAGE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     kRing + (IMAGE ? 2 * kChunkBytes : kWholeBytes));
            if (e != cudaSuccess) return e;
            ready[dev] = true;
        }
    }
    if (IMAGE) {
        e = launch_chained(gemv_image_kernel<NT>, dim3((unsigned)p.m), 256, 0, st, p);
        if (e != cudaSuccess) return e;
    }
    const long blocks = ((long)p.n + 127) / 128 * (4 / RG);
    const dim3 grid((unsigned)blocks, (unsigned)((p.m + 8 * NT - 1) / (8 * NT)));
    const int x_bytes = IMAGE ? 2 * kChunkBytes : std::min(p.m, 8 * NT) * 2 * ((p.k + kStep - 1) / kStep * kStep);
    return launch_chained(gemv_kernel<NT, RG, W, IMAGE>, grid, 32 * W, kRing + x_bytes, st, p);
}

// Rows of x that share a tile's products: 8 or 16.
int tile_rows(int m) { return m <= 8 ? 8 : 16; }

// Whether every CTA converts x for itself.
bool x_whole(int m, int k) { return (long)std::min(m, tile_rows(m)) * 2 * ((k + kStep - 1) / kStep * kStep) <= kWholeBytes; }

template <int NT, bool IMAGE>
cudaError_t launch_rows(const GemvParams& p, cudaStream_t st) {
    const long blocks = ((long)p.n + 127) / 128;
    if (blocks >= 120) return launch<NT, 4, 16, IMAGE>(p, st);
    if (blocks >= 74) return launch<NT, 2, 8, IMAGE>(p, st);
    return launch<NT, 1, 8, IMAGE>(p, st);
}

template <int NT>
cudaError_t launch_x(const GemvParams& p, cudaStream_t st) {
    return p.image ? launch_rows<NT, true>(p, st) : launch_rows<NT, false>(p, st);
}

}  // namespace
}  // namespace fp4b

using namespace fp4b;

FP4B_EXPORT long fp4b_gemv_workspace(int m, int k_in) {
    if (m <= 0 || k_in <= 0) {
        set_last_error("fp4b_gemv_workspace: m and k must be positive");
        return -1;
    }
    if (x_whole(m, k_in)) return 0;
    const int rows = tile_rows(m), chunk = kChunkBytes / (2 * rows);
    return (long)((m + rows - 1) / rows) * ((k_in + chunk - 1) / chunk) * kChunkBytes + 4l * m;
}

FP4B_EXPORT int fp4b_gemv_cached(const void* x, int m, int k_in, long ldx, const void* handle, int n_out, void* y,
                                 long ldy, const void* bias, void* workspace, long workspace_bytes, void* stream) {
    CacheView c;
    if (!cache_view(handle, &c)) {
        set_last_error("null or invalid cache handle");
        return -1;
    }
    if (!x || !y || m <= 0 || m > 8 * 65535 || k_in <= 0 || k_in > c.K || ldx < k_in || n_out <= 0 || n_out > c.N ||
        ldy < n_out) {
        set_last_error("fp4b_gemv_cached: bad shape (m=%d k=%d n=%d vs cache %dx%d)", m, k_in, n_out, c.N, c.K);
        return -1;
    }
    const long need = fp4b_gemv_workspace(m, k_in);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))) {
        set_last_error("fp4b_gemv_cached: needs a 16-byte aligned workspace of %ld bytes", need);
        return -1;
    }
    const bool vec = ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    uint8_t* image = need > 0 ? static_cast<uint8_t*>(workspace) : nullptr;
    const GemvParams p{static_cast<const uint16_t*>(x), c.fp4, c.sf, static_cast<uint16_t*>(y),
                       static_cast<const uint16_t*>(bias), ldx, ldy, m, n_out, k_in, c.K, vec, c.w_alpha * kScaleUnit, image,
                       image ? reinterpret_cast<float*>(image + (need - 4l * m)) : nullptr};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return launch_status(tile_rows(m) == 8 ? launch_x<1>(p, st) : launch_x<2>(p, st), "fp4b_gemv_cached");
}
