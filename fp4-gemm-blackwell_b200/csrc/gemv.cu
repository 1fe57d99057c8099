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
// Split.  A CTA's 8 warps are RG groups of 32 rows times 8 / RG slices of K (its
// steps in turn), joined in shared memory: more rows in a CTA read x less
// often, fewer rows give more CTAs.
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
constexpr int kChunkBytes = 16384;             // a chunk of x in FP16

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
};

// Chunk c (8 elements) of row g of a chunk of x: where it lies, so that the
// eight lanes of one phase of the reads meet distinct banks.
__device__ __forceinline__ int x_offset(int row_bytes, int g, int c) { return g * row_bytes + 16 * (c ^ ((c >> 3) & 1) ^ ((g & 1) << 1)); }

template <int NT, int RG, int W>
__global__ void __launch_bounds__(32 * W) gemv_kernel(const __grid_constant__ GemvParams p) {
    constexpr int kWarps = W, kThreads = 32 * W;
    constexpr int KS = kWarps / RG;                   // slices of K
    constexpr int KC = kChunkBytes / (2 * 8 * NT);    // elements of a chunk
    constexpr int kChunkSteps = KC / kStep;
    constexpr int kRowBytes = 2 * KC;
    constexpr int kPieces = KC / 8 / 32;              // 16-byte pieces of a row's chunk a lane
    constexpr int kHeld = (8 * NT + kWarps - 1) / kWarps;  // rows of x that a warp converts
    static_assert(kChunkSteps % KS == 0 || KS % kChunkSteps == 0, "slices take whole chunks in turn");
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_factor[2][8 * NT];
    chain();
    uint8_t* sx = smem + kWarps * kStages * kStageBytes;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int rg = warp % RG, ks = warp / RG;
    const int part = blockIdx.x % (4 / RG), block = blockIdx.x / (4 / RG);  // which of the 128 rows' r
    const int r0 = 8 * (part * RG + rg);                                    // the warp's first r
    const int m0 = blockIdx.y * 8 * NT, rows = min(8 * NT, p.m - m0);
    const int steps = p.k_pad / kStep, chunks = (p.k + KC - 1) / KC;
    const int nsb = p.k_pad / 16;

    // ---- the stream of the warp's weights: steps ks, ks + KS, ...
    const uint8_t* w_src = p.w + ((size_t)(block * 128 + r0 + g) * p.k_pad >> 1) + 16 * t;
    const size_t w_row32 = (size_t)16 * p.k_pad;  // 32 rows further
    const uint8_t* s_src = p.sf + (size_t)block * 128 * nsb + (r0 + g) * 16 + (t >> 1) * 512;
    uint8_t* ring = smem + warp * kStages * kStageBytes + 16 * lane;
    const uint32_t ring_addr = ptx::smem_u32(ring);
    const int mine = (steps - ks + KS - 1) / KS;
    auto issue = [&](int i) {
        if (i < mine) {
            const int step = ks + i * KS;
            const uint32_t dst = ring_addr + (i % kStages) * kStageBytes;
#pragma unroll
            for (int q = 0; q < 4; ++q) copy_async<16>(dst + 512 * q, w_src + q * w_row32 + (size_t)step * (kStep / 2), true);
            copy_async<16>(dst + 2048, s_src + (size_t)step * 1024, true);
        }
        copy_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);

    // ---- x, chunk by chunk: warp w holds rows w, w + W between the global read and the shared write
    uint4 held[kHeld][kPieces];
    auto fetch = [&](int c) {
#pragma unroll
        for (int nt = 0; nt < kHeld; ++nt) {
            const int row = warp + kWarps * nt;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                held[nt][i] = make_uint4(0u, 0u, 0u, 0u);
                const int k = c * KC + 8 * (lane + 32 * i);
                if (row < rows && k < p.k) {
                    const uint16_t* src = p.x + (size_t)(m0 + row) * p.ldx + k;
                    if (p.x_vec && k + 8 <= p.k) {
                        held[nt][i] = __ldg(reinterpret_cast<const uint4*>(src));
                    } else {
                        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (k + e < p.k) w[e / 2] |= (uint32_t)src[e] << (16 * (e & 1));
                        held[nt][i] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
        }
    };
    auto put = [&](int c) {
        uint8_t* to = sx + (c & 1) * kChunkBytes;
#pragma unroll
        for (int nt = 0; nt < kHeld; ++nt) {
            const int row = warp + kWarps * nt;
            if (row >= rows) continue;  // such columns are never stored
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                top = max_abs_bf16x2(max_abs_bf16x2(top, held[nt][i].x), held[nt][i].y);
                top = max_abs_bf16x2(max_abs_bf16x2(top, held[nt][i].z), held[nt][i].w);
            }
            top = group_umax<32>(max((top << 16) & 0x7FFF0000u, top & 0x7FFF0000u));
            const int up = min(max(141 - (int)(top >> 23), -126), 126);
            const float f = __int_as_float((127 + up) << 23);
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const uint4 w = held[nt][i];
                *reinterpret_cast<uint4*>(to + x_offset(kRowBytes, row, lane + 32 * i)) =
                    make_uint4(pack_f16(bf16_lo(w.x) * f, bf16_hi(w.x) * f), pack_f16(bf16_lo(w.y) * f, bf16_hi(w.y) * f),
                               pack_f16(bf16_lo(w.z) * f, bf16_hi(w.z) * f), pack_f16(bf16_lo(w.w) * f, bf16_hi(w.w) * f));
            }
            if (lane == 0) s_factor[c & 1][row] = __int_as_float((127 - up) << 23);
        }
    };
    fetch(0);
    put(0);
    __syncthreads();

    float sum[2][NT][4];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[a][nt][i] = 0.0f;

    const uint32_t pick0 = t & 1 ? 0x4242u : 0x4040u, pick1 = t & 1 ? 0x4343u : 0x4141u;  // the lane's two scale bytes
    // x_offset of chunk 4 t + u of the lane's row: the permutation moves u alone
    const uint8_t* x_lane = sx + g * kRowBytes + 64 * t;
    const int x_swap = 16 * ((t >> 1) ^ ((g & 1) << 1));
    int i = 0;
    for (int c = 0; c < chunks; ++c) {
        if (c + 1 < chunks) fetch(c + 1);
        float acc[2][NT][4];
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[a][nt][e] = 0.0f;
        const int end = min(steps, (c + 1) * kChunkSteps);
        for (; ks + i * KS < end; ++i) {
            copy_wait<kStages - 2>();
            const uint8_t* st = ring + (i % kStages) * kStageBytes;
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
            issue(i + kStages - 1);
            const uint8_t* xs = x_lane + (c & 1) * kChunkBytes + (ks + i * KS - c * kChunkSteps) * 256;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                uint4 xv[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) xv[nt] = lds128(xs + 8 * nt * kRowBytes + ((16 * u) ^ x_swap));
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
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float f0 = s_factor[c & 1][8 * nt + 2 * t], f1 = s_factor[c & 1][8 * nt + 2 * t + 1];
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                sum[a][nt][0] += acc[a][nt][0] * f0, sum[a][nt][1] += acc[a][nt][1] * f1;
                sum[a][nt][2] += acc[a][nt][2] * f0, sum[a][nt][3] += acc[a][nt][3] * f1;
            }
        }
        if (c + 1 < chunks) put(c + 1);  // the other buffer: its readers passed the last barrier
        __syncthreads();
    }
    copy_wait<0>();

    // ---- the slices of K joined in their order; row 8 RG q + 8 rg + g of the CTA is weight row
    // 128 block + 32 q + 8 (part RG + rg) + g
    float* red = reinterpret_cast<float*>(sx);
    constexpr int kRows = 32 * RG;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 8 * RG * (2 * a + (e >> 1)) + 8 * rg + g, col = 8 * nt + 2 * t + (e & 1);
                red[(ks * 8 * NT + col) * kRows + row] = sum[a][nt][e];
            }
    __syncthreads();
    for (int j = tid; j < rows * kRows; j += kThreads) {
        const int col = j / kRows, row = j - col * kRows;
        const int n = 128 * block + 32 * (row / (8 * RG)) + 8 * part * RG + row % (8 * RG);
        if (n >= p.n) continue;
        float y = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) y += red[(s * 8 * NT + col) * kRows + row];
        y *= p.alpha;
        if (p.bias) y += bf16_lo(p.bias[n]);
        p.y[(size_t)(m0 + col) * p.ldy + n] = (uint16_t)(pack_bf16(y, 0.0f) & 0xFFFFu);
    }
}

constexpr int kMaxDevices = 64;

template <int NT, int RG, int W>
cudaError_t launch(const GemvParams& p, cudaStream_t st) {
    constexpr int kSmem = W * kStages * kStageBytes + 2 * kChunkBytes;
    static std::mutex mu;
    static bool ready[kMaxDevices];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= kMaxDevices) return cudaErrorInvalidDevice;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (!ready[dev]) {
            e = cudaFuncSetAttribute(gemv_kernel<NT, RG, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
            if (e != cudaSuccess) return e;
            ready[dev] = true;
        }
    }
    const long blocks = ((long)p.n + 127) / 128 * (4 / RG);
    const dim3 grid((unsigned)blocks, (unsigned)((p.m + 8 * NT - 1) / (8 * NT)));
    return launch_chained(gemv_kernel<NT, RG, W>, grid, 32 * W, kSmem, st, p);
}

template <int NT>
cudaError_t launch_rows(const GemvParams& p, cudaStream_t st) {
    const long blocks = ((long)p.n + 127) / 128;
    if (blocks >= 120) return launch<NT, 4, 16>(p, st);
    if (blocks >= 74) return launch<NT, 2, 8>(p, st);
    return launch<NT, 1, 8>(p, st);
}

}  // namespace
}  // namespace fp4b

using namespace fp4b;

FP4B_EXPORT int fp4b_gemv_cached(const void* x, int m, int k_in, long ldx, const void* handle, int n_out, void* y,
                                 long ldy, const void* bias, void* stream) {
    CacheView c;
    if (!cache_view(handle, &c)) {
        set_last_error("null or invalid cache handle");
        return -1;
    }
    if (!x || !y || m <= 0 || m > 16 * 65535 || k_in <= 0 || k_in > c.K || ldx < k_in || n_out <= 0 || n_out > c.N ||
        ldy < n_out) {
        set_last_error("fp4b_gemv_cached: bad shape (m=%d k=%d n=%d vs cache %dx%d)", m, k_in, n_out, c.N, c.K);
        return -1;
    }
    const bool vec = ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    const GemvParams p{static_cast<const uint16_t*>(x), c.fp4, c.sf, static_cast<uint16_t*>(y),
                       static_cast<const uint16_t*>(bias), ldx, ldy, m, n_out, k_in, c.K, vec, c.w_alpha * kScaleUnit};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return launch_status(m <= 8 ? launch_rows<1>(p, st) : launch_rows<2>(p, st), "fp4b_gemv_cached");
}
