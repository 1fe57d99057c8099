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
// lose bits, as they do in fp32 sums unless the largest meets a weight of zero); the chunk's sums are multiplied back.
//
// Reads.  A warp takes 32 weight rows, the four rows r, r + 32, r + 64, r + 96
// of eight r: their scales for 64 elements of K are 16 neighbouring bytes of
// the scale layout, so the cache is read as it lies, each byte once.  Per 128
// elements of K a lane copies the 16 code bytes of its four rows and its 16
// scale bytes to shared memory with cp.async, several steps ahead, and reads
// back only what it copied itself: no barrier for the weights.  The order of K
// inside a step is free; a lane's 32 elements are the ones that it holds.
//
// Split.  Every CTA converts the x that it needs itself, before its first step.
// Its 8 or 16 warps are RG groups of 32 rows of the weight times slices of K,
// joined in shared memory.  Where there are too few rows for all SMs, or x does
// not fit beside the rings, K is cut into slices of CTAs of their own too, whose
// sums go to the workspace, and a second kernel adds them in their order.
// Large weights: a CTA keeps one slice of x and walks groups of rows with it, each
// warp a group at a time and without a barrier, so that x is converted 148 times at
// most.  (x by chunks through shared memory instead, all of it for every CTA, took
// a barrier every two steps and as many bytes of x as of the weight from L2: 53.5 us
// for 16 rows of x, 16384 x 16384, now 40.)
//
// Measured on B200 (copy bandwidth 6.54 TB/s): one row, 28672 x 8192 29.4 us = 4.5
// TB/s; 16 rows, 16384 x 16384 40.1 us = 3.8 TB/s, where the copies alone take 30
// and the products alone 31: beside mma.sync the decoding's instructions cost a
// scheduler nearly their own time more.  6 rows, 19072 x 16384 39.1 us; 5 rows, 15360 x
// 2880 9.9 us, on 120 SMs and with x converted before the weights' third step is asked
// for; one row, 2880 x 2880 4.5 us, a launch and one chain of waits.
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
constexpr int kWalkBytes = 65536;              // of x in FP16 that a CTA keeps that walks rows
constexpr int kSliceBytes = 49152;             // that any other keeps

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
    // Slices of K: their number, their steps (the first `slice_more` have one more),
    // the row groups' CTAs of each, and the slices' sums [tiles of rows of
    // x][slices][8 NT][n_pad].
    int slices, slice_steps, slice_more, ctas;
    float* sums;
    int n_pad;
};

// x in shared memory: 16 bytes more after every 128, and rows 32 bytes more than a
// multiple of 128, so that the eight lanes of one phase of the reads (two rows, every
// fourth chunk of 8 elements) meet distinct banks, at constant offsets from a step's
// start.
constexpr int kXStep = 2 * kStep + 32;  // bytes of a step of one row
__host__ __device__ constexpr int x_row_bytes(int steps) { return steps * kXStep + 32 * ((1 - steps) & 3); }
__device__ __forceinline__ int x_offset(int row_bytes, int g, int c) { return g * row_bytes + 16 * (c + (c >> 3)); }
// Room for `bytes` of x.
constexpr int x_room(int bytes) { return bytes / 8 * 9 + 16 * 96; }

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

// Elements [k0, k0 + steps * kStep) of `rows` rows of x to shared memory in FP16 (at
// most kBytes), each row by its own power of two; factor: what undoes it.  All
// threads of the CTA call it; the reads of all pieces are in flight together.
template <int kThreads, int kBytes>
__device__ __forceinline__ void convert_x(const GemvParams& p, int m0, int rows, int k0, int steps, uint8_t* sx, uint32_t* s_top,
                                          float* factor) {
    constexpr int kHeld = kBytes / 16 / kThreads;
    const int per_row = steps * (kStep / 8), pieces = rows * per_row;
    const float inv = 1.0f / (float)per_row;
    auto row_of = [&](int piece) { return (int)(((float)piece + 0.5f) * inv); };  // exact: half a piece from a boundary at least
    if (threadIdx.x < 16) s_top[threadIdx.x] = 0;
    uint4 v[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int piece = threadIdx.x + i * kThreads, row = row_of(piece), k = k0 + 8 * (piece - row * per_row);
        v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (piece < pieces && k < p.k) v[i] = x_eight(p, p.x + (size_t)(m0 + row) * p.ldx, k);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        if (i * kThreads >= pieces) break;
        const int piece = threadIdx.x + i * kThreads, row = row_of(min(piece, pieces - 1));
        uint32_t top = max_magnitudes(0u, v[i]);
        top = max((top << 16) & 0x7FFF0000u, top & 0x7FFF0000u);
        if (__all_sync(0xffffffffu, row == __shfl_sync(0xffffffffu, row, 0))) {
            top = __reduce_max_sync(0xffffffffu, top);
            if ((threadIdx.x & 31) == 0) atomicMax(&s_top[row], top);
        } else {
            atomicMax(&s_top[row], top);
        }
    }
    __syncthreads();
    if (threadIdx.x < rows) factor[threadIdx.x] = power_of_two(-scale_exponent(s_top[threadIdx.x]));
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int piece = threadIdx.x + i * kThreads;
        if (piece >= pieces) break;
        const int row = row_of(piece);
        *reinterpret_cast<uint4*>(sx + x_offset(x_row_bytes(steps), row, piece - row * per_row)) =
            eight_to_f16(v[i], power_of_two(scale_exponent(s_top[row])));
    }
    __syncthreads();
}

// A lane's view of the weights of a warp's 32 rows, r0 + g + 32 q of block `block`:
// where its 16-byte pieces of step 0 lie.
struct WeightLane {
    const uint8_t *w, *s;
    size_t row32;  // 32 rows further
};
__device__ __forceinline__ WeightLane weight_lane(const GemvParams& p, int block, int r0, int g, int t) {
    return WeightLane{p.w + ((size_t)(block * 128 + r0 + g) * p.k_pad >> 1) + 16 * t,
                      p.sf + (size_t)block * 8 * p.k_pad + (r0 + g) * 16 + (t >> 1) * 512, (size_t)16 * p.k_pad};
}
// The lane's copies of one step into its place of a stage.
__device__ __forceinline__ void copy_step(uint32_t dst, const WeightLane& from, int step) {
#pragma unroll
    for (int q = 0; q < 4; ++q) copy_async<16>(dst + 512 * q, from.w + q * from.row32 + (size_t)step * (kStep / 2), true);
    copy_async<16>(dst + 2048, from.s + (size_t)step * 1024, true);
}

// A lane's view of x in shared memory: chunk 4 t + u of its row in a step lies at
// base[nt] + kXStep step + 16 u.  Lanes whose row does not exist read another one;
// their columns are never stored.
template <int NT>
struct XLane {
    const uint8_t* base[NT];
};
template <int NT>
__device__ __forceinline__ XLane<NT> x_lane(const uint8_t* sx, int rows, int row_bytes, int g, int t) {
    XLane<NT> x;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) x.base[nt] = sx + (8 * nt + g < rows ? 8 * nt + g : rows > 1 ? g & 1 : 0) * row_bytes + 64 * t + 16 * (t >> 1);
    return x;
}

// The products of one step: the lane's stage (already complete) with x at `step`.
template <int NT>
__device__ __forceinline__ void step_products(float (&acc)[2][NT][4], const uint4 (&v)[4], uint4 sc, const XLane<NT>& x, int step, int t) {
    // the lane's two scale bytes of each of its four rows
    const uint32_t pick0 = t & 1 ? 0x4242u : 0x4040u, pick1 = t & 1 ? 0x4343u : 0x4141u;
    const uint32_t sw[4] = {sc.x, sc.y, sc.z, sc.w};
    uint32_t s0[4], s1[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        s0[q] = ue4m3x2_to_f16(__byte_perm(sw[q], 0u, pick0));
        s1[q] = ue4m3x2_to_f16(__byte_perm(sw[q], 0u, pick1));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        uint4 xv[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) xv[nt] = lds128(x.base[nt] + kXStep * step + 16 * u);
        uint32_t a[4][4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            e2m1x8_to_f16(u == 0 ? v[q].x : u == 1 ? v[q].y : u == 2 ? v[q].z : v[q].w, a[q]);
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

template <int NT>
__device__ __forceinline__ void clear(float (&acc)[2][NT][4]) {
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[a][nt][e] = 0.0f;
}

// First step and steps of a slice of K.
__device__ __forceinline__ void slice_steps(const GemvParams& p, int slice, int& first, int& steps) {
    first = slice * p.slice_steps + min(slice, p.slice_more);
    steps = p.slice_steps + (slice < p.slice_more ? 1 : 0);
}

// A CTA's warps are RG row groups times W / RG parts of its slice of K, which take
// the steps in turn.
template <int NT, int RG, int W>
__global__ void __launch_bounds__(32 * W) gemv_kernel(const __grid_constant__ GemvParams p) {
    constexpr int kThreads = 32 * W, KS = W / RG, kRows = 32 * RG;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_factor[16];
    __shared__ uint32_t s_top[16];
    uint8_t* sx = smem + W * kStages * kStageBytes;

    chain();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int rg = warp % RG, ks = warp / RG;
    const int part = blockIdx.x % (4 / RG), block = blockIdx.x / (4 / RG);  // which of the block's rows r
    const int m0 = blockIdx.y * 8 * NT, rows = min(8 * NT, p.m - m0);
    int first, steps;
    slice_steps(p, blockIdx.z, first, steps);
    const int mine = (steps - ks + KS - 1) / KS;  // the warp's: ks, ks + KS, ...

    const WeightLane from = weight_lane(p, block, 8 * (part * RG + rg), g, t);
    uint8_t* ring = smem + warp * kStages * kStageBytes + 16 * lane;
    const uint32_t ring_addr = ptx::smem_u32(ring);
    auto issue = [&](int i, int slot) {
        if (i < mine) copy_step(ring_addr + slot * kStageBytes, from, first + ks + i * KS);
        copy_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i, i);
    convert_x<kThreads, kSliceBytes>(p, m0, rows, first * kStep, steps, sx, s_top, s_factor);

    float acc[2][NT][4];
    clear(acc);
    const XLane<NT> x = x_lane<NT>(sx, rows, x_row_bytes(steps), g, t);
    int slot = 0;
    for (int i = 0; i < mine; ++i) {
        copy_wait<kStages - 2>();
        const uint8_t* st = ring + slot * kStageBytes;
        const uint4 v[4] = {lds128(st), lds128(st + 512), lds128(st + 1024), lds128(st + 1536)}, sc = lds128(st + 2048);
        issue(i + kStages - 1, slot == 0 ? kStages - 1 : slot - 1);
        slot = slot == kStages - 1 ? 0 : slot + 1;
        step_products(acc, v, sc, x, ks + i * KS, t);
    }

    // The parts joined in their order; row 8 RG q + 8 rg + g of the CTA is weight row
    // 128 block + 32 q + 8 (part RG + rg) + g.
    copy_wait<0>();
    __syncthreads();  // the rings are idle
    float* red = reinterpret_cast<float*>(smem);
    static_assert(KS * 8 * NT * kRows * 4 <= W * kStages * kStageBytes, "the rings hold the parts' sums");
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
        y *= s_factor[col];
        if (p.slices > 1) {
            p.sums[(((size_t)blockIdx.y * p.slices + blockIdx.z) * 8 * NT + col) * p.n_pad + n] = y;
            continue;
        }
        y *= p.alpha;
        if (p.bias) y += bf16_lo(p.bias[n]);
        p.y[(size_t)(m0 + col) * p.ldy + n] = (uint16_t)(pack_bf16(y, 0.0f) & 0xFFFFu);
    }
}

// A CTA with one slice of x walks rows: its warps draw row groups (of its share:
// every p.ctas-th) from a counter, each through a stream of its own that runs on
// over the groups' ends.
constexpr int kWalkWarps = 16;
constexpr int kWalkSteps = 5;  // of a slice at least
template <int NT>
__global__ void __launch_bounds__(32 * kWalkWarps, 1) gemv_walk_kernel(const __grid_constant__ GemvParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_factor[16];
    __shared__ uint32_t s_top[16];
    __shared__ int s_next;
    uint8_t* sx = smem + kWalkWarps * kStages * kStageBytes;

    chain();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int slice = blockIdx.x % p.slices, cta = blockIdx.x / p.slices;  // the slices of a row run side by side
    const int m0 = blockIdx.y * 8 * NT, rows = min(8 * NT, p.m - m0);
    int first, steps;
    slice_steps(p, slice, first, steps);
    const int groups = (p.n + 127) / 128 * 4;  // group 4 b + i: rows 8 i + g + 32 q of block b
    const int share = (groups - cta + p.ctas - 1) / p.ctas;

    uint8_t* ring = smem + warp * kStages * kStageBytes + 16 * lane;
    const uint32_t ring_addr = ptx::smem_u32(ring);
    // What is copied: step `ahead` of group `to`.
    int to = warp, ahead = 0;
    if (tid == 0) s_next = kWalkWarps;
    auto lane_of = [&](int i) {
        const int group = cta + i * p.ctas;
        return weight_lane(p, group >> 2, 8 * (group & 3), g, t);
    };
    WeightLane from = lane_of(min(to, share - 1));
    int queued = -1;  // the group after the one at hand, once its first step is copied
    auto issue = [&](int slot) {
        if (to < share) {
            copy_step(ring_addr + slot * kStageBytes, from, first + ahead);
            if (++ahead == steps) {
                int next = 0;
                if (lane == 0) next = atomicAdd(&s_next, 1);
                to = __shfl_sync(0xffffffffu, next, 0);
                queued = to;
                ahead = 0;
                if (to < share) from = lane_of(to);
            }
        }
        copy_commit();
    };
    __syncthreads();  // s_next
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);
    int now = warp;
    convert_x<32 * kWalkWarps, kWalkBytes>(p, m0, rows, first * kStep, steps, sx, s_top, s_factor);

    const XLane<NT> x = x_lane<NT>(sx, rows, x_row_bytes(steps), g, t);
    float* sums = p.sums + ((size_t)blockIdx.y * p.slices + slice) * 8 * NT * p.n_pad;
    int slot = 0;
    while (now < share) {
        float acc[2][NT][4];
        clear(acc);
        for (int step = 0; step < steps; ++step) {
            copy_wait<kStages - 2>();
            const uint8_t* st = ring + slot * kStageBytes;
            const uint4 v[4] = {lds128(st), lds128(st + 512), lds128(st + 1024), lds128(st + 1536)}, sc = lds128(st + 2048);
            issue(slot == 0 ? kStages - 1 : slot - 1);
            slot = slot == kStages - 1 ? 0 : slot + 1;
            step_products(acc, v, sc, x, step, t);
        }
        const int group = cta + now * p.ctas, n0 = (group >> 2) * 128 + 8 * (group & 3) + g;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int col = 8 * nt + 2 * t + e;
                if (col < rows) {
                    float* out = sums + (size_t)col * p.n_pad + n0;
                    const float f = s_factor[col];
                    out[0] = acc[0][nt][e] * f, out[32] = acc[0][nt][2 + e] * f;
                    out[64] = acc[1][nt][e] * f, out[96] = acc[1][nt][2 + e] * f;
                }
            }
        now = queued;
    }
    copy_wait<0>();
}

// The slices' sums added in their order.
template <int NT>
__global__ void __launch_bounds__(128) gemv_join_kernel(const __grid_constant__ GemvParams p) {
    chain();
    const int n = blockIdx.x * 128 + threadIdx.x, m = blockIdx.y;
    if (n >= p.n) return;
    const float* sums = p.sums + ((size_t)(m / (8 * NT)) * p.slices * 8 * NT + m % (8 * NT)) * p.n_pad + n;
    float y = 0.0f;
#pragma unroll 8
    for (int s = 0; s < p.slices; ++s) y += __ldcg(sums + (size_t)s * 8 * NT * p.n_pad);
    y *= p.alpha;
    if (p.bias) y += bf16_lo(p.bias[n]);
    p.y[(size_t)m * p.ldy + n] = (uint16_t)(pack_bf16(y, 0.0f) & 0xFFFFu);
}

constexpr int kMaxDevices = 64;

template <typename Kernel>
cudaError_t allow_smem(Kernel* kernel, int bytes, bool (&ready)[kMaxDevices]) {
    static std::mutex mu;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= kMaxDevices) return cudaErrorInvalidDevice;
    std::lock_guard<std::mutex> lk(mu);
    if (!ready[dev]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        ready[dev] = e == cudaSuccess;
    }
    return e;
}

// Rows of x that share a tile's products: 8 or 16.
int tile_rows(int m) { return m <= 8 ? 8 : 16; }

// How a call is cut.
struct Cut {
    bool walk;
    int rows_per_cta;  // 32 RG
    int slices, ctas;
};
Cut cut_of(int m, int n, int k) {
    const int all = (k - 1) / kStep + 1, groups = ((n - 1) / 128 + 1) * 4, step_bytes = std::min(m, tile_rows(m)) * 2 * kStep;
    // Slices are whole steps and differ by one: the longest fits where there are as many
    // slices as it takes of the whole steps that fit (by bytes it would not: 9 rows x 113
    // steps are 4 times 65536 bytes nearly, but one of 4 slices has 29 steps, 66816).
    const int walk_fit = kWalkBytes / step_bytes, slice_fit = kSliceBytes / step_bytes;
    auto slices_of = [&](int most_steps) { return (all - 1) / most_steps + 1; };
    Cut c{};
    // Walked where slices of a few steps give (nearly) every warp of a full GPU a
    // group: rows x 28672 x 8192 28.8 us walked and 34.4 not with one row of x, 37.7 and
    // over 60 with 16; 8 rows, 28672 x 4096 19.4 and 32.7.  Slices of 5 steps do where x
    // does not fit beside the rings otherwise (16 rows, 15360 x 2880: 13.4 us walked,
    // 19.2 not), of 8 where it would (5 rows: 11.1 and 9.8).  Of the numbers of slices
    // the one that lets a CTA's warps end together: the rounds of its groups times the
    // steps of each, and a third of a step for a slice's sums (16 rows, 16384 x 16384, in
    // one session: 8 slices 42.0 us, 9 39.4, 18 43.9).
    const int shortest = all > slice_fit ? kWalkSteps : 8;
    const int from = std::max(slices_of(walk_fit), (148 * kWalkWarps * 3 / 4 - 1) / groups + 1);
    int least = 0;
    for (int slices = from; slices <= std::min(148, 2 * from) && all / slices >= shortest; ++slices) {
        const int ctas = std::max(1, std::min(148 / slices, groups)), share = (groups + ctas - 1) / ctas;
        const int cost = 3 * ((share + kWalkWarps - 1) / kWalkWarps) * ((all + slices - 1) / slices) + slices;
        if (!least || cost < least) least = cost, c.walk = true, c.slices = slices, c.ctas = ctas;
    }
    if (c.walk) return c;
    // Slices that fit, of 16 steps or more, and as many as still make one wave of two
    // CTAs an SM; then 32, 64 or 128 rows of the weight a CTA, as many as leave about
    // a CTA for each SM (15360 rows x 2880, 5 rows of x: 17.1 / 12.6 / 10.7 us; 2880
    // rows, one row of x: 4.4 / 5.9 / 8.7 us).
    c.slices = std::max(slices_of(slice_fit), std::min(296 / groups, all / 16));
    c.rows_per_cta = groups * c.slices < 296 ? 32 : groups * c.slices < 480 ? 64 : 128;
    return c;
}
static_assert(kWalkSteps > kStages, "a walk's stream runs into one further group at most");

int padded_rows(int n) { return ((n - 1) / 128 + 1) * 128; }

// Rows of x of one launch; more than that take several, one after the other, with one
// workspace.  A grid's second dimension ends at 65535 (the join's are rows), and slices'
// sums of many rows would be gigabytes that a GPU full of tiles does not need: 256 MB of
// them, or one tile's.
constexpr long kMostRows = 65520, kMostSums = 256l << 20;
int launch_rows(int m, int n, const Cut& c) {
    const int tile = tile_rows(m);
    long rows = kMostRows;
    if (c.slices > 1 || c.walk) rows = std::min(rows, std::max(1l, kMostSums / ((long)c.slices * padded_rows(n) * 4 * tile)) * tile);
    return (int)std::min<long>(m, rows);
}

int longest_slice(const GemvParams& p) { return p.slice_steps + (p.slice_more > 0 ? 1 : 0); }
int x_bytes(const GemvParams& p) { return std::min(p.m, tile_rows(p.m)) * x_row_bytes(longest_slice(p)); }
// A slice of `bytes` at most: what convert_x's threads hold and x_room has room for.
bool slice_fits(const GemvParams& p, int bytes) { return (long)std::min(p.m, tile_rows(p.m)) * longest_slice(p) * 2 * kStep <= bytes; }

template <int NT, int RG, int W>
cudaError_t launch(const GemvParams& p, cudaStream_t st) {
    constexpr int kRing = W * kStages * kStageBytes;
    static bool ready[kMaxDevices];
    if (!slice_fits(p, kSliceBytes)) return cudaErrorInvalidConfiguration;
    if (const cudaError_t e = allow_smem(gemv_kernel<NT, RG, W>, kRing + x_room(kSliceBytes), ready)) return e;
    const long blocks = ((long)p.n + 127) / 128 * (4 / RG);
    const dim3 grid((unsigned)blocks, (unsigned)((p.m + 8 * NT - 1) / (8 * NT)), (unsigned)p.slices);
    return launch_chained(gemv_kernel<NT, RG, W>, grid, 32 * W, kRing + x_bytes(p), st, p);
}

template <int NT>
cudaError_t launch_walk(const GemvParams& p, cudaStream_t st) {
    constexpr int kRing = kWalkWarps * kStages * kStageBytes;
    static bool ready[kMaxDevices];
    if (!slice_fits(p, kWalkBytes)) return cudaErrorInvalidConfiguration;
    if (const cudaError_t e = allow_smem(gemv_walk_kernel<NT>, kRing + x_room(kWalkBytes), ready)) return e;
    const dim3 grid((unsigned)(p.slices * p.ctas), (unsigned)((p.m + 8 * NT - 1) / (8 * NT)));
    return launch_chained(gemv_walk_kernel<NT>, grid, 32 * kWalkWarps, kRing + x_bytes(p), st, p);
}

template <int NT>
cudaError_t launch_all(const GemvParams& p, const Cut& c, cudaStream_t st) {
    const cudaError_t e = c.walk                  ? launch_walk<NT>(p, st)
                          : c.rows_per_cta == 128 ? launch<NT, 4, 16>(p, st)
                          : c.rows_per_cta == 64  ? launch<NT, 2, 8>(p, st)
                                                  : launch<NT, 1, 8>(p, st);
    if (e != cudaSuccess || (p.slices == 1 && !c.walk)) return e;
    return launch_chained(gemv_join_kernel<NT>, dim3((p.n + 127) / 128, p.m), 128, 0, st, p);
}

}  // namespace
}  // namespace fp4b

using namespace fp4b;

FP4B_EXPORT long fp4b_gemv_workspace(int m, int k_in, int n_out) {
    if (m <= 0 || k_in <= 0 || n_out <= 0) {
        set_last_error("fp4b_gemv_workspace: m, k and n must be positive");
        return -1;
    }
    const Cut c = cut_of(m, n_out, k_in);
    const long tile = tile_rows(m);
    return c.slices == 1 && !c.walk ? 0 : (launch_rows(m, n_out, c) + tile - 1) / tile * tile * c.slices * padded_rows(n_out) * 4;
}

FP4B_EXPORT int fp4b_gemv_cached(const void* x, int m, int k_in, long ldx, const void* handle, int n_out, void* y,
                                 long ldy, const void* bias, void* workspace, long workspace_bytes, void* stream) {
    CacheView c;
    if (!cache_view(handle, &c)) {
        set_last_error("null or invalid cache handle");
        return -1;
    }
    if (!x || !y || m <= 0 || k_in <= 0 || k_in > c.K || ldx < k_in || n_out <= 0 || n_out > c.N ||
        ldy < n_out) {
        set_last_error("fp4b_gemv_cached: bad shape (m=%d k=%d n=%d vs cache %dx%d)", m, k_in, n_out, c.N, c.K);
        return -1;
    }
    const long need = fp4b_gemv_workspace(m, k_in, n_out);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))) {
        set_last_error("fp4b_gemv_cached: needs a 16-byte aligned workspace of %ld bytes", need);
        return -1;
    }
    GemvParams p{};
    p.ldx = ldx;
    p.w = c.fp4, p.sf = c.sf, p.k_pad = c.K;
    p.ldy = ldy;
    p.bias = static_cast<const uint16_t*>(bias);
    p.n = n_out, p.k = k_in;
    p.x_vec = ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    p.alpha = c.w_alpha * kScaleUnit;
    const Cut cut = cut_of(m, n_out, k_in);
    const int all = (k_in - 1) / kStep + 1;
    p.slices = cut.slices, p.slice_steps = all / cut.slices, p.slice_more = all % cut.slices, p.ctas = cut.ctas;
    p.sums = static_cast<float*>(workspace);
    p.n_pad = padded_rows(n_out);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int most = launch_rows(m, n_out, cut);
    cudaError_t e = cudaSuccess;
    for (long at = 0; at < m && e == cudaSuccess; at += most) {
        p.m = (int)std::min<long>(most, m - at);
        p.x = static_cast<const uint16_t*>(x) + at * ldx;
        p.y = static_cast<uint16_t*>(y) + at * ldy;
        e = tile_rows(m) == 8 ? launch_all<1>(p, cut, st) : launch_all<2>(p, cut, st);
    }
    return launch_status(e, "fp4b_gemv_cached");
}
