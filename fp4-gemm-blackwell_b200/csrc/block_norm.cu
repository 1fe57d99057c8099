// block_norm.cu -- what lies between two blocks of a decoder layer: the norm
// after a block, its gate, its residual and the norm before the next block.
//
// Per row of H elements, x the block's output and r the residual stream:
//   y  = x / sqrt(mean(x^2) + eps) * post_weight    (without post_weight: y = x)
//   r' = r + scale * gate * y                       (without gate: 1)
//   h  = r' / sqrt(mean(r'^2) + eps) * weight
// in fp32 from the inputs to the one rounding of r' and of h; the second mean
// and h are of r' as it was before its rounding.  Without x: h from r alone.
//
// Memory-bound: 2 bytes of x, 2 or 4 of r in and out, 2 of h (and 2 of a gate
// that differs by row) for about 10 operations an element, so a row is read
// once and stays in its threads' registers over both means.  A thread has 1, 2,
// 4 or 8 pieces of 8 elements (16 bytes of BF16), loaded before anything is
// computed; a row of at most 32 pieces a warp is one warp's, a longer one a
// CTA's.  Rows that do not start on 16 bytes, or whose width is not a multiple
// of 8, go by single elements, up to 64 a thread.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>

#include "decode_core.cuh"
#include "fp4b_internal.h"

#define FP4B_EXPORT extern "C" __attribute__((visibility("default")))

namespace fp4b {
namespace {

using namespace decode;

constexpr int kMaxThreads = 512;
constexpr int kMaxWidth = 32768;
constexpr int kRowsPerCta = 4;  // of one warp each

struct NormParams {
    const uint16_t* x;  // null: no block before
    long x_stride;
    const void* residual;
    long residual_stride;
    const uint16_t* gate;  // null: none
    long gate_stride;      // 0: one for all rows
    const uint16_t* weight;
    const uint16_t* post_weight;  // null: none
    uint16_t* normed;
    void* residual_out;
    int rows, width;
    float scale, eps, inv_width;
};

// A piece of VEC elements as it is loaded: BF16, or FP32 for a residual.
template <int VEC>
struct Piece16 {
    uint32_t w[VEC > 1 ? VEC / 2 : 1];
    __device__ __forceinline__ void load(const uint16_t* p) {
        if constexpr (VEC == 8) {
            const uint4 v = *reinterpret_cast<const uint4*>(p);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
            w[0] = *p;
        }
    }
    __device__ __forceinline__ float get(int i) const { return i & 1 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]); }
};
template <int VEC>
struct Piece32 {
    float f[VEC];
    __device__ __forceinline__ void load(const float* p) {
        if constexpr (VEC == 8) {
            const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
            f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
        } else {
            f[0] = *p;
        }
    }
    __device__ __forceinline__ float get(int i) const { return f[i]; }
};

template <int VEC>
__device__ __forceinline__ void store16(uint16_t* p, const float (&v)[VEC]) {
    if constexpr (VEC == 8)
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    else
        *p = (uint16_t)pack_bf16(v[0], 0.0f);
}
template <int VEC>
__device__ __forceinline__ void store32(float* p, const float (&v)[VEC]) {
    if constexpr (VEC == 8) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *p = v[0];
    }
}

// Sum over the row's threads (all of them get it).
__device__ __forceinline__ float row_sum(float v, float* slots) {
    v = group_sum<32>(v);
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) slots[warp] = v;
    __syncthreads();
    return group_sum<32>(lane < warps ? slots[lane] : 0.0f);
}

// VEC elements a piece, ITEMS pieces a thread; R32: the residual is fp32.
template <int VEC, int ITEMS, bool R32>
__global__ void __launch_bounds__(kMaxThreads) block_norm_kernel(const __grid_constant__ NormParams p) {
    __shared__ float sums[2][32];
    chain();
    const long row = (long)blockIdx.x * blockDim.y + threadIdx.y;
    if (row >= p.rows) return;  // (whole warps: a CTA of several rows has a warp for each)
    using Res = typename std::conditional<R32, Piece32<VEC>, Piece16<VEC>>::type;
    using R = typename std::conditional<R32, float, uint16_t>::type;
    const R* residual = static_cast<const R*>(p.residual) + row * p.residual_stride;
    const uint16_t* x = p.x + row * p.x_stride;
    const uint16_t* gate = p.gate + row * p.gate_stride;

    Res res[ITEMS];
    Piece16<VEC> in[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int i = (k * (int)blockDim.x + (int)threadIdx.x) * VEC;
        if (i < p.width) {
            if (p.x) in[k].load(x + i);
            res[k].load(residual + i);
        }
    }
    float post = p.scale;  // what y is multiplied by besides the weights
    if (p.x && p.post_weight) {
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k)
            if ((k * (int)blockDim.x + (int)threadIdx.x) * VEC < p.width)
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum = fmaf(in[k].get(e), in[k].get(e), sum);
        post *= rsqrtf(fmaf(row_sum(sum, sums[0]), p.inv_width, p.eps));
    }
    float r[ITEMS][VEC];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int i = (k * (int)blockDim.x + (int)threadIdx.x) * VEC;
        if (i < p.width) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) r[k][e] = res[k].get(e);
            if (p.x) {
                float f[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) f[e] = in[k].get(e) * post;
                if (p.post_weight) {
                    Piece16<VEC> w;
                    w.load(p.post_weight + i);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) f[e] *= w.get(e);
                }
                if (p.gate) {
                    Piece16<VEC> w;
                    w.load(gate + i);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) f[e] *= w.get(e);
                }
#pragma unroll
                for (int e = 0; e < VEC; ++e) r[k][e] += f[e];
                R* to = static_cast<R*>(p.residual_out) + row * p.width + i;
                if constexpr (R32) store32<VEC>(to, r[k]);
                else store16<VEC>(to, r[k]);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum = fmaf(r[k][e], r[k][e], sum);
        }
    }
    const float factor = rsqrtf(fmaf(row_sum(sum, sums[1]), p.inv_width, p.eps));
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int i = (k * (int)blockDim.x + (int)threadIdx.x) * VEC;
        if (i < p.width) {
            Piece16<VEC> w;
            w.load(p.weight + i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) r[k][e] = r[k][e] * factor * w.get(e);
            store16<VEC>(p.normed + row * p.width + i, r[k]);
        }
    }
}

template <int VEC, int ITEMS, bool R32>
cudaError_t launch(const NormParams& p, cudaStream_t st) {
    const int pieces = (p.width + VEC - 1) / VEC;
    const int threads = ((pieces + ITEMS - 1) / ITEMS + 31) / 32 * 32;
    const int per = threads == 32 ? kRowsPerCta : 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)((p.rows + per - 1) / per));
    config.blockDim = dim3(threads, per);
    config.stream = st;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, block_norm_kernel<VEC, ITEMS, R32>, p);
}

template <bool R32>
cudaError_t launch_width(const NormParams& p, bool pieces, cudaStream_t st) {
    if (pieces) {
        const int n = p.width / 8;
        return n <= 2 * kMaxThreads ? launch<8, 2, R32>(p, st) : n <= 4 * kMaxThreads ? launch<8, 4, R32>(p, st) : launch<8, 8, R32>(p, st);
    }
    return p.width <= 8 * kMaxThreads ? launch<1, 8, R32>(p, st) : p.width <= 16 * kMaxThreads ? launch<1, 16, R32>(p, st) : launch<1, 64, R32>(p, st);
}

bool whole(const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }
bool sixteen(const void* p, long stride, int size) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * size % 16 == 0; }

}  // namespace
}  // namespace fp4b

using namespace fp4b;

FP4B_EXPORT int fp4b_block_norm(const fp4b_norm* call, void* stream) {
    const char* why = nullptr;
    if (!call) {
        why = "null arguments";
    } else {
        const fp4b_norm& c = *call;
        if (c.rows < 0) why = "negative rows";
        else if (c.width <= 0 || c.width > kMaxWidth) why = "the width must be 1 to 32768";
        else if (c.rows > 0 && (!c.residual || !c.weight || !c.normed || (c.x && !c.residual_out))) why = "null tensor";
        else if (!c.x && (c.post_weight || c.gate)) why = "a gate and a norm after the block need the block's output";
        else if (!whole(c.x, 2) || !whole(c.residual, c.residual_fp32 ? 4 : 2) || !whole(c.gate, 2) || !whole(c.weight, 2) ||
                 !whole(c.post_weight, 2) || !whole(c.normed, 2) || !whole(c.residual_out, c.residual_fp32 ? 4 : 2))
            why = "tensors must be aligned to their elements";
        else if (!std::isfinite(c.scale) || !std::isfinite(c.eps) || c.eps < 0.0f) why = "scale and eps must be finite, eps not negative";
    }
    if (why) {
        set_last_error("fp4b_block_norm: %s", why);
        return -1;
    }
    const fp4b_norm& c = *call;
    if (c.rows == 0) return 0;
    NormParams p{};
    p.x = static_cast<const uint16_t*>(c.x), p.x_stride = c.x_stride;
    p.residual = c.residual, p.residual_stride = c.residual_stride;
    p.gate = static_cast<const uint16_t*>(c.gate), p.gate_stride = c.gate_stride;
    p.weight = static_cast<const uint16_t*>(c.weight), p.post_weight = static_cast<const uint16_t*>(c.post_weight);
    p.normed = static_cast<uint16_t*>(c.normed), p.residual_out = c.residual_out;
    p.rows = c.rows, p.width = c.width, p.scale = c.scale, p.eps = c.eps, p.inv_width = 1.0f / (float)c.width;
    const int size = c.residual_fp32 ? 4 : 2;
    const bool pieces = c.width % 8 == 0 && sixteen(c.x, c.x_stride, 2) && sixteen(c.residual, c.residual_stride, size) &&
                        sixteen(c.gate, c.gate_stride, 2) && sixteen(c.weight, 0, 2) && sixteen(c.post_weight, 0, 2) &&
                        sixteen(c.normed, 0, 2) && sixteen(c.residual_out, 0, size);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return launch_status(c.residual_fp32 ? launch_width<true>(p, pieces, st) : launch_width<false>(p, pieces, st), "fp4b_block_norm");
}
