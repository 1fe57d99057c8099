// gemv.cu -- few rows of BF16 activations times a cached NVFP4 weight.
//
//   y[m, n] = w_alpha * sum_k x[m, k] * W[n, k] (+ bias[n]),
//   W[n, k] = e2m1[n, k] * ue4m3[n, k / 16]
//
// with the activations as they are: at one to a few rows the time is that of
// the weight's N * K * 9 / 16 bytes, so nothing is gained by quantizing x.
#include <cuda_runtime.h>

#include <cstdio>

#include "decode_core.cuh"
#include "fp4b_internal.h"

#define FP4B_EXPORT extern "C" __attribute__((visibility("default")))

namespace fp4b {
namespace {

constexpr int kThreads = 256;

struct GemvParams {
    const uint16_t* x;
    const uint8_t* w;
    const uint8_t* sf;
    uint16_t* y;
    const uint16_t* bias;
    long ldx, ldy;
    int m, n, k, k_pad;
    float alpha;
};

// One warp per weight row and row of x; lanes stride over 16-element blocks.
__global__ void __launch_bounds__(kThreads) gemv_kernel(const __grid_constant__ GemvParams p) {
    const int lane = threadIdx.x & 31;
    const long n = (long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    if (n >= p.n) return;
    const uint32_t nsb = p.k_pad / 16;
    for (int m = blockIdx.y; m < p.m; m += gridDim.y) {
        const uint16_t* x = p.x + (size_t)m * p.ldx;
        float sum = 0.0f;
        for (uint32_t kb = lane; kb * 16 < (uint32_t)p.k; kb += 32) {
            const uint2 w = *reinterpret_cast<const uint2*>(p.w + ((size_t)n * p.k_pad >> 1) + kb * 8);
            const float s = decode::ue4m3_float(p.sf[sf_offset((uint32_t)n, kb, nsb)]);
            float part = 0.0f;
            for (int i = 0; i < 8; ++i) {
                const float2 f = decode::f16x2_to_float2(decode::e2m1x2_to_f16x2(((i < 4 ? w.x : w.y) >> (8 * (i & 3))) & 0xFFu));
                const int k = kb * 16 + 2 * i;
                if (k < p.k) part += f.x * __uint_as_float((uint32_t)x[k] << 16);
                if (k + 1 < p.k) part += f.y * __uint_as_float((uint32_t)x[k + 1] << 16);
            }
            sum += part * s;
        }
        sum = decode::group_sum<32>(sum);
        if (lane == 0) {
            float y = sum * p.alpha;
            if (p.bias) y += __uint_as_float((uint32_t)p.bias[n] << 16);
            p.y[(size_t)m * p.ldy + n] = (uint16_t)(decode::pack_bf16(y, 0.0f) & 0xFFFFu);
        }
    }
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
    if (!x || !y || m <= 0 || k_in <= 0 || k_in > c.K || ldx < k_in || n_out <= 0 || n_out > c.N || ldy < n_out) {
        set_last_error("fp4b_gemv_cached: bad shape (m=%d k=%d n=%d vs cache %dx%d)", m, k_in, n_out, c.N, c.K);
        return -1;
    }
    GemvParams p{static_cast<const uint16_t*>(x), c.fp4, c.sf, static_cast<uint16_t*>(y),
                 static_cast<const uint16_t*>(bias), ldx, ldy, m, n_out, k_in, c.K, c.w_alpha};
    const dim3 grid((n_out + kThreads / 32 - 1) / (kThreads / 32), m < 65535 ? m : 65535);
    gemv_kernel<<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return launch_status(cudaGetLastError(), "fp4b_gemv_cached");
}
