// decode_attention.cu -- attention of one new token a sequence over a paged
// key-value cache.
//
//   out[b, h] = sum_i p_i v_i / l,  p_i = exp(scale * q . k_i - m),
//   l = sum_i p_i (+ exp(sink_h - m)),  m = the running maximum
//
// over the keys i of [max(0, len - window), len), K and V decoded from the
// cache's format as they are read.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>

#include "decode_core.cuh"
#include "fp4b_internal.h"

#define FP4B_EXPORT extern "C" __attribute__((visibility("default")))

namespace fp4b {
namespace {

struct AttentionParams {
    const uint16_t* q;
    long q_sb, q_sh;
    int batch, q_heads, group;
    fp4b_kv_cache cache;
    int page_shift;
    const int* table;
    long table_stride;
    int table_width;
    const int* lens;
    float scale;
    int window;
    const float* sinks;
    uint16_t* out;
    float* lse;
    int* err;
};

// Two neighbouring elements of a row.
template <int KIND>
__device__ __forceinline__ float2 read_two(const void* base, const void* scales, long row, int d, int e) {
    if constexpr (KIND == kKvBf16) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(base) + (size_t)row * d + e);
        return make_float2(decode::bf16_lo(w), decode::bf16_hi(w));
    } else if constexpr (KIND == kKvFp8) {
        const uint16_t w = *reinterpret_cast<const uint16_t*>(static_cast<const uint8_t*>(base) + (size_t)row * d + e);
        const float2 f = decode::f16x2_to_float2(decode::e4m3x2_to_f16x2(w));
        const float s = static_cast<const float*>(scales)[row];
        return make_float2(f.x * s, f.y * s);
    } else {
        const uint8_t w = static_cast<const uint8_t*>(base)[((size_t)row * d + e) >> 1];
        const float2 f = decode::f16x2_to_float2(decode::e2m1x2_to_f16x2(w));
        const float s = decode::ue4m3_float(static_cast<const uint8_t*>(scales)[((size_t)row * d + e) >> 4]);
        return make_float2(f.x * s, f.y * s);
    }
}

// One warp per (sequence, query head), one key at a time; lane l holds the
// elements 2l, 2l + 1 of each run of 64.
template <int KIND, int D>
__global__ void __launch_bounds__(128) decode_attention_kernel(const __grid_constant__ AttentionParams p) {
    const int lane = threadIdx.x & 31;
    const long unit = (long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (unit >= (long)p.batch * p.q_heads) return;
    const int b = (int)(unit / p.q_heads), h = (int)(unit - (long)b * p.q_heads), hk = h / p.group;
    constexpr int R = D / 64;
    float2 q[R], acc[R];
    const uint16_t* qr = p.q + b * p.q_sb + h * p.q_sh;
    for (int r = 0; r < R; ++r) {
        q[r] = make_float2(__uint_as_float((uint32_t)qr[64 * r + 2 * lane] << 16), __uint_as_float((uint32_t)qr[64 * r + 2 * lane + 1] << 16));
        acc[r] = make_float2(0.f, 0.f);
    }
    int len = p.lens[b];
    const long most = (long)p.table_width << p.page_shift;
    if (len < 0 || len > most) {
        if (lane == 0) decode::report(p.err, kErrPageRange);
        len = len < 0 ? 0 : (int)most;
    }
    const int first = p.window > 0 && len > p.window ? len - p.window : 0;
    float m = -INFINITY, l = 0.0f;
    for (int i = first; i < len; ++i) {
        const int page = p.table[b * p.table_stride + (i >> p.page_shift)];
        if (page < 0 || page >= p.cache.num_pages) {
            if (lane == 0) decode::report(p.err, kErrPageRange);
            continue;
        }
        const long row = ((long)page * p.cache.kv_heads + hk) * p.cache.page_size + (i & (p.cache.page_size - 1));
        float dot = 0.0f;
        for (int r = 0; r < R; ++r) {
            const float2 k = read_two<KIND>(p.cache.k, p.cache.k_scale, row, D, 64 * r + 2 * lane);
            dot += q[r].x * k.x + q[r].y * k.y;
        }
        const float s = decode::group_sum<32>(dot) * p.scale;
        const float top = fmaxf(m, s);
        const float keep = m == -INFINITY ? 0.0f : __expf(m - top), w = top == -INFINITY ? 0.0f : __expf(s - top);
        for (int r = 0; r < R; ++r) {
            const float2 v = read_two<KIND>(p.cache.v, p.cache.v_scale, row, D, 64 * r + 2 * lane);
            acc[r].x = acc[r].x * keep + w * v.x;
            acc[r].y = acc[r].y * keep + w * v.y;
        }
        l = l * keep + w;
        m = top;
    }
    if (p.sinks) {
        const float sink = p.sinks[h], top = fmaxf(m, sink);
        const float keep = m == -INFINITY ? 0.0f : __expf(m - top);
        for (int r = 0; r < R; ++r) acc[r].x *= keep, acc[r].y *= keep;
        l = l * keep + (top == -INFINITY ? 0.0f : __expf(sink - top));
        m = top;
    }
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
    for (int r = 0; r < R; ++r)
        *reinterpret_cast<uint32_t*>(p.out + ((size_t)b * p.q_heads + h) * D + 64 * r + 2 * lane) =
            decode::pack_bf16(acc[r].x * inv, acc[r].y * inv);
    if (p.lse && lane == 0) p.lse[(size_t)b * p.q_heads + h] = m == -INFINITY ? -INFINITY : m + logf(l);
}

template <int KIND>
cudaError_t launch(const AttentionParams& p, cudaStream_t st) {
    const unsigned blocks = (unsigned)(((long)p.batch * p.q_heads + 3) / 4);
    if (p.cache.head_dim == 64) decode_attention_kernel<KIND, 64><<<blocks, 128, 0, st>>>(p);
    else if (p.cache.head_dim == 128) decode_attention_kernel<KIND, 128><<<blocks, 128, 0, st>>>(p);
    else decode_attention_kernel<KIND, 256><<<blocks, 128, 0, st>>>(p);
    return cudaGetLastError();
}

}  // namespace
}  // namespace fp4b

using namespace fp4b;

FP4B_EXPORT long fp4b_decode_attention_workspace(int q_heads, int kv_heads, int head_dim) {
    if (q_heads <= 0 || kv_heads <= 0 || head_dim <= 0) return -1;
    return 16;
}

FP4B_EXPORT int fp4b_decode_attention(const void* q, long q_sb, long q_sh, int batch, int q_heads,
                                      const fp4b_kv_cache* cache, const int* page_table, long table_stride,
                                      int table_width, const int* seq_lens, float scale, int window,
                                      const float* sinks, void* out, float* lse, void* workspace,
                                      long workspace_bytes, void* stream) {
    const char* why = kv_cache_check(cache);
    if (!why && (batch < 0 || q_heads <= 0 || q_heads % cache->kv_heads))
        why = "query heads must be a multiple of the cache's heads";
    if (!why && batch > 0 && (!q || !out || !seq_lens || (table_width > 0 && !page_table))) why = "null tensor";
    if (!why && (table_width < 0 || table_stride < table_width)) why = "bad page table";
    if (!why && (long)table_width * cache->page_size > 0x7fffffffL) why = "more than 2^31 keys in one sequence";
    if (!why && (long)batch * q_heads > 0x7fffffffL) why = "more than 2^31 output rows";
    if (!why && (window < 0 || !std::isfinite(scale))) why = "window must not be negative, scale finite";
    if (!why && ((reinterpret_cast<uintptr_t>(q) & 7) || q_sb % 4 || q_sh % 4 || (reinterpret_cast<uintptr_t>(out) & 15)))
        why = "queries must be 8-byte aligned rows, the output 16-byte aligned";
    if (!why && batch > 0 &&
        (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) ||
         workspace_bytes < fp4b_decode_attention_workspace(q_heads, cache->kv_heads, cache->head_dim)))
        why = "workspace too small or misaligned";
    if (why) {
        set_last_error("fp4b_decode_attention: %s", why);
        return -1;
    }
    if (batch == 0) return 0;
    AttentionParams p{static_cast<const uint16_t*>(q), q_sb, q_sh, batch, q_heads, q_heads / cache->kv_heads, *cache, 0,
                      page_table, table_stride, table_width, seq_lens, scale, window, sinks,
                      static_cast<uint16_t*>(out), lse, device_error_word()};
    while ((1 << p.page_shift) < cache->page_size) ++p.page_shift;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = cache->kind == kKvBf16 ? launch<kKvBf16>(p, st)
                          : cache->kind == kKvFp8 ? launch<kKvFp8>(p, st)
                                                  : launch<kKvNvfp4>(p, st);
    return launch_status(e, "fp4b_decode_attention");
}
