// kv_cache.cu -- what lies between the QKV linear and the attention of a
// decoder layer: the norm and rotation of queries and keys, and the paged
// key-value cache as it is written (quantized) and read back.
//
// Per (token, head) row x of D elements:
//   norm      y = x / sqrt(mean(x^2) + eps) * w          (optional)
//   rotation  (y_i, y_j) -> (y_i c - y_j s, y_j c + y_i s), j = i + R/2 for
//             i < R/2 (or the pairs 2i, 2i + 1), c and s from the table row of
//             the token's position; elements from R up stay (optional)
// in fp32 from the BF16 input to the one rounding: to BF16 for a query (and a
// key without a cache), to the cache's format for a key or value.
//
// Memory-bound: 2 bytes in, 2 (or 1 + 4/D, or 9/16) out per element.  A row
// belongs to L = 8, 16 or 32 lanes of a warp (D / 8 rounded up to a power of
// two): lane l holds elements 4l .. 4l+3 of each half of the row, so that the
// two elements of a rotated pair meet in one lane (when all of the row is
// rotated, or in pairs), a half's 16-element blocks are four lanes each, and
// the loads of a row are two runs of 8 bytes a lane.  A warp stays with one
// token and walks several of its heads, kBatch rounds of 32 / L heads in
// flight at a time; the table row is read once and held.  With few tokens each
// warp has one round, so that a single token's heads still spread over the GPU.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>

#include "decode_core.cuh"
#include "fp4b_internal.h"
#include "quantize_core.cuh"

#define FP4B_EXPORT extern "C" __attribute__((visibility("default")))

namespace fp4b {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBatch = 4;

struct RowsParams {
    const uint16_t *q, *k, *v;  // BF16 rows, null where absent
    long q_st, q_sh, k_st, k_sh, v_st, v_sh;  // token and head strides, elements
    int tokens, q_heads, kv_heads, d;
    const void* positions;
    const void* slots;
    int pos64, slot64;
    const float* rope;  // [rope_rows, rot]: cosines, then sines; null for no rotation
    int rope_rows, rot, pairs;
    const uint16_t *q_weight, *k_weight;  // BF16 [d], null for no norm
    float eps;
    uint16_t *q_out, *k_out;  // BF16 [tokens, heads, d]
    fp4b_kv_cache cache;      // keys and values go here unless KIND is kKvNone
    int page_shift;
    float inv_d;
    int q_rounds, k_rounds, all_rounds;  // rounds of 32 / L heads: the queries', the keys' and all
    int rounds;                          // of which one warp walks these many
    int walks;                           // warps a token
    int* err;
};

__device__ __forceinline__ void unpack4(uint2 w, float (&x)[4]) {
    x[0] = decode::bf16_lo(w.x);
    x[1] = decode::bf16_hi(w.x);
    x[2] = decode::bf16_lo(w.y);
    x[3] = decode::bf16_hi(w.y);
}

// Rotates the lane's two chunks.  c, s: the table's factors for the lane's
// elements (a: first chunk, b: second; with FULL, the whole row in halves, b's
// are a's).
template <int L, bool FULL>
__device__ __forceinline__ void rotate(const RowsParams& p, float (&a)[4], float (&b)[4], const float (&ca)[4],
                                       const float (&sa)[4], const float (&cb)[4], const float (&sb)[4], int l) {
    if constexpr (FULL) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = a[i], y = b[i];
            a[i] = x * ca[i] - y * sa[i];
            b[i] = y * ca[i] + x * sa[i];
        }
    } else if (p.pairs) {
        // Pair (2i, 2i + 1) lies in one lane; ca[2i] = ca[2i + 1].
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const float x = a[i], y = a[i + 1];
            a[i] = x * ca[i] - y * sa[i];
            a[i + 1] = y * ca[i] + x * sa[i];
            const float u = b[i], v = b[i + 1];
            b[i] = u * cb[i] - v * sb[i];
            b[i + 1] = v * cb[i] + u * sb[i];
        }
    } else {
        // Part of the row is rotated: chunk c's partner is chunk c +- rot / 8,
        // held by another lane.  Chunks 0 .. d/8 - 1 are the lanes' first
        // ones, d/8 .. d/4 - 1 their second ones.
        const int half = p.rot >> 1, shift = half >> 2, lanes = p.d >> 3;
        const int group = (threadIdx.x & 31) & ~(L - 1);
        float pa[4], pb[4];
        const int ta = l < shift ? l + shift : l - shift;  // partner of the first chunk
        const int tb = l + lanes - shift;                  // of the second (never in the row's first rot / 8 chunks)
        const int la = group + (ta >= lanes ? ta - lanes : ta), lb = group + (tb >= lanes ? tb - lanes : tb);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float fa = __shfl_sync(0xffffffffu, a[i], la), sa2 = __shfl_sync(0xffffffffu, b[i], la);
            const float fb = __shfl_sync(0xffffffffu, a[i], lb), sb2 = __shfl_sync(0xffffffffu, b[i], lb);
            pa[i] = ta >= lanes ? sa2 : fa;
            pb[i] = tb >= lanes ? sb2 : fb;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int da = 4 * l + i, db = (p.d >> 1) + 4 * l + i;
            if (da < p.rot) a[i] = da < half ? a[i] * ca[i] - pa[i] * sa[i] : a[i] * ca[i] + pa[i] * sa[i];
            if (db < p.rot) b[i] = db < half ? b[i] * cb[i] - pb[i] * sb[i] : b[i] * cb[i] + pb[i] * sb[i];
        }
    }
}

// Table factors of element d of a rotated row.
__device__ __forceinline__ void factors(const RowsParams& p, const float* row, int d, float& c, float& s) {
    c = 1.0f;
    s = 0.0f;
    if (d < p.rot) {
        const int half = p.rot >> 1;
        const int i = p.pairs ? d >> 1 : (d < half ? d : d - half);
        c = row[i];
        s = row[half + i];
    }
}

// |x|max of a block from its four lanes' values, as the codec takes it: NaN is
// skipped.  `literal`: the block holds a NaN, an infinity or a huge value.
__device__ __forceinline__ float block_absmax(const float (&x)[4], bool& literal) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    top = decode::group_umax<4>(top);
    literal = top >= kFastAbsmaxF32Limit;
    float amax = __uint_as_float(top);
    if (__any_sync(0xffffffffu, literal)) {
        float f = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
        f = fmaxf(f, __shfl_xor_sync(0xffffffffu, f, 2));
        f = fmaxf(f, __shfl_xor_sync(0xffffffffu, f, 1));
        if (literal) amax = f == f ? f : 0.0f;
    }
    return amax;
}

__device__ __forceinline__ uint32_t block_codes(const float (&x)[4], float inv, bool literal) {
    if (literal) {
        uint32_t codes = 0;
        for (int i = 0; i < 4; ++i) codes |= (uint32_t)e2m1_scan(__fmul_rn(x[i], inv)) << (4 * i);
        return codes;
    }
    return decode::e2m1x4(__fmul_rn(x[0], inv), __fmul_rn(x[1], inv), __fmul_rn(x[2], inv), __fmul_rn(x[3], inv));
}

// Writes one row's lane share into the cache.  All lanes of the warp call it;
// `live`: the lane has elements and its slot is valid.
template <int KIND, int L>
__device__ __forceinline__ void store_row(const RowsParams& p, bool value, long row, bool live, int l,
                                          const float (&a)[4], const float (&b)[4]) {
    void* base = value ? p.cache.v : p.cache.k;
    void* scales = value ? p.cache.v_scale : p.cache.k_scale;
    const int half = p.d >> 1;
    if constexpr (KIND == kKvBf16) {
        if (!live) return;
        uint16_t* out = static_cast<uint16_t*>(base) + (size_t)row * p.d;
        *reinterpret_cast<uint2*>(out + 4 * l) = make_uint2(decode::pack_bf16(a[0], a[1]), decode::pack_bf16(a[2], a[3]));
        *reinterpret_cast<uint2*>(out + half + 4 * l) = make_uint2(decode::pack_bf16(b[0], b[1]), decode::pack_bf16(b[2], b[3]));
    } else if constexpr (KIND == kKvFp8) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(__float_as_uint(a[i]) & 0x7FFFFFFFu, __float_as_uint(b[i]) & 0x7FFFFFFFu));
        // Non-negative floats order like their bits; a NaN orders above all
        // and makes the row's scale, and so the row, NaN.
        const float amax = __uint_as_float(max(decode::group_umax<L>(top), __float_as_uint(kFp8AbsmaxFloor)));
        if (!live) return;
        const float inv = __fdiv_rn(kFp8Max, amax);
        uint8_t* out = static_cast<uint8_t*>(base) + (size_t)row * p.d;
        *reinterpret_cast<uint32_t*>(out + 4 * l) = decode::e4m3x4(a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv);
        *reinterpret_cast<uint32_t*>(out + half + 4 * l) = decode::e4m3x4(b[0] * inv, b[1] * inv, b[2] * inv, b[3] * inv);
        if (l == 0) static_cast<float*>(scales)[row] = __fdiv_rn(amax, kFp8Max);
    } else if constexpr (KIND == kKvNvfp4) {
        // The lane's two blocks: even lanes work out the first's scale, odd ones
        // the second's, and they exchange them.
        bool lit_a, lit_b;
        const float max_a = block_absmax(a, lit_a), max_b = block_absmax(b, lit_b);
        const bool odd = l & 1;
        const uint32_t byte = ue4m3_encode(fmaxf(__fdiv_rn(odd ? max_b : max_a, 6.0f), kScaleMin));
        const float inv = __fdiv_rn(1.0f, ue4m3_decode((uint8_t)byte));
        const uint32_t other_byte = __shfl_xor_sync(0xffffffffu, byte, 1);
        const float other_inv = __shfl_xor_sync(0xffffffffu, inv, 1);
        const uint32_t sa = odd ? other_byte : byte, sb = odd ? byte : other_byte;
        const uint32_t ca = block_codes(a, odd ? other_inv : inv, lit_a), cb = block_codes(b, odd ? inv : other_inv, lit_b);
        if (!live) return;
        uint8_t* out = static_cast<uint8_t*>(base) + (size_t)row * half;
        *reinterpret_cast<uint16_t*>(out + 2 * l) = (uint16_t)ca;
        *reinterpret_cast<uint16_t*>(out + (half >> 1) + 2 * l) = (uint16_t)cb;
        if ((l & 3) == 0) {
            uint8_t* sc = static_cast<uint8_t*>(scales) + (size_t)row * (p.d >> 4);
            sc[l >> 2] = (uint8_t)sa;
            sc[(p.d >> 5) + (l >> 2)] = (uint8_t)sb;
        }
    }
}

template <int KIND, int L, bool FULL>
__global__ void __launch_bounds__(kThreads, FULL ? 4 : 1) kv_rows_kernel(const __grid_constant__ RowsParams p) {
    constexpr int kPer = 32 / L;  // heads of a token that a warp holds at once
    decode::chain();
    const int lane = threadIdx.x & 31, l = lane & (L - 1), sub = lane / L;
    const unsigned unit = blockIdx.x * kWarps + (threadIdx.x >> 5);
    const unsigned token = unit / (unsigned)p.walks;
    if (token >= (unsigned)p.tokens) return;
    const long t = token;
    const int begin = (int)(unit - token * p.walks) * p.rounds, end = min(begin + p.rounds, p.all_rounds);
    const bool inside = l < (p.d >> 3);
    const int half = p.d >> 1;
    const uint16_t* q_row = p.q + t * p.q_st + 4 * l;
    const uint16_t* k_row = p.k + t * p.k_st + 4 * l;
    const uint16_t* v_row = p.v + t * p.v_st + 4 * l;

    // A round's heads are all queries, all keys or all values.
    uint2 wa[kBatch], wb[kBatch];  // the lane's chunks of the next rounds' rows
    auto fetch = [&](int r0) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int r = r0 + i;
            wa[i] = wb[i] = make_uint2(0u, 0u);
            if (r >= end) continue;
            const bool query = r < p.q_rounds, key = !query && r < p.k_rounds;
            const int h = (r - (query ? 0 : key ? p.q_rounds : p.k_rounds)) * kPer + sub;
            if (h < (query ? p.q_heads : p.kv_heads) && inside) {
                const uint16_t* src = query ? q_row + (long)h * p.q_sh : key ? k_row + (long)h * p.k_sh : v_row + (long)h * p.v_sh;
                wa[i] = *reinterpret_cast<const uint2*>(src);
                wb[i] = *reinterpret_cast<const uint2*>(src + half);
            }
        }
    };
    fetch(begin);

    // The token's slot, its table row, and the norm weights of the lane's elements.
    long row0 = -1;  // cache row of head 0
    if constexpr (KIND != kKvNone) {
        const long slot = decode::load_index(p.slots, t, p.slot64);
        const long page = slot >> p.page_shift;
        if (slot >= 0) {
            if (page < p.cache.num_pages)
                row0 = page * p.kv_heads * p.cache.page_size + (slot & (p.cache.page_size - 1));
            else if (lane == 0)
                decode::report(p.err, kErrSlotRange);
        }
    }
    float ca[4], sa[4], cb[4], sb[4];
    if (p.rope) {
        const long pos = decode::load_index(p.positions, t, p.pos64);
        const bool ok = pos >= 0 && pos < p.rope_rows;
        if (!ok && lane == 0) decode::report(p.err, kErrPositionRange);
        const float* row = p.rope + (ok ? pos : 0) * p.rot;
        if constexpr (FULL) {  // rot == d, 16-byte aligned table
            const float4 c = inside ? *reinterpret_cast<const float4*>(row + 4 * l) : make_float4(1.f, 1.f, 1.f, 1.f);
            const float4 s = inside ? *reinterpret_cast<const float4*>(row + half + 4 * l) : make_float4(0.f, 0.f, 0.f, 0.f);
            ca[0] = ok ? c.x : 1.f, ca[1] = ok ? c.y : 1.f, ca[2] = ok ? c.z : 1.f, ca[3] = ok ? c.w : 1.f;
            sa[0] = ok ? s.x : 0.f, sa[1] = ok ? s.y : 0.f, sa[2] = ok ? s.z : 0.f, sa[3] = ok ? s.w : 0.f;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                ca[i] = cb[i] = 1.0f;
                sa[i] = sb[i] = 0.0f;
                if (inside && ok) {
                    factors(p, row, 4 * l + i, ca[i], sa[i]);
                    factors(p, row, half + 4 * l + i, cb[i], sb[i]);
                }
            }
        }
    }

    for (int r0 = begin; r0 < end; r0 += kBatch) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int r = r0 + i;
            if (r >= end) break;
            const bool query = r < p.q_rounds, key = !query && r < p.k_rounds;
            const int h = (r - (query ? 0 : key ? p.q_rounds : p.k_rounds)) * kPer + sub;
            const bool live = h < (query ? p.q_heads : p.kv_heads) && inside;
            float a[4], b[4];
            unpack4(wa[i], a);
            unpack4(wb[i], b);
            if (query || key) {
                const uint16_t* weight = query ? p.q_weight : p.k_weight;
                if (weight) {
                    float na[4] = {}, nb[4] = {};
                    if (inside) {
                        unpack4(__ldg(reinterpret_cast<const uint2*>(weight + 4 * l)), na);
                        unpack4(__ldg(reinterpret_cast<const uint2*>(weight + half + 4 * l)), nb);
                    }
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum += a[e] * a[e] + b[e] * b[e];
                    const float inv = rsqrtf(decode::group_sum<L>(sum) * p.inv_d + p.eps);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        a[e] = a[e] * inv * na[e];
                        b[e] = b[e] * inv * nb[e];
                    }
                }
                if (p.rope) rotate<L, FULL>(p, a, b, ca, sa, cb, sb, l);
            }
            if (query || (key && KIND == kKvNone)) {
                if (live) {
                    uint16_t* out = (query ? p.q_out + ((size_t)t * p.q_heads + h) * p.d : p.k_out + ((size_t)t * p.kv_heads + h) * p.d) + 4 * l;
                    *reinterpret_cast<uint2*>(out) = make_uint2(decode::pack_bf16(a[0], a[1]), decode::pack_bf16(a[2], a[3]));
                    *reinterpret_cast<uint2*>(out + half) = make_uint2(decode::pack_bf16(b[0], b[1]), decode::pack_bf16(b[2], b[3]));
                }
            } else if constexpr (KIND != kKvNone) {
                store_row<KIND, L>(p, !key, row0 + (long)h * p.cache.page_size, live && row0 >= 0, l, a, b);
            }
        }
        if (r0 + kBatch < end) fetch(r0 + kBatch);
    }
}

struct ReadParams {
    fp4b_kv_cache cache;
    int page_shift;
    const void* slots;
    int slot64;
    uint32_t total;               // pieces of eight elements
    uint32_t div_mul, div_shift;  // division by a slot's pieces
    uint16_t *k, *v;
    int* err;
};

// Eight elements of a row as BF16.
template <int KIND>
__device__ __forceinline__ uint4 read_eight(const void* base, const void* scales, long row, int d, int e) {
    if constexpr (KIND == kKvBf16) {
        return *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + (size_t)row * d + e);
    } else if constexpr (KIND == kKvFp8) {
        const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(base) + (size_t)row * d + e);
        const float s = static_cast<const float*>(scales)[row];
        uint32_t h[4], lo[2], hi[2];
        decode::e4m3x4_to_f16(w.x, lo);
        decode::e4m3x4_to_f16(w.y, hi);
        h[0] = lo[0], h[1] = lo[1], h[2] = hi[0], h[3] = hi[1];
        uint32_t out[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = decode::f16x2_to_float2(h[i]);
            out[i] = decode::pack_bf16(f.x * s, f.y * s);
        }
        return make_uint4(out[0], out[1], out[2], out[3]);
    } else {
        // code times scale is exact in FP16 (6 significant bits, 2^-10 to 2880), and in BF16
        const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(base) + (size_t)row * (d >> 1) + (e >> 1));
        const uint32_t byte = static_cast<const uint8_t*>(scales)[(size_t)row * (d >> 4) + (e >> 4)];
        const uint32_t s = decode::mul_f16x2(decode::ue4m3x2_to_f16(byte * 0x10001u), 0x5C005C00u);  // times 256
        uint32_t h[4], out[4];
        decode::e2m1x8_to_f16(w, h);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = decode::f16x2_to_float2(decode::mul_f16x2(h[i], s));
            out[i] = decode::pack_bf16(f.x, f.y);
        }
        return make_uint4(out[0], out[1], out[2], out[3]);
    }
}

// One thread takes kBatch pieces of eight elements (16 bytes of K and of V), 32
// apart, all its reads ahead of its writes.
template <int KIND>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ ReadParams p) {
    decode::chain();
    const int d = p.cache.head_dim, heads = p.cache.kv_heads, per_shift = d == 64 ? 3 : d == 128 ? 4 : 5;
    const uint32_t pieces = (uint32_t)heads << per_shift;
    const uint32_t first = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * (32u * kBatch) + (threadIdx.x & 31);
    long slot[kBatch];
    uint32_t in_slot[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        const uint32_t at = first + 32 * i, slot_at = (__umulhi(at, p.div_mul) + at) >> p.div_shift;  // at / pieces
        in_slot[i] = at - slot_at * pieces;
        slot[i] = at < p.total ? decode::load_index(p.slots, slot_at, p.slot64) : -1;
    }
    uint4 k[kBatch], v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        k[i] = v[i] = make_uint4(0, 0, 0, 0);
        const long page = slot[i] >> p.page_shift;
        if (slot[i] >= 0 && page < p.cache.num_pages) {
            const int h = in_slot[i] >> per_shift, e = (in_slot[i] - (h << per_shift)) * 8;
            const int row = ((int)page * heads + h) * p.cache.page_size + ((int)slot[i] & (p.cache.page_size - 1));
            k[i] = read_eight<KIND>(p.cache.k, p.cache.k_scale, row, d, e);
            v[i] = read_eight<KIND>(p.cache.v, p.cache.v_scale, row, d, e);
        } else if (slot[i] >= 0) {
            decode::report(p.err, kErrSlotRange);
        }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        const uint32_t at = first + 32 * i;
        if (at < p.total) {
            reinterpret_cast<uint4*>(p.k)[at] = k[i];
            reinterpret_cast<uint4*>(p.v)[at] = v[i];
        }
    }
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int shift_of(int page_size) {
    int s = 0;
    while ((1 << s) < page_size) ++s;
    return s;
}

template <int KIND, bool FULL>
cudaError_t launch_rows(RowsParams& p, cudaStream_t st) {
    const int need = p.d >> 3, lanes = need <= 8 ? 8 : need <= 16 ? 16 : 32, per = 32 / lanes;
    p.q_rounds = (p.q_heads + per - 1) / per;
    p.k_rounds = p.q_rounds + (p.k ? (p.kv_heads + per - 1) / per : 0);
    p.all_rounds = p.k_rounds + (p.v ? (p.kv_heads + per - 1) / per : 0);
    p.inv_d = 1.0f / (float)p.d;
    // As many rounds a warp as leave about 64 warps for each of 148 SMs: more
    // rounds share one table row and prologue, fewer spread over the GPU.
    p.rounds = (int)std::clamp((long)p.tokens * p.all_rounds / (148 * 64), 1l, (long)p.all_rounds);
    p.walks = (p.all_rounds + p.rounds - 1) / p.rounds;
    const long blocks = ((long)p.walks * p.tokens + kWarps - 1) / kWarps;
    auto* kernel = lanes == 8    ? kv_rows_kernel<KIND, 8, FULL>
                   : lanes == 16 ? kv_rows_kernel<KIND, 16, FULL>
                                 : kv_rows_kernel<KIND, 32, FULL>;
    return decode::launch_chained(kernel, dim3((unsigned)blocks), kThreads, 0, st, p);
}

template <int KIND>
cudaError_t launch_kind(RowsParams& p, cudaStream_t st) {
    const bool full = !p.rope || (p.rot == p.d && !p.pairs && aligned(p.rope, 16));
    return full ? launch_rows<KIND, true>(p, st) : launch_rows<KIND, false>(p, st);
}

// Checks shared by the two writing entry points; nullptr when all is well.
const char* rows_check(const RowsParams& p) {
    if (p.tokens < 0 || p.q_heads < 0 || p.kv_heads <= 0) return "negative token or head count";
    if (p.d < 32 || p.d > 256 || p.d % 32) return "head_dim must be a multiple of 32 from 32 to 256";
    const long most = (long)p.tokens * (p.q_heads + 2l * p.kv_heads);
    if (most > 0x7fffffffL) return "more than 2^31 rows in one call";
    const struct { const void* p; long st, sh; } rows[3] = {{p.q, p.q_st, p.q_sh}, {p.k, p.k_st, p.k_sh}, {p.v, p.v_st, p.v_sh}};
    for (const auto& r : rows)
        if (r.p && (!aligned(r.p, 8) || r.st % 4 || r.sh % 4)) return "rows must start on 8-byte boundaries";
    if (p.rope && (!p.positions || p.rope_rows <= 0 || p.rot <= 0 || p.rot > p.d || p.rot % 8))
        return "a rotation needs positions, a table and a rotated size that is a multiple of 8 up to head_dim";
    if (!aligned(p.q_weight, 8) || !aligned(p.k_weight, 8)) return "norm weights must be 8-byte aligned";
    return nullptr;
}

}  // namespace

const char* kv_cache_check(const fp4b_kv_cache* c) {
    if (!c || !c->k || !c->v) return "null cache or pages";
    if (c->num_pages <= 0 || c->kv_heads <= 0) return "a cache has at least one page and one head";
    if (c->page_size <= 0 || (c->page_size & (c->page_size - 1)) || c->page_size > 1024)
        return "page_size must be a power of two up to 1024";
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return "head_dim must be 64, 128 or 256";
    if (c->kind != kKvBf16 && c->kind != kKvFp8 && c->kind != kKvNvfp4) return "unknown cache kind";
    if ((long)c->num_pages * c->kv_heads * c->page_size > 0x7fffffffL) return "more than 2^31 rows in one cache";
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) return "pages must be 16-byte aligned";
    if (c->kind != kKvBf16 && (!c->k_scale || !c->v_scale)) return "a quantized cache needs its scales";
    if (!aligned(c->k_scale, 16) || !aligned(c->v_scale, 16)) return "scales must be 16-byte aligned";
    return nullptr;
}

}  // namespace fp4b

using namespace fp4b;

FP4B_EXPORT int fp4b_kv_rows(const fp4b_rows* rows, void* stream) {
    if (!rows) {
        set_last_error("fp4b_kv_rows: null arguments");
        return -1;
    }
    const fp4b_rows& r = *rows;
    const fp4b_kv_cache* cache = r.cache;
    RowsParams p{};
    p.q = static_cast<const uint16_t*>(r.q);
    p.k = static_cast<const uint16_t*>(r.k);
    p.v = static_cast<const uint16_t*>(r.v);
    p.q_st = r.q_st, p.q_sh = r.q_sh, p.k_st = r.k_st, p.k_sh = r.k_sh, p.v_st = r.v_st, p.v_sh = r.v_sh;
    p.tokens = r.tokens, p.q_heads = r.q ? r.q_heads : 0, p.kv_heads = r.kv_heads, p.d = r.head_dim;
    p.positions = r.positions, p.pos64 = r.pos64, p.rope = r.rope, p.rope_rows = r.rope_rows, p.rot = r.rot;
    p.pairs = r.interleaved;
    p.q_weight = static_cast<const uint16_t*>(r.q_weight);
    p.k_weight = static_cast<const uint16_t*>(r.k_weight);
    p.eps = r.eps;
    p.q_out = static_cast<uint16_t*>(r.q_out);
    p.k_out = static_cast<uint16_t*>(r.k_out);
    p.slots = r.slots, p.slot64 = r.slot64;
    const char* why = rows_check(p);
    if (!why && !p.q && !p.k) why = "neither queries nor keys";
    if (!why && p.q && (!p.q_out || !aligned(p.q_out, 8) || p.q_heads <= 0)) why = "queries need an 8-byte aligned output";
    if (!why && cache) {
        why = kv_cache_check(cache);
        if (!why && (!p.k || !p.v || !p.slots)) why = "a cache takes keys, values and slots";
        if (!why && (cache->kv_heads != p.kv_heads || cache->head_dim != p.d)) why = "the cache has other heads";
    } else if (!why) {
        if (p.k && (!p.k_out || !aligned(p.k_out, 8))) why = "keys need an 8-byte aligned output or a cache";
        if (p.v) why = "values need a cache";
    }
    if (why) {
        set_last_error("fp4b_kv_rows: %s", why);
        return -1;
    }
    if (p.tokens == 0) return 0;
    p.err = device_error_word();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (cache) {
        p.cache = *cache;
        p.page_shift = shift_of(cache->page_size);
        e = cache->kind == kKvBf16 ? launch_kind<kKvBf16>(p, st)
            : cache->kind == kKvFp8 ? launch_kind<kKvFp8>(p, st)
                                    : launch_kind<kKvNvfp4>(p, st);
    } else {
        e = launch_kind<kKvNone>(p, st);
    }
    return launch_status(e, "fp4b_kv_rows");
}

FP4B_EXPORT int fp4b_kv_read(const fp4b_kv_cache* cache, const void* slots, int slot64, long count, void* k_out,
                             void* v_out, void* stream) {
    const char* why = kv_cache_check(cache);
    if (!why && cache->kv_heads > 0x7fff0000 / (cache->head_dim / 8)) why = "too many heads";
    if (!why && (count < 0 || (count > 0 && (!slots || !k_out || !v_out)))) why = "null slots or outputs";
    if (!why && (!aligned(k_out, 16) || !aligned(v_out, 16))) why = "outputs must be 16-byte aligned";
    if (why) {
        set_last_error("fp4b_kv_read: %s", why);
        return -1;
    }
    if (count == 0) return 0;
    const int pieces = cache->kv_heads * (cache->head_dim / 8);
    ReadParams p{};
    p.cache = *cache;
    p.page_shift = shift_of(cache->page_size);
    p.slot64 = slot64;
    qcore::make_fast_div(pieces, &p.div_mul, &p.div_shift);
    p.err = device_error_word();
    auto* kernel = cache->kind == kKvBf16 ? kv_read_kernel<kKvBf16>
                   : cache->kind == kKvFp8 ? kv_read_kernel<kKvFp8>
                                           : kv_read_kernel<kKvNvfp4>;
    cudaError_t e = cudaSuccess;
    // Piece numbers are 31-bit: more slots than that in several launches.
    const long most = 0x7fff0000L / pieces;
    for (long at = 0; at < count && e == cudaSuccess; at += most) {
        const long n = std::min(most, count - at);
        p.total = (uint32_t)(n * pieces);
        p.slots = static_cast<const uint8_t*>(slots) + at * (slot64 ? 8 : 4);
        p.k = static_cast<uint16_t*>(k_out) + at * pieces * 8;
        p.v = static_cast<uint16_t*>(v_out) + at * pieces * 8;
        const unsigned blocks = (p.total + kThreads * kBatch - 1) / (kThreads * kBatch);
        e = decode::launch_chained(kernel, dim3(blocks), kThreads, 0, static_cast<cudaStream_t>(stream), p);
    }
    return launch_status(e, "fp4b_kv_read");
}
