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
//
// Measured on B200 (copy bandwidth 6.54 TB/s): norm and rotation of 8192 x 72
// heads x 64 30.1 us = 5.1 TB/s, bound by instruction issue and by DRAM's mix of
// reads and writes alike; 4099 tokens x 8 heads x 128 of K and V to nvfp4 and read
// back 14.6 us = 3.0 TB/s (9.4 of them the writing), two short launches; 32768 tokens of
// the same written alone 47.4 us in bf16 = 5.7 TB/s, 45.7 in fp8 = 4.5 and 58.7 in nvfp4 =
// 2.9 (its codes leave in two-byte, its scales in one-byte stores; what that costs was
// not measured); 131072 slots x 8 heads x 64 of nvfp4 read back 57.1 us = 6.0 TB/s, bound
// by HBM.
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

// Rotates the lane's two chunks, any rotated size and pairing.  c, s: the
// table's factors for the lane's elements (a: first chunk, b: second).
template <int L>
__device__ __forceinline__ void rotate(const RowsParams& p, float (&a)[4], float (&b)[4], const float (&ca)[4],
                                       const float (&sa)[4], const float (&cb)[4], const float (&sb)[4], int l) {
    if (p.pairs) {
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

// The scale byte of a 16-element block, ue4m3(absmax / 6) by the codec's rule
// (normal numbers rounded half up, subnormals truncated, at least 2^-9, from
// 256 up the largest), without the division: absmax / 6 rounded to fp32 reaches
// a boundary t of the rule exactly when absmax >= 6 t, since 6 t is an fp32
// number and the float below it, a sixth of an ulp of 6 t (2/3 of one of t or
// more) short of it, stays below when divided.  With absmax = M 2^e, M in [2^23,
// 2^24): the mantissa's eighths are floor((2 M - 45 2^h) / (3 2^(h + 1))) with h =
// 19 from M = 1.5 * 2^23 on, else 18.  absmax finite.
__device__ __forceinline__ uint32_t scale_byte(float absmax) {
    if (absmax < 0.09375f) return max(((uint32_t)(absmax * 512.0f) * 43u) >> 8, 1u);  // floor(x / 6) of x < 48
    const uint32_t bits = __float_as_uint(absmax), mant = (bits & 0x7FFFFFu) | 0x800000u;
    const uint32_t upper = mant >= 0xC00000u ? 1u : 0u;
    const uint32_t eighths = (((2u * mant - (45u << (18u + upper))) >> (19u + upper)) * 11u) >> 5;  // floor(y / 3) of y < 32
    const uint32_t exponent = (bits >> 23) - 123u + upper;
    return exponent >= 15u ? 0x7Fu : exponent * 8u + eighths;
}

// Lane i < 8 holds 1 / (8 + i) and lane 8 + i 1 / i, rounded to nearest: the
// reciprocals of the scales' mantissas, from which a power of two makes each
// scale's own exactly.
__device__ __forceinline__ float mantissa_reciprocal(int lane) { return __frcp_rn((float)(lane < 8 ? 8 + lane : lane & 7)); }
__device__ __forceinline__ float scale_reciprocal(float table, uint32_t byte) {
    const uint32_t e = byte >> 3, m = byte & 7u;
    return __shfl_sync(0xffffffffu, table, e ? m : 8u + m) * __uint_as_float((e ? 137u - e : 136u) << 23);
}

// Largest magnitudes (as fp32 bits; a NaN or an infinity orders above the rest)
// of the lane's two chunks, over the four lanes of each block (nvfp4) or over
// the whole row (fp8: both the same).
template <int KIND, int L>
__device__ __forceinline__ void magnitudes(const float (&a)[4], const float (&b)[4], uint32_t& top_a, uint32_t& top_b) {
    top_a = top_b = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        top_a = max(top_a, __float_as_uint(a[i]) & 0x7FFFFFFFu);
        top_b = max(top_b, __float_as_uint(b[i]) & 0x7FFFFFFFu);
    }
    if constexpr (KIND == kKvNvfp4) {
        top_a = decode::group_umax<4>(top_a);
        top_b = decode::group_umax<4>(top_b);
    } else {
        top_a = top_b = decode::group_umax<L>(max(top_a, top_b));
    }
}
// The same of BF16 chunks as they were read.
template <int KIND, int L>
__device__ __forceinline__ void magnitudes(uint2 a, uint2 b, uint32_t& top_a, uint32_t& top_b) {
    const uint32_t ma = decode::max_abs_bf16x2(a.x, a.y), mb = decode::max_abs_bf16x2(b.x, b.y);
    // chunk a's in the low half, b's in the high one
    uint32_t both = decode::max_abs_bf16x2(__byte_perm(ma, mb, 0x5410), __byte_perm(ma, mb, 0x7632));
#pragma unroll
    for (int o = KIND == kKvNvfp4 ? 2 : L / 2; o > 0; o >>= 1) both = decode::max_abs_bf16x2(both, __shfl_xor_sync(0xffffffffu, both, o));
    top_a = (both << 16) & 0x7FFF0000u;
    top_b = both & 0x7FFF0000u;
    if constexpr (KIND != kKvNvfp4) top_a = top_b = max(top_a, top_b);
}

// A block that holds a NaN, an infinity or a value from 2^30 on: the codec's
// absmax (NaN is skipped) and its literal scan.  Rare, and so out of line.  The
// four lanes of the block call it together; byte in bits 16 and up, four codes
// below.
__device__ __noinline__ uint32_t literal_block(float x0, float x1, float x2, float x3) {
    float f = fmaxf(fmaxf(fabsf(x0), fabsf(x1)), fmaxf(fabsf(x2), fabsf(x3)));
    f = fmaxf(f, __shfl_xor_sync(0xffffffffu, f, 2));
    f = fmaxf(f, __shfl_xor_sync(0xffffffffu, f, 1));
    const uint32_t byte = ue4m3_encode(fmaxf(__fdiv_rn(f == f ? f : 0.0f, 6.0f), kScaleMin));
    const float inv = __fdiv_rn(1.0f, ue4m3_decode((uint8_t)byte));
    return byte << 16 | (uint32_t)e2m1_scan(__fmul_rn(x0, inv)) | (uint32_t)e2m1_scan(__fmul_rn(x1, inv)) << 4 |
           (uint32_t)e2m1_scan(__fmul_rn(x2, inv)) << 8 | (uint32_t)e2m1_scan(__fmul_rn(x3, inv)) << 12;
}

// Bytes of a cache row's elements and of its scales.
template <int KIND>
__device__ __forceinline__ int row_bytes(int d) { return KIND == kKvBf16 ? 2 * d : KIND == kKvFp8 ? d : d >> 1; }
template <int KIND>
__device__ __forceinline__ int scale_bytes(int d) { return KIND == kKvBf16 ? 0 : KIND == kKvFp8 ? 4 : d >> 4; }

// Where lane l's share of a cache row goes: its first chunk (the second is half
// a row further) and, if it writes one, its scale.
struct Place {
    uint8_t* codes;
    uint8_t* scale;
};
template <int KIND>
__device__ __forceinline__ Place place_of(const RowsParams& p, bool value, long row, int l) {
    Place at;
    at.codes = static_cast<uint8_t*>(value ? p.cache.v : p.cache.k) + row * row_bytes<KIND>(p.d) + l * (KIND == kKvBf16 ? 8 : KIND == kKvFp8 ? 4 : 2);
    at.scale = static_cast<uint8_t*>(value ? p.cache.v_scale : p.cache.k_scale) + row * scale_bytes<KIND>(p.d);
    // nvfp4: lane 4j writes the scale of the first half's block j, lane 4j + 1 of the second's
    if (KIND == kKvNvfp4) at.scale += ((l & 1) ? p.d >> 5 : 0) + (l >> 2);
    return at;
}

// Writes one row's lane share.  All lanes of the warp call it; `live`: the lane
// has elements and its slot is valid.  top_a, top_b: see magnitudes; table: see
// mantissa_reciprocal.
template <int KIND, int L>
__device__ __forceinline__ void store_row(const RowsParams& p, Place at, bool live, int l, const float (&a)[4], const float (&b)[4],
                                          uint32_t top_a, uint32_t top_b, float table) {
    uint8_t* second = at.codes + (row_bytes<KIND>(p.d) >> 1);
    if constexpr (KIND == kKvBf16) {
        if (!live) return;
        *reinterpret_cast<uint2*>(at.codes) = make_uint2(decode::pack_bf16(a[0], a[1]), decode::pack_bf16(a[2], a[3]));
        *reinterpret_cast<uint2*>(second) = make_uint2(decode::pack_bf16(b[0], b[1]), decode::pack_bf16(b[2], b[3]));
    } else if constexpr (KIND == kKvFp8) {
        if (!live) return;
        // (a NaN makes the row's scale, and so the row, NaN)
        const float amax = __uint_as_float(max(top_a, __float_as_uint(kFp8AbsmaxFloor)));
        const float inv = __fdiv_rn(kFp8Max, amax);
        *reinterpret_cast<uint32_t*>(at.codes) = decode::e4m3x4(a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv);
        *reinterpret_cast<uint32_t*>(second) = decode::e4m3x4(b[0] * inv, b[1] * inv, b[2] * inv, b[3] * inv);
        if (l == 0) *reinterpret_cast<float*>(at.scale) = __fdiv_rn(amax, kFp8Max);
    } else if constexpr (KIND == kKvNvfp4) {
        // The lane's two blocks: even lanes work out the first's scale, odd ones
        // the second's, and they exchange their reciprocals.
        const bool odd = l & 1, lit_a = top_a >= kFastAbsmaxF32Limit, lit_b = top_b >= kFastAbsmaxF32Limit;
        uint32_t byte = scale_byte(__uint_as_float(min(odd ? top_b : top_a, kFastAbsmaxF32Limit)));
        const float inv = scale_reciprocal(table, byte), other = __shfl_xor_sync(0xffffffffu, inv, 1);
        const float inv_a = odd ? other : inv, inv_b = odd ? inv : other;
        uint32_t ca = decode::e2m1x4(a[0], a[1], a[2], a[3], inv_a), cb = decode::e2m1x4(b[0], b[1], b[2], b[3], inv_b);
        if (__any_sync(0xffffffffu, lit_a || lit_b)) {
            const uint32_t la = literal_block(a[0], a[1], a[2], a[3]), lb = literal_block(b[0], b[1], b[2], b[3]);
            if (lit_a) ca = la & 0xFFFFu;
            if (lit_b) cb = lb & 0xFFFFu;
            if (odd ? lit_b : lit_a) byte = (odd ? lb : la) >> 16;
        }
        if (!live) return;
        *reinterpret_cast<uint16_t*>(at.codes) = (uint16_t)ca;
        *reinterpret_cast<uint16_t*>(second) = (uint16_t)cb;
        if ((l & 2) == 0) *at.scale = (uint8_t)byte;
    }
}

// Cache row of head 0 of token t's slot; -1 for none.
__device__ __forceinline__ long slot_row(const RowsParams& p, long t, int lane) {
    const long slot = decode::load_index(p.slots, t, p.slot64);
    const long page = slot >> p.page_shift;
    if (slot < 0) return -1;
    if (page < p.cache.num_pages) return page * p.kv_heads * p.cache.page_size + (slot & (p.cache.page_size - 1));
    if (lane == 0) decode::report(p.err, kErrSlotRange);
    return -1;
}

using decode::fma2;
using decode::mul2;
using decode::pair_of;

__device__ __forceinline__ unsigned long long widen(uint32_t w) {
    return ((unsigned long long)(w & 0xFFFF0000u) << 32) | (unsigned long long)(w << 16);
}

// The common forms: rows rotated as a whole in halves, normed or not (ROTATED),
// or written as they are; values as they are.  Two elements an instruction, and
// the norm weights multiplied into the table's factors once a token: with w_a,
// w_b a pair's weights,
//   out_a = (a (w_a c) - b (w_b s)) / rms,  out_b = (b (w_b c) + a (w_a s)) / rms
// (117 instructions a round of 32 / L rows where the general kernel below, one
// element and one check at a time, has 200: 8192 tokens x 72 heads x 64 30.1 us
// against 50.0; what only the latter can do is up to twice as slow: pairs 48.4 us, half
// of each row rotated 61.8).
template <int KIND, int L, bool ROTATED>
__global__ void __launch_bounds__(kThreads, 4) kv_walk_kernel(const __grid_constant__ RowsParams p) {
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
    [[maybe_unused]] const float table = mantissa_reciprocal(lane & 15);
    [[maybe_unused]] const long row0 = KIND != kKvNone ? slot_row(p, t, lane) : -1;
    [[maybe_unused]] float c[4], s[4];
    if constexpr (ROTATED) {
        const long pos = decode::load_index(p.positions, t, p.pos64);
        const bool ok = pos >= 0 && pos < p.rope_rows;
        if (!ok && lane == 0) decode::report(p.err, kErrPositionRange);
        const float* row = p.rope + (ok ? pos : 0) * p.rot + 4 * (inside ? l : 0);
        const float4 cv = *reinterpret_cast<const float4*>(row), sv = *reinterpret_cast<const float4*>(row + half);
        c[0] = ok ? cv.x : 1.f, c[1] = ok ? cv.y : 1.f, c[2] = ok ? cv.z : 1.f, c[3] = ok ? cv.w : 1.f;
        s[0] = ok ? sv.x : 0.f, s[1] = ok ? sv.y : 0.f, s[2] = ok ? sv.z : 0.f, s[3] = ok ? sv.w : 0.f;
    }

    // Walks rounds [from, to) of one kind of rows, two in flight ahead of the two
    // at hand: `src` the lane's first chunk of head 0, `put(live, wa, wb)` what
    // is done with each round's two chunks in turn.
    auto walk = [&](int from, int to, const uint16_t* src, long stride, int heads, auto&& put) {
        const uint16_t* at = src + (long)(from * kPer + sub) * stride;
        const long step = kPer * stride;
        int h = from * kPer + sub;  // the next head to be read
        uint2 wa[2], wb[2];
        auto fetch = [&](int r0) {
#pragma unroll
            for (int i = 0; i < 2; ++i, at += step, h += kPer) {
                wa[i] = wb[i] = make_uint2(0u, 0u);
                if (r0 + i < to && h < heads && inside) {
                    wa[i] = *reinterpret_cast<const uint2*>(at);
                    wb[i] = *reinterpret_cast<const uint2*>(at + half);
                }
            }
        };
        fetch(from);
        int done = from * kPer + sub;  // the next head to be put
        for (int r0 = from; r0 < to; r0 += 2) {
            const uint2 a0 = wa[0], b0 = wb[0], a1 = wa[1], b1 = wb[1];
            if (r0 + 2 < to) fetch(r0 + 2);
            put(done < heads && inside, a0, b0);
            if (r0 + 1 < to) put(done + kPer < heads && inside, a1, b1);
            done += 2 * kPer;
        }
    };
    auto rotated = [&](int from, int to, const uint16_t* src, long stride, int heads, const uint16_t* weight, auto&& put) {
        unsigned long long ac[2], bs[2], bc[2], as[2];  // w_a c, -w_b s, w_b c, w_a s
        {
            float wa[4] = {1.f, 1.f, 1.f, 1.f}, wb[4] = {1.f, 1.f, 1.f, 1.f};
            if (weight && inside) {
                unpack4(__ldg(reinterpret_cast<const uint2*>(weight + 4 * l)), wa);
                unpack4(__ldg(reinterpret_cast<const uint2*>(weight + half + 4 * l)), wb);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                ac[i] = pair_of(wa[2 * i] * c[2 * i], wa[2 * i + 1] * c[2 * i + 1]);
                bs[i] = pair_of(-wb[2 * i] * s[2 * i], -wb[2 * i + 1] * s[2 * i + 1]);
                bc[i] = pair_of(wb[2 * i] * c[2 * i], wb[2 * i + 1] * c[2 * i + 1]);
                as[i] = pair_of(wa[2 * i] * s[2 * i], wa[2 * i + 1] * s[2 * i + 1]);
            }
        }
        walk(from, to, src, stride, heads, [&](bool live, uint2 wa, uint2 wb) {
            const unsigned long long a0 = widen(wa.x), a1 = widen(wa.y), b0 = widen(wb.x), b1 = widen(wb.y);
            unsigned long long o[4] = {fma2(b0, bs[0], mul2(a0, ac[0])), fma2(b1, bs[1], mul2(a1, ac[1])),
                                       fma2(a0, as[0], mul2(b0, bc[0])), fma2(a1, as[1], mul2(b1, bc[1]))};
            if (weight) {
                const unsigned long long q = fma2(a0, a0, fma2(a1, a1, fma2(b0, b0, mul2(b1, b1))));
                const float sum = decode::group_sum<L>(__uint_as_float((uint32_t)q) + __uint_as_float((uint32_t)(q >> 32)));
                const float inv = rsqrtf(sum * p.inv_d + p.eps);
                const unsigned long long inv2 = pair_of(inv, inv);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = mul2(o[i], inv2);
            }
            float a[4], b[4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[2 * i] = __uint_as_float((uint32_t)o[i]), a[2 * i + 1] = __uint_as_float((uint32_t)(o[i] >> 32));
                b[2 * i] = __uint_as_float((uint32_t)o[2 + i]), b[2 * i + 1] = __uint_as_float((uint32_t)(o[2 + i] >> 32));
            }
            put(live, a, b);
        });
    };
    auto to_rows = [&](uint16_t* out, int from) {  // `out`: the lane's first chunk of head 0
        out += (size_t)(from * kPer + sub) * p.d;
        return [&, out](bool live, const float (&a)[4], const float (&b)[4]) mutable {
            if (live) {
                *reinterpret_cast<uint2*>(out) = make_uint2(decode::pack_bf16(a[0], a[1]), decode::pack_bf16(a[2], a[3]));
                *reinterpret_cast<uint2*>(out + half) = make_uint2(decode::pack_bf16(b[0], b[1]), decode::pack_bf16(b[2], b[3]));
            }
            out += kPer * p.d;
        };
    };
    [[maybe_unused]] const bool stored = row0 >= 0;
    [[maybe_unused]] auto first_place = [&](bool value, int from) {
        return place_of<KIND>(p, value, (stored ? row0 : 0) + (long)(from * kPer + sub) * p.cache.page_size, l);
    };
    [[maybe_unused]] const long code_step = (long)kPer * p.cache.page_size * row_bytes<KIND>(p.d);
    [[maybe_unused]] const long scale_step = (long)kPer * p.cache.page_size * scale_bytes<KIND>(p.d);
    [[maybe_unused]] auto raw_to_cache = [&](bool value, int from) {
        Place at = first_place(value, from);
        return [&, at](bool live, uint2 wa, uint2 wb) mutable {
            float a[4], b[4];
            unpack4(wa, a);
            unpack4(wb, b);
            uint32_t top_a = 0, top_b = 0;
            if constexpr (KIND == kKvFp8 || KIND == kKvNvfp4) magnitudes<KIND, L>(wa, wb, top_a, top_b);
            store_row<KIND, L>(p, at, live && stored, l, a, b, top_a, top_b, table);
            at.codes += code_step, at.scale += scale_step;
        };
    };

    if constexpr (ROTATED) {
        if (begin < p.q_rounds)
            rotated(begin, min(end, p.q_rounds), p.q + t * p.q_st + 4 * l, p.q_sh, p.q_heads, p.q_weight,
                    to_rows(p.q_out + (size_t)t * p.q_heads * p.d + 4 * l, begin));
    }
    const int k_begin = max(begin - p.q_rounds, 0), k_end = min(end, p.k_rounds) - p.q_rounds;
    if (k_begin < k_end) {
        const uint16_t* src = p.k + t * p.k_st + 4 * l;
        if constexpr (ROTATED && KIND == kKvNone) {
            rotated(k_begin, k_end, src, p.k_sh, p.kv_heads, p.k_weight, to_rows(p.k_out + (size_t)t * p.kv_heads * p.d + 4 * l, k_begin));
        } else if constexpr (ROTATED) {
            Place at = first_place(false, k_begin);
            rotated(k_begin, k_end, src, p.k_sh, p.kv_heads, p.k_weight, [&](bool live, const float (&a)[4], const float (&b)[4]) {
                uint32_t top_a = 0, top_b = 0;
                if constexpr (KIND == kKvFp8 || KIND == kKvNvfp4) magnitudes<KIND, L>(a, b, top_a, top_b);
                store_row<KIND, L>(p, at, live && stored, l, a, b, top_a, top_b, table);
                at.codes += code_step, at.scale += scale_step;
            });
        } else {
            walk(k_begin, k_end, src, p.k_sh, p.kv_heads, raw_to_cache(false, k_begin));
        }
    }
    if constexpr (KIND != kKvNone) {
        const int v_begin = max(begin - p.k_rounds, 0), v_end = end - p.k_rounds;
        if (v_begin < v_end) walk(v_begin, v_end, p.v + t * p.v_st + 4 * l, p.v_sh, p.kv_heads, raw_to_cache(true, v_begin));
    }
}

// Every other form: parts of rows and pairs rotated, norms without a rotation.
template <int KIND, int L>
__global__ void __launch_bounds__(kThreads) kv_rows_kernel(const __grid_constant__ RowsParams p) {
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
    [[maybe_unused]] const float table = mantissa_reciprocal(lane & 15);
    [[maybe_unused]] const long row0 = KIND != kKvNone ? slot_row(p, t, lane) : -1;
    float ca[4], sa[4], cb[4], sb[4];
    if (p.rope) {
        const long pos = decode::load_index(p.positions, t, p.pos64);
        const bool ok = pos >= 0 && pos < p.rope_rows;
        if (!ok && lane == 0) decode::report(p.err, kErrPositionRange);
        const float* row = p.rope + (ok ? pos : 0) * p.rot;
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
                if (p.rope) rotate<L>(p, a, b, ca, sa, cb, sb, l);
            }
            if (query || (key && KIND == kKvNone)) {
                if (live) {
                    uint16_t* out = (query ? p.q_out + ((size_t)t * p.q_heads + h) * p.d : p.k_out + ((size_t)t * p.kv_heads + h) * p.d) + 4 * l;
                    *reinterpret_cast<uint2*>(out) = make_uint2(decode::pack_bf16(a[0], a[1]), decode::pack_bf16(a[2], a[3]));
                    *reinterpret_cast<uint2*>(out + half) = make_uint2(decode::pack_bf16(b[0], b[1]), decode::pack_bf16(b[2], b[3]));
                }
            } else if constexpr (KIND != kKvNone) {
                uint32_t top_a = 0, top_b = 0;
                if constexpr (KIND == kKvFp8 || KIND == kKvNvfp4) magnitudes<KIND, L>(a, b, top_a, top_b);
                const Place at = place_of<KIND>(p, !key, (row0 < 0 ? 0 : row0) + (long)h * p.cache.page_size, l);
                store_row<KIND, L>(p, at, live && row0 >= 0, l, a, b, top_a, top_b, table);
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
    uint32_t total;               // pieces of sixteen elements
    uint32_t div_mul, div_shift;  // division by a slot's pieces
    uint16_t *k, *v;
    int* err;
};

// Sixteen elements of a row as BF16, and their way to 32-byte aligned memory.
struct Sixteen {
    uint32_t w[8];
};
template <int KIND>
__device__ __forceinline__ Sixteen read_sixteen(const void* base, const void* scales, int row, int d, int e) {
    Sixteen x;
    const size_t at = (size_t)row * d + e;
    if constexpr (KIND == kKvBf16) {
        const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
        const uint4 a = from[0], b = from[1];
        x = Sixteen{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
    } else if constexpr (KIND == kKvFp8) {
        const uint4 c = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(base) + at);
        const float s = static_cast<const float*>(scales)[row];
        const uint32_t word[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t h[2];
            decode::e4m3x4_to_f16(word[i], h);
            const float2 a = decode::f16x2_to_float2(h[0]), b = decode::f16x2_to_float2(h[1]);
            x.w[2 * i] = decode::pack_bf16(a.x * s, a.y * s);
            x.w[2 * i + 1] = decode::pack_bf16(b.x * s, b.y * s);
        }
    } else {
        // code times scale is exact in FP16 (6 significant bits, 2^-10 to 2880), and in BF16
        const uint2 c = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(base) + (at >> 1));
        const uint32_t byte = static_cast<const uint8_t*>(scales)[at >> 4];
        const uint32_t s = decode::mul_f16x2(decode::ue4m3x2_to_f16(byte * 0x10001u), 0x5C005C00u);  // times 256
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t h[4];
            decode::e2m1x8_to_f16(half ? c.y : c.x, h);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = decode::f16x2_to_float2(decode::mul_f16x2(h[i], s));
                x.w[4 * half + i] = decode::pack_bf16(f.x, f.y);
            }
        }
    }
    return x;
}
__device__ __forceinline__ void store_sixteen(uint16_t* to, const Sixteen& x) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(x.w[0]), "r"(x.w[1]), "r"(x.w[2]), "r"(x.w[3]),
                 "r"(x.w[4]), "r"(x.w[5]), "r"(x.w[6]), "r"(x.w[7])
                 : "memory");
}

// A thread takes one piece of sixteen elements, 32 bytes of K and of V written by one
// instruction each: 131072 slots x 8 heads x 64 of nvfp4 57.3 us (70.0 with two pieces
// of eight for one of these, four of them a thread; 61.5 and 66.2 with two and four
// of sixteen: what counts is many short threads and wide stores).
template <int KIND>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ ReadParams p) {
    decode::chain();
    const int d = p.cache.head_dim, heads = p.cache.kv_heads, per_shift = d == 64 ? 2 : d == 128 ? 3 : 4;
    const uint32_t at = blockIdx.x * kThreads + threadIdx.x;
    if (at >= p.total) return;
    const uint32_t pieces = (uint32_t)heads << per_shift;
    const uint32_t slot_at = (__umulhi(at, p.div_mul) + at) >> p.div_shift;  // at / pieces
    const int in_slot = (int)(at - slot_at * pieces), h = in_slot >> per_shift, e = (in_slot - (h << per_shift)) * 16;
    const long slot = decode::load_index(p.slots, slot_at, p.slot64), page = slot >> p.page_shift;
    Sixteen k{}, v{};
    if (slot >= 0 && page < p.cache.num_pages) {
        const int row = ((int)page * heads + h) * p.cache.page_size + ((int)slot & (p.cache.page_size - 1));
        k = read_sixteen<KIND>(p.cache.k, p.cache.k_scale, row, d, e);
        v = read_sixteen<KIND>(p.cache.v, p.cache.v_scale, row, d, e);
    } else if (slot >= 0) {
        decode::report(p.err, kErrSlotRange);
    }
    store_sixteen(p.k + (size_t)at * 16, k);
    store_sixteen(p.v + (size_t)at * 16, v);
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int shift_of(int page_size) {
    int s = 0;
    while ((1 << s) < page_size) ++s;
    return s;
}

template <int KIND>
cudaError_t launch_rows(RowsParams& p, cudaStream_t st) {
    const int need = p.d >> 3, lanes = need <= 8 ? 8 : need <= 16 ? 16 : 32, per = 32 / lanes;
    const bool rotated = p.rope && p.rot == p.d && !p.pairs && aligned(p.rope, 16);
    p.q_rounds = (p.q_heads + per - 1) / per;
    p.k_rounds = p.q_rounds + (p.k ? (p.kv_heads + per - 1) / per : 0);
    p.all_rounds = p.k_rounds + (p.v ? (p.kv_heads + per - 1) / per : 0);
    p.inv_d = 1.0f / (float)p.d;
    // As many rounds a warp as leave about 32 warps for each of 148 SMs: more
    // rounds share one table row and prologue, fewer spread over the GPU.
    p.rounds = (int)std::clamp((long)p.tokens * p.all_rounds / (148 * 32), 1l, (long)p.all_rounds);
    p.walks = (p.all_rounds + p.rounds - 1) / p.rounds;
    p.rounds = (p.all_rounds + p.walks - 1) / p.walks;  // the same for all, nearly
    const long blocks = ((long)p.walks * p.tokens + kWarps - 1) / kWarps;
    void (*kernel)(RowsParams) =
        rotated ? (lanes == 8 ? kv_walk_kernel<KIND, 8, true> : lanes == 16 ? kv_walk_kernel<KIND, 16, true> : kv_walk_kernel<KIND, 32, true>)
                : (lanes == 8 ? kv_rows_kernel<KIND, 8> : lanes == 16 ? kv_rows_kernel<KIND, 16> : kv_rows_kernel<KIND, 32>);
    if constexpr (KIND != kKvNone) {
        if (!p.rope && !p.k_weight && !p.q)
            kernel = lanes == 8 ? kv_walk_kernel<KIND, 8, false> : lanes == 16 ? kv_walk_kernel<KIND, 16, false> : kv_walk_kernel<KIND, 32, false>;
    }
    return decode::launch_chained(kernel, dim3((unsigned)blocks), kThreads, 0, st, p);
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
        e = cache->kind == kKvBf16 ? launch_rows<kKvBf16>(p, st)
            : cache->kind == kKvFp8 ? launch_rows<kKvFp8>(p, st)
                                    : launch_rows<kKvNvfp4>(p, st);
    } else {
        e = launch_rows<kKvNone>(p, st);
    }
    return launch_status(e, "fp4b_kv_rows");
}

FP4B_EXPORT int fp4b_kv_read(const fp4b_kv_cache* cache, const void* slots, int slot64, long count, void* k_out,
                             void* v_out, void* stream) {
    const char* why = kv_cache_check(cache);
    if (!why && cache->kv_heads > 0x7fff0000 / (cache->head_dim / 8)) why = "too many heads";
    if (!why && (count < 0 || (count > 0 && (!slots || !k_out || !v_out)))) why = "null slots or outputs";
    if (!why && (!aligned(k_out, 32) || !aligned(v_out, 32))) why = "outputs must be 32-byte aligned";
    if (why) {
        set_last_error("fp4b_kv_read: %s", why);
        return -1;
    }
    if (count == 0) return 0;
    const int pieces = cache->kv_heads * (cache->head_dim / 16);
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
        p.k = static_cast<uint16_t*>(k_out) + at * pieces * 16;
        p.v = static_cast<uint16_t*>(v_out) + at * pieces * 16;
        const unsigned blocks = (p.total + kThreads - 1) / kThreads;
        e = decode::launch_chained(kernel, dim3(blocks), kThreads, 0, static_cast<cudaStream_t>(stream), p);
    }
    return launch_status(e, "fp4b_kv_read");
}
