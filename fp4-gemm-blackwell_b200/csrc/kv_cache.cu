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
// token and walks its heads, so the table row and the norm weights are read
// once a token.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>

#include "decode_core.cuh"
#include "fp4b_internal.h"

#define FP4B_EXPORT extern "C" __attribute__((visibility("default")))

namespace fp4b {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

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
    int rounds;  // head groups of 32 / L heads that one warp walks
    int* err;
};

__device__ __forceinline__ void unpack4(uint2 w, float (&x)[4]) {
    x[0] = decode::bf16_lo(w.x);
    x[1] = decode::bf16_hi(w.x);
    x[2] = decode::bf16_lo(w.y);
    x[3] = decode::bf16_hi(w.y);
}

// Rotates the lane's two chunks.  c, s: the table's factors for the lane's
// elements (a: first chunk, b: second).
template <int L>
__device__ __forceinline__ void rotate(const RowsParams& p, float (&a)[4], float (&b)[4], const float (&ca)[4],
                                       const float (&sa)[4], const float (&cb)[4], const float (&sb)[4], int l) {
    const int half = p.rot >> 1;
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
    } else if (p.rot == p.d) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = a[i], y = b[i];
            a[i] = x * ca[i] - y * sa[i];
            b[i] = y * ca[i] + x * sa[i];
        }
    } else {
        // Part of the row is rotated: chunk c's partner is chunk c +- rot / 8,
        // held by another lane.  Chunks 0 .. d/8 - 1 are the lanes' first
        // ones, d/8 .. d/4 - 1 their second ones.
        const int shift = half >> 2, lanes = p.d >> 3;
        const int group = (threadIdx.x & 31) & ~(L - 1);
        float pa[4], pb[4];
        const int ta = l < shift ? l + shift : l - shift;                  // partner of the first chunk
        const int tb = l + lanes < shift ? l + lanes + shift : l + lanes - shift;  // of the second
        const int la = group + (ta >= lanes ? ta - lanes : max(ta, 0)), lb = group + (tb >= lanes ? tb - lanes : max(tb, 0));
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

// Four values of a block's lane -> its four E2M1 codes; `byte`: the block's
// scale.  The four lanes of the block call it together.
__device__ __forceinline__ uint32_t nvfp4_four(const float (&x)[4], uint32_t& byte) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    top = decode::group_umax<4>(top);
    float amax = __uint_as_float(top);
    const bool literal = top >= kFastAbsmaxF32Limit;
    if (literal) {  // the codec's absmax skips NaN
        amax = 0.0f;
        for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(x[i]));
    }
    if (__any_sync(0xffffffffu, literal)) {
        float other = amax;
        other = fmaxf(other, __shfl_xor_sync(0xffffffffu, other, 2));
        other = fmaxf(other, __shfl_xor_sync(0xffffffffu, other, 1));
        if (literal) amax = other;
    }
    byte = ue4m3_encode(fmaxf(__fdiv_rn(amax, 6.0f), kScaleMin));
    const float inv = __fdiv_rn(1.0f, ue4m3_decode((uint8_t)byte));
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
        uint32_t sa, sb;
        const uint32_t ca = nvfp4_four(a, sa), cb = nvfp4_four(b, sb);
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

template <int KIND, int L>
__global__ void __launch_bounds__(kThreads) kv_rows_kernel(const __grid_constant__ RowsParams p) {
    constexpr int kPer = 32 / L;  // heads of a token that a warp holds at once
    const int lane = threadIdx.x & 31, l = lane & (L - 1), sub = lane / L;
    const int heads = p.q_heads + (p.k ? p.kv_heads : 0) + (p.v ? p.kv_heads : 0);
    const int walks = (heads + kPer * p.rounds - 1) / (kPer * p.rounds);  // warps a token
    const long unit = (long)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const long t = unit / walks;
    if (t >= p.tokens) return;
    const int first = (int)(unit - t * walks) * kPer * p.rounds + sub;
    const bool inside = l < (p.d >> 3);
    const int half = p.d >> 1;

    // The token's table row, its slot, and the norm weights of the lane's elements.
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
    for (int r = 0; r < p.rounds; ++r) {
        const int h = first + r * kPer;
        const bool query = h < p.q_heads;
        const int hk = h - p.q_heads;
        const bool key = !query && p.k && hk < p.kv_heads;
        const int hv = p.k ? hk - p.kv_heads : hk;
        const bool live = h < heads && inside;
        const uint16_t* src = query ? p.q + t * p.q_st + h * p.q_sh
                              : key ? p.k + t * p.k_st + hk * p.k_sh
                                    : p.v + t * p.v_st + hv * p.v_sh;
        float a[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
        if (live) {
            unpack4(*reinterpret_cast<const uint2*>(src + 4 * l), a);
            unpack4(*reinterpret_cast<const uint2*>(src + half + 4 * l), b);
        }
        const uint16_t* weight = query ? p.q_weight : p.k_weight;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += a[i] * a[i] + b[i] * b[i];
        sum = decode::group_sum<L>(sum);
        if ((query || key) && weight && live) {
            const float inv = rsqrtf(sum / (float)p.d + p.eps);
            float wa[4], wb[4];
            unpack4(*reinterpret_cast<const uint2*>(weight + 4 * l), wa);
            unpack4(*reinterpret_cast<const uint2*>(weight + half + 4 * l), wb);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = a[i] * inv * wa[i];
                b[i] = b[i] * inv * wb[i];
            }
        }
        if (p.rope) {
            float ra[4] = {a[0], a[1], a[2], a[3]}, rb[4] = {b[0], b[1], b[2], b[3]};
            rotate<L>(p, ra, rb, ca, sa, cb, sb, l);
            if (query || key) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[i] = ra[i];
                    b[i] = rb[i];
                }
            }
        }
        if (live && (query || (key && KIND == kKvNone))) {
            uint16_t* out = query ? p.q_out + ((size_t)t * p.q_heads + h) * p.d : p.k_out + ((size_t)t * p.kv_heads + hk) * p.d;
            *reinterpret_cast<uint2*>(out + 4 * l) = make_uint2(decode::pack_bf16(a[0], a[1]), decode::pack_bf16(a[2], a[3]));
            *reinterpret_cast<uint2*>(out + half + 4 * l) =
                make_uint2(decode::pack_bf16(b[0], b[1]), decode::pack_bf16(b[2], b[3]));
        }
        if constexpr (KIND != kKvNone) {
            const long row = row0 + (long)(key ? hk : hv) * p.cache.page_size;
            if (__any_sync(0xffffffffu, live && !query))
                store_row<KIND, L>(p, !key, row, live && !query && row0 >= 0, l, a, b);
        }
    }
}

struct ReadParams {
    fp4b_kv_cache cache;
    int page_shift;
    const void* slots;
    int slot64;
    long rows;  // slots x heads
    uint16_t *k, *v;
    int* err;
};

// Eight elements of a row as BF16.
template <int KIND>
__device__ __forceinline__ uint4 read_eight(const void* base, const void* scales, long row, int d, int e) {
    float x[8];
    if constexpr (KIND == kKvBf16) {
        return *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + (size_t)row * d + e);
    } else if constexpr (KIND == kKvFp8) {
        const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(base) + (size_t)row * d + e);
        const float s = static_cast<const float*>(scales)[row];
        uint32_t h[4], lo[2], hi[2];
        decode::e4m3x4_to_f16(w.x, lo);
        decode::e4m3x4_to_f16(w.y, hi);
        h[0] = lo[0], h[1] = lo[1], h[2] = hi[0], h[3] = hi[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = decode::f16x2_to_float2(h[i]);
            x[2 * i] = f.x * s, x[2 * i + 1] = f.y * s;
        }
    } else {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(base) + (size_t)row * (d >> 1) + (e >> 1));
        const float s = decode::ue4m3_float(static_cast<const uint8_t*>(scales)[(size_t)row * (d >> 4) + (e >> 4)]);
        uint32_t h[4];
        decode::e2m1x8_to_f16(w, h);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = decode::f16x2_to_float2(h[i]);
            x[2 * i] = f.x * s, x[2 * i + 1] = f.y * s;
        }
    }
    return make_uint4(decode::pack_bf16(x[0], x[1]), decode::pack_bf16(x[2], x[3]), decode::pack_bf16(x[4], x[5]),
                      decode::pack_bf16(x[6], x[7]));
}

// One thread per eight elements of an output row (16 bytes of K and of V).
template <int KIND>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ ReadParams p) {
    const int d = p.cache.head_dim, per = d >> 3, heads = p.cache.kv_heads;
    const long total = p.rows * per;
    for (long i = (long)blockIdx.x * kThreads + threadIdx.x; i < total; i += (long)gridDim.x * kThreads) {
        const long r = i / per;
        const int e = (int)(i - r * per) * 8;
        const long t = r / heads;
        const int h = (int)(r - t * heads);
        const long slot = decode::load_index(p.slots, t, p.slot64);
        const long page = slot >> p.page_shift;
        uint4 k = make_uint4(0, 0, 0, 0), v = k;
        if (slot >= 0 && page < p.cache.num_pages) {
            const long row = (page * heads + h) * p.cache.page_size + (slot & (p.cache.page_size - 1));
            k = read_eight<KIND>(p.cache.k, p.cache.k_scale, row, d, e);
            v = read_eight<KIND>(p.cache.v, p.cache.v_scale, row, d, e);
        } else if (slot >= 0) {
            decode::report(p.err, kErrSlotRange);
        }
        *reinterpret_cast<uint4*>(p.k + (size_t)r * d + e) = k;
        *reinterpret_cast<uint4*>(p.v + (size_t)r * d + e) = v;
    }
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

int shift_of(int page_size) {
    int s = 0;
    while ((1 << s) < page_size) ++s;
    return s;
}

template <int KIND>
cudaError_t launch_rows(const RowsParams& p, cudaStream_t st) {
    const int need = p.d >> 3, lanes = need <= 8 ? 8 : need <= 16 ? 16 : 32, per = 32 / lanes;
    const int heads = p.q_heads + (p.k ? p.kv_heads : 0) + (p.v ? p.kv_heads : 0);
    const long walks = (heads + per * p.rounds - 1) / (per * p.rounds);
    const long blocks = (walks * p.tokens + kWarps - 1) / kWarps;
    auto* kernel = lanes == 8 ? kv_rows_kernel<KIND, 8> : lanes == 16 ? kv_rows_kernel<KIND, 16> : kv_rows_kernel<KIND, 32>;
    kernel<<<(unsigned)blocks, kThreads, 0, st>>>(p);
    return cudaGetLastError();
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

FP4B_EXPORT int fp4b_kv_rows(const void* q, long q_st, long q_sh, const void* k, long k_st, long k_sh, const void* v,
                             long v_st, long v_sh, int tokens, int q_heads, int kv_heads, int head_dim,
                             const void* positions, int pos64, const float* rope, int rope_rows, int rot,
                             int interleaved, const void* q_weight, const void* k_weight, float eps, void* q_out,
                             void* k_out, const fp4b_kv_cache* cache, const void* slots, int slot64, void* stream) {
    RowsParams p{};
    p.q = static_cast<const uint16_t*>(q);
    p.k = static_cast<const uint16_t*>(k);
    p.v = static_cast<const uint16_t*>(v);
    p.q_st = q_st, p.q_sh = q_sh, p.k_st = k_st, p.k_sh = k_sh, p.v_st = v_st, p.v_sh = v_sh;
    p.tokens = tokens, p.q_heads = q ? q_heads : 0, p.kv_heads = kv_heads, p.d = head_dim;
    p.positions = positions, p.pos64 = pos64, p.rope = rope, p.rope_rows = rope_rows, p.rot = rot, p.pairs = interleaved;
    p.q_weight = static_cast<const uint16_t*>(q_weight);
    p.k_weight = static_cast<const uint16_t*>(k_weight);
    p.eps = eps;
    p.q_out = static_cast<uint16_t*>(q_out);
    p.k_out = static_cast<uint16_t*>(k_out);
    p.slots = slots, p.slot64 = slot64;
    const char* why = rows_check(p);
    if (!why && !q && !k) why = "neither queries nor keys";
    if (!why && q && (!q_out || !aligned(q_out, 8) || q_heads <= 0)) why = "queries need an 8-byte aligned output";
    if (!why && cache) {
        why = kv_cache_check(cache);
        if (!why && (!k || !v || !slots)) why = "a cache takes keys, values and slots";
        if (!why && (cache->kv_heads != kv_heads || cache->head_dim != head_dim)) why = "the cache has other heads";
    } else if (!why) {
        if (k && (!k_out || !aligned(k_out, 8))) why = "keys need an 8-byte aligned output or a cache";
        if (v) why = "values need a cache";
    }
    if (why) {
        set_last_error("fp4b_kv_rows: %s", why);
        return -1;
    }
    if (tokens == 0) return 0;
    p.rounds = 1;
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
    if (!why && (count < 0 || (count > 0 && (!slots || !k_out || !v_out)))) why = "null slots or outputs";
    if (!why && (!aligned(k_out, 16) || !aligned(v_out, 16))) why = "outputs must be 16-byte aligned";
    if (why) {
        set_last_error("fp4b_kv_read: %s", why);
        return -1;
    }
    if (count == 0) return 0;
    ReadParams p{*cache, shift_of(cache->page_size), slots, slot64, count * cache->kv_heads,
                 static_cast<uint16_t*>(k_out), static_cast<uint16_t*>(v_out), device_error_word()};
    const long threads = p.rows * (cache->head_dim / 8);
    const unsigned blocks = (unsigned)std::min<long>((threads + kThreads - 1) / kThreads, 1l << 30);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (cache->kind == kKvBf16) kv_read_kernel<kKvBf16><<<blocks, kThreads, 0, st>>>(p);
    else if (cache->kind == kKvFp8) kv_read_kernel<kKvFp8><<<blocks, kThreads, 0, st>>>(p);
    else kv_read_kernel<kKvNvfp4><<<blocks, kThreads, 0, st>>>(p);
    return launch_status(cudaGetLastError(), "fp4b_kv_read");
}
