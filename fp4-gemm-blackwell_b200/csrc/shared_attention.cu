// shared_attention.cu -- attention of one new token a sequence where sequences
// share a prefix: the prefix's keys and values are read once for every 128 rows
// (sequence, query head of a key head) instead of once for each sequence.
//
// Two kernels.  The first goes over the prefixes: the query heads of a key head
// of all sequences of a prefix are the rows of one matrix, so that
//   S = Q K^T,  P = exp(S - reference),  O = P V
// are matrix products on tcgen05 with 128 rows.  The second is
// decode_attention's over each sequence's own keys, which joins every output row
// at its end with what the first one found for it.
//
// A CTA, one an SM, takes a share of all tiles of keys (128, or 64 of 256
// elements): unit by unit (prefix, key head, 128 rows), a tile at a time.
//   the first 8 (4)    two slots of 128 threads, a row a thread, take the tiles in
//                      turn: each has scores, sums and an O of its own, so that
//                      neither waits for the other (256 elements: one);
//   4 or 8 feeders     bring K and V in 16 bits and the 128-byte swizzle, half of them
//                      each: bf16 by TMA boxes of whole pages, fp8 and nvfp4 decoded
//                      on the way (two warps each took 74 us where four take 66:
//                      32 sequences, 32768 keys x 8 x 64 of nvfp4, 64 heads);
//   one warp           issues the products: S of the next tiles before O of this.
// O stays in TMEM over a unit; S (128 columns of fp32) is read once, a row's into
// its thread's registers, and its weights go back over it as the A operand of the
// second product.  (Read twice, in loops of 16 or 32 columns with fewer registers
// and more warps: 128 sequences over 65536 keys of bf16 in 337 us, 268 so at that time.)
//
// Formats, the reference exponent (moved when a score passes it by 2^10) and the
// weights' two terms are decode_attention's: bf16 in BF16 (16 bits), fp8 and nvfp4
// in FP16 (22 bits); see there for why.
//
// What the parts of a unit found (two for each CTA that has tiles of it) goes to
// the workspace, with the place and the number of each unit's parts.
//
// O is a sum of the tensor cores' fp32 over a CTA's tiles of a unit. Over 65536 keys of
// bf16 outputs lie 2e-5 of their size nearer to zero than fp32 products of the library,
// as cut sums would (half a step of BF16 is 2e-3 to 4e-3), and one in seventy is rounded
// the other way; their error against 64 bits is the same, 1.653e-3.
//
// Measured on B200, both kernels: 128 sequences over 65536 shared keys x 8 x 64 of bf16
// and up to 2048 own ones, 64 heads, 275 us queued back to back: about 230 of them the
// prefix's, whose exponentials alone take 121 at 16 a cycle an SM (61 % of that pipe
// in use, the tensor pipe 45 %), 45 the own keys' (236 MB). 32 over 32768 of nvfp4
// 66 us: decoding (four warps each) and softmax alike, 5 us of joining. Four prefixes
// of up to 8000 keys of fp8 x 8 x 128 with 16 sequences each 83 us: 64 rows leave half
// of each tile empty, ten tiles a CTA behind loads of queries and joining; 19 of them
// the own keys'. Two sequences over 500 keys 12.5 us: two launches, two chains of waits.
#include <cuda.h>

#include "decode_attention.cuh"

#define FP4B_EXPORT extern "C" __attribute__((visibility("default")))

namespace fp4b {
namespace {

constexpr int kErrPrefixTimeout = 14;
constexpr int kTileRows = 128;
constexpr int kSmemMost = 232448;

struct PrefixParams {
    const uint16_t* q;
    long q_sb, q_sh;
    fp4b_kv_cache cache;
    int page_shift;
    const int* table;
    long table_stride;
    int table_width;
    const int* lens;
    int prefixes, each, group, rows, tiles;  // rows: of a key head of a prefix; tiles of 128 of them
    int part_rows;                           // rows of a part: min(rows, 128)
    float scale2;
    int* err;
    int2* units;
    float2* ml;
    float* acc;
    int runs;           // of a tile's rows that are copied as boxes; 0: row by row
    alignas(64) CUtensorMap k_map, v_map;  // of the pages' rows (bf16)
};

template <int KIND, int D>
struct PrefixCfg {
    static constexpr int TK = D == 256 ? 64 : 128;                                   // keys of a tile
    static constexpr int SLOTS = D == 256 ? 1 : 2;                                   // tiles that are worked on at once
    // Warps for K, and as many for V: decoding takes time, starting boxes does not.
    static constexpr int FEEDERS = KIND == kKvBf16 ? 2 : 4;
    static constexpr int ROW_THREADS = SLOTS * 128, THREADS = ROW_THREADS + 2 * FEEDERS * 32 + 128;
    static constexpr int RB = KIND == kKvBf16 ? 2 * D : KIND == kKvFp8 ? D : D / 2;  // bytes of a row
    static constexpr int SB = KIND == kKvBf16 ? 0 : KIND == kKvFp8 ? 4 : D / 16;     // bytes of its scales
    static constexpr int Q = kTileRows * D * 2;
    static constexpr int PIECE = TK * D * 2;                                         // K or V of a tile in 16 bits
    static constexpr int K_STAGES = KIND == kKvBf16 ? (D == 64 ? 5 : D == 128 ? 3 : 2) : D == 64 ? 3 : KIND == kKvNvfp4 && D == 128 ? 2 : 1;
    static constexpr int V_STAGES = KIND == kKvBf16 ? (D == 64 ? 5 : 2) : D == 64 ? 3 : KIND == kKvFp8 && D == 256 ? 1 : 2;
    // fp8 and nvfp4 come through rings as they lie in the cache, of each producing warp's
    // own: its rows' codes and scales (with V fp8's scales of both).
    static constexpr int ROWS = TK / FEEDERS;
    static constexpr int RAW_K = KIND == kKvBf16 ? 0 : ROWS * (RB + (KIND == kKvFp8 ? 0 : SB));
    static constexpr int RAW_V = KIND == kKvBf16 ? 0 : ROWS * (RB + (KIND == kKvFp8 ? 2 * SB : SB));
    static constexpr int RAWS = KIND == kKvBf16 ? 0 : D == 64 ? 4 : KIND == kKvFp8 ? 2 : 3;
    static constexpr int SCALES = KIND == kKvFp8 ? 3 * TK * 4 : 0;                   // of a stage: key scales, value scales, their logarithms
    static constexpr int BUFFERS = D == 64 ? 3 : 2;                                  // of S in TMEM
    static constexpr int S_COLUMNS = BUFFERS * TK;
    static constexpr int BARS = 2 * K_STAGES + 2 * V_STAGES + 2 * BUFFERS + 5 + 8 * RAWS;
    static constexpr int OFF_K = Q, OFF_V = OFF_K + K_STAGES * PIECE, OFF_RAW_K = OFF_V + V_STAGES * PIECE, OFF_RAW_V = OFF_RAW_K + 4 * RAWS * RAW_K;
    static constexpr int OFF_SCALES = OFF_RAW_V + 4 * RAWS * RAW_V, OFF_BARS = OFF_SCALES + V_STAGES * SCALES;
    static constexpr int OFF_FACTORS = OFF_BARS + BARS * 8, OFF_VARS = OFF_FACTORS + kTileRows * 4;
    static constexpr int SMEM = OFF_VARS + 32;
    static_assert(SMEM <= kSmemMost, "shared memory");
    static_assert(S_COLUMNS + SLOTS * D <= 512, "TMEM");
    static_assert(RAW_K % 16 == 0 && RAW_V % 16 == 0 && OFF_SCALES % 16 == 0 && OFF_BARS % 8 == 0, "alignment");
};

// The tiles of this CTA, unit by unit: every role goes over them by itself.
struct Walk {
    int u, end;         // tiles of all units, in order
    int g, before;      // prefix at hand, tiles before its units
    int unit, kv_head, tile, length, r0, r1;  // rows' tile, tiles of the unit, and those at hand
    int valid;          // keys of the prefix
};

__device__ __forceinline__ int prefix_len(const PrefixParams& p, int g) {
    const int most = p.table_width << p.page_shift, n = p.lens[g];
    return n < 0 ? 0 : min(n, most);
}

template <int TK>
__device__ __forceinline__ bool next_unit(const PrefixParams& p, Walk& w) {
    if (w.u >= w.end) return false;
    const int units = p.cache.kv_heads * p.tiles;
    for (;;) {
        w.valid = prefix_len(p, w.g);
        w.length = (w.valid + TK - 1) / TK;
        if (w.u < w.before + w.length * units) break;
        w.before += w.length * units;
        ++w.g;
    }
    const int at = w.u - w.before, local = at / w.length;
    w.unit = w.g * units + local;
    w.kv_head = local / p.tiles;
    w.tile = local - w.kv_head * p.tiles;
    w.r0 = at - local * w.length;
    w.r1 = min(w.length, w.r0 + w.end - w.u);
    w.u += w.r1 - w.r0;
    return true;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

template <int KIND, int D>
__global__ void __launch_bounds__(PrefixCfg<KIND, D>::THREADS, 1) prefix_attention_kernel(const __grid_constant__ PrefixParams p) {
    using C = PrefixCfg<KIND, D>;
    constexpr int TK = C::TK, SLOTS = C::SLOTS, RB = C::RB, SB = C::SB;
    constexpr bool kBf16 = KIND == kKvBf16;
    extern __shared__ __align__(1024) uint8_t tiles_smem[];
    uint8_t* const smem = tiles_smem;
    // (no other shared memory: the swizzle wants this at a multiple of 1024)
    float* const s_factor = reinterpret_cast<float*>(smem + C::OFF_FACTORS);
    int* const vars = reinterpret_cast<int*>(smem + C::OFF_VARS);
    uint32_t& s_tmem = reinterpret_cast<uint32_t&>(vars[0]);
    int &s_abort = vars[1], &s_total = vars[2], &s_g = vars[3], &s_before = vars[4];
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BARS);
    uint64_t *const k_full = bars, *const k_empty = k_full + C::K_STAGES, *const v_full = k_empty + C::K_STAGES, *const v_empty = v_full + C::V_STAGES;
    uint64_t *const s_full = v_empty + C::V_STAGES, *const p_full = s_full + C::BUFFERS, *const q_full = p_full + C::BUFFERS, *const o_done = q_full + 1;
    uint64_t *const unit_done = q_full + 3, *const drained = q_full + 4, *const raw_full = q_full + 5;  // (o_done: of each slot)

    chain();
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    constexpr int kProducerWarp = SLOTS * 4, kMmaWarp = kProducerWarp + 2 * C::FEEDERS;

    // ---- set up: barriers, TMEM, this CTA's share
    if (tid == 0) {
        s_abort = 0;
        for (int i = 0; i < C::K_STAGES; ++i) ptx::mbar_init(k_full + i, 32 * C::FEEDERS), ptx::mbar_init(k_empty + i, 1);
        for (int i = 0; i < C::V_STAGES; ++i) ptx::mbar_init(v_full + i, 32 * C::FEEDERS), ptx::mbar_init(v_empty + i, 1);
        for (int i = 0; i < C::BUFFERS; ++i) ptx::mbar_init(s_full + i, 1), ptx::mbar_init(p_full + i, 128);
        ptx::mbar_init(q_full, C::ROW_THREADS), ptx::mbar_init(o_done, 1), ptx::mbar_init(o_done + 1, 1), ptx::mbar_init(unit_done, 1), ptx::mbar_init(drained, 1);
        for (int i = 0; i < 8 * C::RAWS; ++i) ptx::mbar_init(raw_full + i, 1);
        ptx::fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        ptx::tmem_alloc(&s_tmem, 512);
        ptx::tmem_relinquish();
    }
    const int units = p.cache.kv_heads * p.tiles;
    if (warp == 0) {
        int total = 0;
        for (int base = 0; base < p.prefixes; base += 32) {
            const int g = base + lane, n = g < p.prefixes ? p.lens[g] : 0;
            if (n < 0 || n > p.table_width << p.page_shift) report(p.err, kErrPageRange);
            const int length = g < p.prefixes ? (prefix_len(p, g) + TK - 1) / TK : 0;
            total += __reduce_add_sync(0xffffffffu, length) * units;
            // prefixes without keys: their units have no parts
            if (g < p.prefixes && length == 0 && blockIdx.x == 0)
                for (int i = 0; i < units; ++i) p.units[(size_t)g * units + i] = make_int2(0, 0);
        }
        if (lane == 0) s_total = total;
    }
    __syncthreads();
    const int total = s_total, ctas = min((int)gridDim.x, total);
    const bool working = (int)blockIdx.x < ctas;
    const int share = working ? total / ctas : 0, extra = total - share * ctas;
    Walk walk{};
    if (working) {
        walk.u = (int)blockIdx.x * share + min((int)blockIdx.x, extra);
        walk.end = walk.u + share + ((int)blockIdx.x < extra ? 1 : 0);
        if (warp == 0) {  // the prefix in which it begins
            int sum = 0;
            for (int base = 0; base < p.prefixes; base += 32) {
                const int g = base + lane, mine = g < p.prefixes ? (prefix_len(p, g) + TK - 1) / TK * units : 0;
                int upto = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int other = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += other;
                }
                if (sum + upto - mine <= walk.u && walk.u < sum + upto) s_g = g, s_before = sum + upto - mine;
                sum += __shfl_sync(0xffffffffu, upto, 31);
                if (sum > walk.u) break;
            }
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = s_tmem;
    walk.g = s_g, walk.before = s_before;
    auto owner = [&](int x) {
        const int cut = extra * (share + 1);
        return x < cut ? x / (share + 1) : extra + (x - cut) / share;
    };
    // A bounded wait of a whole warp; false when it gave up or another role did.
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        bool ok;
        uint64_t t0 = 0;
        for (uint32_t i = 1; !(ok = ptx::mbar_try_wait(bar, parity)); ++i) {
            if ((i & 63u) == 0) {  // (the timer is slow to read)
                if (*(volatile int*)&s_abort) break;
                const uint64_t t = ptx::global_timer_ns();
                if (t0 == 0) {
                    t0 = t;
                } else if (t - t0 > ptx::kSpinLimitNs) {
                    *(volatile int*)&s_abort = 1;
                    report(p.err, kErrPrefixTimeout);
                    break;
                }
            }
        }
        return (bool)__all_sync(0xffffffffu, ok);
    };

    // Rows take more registers than a block has for each thread, the others fewer:
    // 256 x 184 + 256 x 72 = 512 x 128, 256 x 168 + 384 x 48 = 640 x 96.
    if constexpr (SLOTS == 2) {
        constexpr int kMore = kBf16 ? 184 : 168, kFewer = kBf16 ? 72 : 48;
        static_assert(256 * kMore + (C::THREADS - 256) * kFewer == C::THREADS * (65536 / C::THREADS / 8 * 8), "registers");
        if (warp < kProducerWarp) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMore));
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewer));
    }

    if (working && warp < kProducerWarp) {
        // ------------------------------------------------------------ a row a thread: queries, softmax, results
        // Where a wait gives up the tiles are gone through without waiting: every barrier is met.
        const int mine = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);  // this warp's 32 lanes
        const uint32_t o_at = lanes + C::S_COLUMNS + mine * D;
        int it = 0, segment = 0;
        bool ok = true;
        while (next_unit<TK>(p, walk)) {
            const int rows = min(kTileRows, p.rows - walk.tile * kTileRows);
            const bool live = (warp & 3) * 32 < rows;
            {
                // ---- Q in 16 bits and swizzled, 8 elements a lane; rows that there are not as zeros
                constexpr int LANES = D / 8, AT_ONCE = C::ROW_THREADS / LANES, PASSES = kTileRows / AT_ONCE;
                const int c = tid % LANES;
                const uint32_t sign = p.scale2 < 0.0f ? 0x80008000u : 0u;  // goes to the queries
#pragma unroll 4
                for (int i = 0; i < PASSES; ++i) {
                    const int r = i * AT_ONCE + tid / LANES, all = walk.tile * kTileRows + r, of = all / p.group;
                    uint2 a = make_uint2(0u, 0u), b = a;
                    if (r < rows) {
                        const uint16_t* from = p.q + (size_t)(walk.g * p.each + of) * p.q_sb + (size_t)(walk.kv_head * p.group + all - of * p.group) * p.q_sh + 8 * c;
                        a = *reinterpret_cast<const uint2*>(from), b = *reinterpret_cast<const uint2*>(from + 4);
                    }
                    float factor = fabsf(p.scale2);
                    if constexpr (!kBf16) {
                        auto largest = [](uint32_t w) { return max((w & 0x7FFFu) << 16, w & 0x7FFF0000u); };
                        const uint32_t top = group_umax<LANES>(max(max(largest(a.x), largest(a.y)), max(largest(b.x), largest(b.y))));
                        const int k = min(max(141 - (int)(top >> 23), -126), 126);
                        const float up = __int_as_float((127 + k) << 23);
                        factor *= __int_as_float((127 - k) << 23);
                        if (KIND == kKvNvfp4) factor *= kScaleUnit;
                        auto half16 = [&](uint32_t w) { return pack_f16(bf16_lo(w) * up, bf16_hi(w) * up); };
                        a = make_uint2(half16(a.x), half16(a.y)), b = make_uint2(half16(b.x), half16(b.y));
                    }
                    if (c == 0) s_factor[r] = fmaxf(factor, 0x1p-126f);  // (masked keys' -inf stays one where scale is 0)
                    const int to = (c >> 3) * (kTileRows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                    *reinterpret_cast<uint4*>(smem + to) = make_uint4(a.x ^ sign, a.y ^ sign, b.x ^ sign, b.y ^ sign);
                }
                ptx::fence_proxy_async_smem();
            }
            ptx::mbar_arrive(q_full);
            ok = ok && wait(q_full, segment & 1);
            const float f = s_factor[row];
            float ref = kNoScore, l = 0.0f;
            bool begun = false;
            for (int j = walk.r0; j < walk.r1; ++j, ++it) {
                if (SLOTS == 2 && (it & 1) != mine) continue;
                const int buf = it % C::BUFFERS, stage = it % C::V_STAGES;
                ok = ok && wait(s_full + buf, (it / C::BUFFERS) & 1);
                if (KIND == kKvFp8) ok = ok && wait(v_full + stage, (it / C::V_STAGES) & 1);
                ptx::tc_fence_after();
                const uint32_t s_at = lanes + buf * TK;
                const float4* const scales = reinterpret_cast<const float4*>(smem + C::OFF_SCALES + stage * C::SCALES);
                const int seen = walk.valid - j * TK;  // keys of the tile that there are
                if (live) {
                    float s[TK];
#pragma unroll
                    for (int c = 0; c < TK / 32; ++c) ptx::tmem_ld_32x32b_x32(s_at + 32 * c, reinterpret_cast<uint32_t(&)[32]>(s[32 * c]));
                    ptx::tmem_ld_wait();
                    if constexpr (KIND == kKvFp8) {
#pragma unroll
                        for (int i = 0; i < TK; i += 4) {
                            const float4 ks = scales[i / 4];
                            s[i] *= ks.x, s[i + 1] *= ks.y, s[i + 2] *= ks.z, s[i + 3] *= ks.w;
                        }
                    }
                    if (seen < TK) {
#pragma unroll
                        for (int i = 0; i < TK; ++i)
                            if (i >= seen) s[i] = -INFINITY;
                    }
                    // ---- the largest score, in base 2 (for fp8 with the value scale's share); f is not negative
                    float top = -INFINITY, other = -INFINITY;
                    const unsigned long long ff = pair_of(f, f);
                    if constexpr (KIND == kKvFp8) {
#pragma unroll
                        for (int i = 0; i < TK; i += 4) {
                            const float4 lv = scales[TK / 2 + i / 4];
                            const unsigned long long a = fma2(pair_of(s[i], s[i + 1]), ff, pair_of(lv.x, lv.y)), b = fma2(pair_of(s[i + 2], s[i + 3]), ff, pair_of(lv.z, lv.w));
                            top = max3(top, first_of(a), second_of(a));
                            other = max3(other, first_of(b), second_of(b));
                        }
                        top = fmaxf(top, other);
                    } else {
#pragma unroll
                        for (int i = 0; i < TK; i += 4) top = max3(top, s[i], s[i + 1]), other = max3(other, s[i + 2], s[i + 3]);
                        top = fmaxf(top, other) * f;
                    }
                    // ---- the reference moves when a score of the warp's passes it by too much
                    if (__any_sync(0xffffffffu, top > ref + kHeadroom)) {
                        const float to = fmaxf(ref, top - kBelowMax), c = exp2_approx(ref - to);
                        ref = to;
                        l *= c;
                        if (begun) {
                            ok = ok && wait(o_done + mine, (it / SLOTS - 1) & 1);  // the slot's last product
                            ptx::tc_fence_after();
#pragma unroll 1
                            for (int d = 0; d < D; d += 32) {
                                uint32_t o[32];
                                ptx::tmem_ld_32x32b_x32(o_at + d, o);
                                ptx::tmem_ld_wait();
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * c);
                                ptx::tmem_st_32x32b_x32(o_at + d, o);
                            }
                        }
                    }
                    // ---- weights: 32 scores to 16 columns of their rounding and 16 of what that left
                    const unsigned long long rr = pair_of(-ref, -ref), less = pair_of(-1.0f, -1.0f);
                    unsigned long long sum[2] = {pair_of(0.0f, 0.0f), pair_of(0.0f, 0.0f)};
#pragma unroll
                    for (int c = 0; c < TK / 32; ++c) {
                        uint32_t w[32];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const int k = 32 * c + i;
                            const unsigned long long x = fma2(pair_of(s[k], s[k + 1]), ff, rr);
                            unsigned long long e = pair_of(exp2_approx(first_of(x)), exp2_approx(second_of(x)));
                            sum[i / 2 % 2] = add2(sum[i / 2 % 2], e);
                            if constexpr (KIND == kKvFp8) {
                                const float4 vs = scales[TK / 4 + k / 4];
                                e = mul2(e, i & 2 ? pair_of(vs.z, vs.w) : pair_of(vs.x, vs.y));
                            }
                            if constexpr (kBf16) {
                                w[i / 2] = pack_bf16(first_of(e), second_of(e));
                                e = fma2(pair_of(bf16_lo(w[i / 2]), bf16_hi(w[i / 2])), less, e);
                                w[16 + i / 2] = pack_bf16(first_of(e), second_of(e));
                            } else {
                                w[i / 2] = pack_f16(first_of(e), second_of(e));
                                const float2 back = f16x2_to_float2(w[i / 2]);
                                e = fma2(pair_of(back.x, back.y), less, e);
                                w[16 + i / 2] = pack_f16(first_of(e), second_of(e));
                            }
                        }
                        ptx::tmem_st_32x32b_x32(s_at + 32 * c, w);
                    }
                    sum[0] = add2(sum[0], sum[1]);
                    l += first_of(sum[0]) + second_of(sum[0]);
                    ptx::tmem_st_wait();
                }
                begun = true;
                ptx::tc_fence_before();
                ptx::mbar_arrive(p_full + buf);
            }
            // ---- the unit's part: (reference, sum) and O
            ok = ok && wait(unit_done, segment & 1);
            ptx::tc_fence_after();
            const int first = owner(walk.u - walk.r1), count = owner(walk.u - walk.r1 + walk.length - 1) - first + 1;
            const size_t part = ((size_t)walk.unit + blockIdx.x) * SLOTS + mine;
            if (walk.r0 == 0 && tid == 0) p.units[walk.unit] = make_int2((walk.unit + first) * SLOTS, count * SLOTS);
            if (live) {
                const size_t to = part * p.part_rows + row;
                if (row < rows) p.ml[to] = make_float2(ref, l);
                if (begun)
#pragma unroll 1
                    for (int d = 0; d < D; d += 32) {
                        uint32_t o[32];
                        ptx::tmem_ld_32x32b_x32(o_at + d, o);
                        ptx::tmem_ld_wait();
                        if (row < rows)
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                *reinterpret_cast<uint4*>(p.acc + to * D + d + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
            }
            ++segment;
        }
    } else if (working && warp < kMmaWarp) {
        // ------------------------------------------------------------ pages to K and V in shared memory
        // Each warp has its share of a tile's rows.
        const bool value = warp >= kProducerWarp + C::FEEDERS;
        const int my = (warp - kProducerWarp) % C::FEEDERS, stages = value ? C::V_STAGES : C::K_STAGES;
        constexpr int ROWS = C::ROWS;
        constexpr int LR = RB / 16, PER = 32 / LR;  // lanes a row, rows an instruction
        const int sub = lane / LR, c = lane % LR;
        uint64_t *const full = value ? v_full : k_full, *const empty = value ? v_empty : k_empty;
        uint8_t* const pieces = smem + (value ? C::OFF_V : C::OFF_K);
        const uint8_t* const from = static_cast<const uint8_t*>(value ? p.cache.v : p.cache.k);
        bool ok = true;
        int stage = 0;
        uint32_t round = 0;  // of the stages, its low bit the barriers' phase
        auto row_of = [&](int page, int key) {  // in the cache; -1: none to read
            if (page >= 0 && page < p.cache.num_pages)
                return (page * p.cache.kv_heads + walk.kv_head) * p.cache.page_size + (key & (p.cache.page_size - 1));
            if (page != -2) report(p.err, kErrPageRange);
            return -1;
        };
        if constexpr (kBf16) {
            // Whole tiles of whole pages come as boxes that TMA swizzles; others row by row,
            // each of which is handed on when the next one's copies are under way.
            int pending = -1;
            ptx::Flights flights;
            auto hand_on = [&]() {
                ptx::fence_proxy_async_smem();
                ptx::mbar_arrive(full + pending);
                pending = -1;
            };
            const int run = p.runs > 0 ? TK / p.runs : TK;
            while (ok && next_unit<TK>(p, walk)) {
                const int* const table = p.table + (size_t)walk.g * p.table_stride;
                // the table's entry of this lane's run of a tile, on its way a tile ahead
                auto look = [&](int j) {
                    const int key = j * TK + lane * run;
                    return lane < p.runs && j < walk.r1 && key < walk.valid ? table[key >> p.page_shift] : 0;
                };
                int next = look(walk.r0);
                for (int j = walk.r0; j < walk.r1; ++j, stage = stage + 1 == stages ? (++round, 0) : stage + 1) {
                    const int key0 = j * TK, entry = next;
                    next = look(j + 1);
                    uint8_t* const to = pieces + stage * C::PIECE;
                    bool boxes = p.runs > 0 && walk.valid - key0 >= TK;
                    int first = -1;  // row of this lane's run
                    if (boxes) {
                        if (lane < p.runs) first = row_of(max(entry, -1), key0 + lane * run);
                        boxes = __all_sync(0xffffffffu, lane >= p.runs || first >= 0);
                    }
                    if (round > 0 && !wait(empty + stage, (round & 1) ^ 1)) {
                        ok = false;
                        break;
                    }
                    if (boxes) {
                        if (my == 0) {  // one warp's alone
                            flights.begin(full, stage, round, C::PIECE, 32 * C::FEEDERS, lane);
                            if (lane < p.runs)
#pragma unroll
                                for (int n = 0; n < D / 64; ++n)
                                    ptx::tma_load_2d(to + n * (TK * 128) + lane * run * 128, value ? &p.v_map : &p.k_map, full + stage, 128 * n, first);
                        }
                    } else {
#pragma unroll 1
                        for (int r0 = my * ROWS; r0 < (my + 1) * ROWS; r0 += min(ROWS, 32)) {
                            const int key = key0 + r0 + lane;
                            const int mine = row_of(lane < ROWS && key < walk.valid ? max(table[key >> p.page_shift], -1) : -2, key);
#pragma unroll 4
                            for (int i = 0; i < min(ROWS, 32) / PER; ++i) {
                                const int r = i * PER + sub, at = __shfl_sync(0xffffffffu, mine, r), tr = r0 + r;
                                copy_async<16>(ptx::smem_u32(to + (c >> 3) * (TK * 128) + tr * 128 + (((c & 7) ^ (tr & 7)) << 4)), from + (size_t)max(at, 0) * RB + 16 * c, at >= 0);
                            }
                        }
                        copy_commit();
                        if (pending >= 0) {
                            copy_wait<1>();
                            hand_on();
                        }
                        pending = stage;
                        if (p.runs > 0) {  // one among boxes
                            copy_wait<0>();
                            hand_on();
                        }
                    }
                }
            }
            copy_wait<0>();
            if (ok && pending >= 0) hand_on();
            if (!ok) flights.land(full, stages);  // (what is under way has to end before shared memory goes)
        } else {
            // Through a ring of the warp's own: bulk copies of whole pages' runs, or row by row
            // where they are not whole.
            constexpr int COPIES = ROWS / PER, AHEAD = C::RAWS - 1;
            constexpr int GROUP = COPIES < 4 ? COPIES : 4;  // decoded at once
            const int raw_bytes = value ? C::RAW_V : C::RAW_K, run = min(p.cache.page_size, ROWS);
            uint8_t* const raw = smem + (value ? C::OFF_RAW_V : C::OFF_RAW_K) + my * C::RAWS * raw_bytes;
            uint64_t* const arrived = raw_full + (warp - kProducerWarp) * C::RAWS;
            const uint8_t* const scales = static_cast<const uint8_t*>(value ? p.cache.v_scale : p.cache.k_scale);
            // `walk` is at the tile whose copies start, `here` at the one that is decoded
            Walk here = walk;
            bool more = next_unit<TK>(p, walk), there = false;
            int tile = walk.r0, slot = 0, entry = 0;
            uint32_t bulk = 0, parity = 0;  // of the slots: whether bulk copies are under way, their phases
            auto look = [&]() {  // the table's entry of this lane's key, on its way (nothing here may wait for it)
                const int key = tile * TK + my * ROWS + lane;
                there = lane < ROWS && key < walk.valid;
                if (there) entry = p.table[(size_t)walk.g * p.table_stride + (key >> p.page_shift)];
            };
            if (more) look();
            auto issue = [&]() {
                if (more) {
                    const int row = row_of(there ? max(entry, -1) : -2, tile * TK + my * ROWS + lane);
                    uint8_t* const to = raw + slot * raw_bytes;
                    if (run >= 8 && __all_sync(0xffffffffu, lane >= ROWS || row >= 0)) {
                        bulk |= 1u << slot;
                        if (lane == 0) ptx::mbar_arrive_expect_tx(arrived + slot, raw_bytes);
                        __syncwarp();
                        if (lane < ROWS && (lane & (run - 1)) == 0) {
                            ptx::bulk_load(to + lane * RB, from + (size_t)row * RB, run * RB, arrived + slot);
                            if (KIND != kKvFp8 || value) ptx::bulk_load(to + ROWS * RB + lane * SB, scales + (size_t)row * SB, run * SB, arrived + slot);
                            if (KIND == kKvFp8 && value)
                                ptx::bulk_load(to + ROWS * (RB + SB) + lane * SB, static_cast<const uint8_t*>(p.cache.k_scale) + (size_t)row * SB, run * SB, arrived + slot);
                        }
                    } else {
                        const uint32_t at_smem = ptx::smem_u32(to);
#pragma unroll
                        for (int i = 0; i < COPIES; ++i) {
                            const int at = __shfl_sync(0xffffffffu, row, i * PER + sub);
                            copy_async<16>(at_smem + (i * 32 + lane) * 16, from + (size_t)max(at, 0) * RB + 16 * c, at >= 0);
                        }
                        if (lane < ROWS) {
                            if (KIND != kKvFp8 || value) copy_async<SB>(at_smem + ROWS * RB + lane * SB, scales + (size_t)max(row, 0) * SB, row >= 0);
                            if (KIND == kKvFp8 && value)
                                copy_async<SB>(at_smem + ROWS * (RB + SB) + lane * SB, static_cast<const uint8_t*>(p.cache.k_scale) + (size_t)max(row, 0) * SB, row >= 0);
                        }
                    }
                    if (++slot == C::RAWS) slot = 0;
                    if (++tile == walk.r1) {
                        more = next_unit<TK>(p, walk);
                        tile = walk.r0;
                    }
                    if (more) look();
                }
                copy_commit();
            };
            for (int i = 0; i < AHEAD; ++i) issue();
            int at_slot = 0;
            while (ok && next_unit<TK>(p, here)) {
                for (int j = here.r0; j < here.r1; ++j, stage = stage + 1 == stages ? (++round, 0) : stage + 1) {
                    issue();
                    copy_wait<AHEAD>();
                    __syncwarp();  // the other lanes' copies
                    if (bulk >> at_slot & 1) {
                        ok = wait(arrived + at_slot, parity >> at_slot & 1);
                        if (!ok) break;
                        parity ^= 1u << at_slot, bulk &= ~(1u << at_slot);
                    }
                    if (round > 0) ok = wait(empty + stage, (round & 1) ^ 1);
                    if (!ok) break;
                    uint8_t* const to = pieces + stage * C::PIECE;
                    const uint8_t* const in = raw + at_slot * raw_bytes;
#pragma unroll
                    for (int i0 = 0; i0 < COPIES; i0 += GROUP) {
                        uint4 w[GROUP];
                        uint32_t sc[GROUP];
#pragma unroll
                        for (int i = 0; i < GROUP; ++i) {
                            w[i] = lds128(in + ((i0 + i) * 32 + lane) * 16);
                            if constexpr (KIND == kKvNvfp4) sc[i] = *reinterpret_cast<const uint16_t*>(in + ROWS * RB + ((i0 + i) * PER + sub) * SB + 2 * c);
                        }
#pragma unroll
                        for (int i = 0; i < GROUP; ++i) {
                            const int r = my * ROWS + (i0 + i) * PER + sub, e = (KIND == kKvFp8 ? 16 : 32) * c;
                            uint8_t* const line = to + (e >> 6) * (TK * 128) + r * 128;
                            const uint32_t words[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                            auto put = [&](int n, uint4 v) { *reinterpret_cast<uint4*>(line + (((((e & 63) >> 3) + n) ^ (r & 7)) << 4)) = v; };
                            if constexpr (KIND == kKvFp8) {
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    uint32_t a[2], b[2];
                                    e4m3x4_to_f16(words[2 * h], a);
                                    e4m3x4_to_f16(words[2 * h + 1], b);
                                    put(h, make_uint4(a[0], a[1], b[0], b[1]));
                                }
                            } else {
#pragma unroll
                                for (int h = 0; h < 4; ++h) {
                                    const uint32_t scale = ue4m3x2_to_f16((h < 2 ? sc[i] & 0xFFu : sc[i] >> 8) * 0x10001u);
                                    uint32_t a[4];
                                    e2m1x8_to_f16(words[h], a);
                                    put(h, make_uint4(mul_f16x2(a[0], scale), mul_f16x2(a[1], scale), mul_f16x2(a[2], scale), mul_f16x2(a[3], scale)));
                                }
                            }
                        }
                    }
                    if constexpr (KIND == kKvFp8) {
                        // (with V: the softmax that reads them ends before V's stage is free again)
                        if (value && lane < ROWS) {
                            float* const s = reinterpret_cast<float*>(smem + C::OFF_SCALES + stage * C::SCALES) + my * ROWS + lane;
                            const float scale = *reinterpret_cast<const float*>(in + ROWS * RB + lane * SB);
                            s[0] = *reinterpret_cast<const float*>(in + ROWS * (RB + SB) + lane * SB);
                            s[TK] = scale, s[2 * TK] = fmaxf(log2_approx(scale), -80.0f);
                        }
                    }
                    if (++at_slot == C::RAWS) at_slot = 0;
                    ptx::fence_proxy_async_smem();
                    ptx::mbar_arrive(full + stage);
                    __syncwarp();  // (the slot may be copied over)
                }
            }
            copy_wait<0>();
            for (int i = 0; i < C::RAWS; ++i)  // (none are after the last tile)
                if (bulk >> i & 1) ptx::mbar_wait(arrived + i, parity >> i & 1);
        }
    } else if (working && warp == kMmaWarp) {
        // ------------------------------------------------------------ the products
        constexpr uint32_t s_desc = ptx::idesc_f16(kBf16, false, TK), o_desc = ptx::idesc_f16(kBf16, true, D);
        const uint64_t q_at = ptx::desc_kmajor_sw128(ptx::smem_u32(smem));
        const uint64_t k_at = ptx::desc_kmajor_sw128(ptx::smem_u32(smem + C::OFF_K));
        const uint64_t v_at = ptx::desc_mnmajor_sw128(ptx::smem_u32(smem + C::OFF_V), TK * 128);
        int it = 0, segment = 0;
        bool ok = true;
        auto scores = [&](int t) {  // S of tile t
            const int stage = t % C::K_STAGES;
            ok = wait(k_full + stage, (t / C::K_STAGES) & 1);
            if (!ok) return;
            ptx::tc_fence_after();
            if (ptx::elect_one()) {
                const uint64_t k = k_at + (uint64_t)((stage * C::PIECE) >> 4);
#pragma unroll
                for (int j = 0; j < D / 16; ++j)
                    ptx::tc_mma_f16(tmem + t % C::BUFFERS * TK, q_at + (uint64_t)(((j >> 2) * kTileRows * 128 + (j & 3) * 32) >> 4),
                                    k + (uint64_t)(((j >> 2) * TK * 128 + (j & 3) * 32) >> 4), s_desc, j > 0);
                ptx::tc_commit(k_empty + stage);
                ptx::tc_commit(s_full + t % C::BUFFERS);
            }
            __syncwarp();
        };
        while (ok && next_unit<TK>(p, walk)) {
            const int n = walk.r1 - walk.r0;
            ok = wait(q_full, segment & 1);
            constexpr int kAhead = C::BUFFERS - 1;  // tiles whose scores come before this one's O
            for (int j = 0; ok && j < min(kAhead, n); ++j) scores(it + j);
            for (int j = 0; ok && j < n; ++j, ++it) {
                if (j + kAhead < n) {
                    // S goes over the weights of tile it - 1, and products of other shapes and results are not bound
                    // to the order in which they were issued: the one that reads the weights has to have ended.  (It
                    // costs 128 sequences over 65536 keys of bf16 about 4 %, 264 to 275 us, the others nothing.)
                    if (j > 0) ok = wait(o_done + (SLOTS == 2 ? (it - 1) & 1 : 0), ((it - 1) / SLOTS) & 1);
                    if (ok) scores(it + kAhead);
                }
                if (!ok) break;
                const int stage = it % C::V_STAGES, buf = it % C::BUFFERS, mine = SLOTS == 2 ? it & 1 : 0;
                ok = wait(p_full + buf, (it / C::BUFFERS) & 1) && wait(v_full + stage, (it / C::V_STAGES) & 1);
                if (!ok) break;
                ptx::tc_fence_after();
                if (ptx::elect_one()) {
                    const uint32_t o = tmem + C::S_COLUMNS + mine * D, w = tmem + buf * TK;
                    const uint64_t v = v_at + (uint64_t)((stage * C::PIECE) >> 4);
#pragma unroll
                    for (int k = 0; k < TK / 16; ++k)
#pragma unroll
                        for (int term = 0; term < 2; ++term)
                            ptx::tc_mma_f16_ts(o, w + 32 * (k >> 1) + 16 * term + 8 * (k & 1), v + (uint64_t)((k * 2048) >> 4), o_desc,
                                               j >= SLOTS || k > 0 || term > 0);
                    ptx::tc_commit(v_empty + stage);
                    ptx::tc_commit(o_done + mine);
                    if (j + 1 == n) ptx::tc_commit(unit_done);
                }
                __syncwarp();
            }
            ++segment;
        }
        if (!ok) {
            // what was issued has to end before TMEM and shared memory go
            if (ptx::elect_one()) ptx::tc_commit(drained);
            __syncwarp();
            ptx::mbar_wait(drained, 0);
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    if (warp == kMmaWarp) ptx::tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------- host side

struct SharedLayout {
    long units, ml, acc, bytes;
};
SharedLayout shared_layout(long own, int sms, int prefixes, int batch, int group, int kv_heads, int d) {
    SharedLayout w;
    const long rows = (long)(batch / prefixes) * group, tiles = (rows + kTileRows - 1) / kTileRows, units = prefixes * kv_heads * tiles;
    const long parts = (units + sms) * (d == 256 ? 1 : 2) * std::min<long>(rows, kTileRows);
    w.units = (own + 15) / 16 * 16;
    w.ml = w.units + (units * 8 + 15) / 16 * 16;
    w.acc = w.ml + (parts * 8 + 15) / 16 * 16;
    w.bytes = w.acc + parts * d * 4;
    return w;
}

template <int KIND, int D>
cudaError_t launch_prefix(PrefixParams& p, int sms, cudaStream_t st) {
    using C = PrefixCfg<KIND, D>;
    // Boxes of the tile's rows in one page, 8 rows (a swizzle's pattern) at least.
    p.runs = 0;
    if (KIND == kKvBf16 && p.cache.page_size >= 8) {
        const int box = std::min(p.cache.page_size, C::TK);
        const long rows = (long)p.cache.num_pages * p.cache.kv_heads * p.cache.page_size;
        if (!make_byte_map(&p.k_map, p.cache.k, rows, 2 * D, box) || !make_byte_map(&p.v_map, p.cache.v, rows, 2 * D, box)) return cudaErrorInvalidValue;
        p.runs = C::TK / box;
    }
    static std::mutex mu;
    static bool ready[kMaxDevices];
    auto* kernel = prefix_attention_kernel<KIND, D>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (!ready[dev]) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
            if (e != cudaSuccess) return e;
            ready[dev] = true;
        }
    }
    const long keys = (long)p.table_width << p.page_shift;
    const long most = (long)p.prefixes * p.cache.kv_heads * p.tiles * ((keys + C::TK - 1) / C::TK);
    return launch_chained(kernel, dim3((unsigned)std::max<long>(1, std::min<long>(sms, most))), C::THREADS, C::SMEM, st, p);
}

template <int KIND>
cudaError_t launch_both(PrefixParams& x, AttentionParams& p, uint8_t* workspace, int sms, cudaStream_t st) {
    const cudaError_t e = p.cache.head_dim == 64    ? launch_prefix<KIND, 64>(x, sms, st)
                          : p.cache.head_dim == 128 ? launch_prefix<KIND, 128>(x, sms, st)
                                                    : launch_prefix<KIND, 256>(x, sms, st);
    return e != cudaSuccess ? e : launch_dim<KIND, true>(p, workspace, st);
}

}  // namespace
}  // namespace fp4b

using namespace fp4b;

FP4B_EXPORT long fp4b_shared_attention_workspace(int prefixes, int batch, int q_heads, int kv_heads, int head_dim) {
    const long own = fp4b_decode_attention_workspace(q_heads, kv_heads, head_dim);
    if (own < 0) return own;
    if (prefixes <= 0 || batch < 0 || batch % prefixes) {
        set_last_error("fp4b_shared_attention_workspace: the batch must be a multiple of the prefixes");
        return -1;
    }
    return shared_layout(own, device_sm_count(), prefixes, batch, q_heads / kv_heads, kv_heads, head_dim).bytes;
}

FP4B_EXPORT int fp4b_shared_attention(const fp4b_shared* call, void* stream) {
    if (!call) {
        set_last_error("fp4b_shared_attention: null arguments");
        return -1;
    }
    const fp4b_shared& s = *call;
    const fp4b_decode& c = s.own;
    const fp4b_kv_cache* cache = c.cache;
    const bool sizes = c.batch > 0 && cache && cache->kv_heads > 0 && s.prefixes > 0;
    const long need = sizes ? fp4b_shared_attention_workspace(s.prefixes, c.batch, c.q_heads, cache->kv_heads, cache->head_dim) : 0;
    const char* why = decode_check(c, need);
    if (!why && c.window != 0) why = "a window does not go with prefixes";
    if (!why && (s.prefixes <= 0 || c.batch % s.prefixes)) why = "the batch must be a multiple of the prefixes";
    if (!why && c.batch > 0 && (!s.prefix_lens || (s.prefix_width > 0 && !s.prefix_table))) why = "null tensor";
    if (!why && (s.prefix_width < 0 || s.prefix_stride < s.prefix_width)) why = "bad page table";
    if (!why && (long)s.prefix_width * cache->page_size > 0x7fff0000L) why = "more than 2^31 keys in one prefix";
    const long rows = why || c.batch == 0 ? 0 : (long)(c.batch / s.prefixes) * (c.q_heads / cache->kv_heads), tiles = (rows + kTileRows - 1) / kTileRows;
    if (!why && rows && (((long)s.prefix_width * cache->page_size + 63) / 64 + 1) * s.prefixes > 0x7fffffffL / (cache->kv_heads * tiles))
        why = "more than 2^31 tiles of 64 keys in one call";
    if (!why && need < 0) why = "no device, or one beyond those that the library knows";
    if (why) {
        set_last_error("fp4b_shared_attention: %s", why);
        return -1;
    }
    if (c.batch == 0) return 0;
    const int sms = device_sm_count(), d = cache->head_dim;
    AttentionParams p = params_of(c);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint8_t* ws = static_cast<uint8_t*>(c.workspace);
    const SharedLayout w = shared_layout(fp4b_decode_attention_workspace(c.q_heads, cache->kv_heads, d), sms, s.prefixes, c.batch, p.group, cache->kv_heads, d);
    PrefixParams x{};
    x.q = p.q, x.q_sb = p.q_sb, x.q_sh = p.q_sh, x.cache = p.cache, x.page_shift = p.page_shift;
    x.table = s.prefix_table, x.table_stride = s.prefix_stride, x.table_width = s.prefix_width, x.lens = s.prefix_lens;
    x.prefixes = s.prefixes, x.each = c.batch / s.prefixes, x.group = p.group, x.rows = (int)rows, x.tiles = (int)tiles;
    x.part_rows = (int)std::min<long>(rows, kTileRows);
    x.scale2 = p.scale2, x.err = p.err;
    x.units = reinterpret_cast<int2*>(ws + w.units), x.ml = reinterpret_cast<float2*>(ws + w.ml), x.acc = reinterpret_cast<float*>(ws + w.acc);
    p.prefix = PrefixParts{x.units, x.ml, reinterpret_cast<const float4*>(x.acc), x.each, x.tiles, x.part_rows};
    const cudaError_t e = cache->kind == kKvBf16  ? launch_both<kKvBf16>(x, p, ws, sms, st)
                          : cache->kind == kKvFp8 ? launch_both<kKvFp8>(x, p, ws, sms, st)
                                                  : launch_both<kKvNvfp4>(x, p, ws, sms, st);
    return launch_status(e, "fp4b_shared_attention");
}
