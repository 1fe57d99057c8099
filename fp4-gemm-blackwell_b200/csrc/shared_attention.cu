// shared_attention.cu -- attention of one new token a sequence where sequences
// share a prefix: the prefix's keys and values are read once for all of them.
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
//   warps 8-11 (4-7)   read pages, decode them to 16 bits, write K and V in the
//                      128-byte swizzle;
//   warp 12 (8)        issues the products: S of the next tile before O of this;
//   warps 0-7 (0-3)    two groups of 128 threads, a row a thread, take the tiles
//                      in turn: each has scores, sums and an O of its own, so
//                      that neither waits for the other (256 elements: one).
// O stays in TMEM over a unit; S (128 columns of fp32) is read twice, for its
// largest and for the weights, which go back over it as the A operand of the
// second product.
//
// Formats, the reference exponent (moved when a score passes it by 2^10) and the
// weights' two terms are decode_attention's: bf16 in BF16 (16 bits), fp8 and nvfp4
// in FP16 (22 bits); see there for why.
//
// What the parts of a unit found (two for each CTA that has tiles of it) goes to
// the workspace, with the place and the number of each unit's parts.
#include "decode_attention.cuh"

#define FP4B_EXPORT extern "C" __attribute__((visibility("default")))

namespace fp4b {
namespace {

constexpr int kErrPrefixTimeout = 14;
constexpr int kTileRows = 128;
constexpr int kProducers = 128;
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
};

template <int KIND, int D>
struct PrefixCfg {
    static constexpr int TK = D == 256 ? 64 : 128;                                   // keys of a tile
    static constexpr int GROUPS = D == 256 ? 1 : 2;
    static constexpr int THREADS = GROUPS * 128 + kProducers + 128;
    static constexpr int RB = KIND == kKvBf16 ? 2 * D : KIND == kKvFp8 ? D : D / 2;  // bytes of a row
    static constexpr int SB = KIND == kKvBf16 ? 0 : KIND == kKvFp8 ? 4 : D / 16;     // bytes of its scales
    static constexpr int Q = kTileRows * D * 2;
    static constexpr int PIECE = TK * D * 2;                                         // K or V of a tile in 16 bits
    static constexpr int STAGES = KIND == kKvBf16 ? (D == 64 ? 5 : D == 128 ? 3 : 2) : D == 64 ? 3 : 2;
    static constexpr int RAW = KIND == kKvBf16 ? 0 : TK * (RB + SB);                 // a piece as it lies in the cache
    static constexpr int RAWS = KIND == kKvBf16 ? 0 : KIND == kKvFp8 ? (D == 64 ? 8 : D == 128 ? 3 : 2) : D == 64 ? 8 : D == 128 ? 6 : 3;
    // Pieces on their way.  BF16 is copied in place: with this many the wait for a
    // free stage is never one for a product that waits for the piece at hand.
    static constexpr int AHEAD = KIND == kKvBf16 ? 2 * STAGES - 3 : RAWS - 1;
    static constexpr int SCALES = KIND == kKvFp8 ? 3 * TK * 4 : 0;                   // of a stage: key scales, value scales, their logarithms
    static constexpr int S_COLUMNS = 2 * TK;
    static constexpr int OFF_K = Q, OFF_V = OFF_K + STAGES * PIECE, OFF_RAW = OFF_V + STAGES * PIECE;
    static constexpr int OFF_SCALES = OFF_RAW + RAWS * RAW, OFF_BARS = OFF_SCALES + STAGES * SCALES;
    static constexpr int OFF_FACTORS = OFF_BARS + (4 * STAGES + 8) * 8, OFF_VARS = OFF_FACTORS + kTileRows * 4;
    static constexpr int SMEM = OFF_VARS + 32;
    static_assert(SMEM <= kSmemMost, "shared memory");
    static_assert(S_COLUMNS + GROUPS * D <= 512, "TMEM");
    static_assert(OFF_RAW % 1024 == 0 && RAW % 16 == 0 && OFF_SCALES % 16 == 0 && OFF_BARS % 8 == 0, "alignment");
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

__device__ __forceinline__ float at(const float4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

template <int KIND, int D>
__global__ void __launch_bounds__(PrefixCfg<KIND, D>::THREADS, 1) prefix_attention_kernel(const __grid_constant__ PrefixParams p) {
    using C = PrefixCfg<KIND, D>;
    constexpr int TK = C::TK, GROUPS = C::GROUPS, STAGES = C::STAGES, RB = C::RB, SB = C::SB;
    constexpr bool kBf16 = KIND == kKvBf16;
    extern __shared__ __align__(1024) uint8_t tiles_smem[];
    uint8_t* const smem = tiles_smem;
    // (no other shared memory: the swizzle wants this at a multiple of 1024)
    float* const s_factor = reinterpret_cast<float*>(smem + C::OFF_FACTORS);
    int* const vars = reinterpret_cast<int*>(smem + C::OFF_VARS);
    uint32_t& s_tmem = reinterpret_cast<uint32_t&>(vars[0]);
    int &s_abort = vars[1], &s_total = vars[2], &s_g = vars[3], &s_before = vars[4];
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BARS);
    uint64_t *const k_full = bars, *const k_empty = bars + STAGES, *const v_full = bars + 2 * STAGES, *const v_empty = bars + 3 * STAGES;
    uint64_t *const s_full = bars + 4 * STAGES, *const p_full = s_full + 2, *const q_full = s_full + 4, *const o_done = s_full + 5, *const unit_done = s_full + 6, *const drained = s_full + 7;

    chain();
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    constexpr int kProducerWarp = GROUPS * 4, kMmaWarp = kProducerWarp + 4;

    // ---- set up: barriers, TMEM, this CTA's share
    if (tid == 0) {
        s_abort = 0;
        for (int i = 0; i < STAGES; ++i) {
            ptx::mbar_init(k_full + i, kProducers), ptx::mbar_init(v_full + i, kProducers);
            ptx::mbar_init(k_empty + i, 1), ptx::mbar_init(v_empty + i, 1);
        }
        for (int i = 0; i < 2; ++i) ptx::mbar_init(s_full + i, 1), ptx::mbar_init(p_full + i, 128);
        ptx::mbar_init(q_full, GROUPS * 128), ptx::mbar_init(o_done, 1), ptx::mbar_init(unit_done, 1), ptx::mbar_init(drained, 1);
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

    if (working && warp < kProducerWarp) {
        // ------------------------------------------------------------ a row a thread: queries, softmax, results
        const int mine = warp >> 2, row = tid & 127;
        const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);  // this warp's 32 lanes
        const uint32_t o_at = lanes + C::S_COLUMNS + mine * D;
        int it = 0, segment = 0;
        bool ok = true;
        while (ok && next_unit<TK>(p, walk)) {
            const int rows = min(kTileRows, p.rows - walk.tile * kTileRows);
            const bool live = (warp & 3) * 32 < rows;
            if (mine == 0) {
                // ---- this row of Q, in 16 bits and swizzled; rows that there are not as zeros
                const int r = walk.tile * kTileRows + row, of = r / p.group;
                const bool there = row < rows;
                const uint16_t* from = p.q + (size_t)(walk.g * p.each + (there ? of : 0)) * p.q_sb +
                                       (size_t)(walk.kv_head * p.group + (there ? r - of * p.group : 0)) * p.q_sh;
                float up = 1.0f, factor = p.scale2;
                if constexpr (!kBf16) {
                    uint32_t top = 0;
                    for (int d = 0; d < D; d += 4) {
                        const uint2 w = *reinterpret_cast<const uint2*>(from + d);
                        top = max(top, max((w.x & 0x7FFFu) << 16, w.x & 0x7FFF0000u));
                        top = max(top, max((w.y & 0x7FFFu) << 16, w.y & 0x7FFF0000u));
                    }
                    const int k = min(max(141 - (int)(top >> 23), -126), 126);
                    up = __int_as_float((127 + k) << 23);
                    factor *= __int_as_float((127 - k) << 23);
                    if (KIND == kKvNvfp4) factor *= kScaleUnit;
                }
                s_factor[row] = factor;
#pragma unroll 4
                for (int c = 0; c < D / 8; ++c) {
                    uint2 a = make_uint2(0u, 0u), b = a;
                    if (there) a = *reinterpret_cast<const uint2*>(from + 8 * c), b = *reinterpret_cast<const uint2*>(from + 8 * c + 4);
                    if constexpr (!kBf16) {
                        a = make_uint2(pack_f16(bf16_lo(a.x) * up, bf16_hi(a.x) * up), pack_f16(bf16_lo(a.y) * up, bf16_hi(a.y) * up));
                        b = make_uint2(pack_f16(bf16_lo(b.x) * up, bf16_hi(b.x) * up), pack_f16(bf16_lo(b.y) * up, bf16_hi(b.y) * up));
                    }
                    const int at = (c >> 3) * (kTileRows * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
                    *reinterpret_cast<uint4*>(smem + at) = make_uint4(a.x, a.y, b.x, b.y);
                }
                ptx::fence_proxy_async_smem();
            }
            ptx::mbar_arrive(q_full);  // (both groups: neither falls a unit behind)
            ok = wait(q_full, segment & 1);
            const float f = s_factor[row];
            float ref = kNoScore, l = 0.0f;
            bool begun = false;
            for (int j = walk.r0; ok && j < walk.r1; ++j, ++it) {
                if (GROUPS == 2 && (it & 1) != mine) continue;
                const int buf = it & 1, stage = it % STAGES;
                ok = wait(s_full + buf, (it >> 1) & 1);
                if (KIND == kKvFp8 && ok) ok = wait(v_full + stage, (it / STAGES) & 1);
                if (!ok) break;
                ptx::tc_fence_after();
                if (live) {
                    const uint32_t s_at = lanes + buf * TK;
                    const float4* const scales = reinterpret_cast<const float4*>(smem + C::OFF_SCALES + stage * C::SCALES);
                    const int seen = walk.valid - j * TK;  // keys of the tile that there are
                    // ---- the largest score, in base 2 (for fp8 with the value scale's share)
                    float top = -INFINITY;
                    auto largest = [&](auto whole) {
#pragma unroll
                        for (int c = 0; c < TK / 32; ++c) {
                            uint32_t s[32];
                            ptx::tmem_ld_32x32b_x32(s_at + 32 * c, s);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                float x[4];
                                [[maybe_unused]] float4 ks, lv;
                                if constexpr (KIND == kKvFp8) ks = scales[8 * c + i / 4], lv = scales[TK / 2 + 8 * c + i / 4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    x[e] = __uint_as_float(s[i + e]);
                                    if constexpr (KIND == kKvFp8) x[e] = fmaf(x[e] * at(ks, e), f, at(lv, e));
                                    else x[e] *= f;
                                    if (!decltype(whole)::value && 32 * c + i + e >= seen) x[e] = -INFINITY;
                                }
                                top = fmaxf(fmaxf(top, fmaxf(x[0], x[1])), fmaxf(x[2], x[3]));
                            }
                        }
                    };
                    if (seen >= TK) largest(std::true_type{});
                    else largest(std::false_type{});
                    // ---- the reference moves when a score of the warp's passes it by too much
                    if (__any_sync(0xffffffffu, top > ref + kHeadroom)) {
                        const float to = fmaxf(ref, top - kBelowMax), c = exp2_approx(ref - to);
                        ref = to;
                        l *= c;
                        if (begun) {
                            if (GROUPS == 1) ok = wait(o_done, (it - 1) & 1);  // (two groups: the scores came after it)
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
                    const unsigned long long ff = pair_of(f, f), rr = pair_of(-ref, -ref);
                    unsigned long long sum = pair_of(0.0f, 0.0f);
                    auto weigh = [&](auto whole) {
#pragma unroll
                        for (int c = 0; c < TK / 32; ++c) {
                            uint32_t s[32], w[32];
                            ptx::tmem_ld_32x32b_x32(s_at + 32 * c, s);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                unsigned long long x = pair_of(__uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                                [[maybe_unused]] float4 ks, vs;
                                if constexpr (KIND == kKvFp8) {
                                    ks = scales[8 * c + i / 4], vs = scales[TK / 4 + 8 * c + i / 4];
                                    x = mul2(x, pair_of(at(ks, i & 2), at(ks, (i & 2) + 1)));
                                }
                                x = fma2(x, ff, rr);
                                float a = exp2_approx(first_of(x)), b = exp2_approx(second_of(x));
                                if constexpr (!decltype(whole)::value) {
                                    if (32 * c + i >= seen) a = 0.0f;
                                    if (32 * c + i + 1 >= seen) b = 0.0f;
                                }
                                sum = add2(sum, pair_of(a, b));
                                if constexpr (KIND == kKvFp8) a *= at(vs, i & 2), b *= at(vs, (i & 2) + 1);
                                if constexpr (kBf16) {
                                    const uint32_t hi = pack_bf16(a, b);
                                    w[i / 2] = hi;
                                    w[16 + i / 2] = pack_bf16(a - bf16_lo(hi), b - bf16_hi(hi));
                                } else {
                                    const uint32_t hi = pack_f16(a, b);
                                    const float2 back = f16x2_to_float2(hi);
                                    w[i / 2] = hi;
                                    w[16 + i / 2] = pack_f16(a - back.x, b - back.y);
                                }
                            }
                            ptx::tmem_st_32x32b_x32(s_at + 32 * c, w);
                        }
                    };
                    if (seen >= TK) weigh(std::true_type{});
                    else weigh(std::false_type{});
                    l += first_of(sum) + second_of(sum);
                    ptx::tmem_st_wait();
                }
                begun = true;
                ptx::tc_fence_before();
                ptx::mbar_arrive(p_full + buf);
            }
            // ---- the unit's part: (reference, sum) and O
            if (ok) ok = wait(unit_done, segment & 1);
            if (!ok) break;
            ptx::tc_fence_after();
            const int first = owner(walk.u - walk.r1), count = owner(walk.u - walk.r1 + walk.length - 1) - first + 1;
            const size_t part = ((size_t)walk.unit + blockIdx.x) * GROUPS + mine;
            if (walk.r0 == 0 && tid == 0) p.units[walk.unit] = make_int2((walk.unit + first) * GROUPS, count * GROUPS);
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
        const int my = warp - kProducerWarp;
        constexpr int ROWS = TK / 4;                     // of a tile, a warp
        constexpr int LR = RB / 16, PER = 32 / LR;       // lanes a row, rows an instruction
        constexpr int COPIES = ROWS / PER;
        const int sub = lane / LR, c = lane % LR;
        uint8_t* const raw = smem + C::OFF_RAW;
        // pieces: K and V of each tile in turn; `there` is on its way, `here` is decoded
        Walk there = walk, here = walk;
        bool more = next_unit<TK>(p, there), ok = true;
        int tile = there.r0, issued = 0, row = -1, page = -2;
        auto look = [&]() {  // the page of this lane's key of the tile, on its way; -2 for no key
            const int key = tile * TK + my * ROWS + lane;
            page = lane < ROWS && key < there.valid ? max(p.table[(size_t)there.g * p.table_stride + (key >> p.page_shift)], -1) : -2;
        };
        if (more) look();
        // Starts the copy of piece `issued` (K where even); false at the end of a wait.
        auto issue = [&]() {
            if (more) {
                const bool value = issued & 1;
                const int t = issued >> 1, stage = t % STAGES;
                if (!value) {  // the key's row in the cache, -1 for none
                    const int slot = (tile * TK + my * ROWS + lane) & (p.cache.page_size - 1);
                    row = -1;
                    if (page >= 0 && page < p.cache.num_pages) row = (page * p.cache.kv_heads + there.kv_head) * p.cache.page_size + slot;
                    else if (page != -2) report(p.err, kErrPageRange);
                }
                uint32_t to;
                if constexpr (kBf16) {
                    if (t >= STAGES && !wait((value ? v_empty : k_empty) + stage, ((t / STAGES) & 1) ^ 1)) return false;
                    to = ptx::smem_u32(smem + (value ? C::OFF_V : C::OFF_K) + stage * C::PIECE);
                } else {
                    to = ptx::smem_u32(raw + issued % C::RAWS * C::RAW);
                }
                const uint8_t* const from = static_cast<const uint8_t*>(value ? p.cache.v : p.cache.k);
#pragma unroll
                for (int i = 0; i < COPIES; ++i) {
                    const int r = i * PER + sub, at = __shfl_sync(0xffffffffu, row, r);
                    const uint8_t* src = from + (size_t)max(at, 0) * RB + 16 * c;
                    if constexpr (kBf16) {
                        const int tr = my * ROWS + r;
                        copy_async<16>(to + (c >> 3) * (TK * 128) + tr * 128 + (((c & 7) ^ (tr & 7)) << 4), src, at >= 0);
                    } else {
                        copy_async<16>(to + ((my * COPIES + i) * 32 + lane) * 16, src, at >= 0);
                    }
                }
                if constexpr (SB > 0)
                    if (lane < ROWS)
                        copy_async<SB>(to + TK * RB + (my * ROWS + lane) * SB,
                                       static_cast<const uint8_t*>(value ? p.cache.v_scale : p.cache.k_scale) + (size_t)max(row, 0) * SB, row >= 0);
                ++issued;
                if (value) {
                    if (++tile == there.r1) {
                        more = next_unit<TK>(p, there);
                        tile = there.r0;
                    }
                    if (more) look();
                }
            }
            copy_commit();
            return true;
        };
        for (int i = 0; ok && i < C::AHEAD; ++i) ok = issue();
        int piece = 0;
        float key_scale = 0.0f;  // of this lane's key (fp8)
        while (ok && next_unit<TK>(p, here)) {
            for (int j = 2 * here.r0; ok && j < 2 * here.r1; ++j, ++piece) {
                const bool value = piece & 1;
                const int t = piece >> 1, stage = t % STAGES;
                if constexpr (kBf16) {
                    copy_wait<C::AHEAD - 1>();
                } else {
                    issue();
                    copy_wait<C::AHEAD>();
                    __syncwarp();  // the other lanes' copies: a row's scales
                    if (t >= STAGES) ok = wait((value ? v_empty : k_empty) + stage, ((t / STAGES) & 1) ^ 1);
                    if (!ok) break;
                    const uint8_t* const from = raw + piece % C::RAWS * C::RAW;
                    uint8_t* const to = smem + (value ? C::OFF_V : C::OFF_K) + stage * C::PIECE;
#pragma unroll
                    for (int i = 0; i < COPIES; ++i) {
                        const int r = my * ROWS + i * PER + sub;
                        const uint4 w = lds128(from + ((my * COPIES + i) * 32 + lane) * 16);
                        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
                        if constexpr (KIND == kKvFp8) {
                            const int e = 16 * c;
                            uint8_t* line = to + (e >> 6) * (TK * 128) + r * 128;
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                uint32_t a[2], b[2];
                                e4m3x4_to_f16(words[2 * h], a);
                                e4m3x4_to_f16(words[2 * h + 1], b);
                                *reinterpret_cast<uint4*>(line + (((((e & 63) >> 3) + h) ^ (r & 7)) << 4)) = make_uint4(a[0], a[1], b[0], b[1]);
                            }
                        } else {
                            const int e = 32 * c;
                            uint8_t* line = to + (e >> 6) * (TK * 128) + r * 128;
                            const uint32_t sc = *reinterpret_cast<const uint16_t*>(from + TK * RB + r * SB + 2 * c);
#pragma unroll
                            for (int h = 0; h < 4; ++h) {
                                const uint32_t scale = ue4m3x2_to_f16((h < 2 ? sc & 0xFFu : sc >> 8) * 0x10001u);
                                uint32_t a[4];
                                e2m1x8_to_f16(words[h], a);
                                *reinterpret_cast<uint4*>(line + (((((e & 63) >> 3) + h) ^ (r & 7)) << 4)) =
                                    make_uint4(mul_f16x2(a[0], scale), mul_f16x2(a[1], scale), mul_f16x2(a[2], scale), mul_f16x2(a[3], scale));
                            }
                        }
                    }
                    if constexpr (KIND == kKvFp8) {
                        if (lane < ROWS) {
                            const int r = my * ROWS + lane;
                            const float scale = *reinterpret_cast<const float*>(from + TK * RB + r * SB);
                            if (value) {
                                float* s = reinterpret_cast<float*>(smem + C::OFF_SCALES + stage * C::SCALES);
                                s[r] = key_scale, s[TK + r] = scale, s[2 * TK + r] = fmaxf(log2_approx(scale), -80.0f);
                            }
                            key_scale = scale;
                        }
                    }
                    __syncwarp();  // (the raw piece may be copied over)
                }
                ptx::fence_proxy_async_smem();
                ptx::mbar_arrive((value ? v_full : k_full) + stage);
                if constexpr (kBf16) ok = issue();
            }
        }
        copy_wait<0>();
    } else if (working && warp == kMmaWarp) {
        // ------------------------------------------------------------ the products
        constexpr uint32_t s_desc = ptx::idesc_f16(kBf16, false, TK), o_desc = ptx::idesc_f16(kBf16, true, D);
        const uint64_t q_at = ptx::desc_kmajor_sw128(ptx::smem_u32(smem));
        const uint64_t k_at = ptx::desc_kmajor_sw128(ptx::smem_u32(smem + C::OFF_K));
        const uint64_t v_at = ptx::desc_mnmajor_sw128(ptx::smem_u32(smem + C::OFF_V), TK * 128);
        int it = 0, segment = 0;
        bool ok = true;
        auto scores = [&](int t) {  // S of tile t
            const int stage = t % STAGES;
            ok = wait(k_full + stage, (t / STAGES) & 1);
            if (!ok) return;
            ptx::tc_fence_after();
            if (ptx::elect_one()) {
                const uint64_t k = k_at + (uint64_t)((stage * C::PIECE) >> 4);
#pragma unroll
                for (int j = 0; j < D / 16; ++j)
                    ptx::tc_mma_f16(tmem + (t & 1) * TK, q_at + (uint64_t)(((j >> 2) * kTileRows * 128 + (j & 3) * 32) >> 4),
                                    k + (uint64_t)(((j >> 2) * TK * 128 + (j & 3) * 32) >> 4), s_desc, j > 0);
                ptx::tc_commit(k_empty + stage);
                ptx::tc_commit(s_full + (t & 1));
            }
            __syncwarp();
        };
        while (ok && next_unit<TK>(p, walk)) {
            const int n = walk.r1 - walk.r0;
            ok = wait(q_full, segment & 1);
            if (ok) scores(it);
            for (int j = 0; ok && j < n; ++j, ++it) {
                if (j + 1 < n) scores(it + 1);
                if (!ok) break;
                const int stage = it % STAGES, buf = it & 1, mine = GROUPS == 2 ? buf : 0;
                ok = wait(p_full + buf, (it >> 1) & 1) && wait(v_full + stage, (it / STAGES) & 1);
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
                                               j >= GROUPS || k > 0 || term > 0);
                    ptx::tc_commit(v_empty + stage);
                    if (GROUPS == 1) ptx::tc_commit(o_done);
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
cudaError_t launch_prefix(const PrefixParams& p, int sms, cudaStream_t st) {
    using C = PrefixCfg<KIND, D>;
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
cudaError_t launch_both(const PrefixParams& x, AttentionParams& p, uint8_t* workspace, int sms, cudaStream_t st) {
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
