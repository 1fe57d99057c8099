// decode_attention.cu -- attention of one new token a sequence over a paged
// key-value cache, split over the cache's length and joined in one launch.
//
//   out[b, h] = sum_i p_i v_i / l,  p_i = exp(scale * q . k_i - m),
//   l = sum_i p_i (+ exp(sink_h - m))
//
// over the keys i of [max(0, len - window), len).  Every cached byte is read
// once for up to 16 query heads of its key head (again for each further 16), so
// the floor is the cache's bytes over the HBM rate; what has to stay below that
// is the work per key.
//
// Products.  Both run on mma.sync m16n8k16 with the keys (then the elements of
// a value) as the 16 rows and up to 8 query heads as the 8 columns:
//   S^T[16 keys, 8 heads]     = K[16, D] Q^T[D, 8]
//   O^T[16 elements, 8 heads] += V^T[16 elements, 16 keys] P^T[16 keys, 8]
// (tcgen05's 128 rows would need 128 query heads for each key head).  The order
// of the contracted index is free as long as both operands agree, so a lane
// reads the 16-byte runs of a row as they lie, and neither K nor V is
// transposed through shared memory: V^T's register pairs, two keys of one
// element, are byte permutes of two rows' words.  P^T comes from S^T's
// accumulators by movmatrix.
//
// Formats.  bf16 multiplies in BF16.  fp8 and nvfp4 multiply in FP16, which
// holds their codes exactly (e2m1 * ue4m3 has 6 significant bits; the scale
// enters as 2^-8 of its value, a shift of its byte), and q times the power of
// two that puts its largest element into [2^14, 2^15).  An fp8 row's scale
// multiplies the score of its key and the weight of its value.  p enters as two
// terms, its rounding and what that left: 16 bits in BF16, 22 in FP16 (less
// below 2^-3, to within 2^-25; the largest weight is 2^4 or more, see below).  One
// term would be 8 bits in BF16, as large an error as the output's own rounding,
// and 11 in FP16: outputs would lie 6.5e-4 of their size from those of 32-bit
// weights, with two they lie 1.2e-4 or less, and values of either sign that nearly
// cancel would leave no right digit.  The second term costs nvfp4 13 % (3 x 131072
// keys, D = 64: 58.5 us, 52.0 without it), fp8 1 % (47.9, 47.5).
//
// Softmax.  In base 2 with a reference exponent per head instead of the exact
// maximum: it moves (to the maximum less 4) only when a score passes it by
// more than 10, so most steps need one vote and no rescaling; p stays below
// 2^14.  For fp8 the reference follows the weighted scale, score + log2(value
// scale), so that p times the scale is what stays in range.
//
// Split.  Sequence lengths are known on the GPU only.  A round is WARPS * TK
// keys of one sequence and head unit, one step for each warp; the rounds of the
// whole batch, in order, are dealt out evenly to the CTAs, each of which finds
// its share by a prefix sum over the lengths.  Lengths of any unevenness fill
// the GPU the same.  A share is cut into segments of one head unit each; a unit
// whose rounds lie in several CTAs has its parts in the workspace, and the CTA
// that arrives last at its counter joins them, in the order of their keys, so
// that results do not depend on the arrival.  A CTA has at most two such parts,
// its first and its last segment, and arrives for both at its end: one fence.
// The first steps of the next segment are under way while one is finished.
// Still a segment costs about as much as kSegmentRounds rounds besides its own
// (a CTA with four short ones ended 15 us behind the others): shares are even
// in rounds with these added to each unit.
//
// Measured on B200 (copy bandwidth 6.54 TB/s): nvfp4, 3 x 131072 keys x 8 heads x 64
// under 64 query heads 58.5 us = 3.9 TB/s, bound by its instructions: 350 for 32 keys,
// in 580 cycles of a scheduler.  24 are matrix instructions of 8 cycles each, 128 decode
// and scale the codes; 60 % of the issue slots are used, as the cycles of matrix
// instructions and of others nearly add up.  fp8, 33 sequences up to 8000 x 8 x 128 under
// 32 heads 47.9 us = 5.3 TB/s and bf16, 8 up to 4095 x 16 x 256 under 16 heads 49 us = 5.6
// TB/s, bound by HBM behind about 7 us of start, first bytes and joining; one sequence of
// 77 keys 4.7 us, a launch and a chain of waits.
//
// A warp streams its steps through a ring of its own in shared memory with
// cp.async: no barrier in the loop.  Masked keys are zero-filled, not read.
// What a step costs besides its keys (its pages, addresses, waits, the loop)
// was 58 of 357 instructions for 32 keys of 32 bytes, where instructions are the
// bound: such steps have 64 keys, worked on in two unrolled parts (3 x 131072 keys
// of nvfp4, D = 64, p in one term: 58 us by 32 keys and four steps in the ring, 53.7
// by 64 and two, 51.6 unrolled).  Pages are looked up for 32 runs of keys at once.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <mutex>

#include "decode_core.cuh"
#include "fp4b_internal.h"
#include "ptx_sm100.cuh"

#define FP4B_EXPORT extern "C" __attribute__((visibility("default")))

namespace fp4b {
namespace {

using namespace decode;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxCtasPerSm = 4;
constexpr int kSegmentRounds = 3;  // of CK keys a warp, as kWholeRounds
constexpr int kWholeRounds = 8;
constexpr float kNoScore = -3.402823466e38f;  // reference exponent before any key: any finite score passes it
constexpr float kHeadroom = 10.0f;    // a score may pass the reference by 2^10 ...
constexpr float kBelowMax = 4.0f;     // ... which is set 2^4 below the maximum
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttentionParams {
    const uint16_t* q;
    long q_sb, q_sh;
    int batch, q_heads, group;
    int group_tiles;  // head units of a key head: ceil(group / heads of a unit)
    fp4b_kv_cache cache;
    int page_shift;
    const int* table;
    long table_stride;
    int table_width;
    const int* lens;
    float scale2;  // scale * log2(e)
    int window;
    const float* sinks;
    uint16_t* out;
    float* lse;
    int* err;
    // Workspace: counters [max_ctas], zero before and after; the parts that go on
    // in CTA c at c, those that begin in it at max_ctas + c: (maximum, sum)
    // [2 * max_ctas][heads of a unit][2] and sums [2 * max_ctas][heads][D].
    int max_ctas;
    uint32_t* counters;
    float* part_ml;
    float* part_acc;
};

template <int KIND, int D, int NT>
struct Cfg {
    static constexpr int RB = KIND == kKvBf16 ? 2 * D : KIND == kKvFp8 ? D : D / 2;  // bytes of a row
    static constexpr int SB = KIND == kKvBf16 ? 0 : KIND == kKvFp8 ? 4 : D / 16;     // bytes of its scales
    static constexpr int CK = RB <= 64 ? 32 : 16;   // keys that are worked on at once: at least 1 KB of K
    static constexpr int KT = CK / 16;
    static constexpr int PARTS = RB <= 64 || KIND == kKvNvfp4 ? 2 : 1;  // of them in a step, which is copied at once
    static constexpr int TK = PARTS * CK;           // keys of a step
    static constexpr int SEGMENT = (kSegmentRounds + PARTS - 1) / PARTS, WHOLE = kWholeRounds / PARTS;
    static constexpr int HEADS = 8 * NT;
    static constexpr int ROUND = kWarps * TK;
    static constexpr int PART = 2 * CK * (RB + SB);
    static constexpr int STAGE = PARTS * PART;
    static constexpr int STAGES = PARTS > 1 ? 2 : STAGE >= 4096 ? 3 : 4;
    static constexpr int RING = STAGES * STAGE;
    static constexpr int LD = D + 8;                // row stride of the merge area
    static constexpr int MERGE = kWarps * HEADS * LD * 4;
    // Where a third stage would not fit beside it, the merge area lies over the
    // rings and the next segment's steps start after it was read.
    static constexpr bool APART = STAGE < 8192;
    static constexpr int SMEM = APART ? kWarps * RING + MERGE : (kWarps * RING > MERGE ? kWarps * RING : MERGE);
    // Elements of one of a lane's runs in a K row (4 lanes share the row) and in a V row (8 lanes).
    static constexpr int EK = KIND == kKvBf16 ? 8 : KIND == kKvFp8 ? 16 : (D == 64 ? 16 : 32);
    static constexpr int EV = KIND == kKvBf16 ? 8 : KIND == kKvFp8 ? (D == 64 ? 8 : 16) : D / 8;
};

// Shared-memory offset of 16-byte chunk c of row r: rows of 128 bytes or more
// (and all V rows) are permuted so that the 8 or 16 lanes of one phase of the
// reads below meet distinct banks.
template <int RB>
__device__ __forceinline__ int k_offset(int r, int c) {
    return r * RB + 16 * (RB >= 128 ? c ^ ((r & 1) << 2) : c);
}
template <int RB>
__device__ __forceinline__ int v_offset(int r, int c) {
    if constexpr (RB == 32) return ((((r >> 1) & 3) | ((r & 1) << 2) | (r & 24)) * RB) + 16 * c;
    else if constexpr (RB == 64) return ((((r >> 1) & 1) | ((r & 1) << 1) | (r & 28)) * RB) + 16 * (c ^ (((r >> 2) & 1) << 1));
    else return r * RB + 16 * (c ^ (((r >> 1) & 3) << 1));
}

// First key of a sequence's rounds, its clamped length and first visible key.
struct Span {
    int start, first, len, rounds;
};
template <int TK, int ROUND>
__device__ __forceinline__ Span span_of(const AttentionParams& p, int b) {
    Span s;
    const int most = p.table_width << p.page_shift;
    s.len = p.lens[b];
    if (s.len < 0 || s.len > most) {
        report(p.err, kErrPageRange);
        s.len = s.len < 0 ? 0 : most;
    }
    s.first = p.window > 0 && s.len > p.window ? s.len - p.window : 0;
    s.start = s.first & ~(TK - 1);
    s.rounds = (s.len - s.start + ROUND - 1) / ROUND;
    return s;
}

// One output row: divides by the softmax's denominator, the sink's share included.
struct Finish {
    float factor, lse;
};
__device__ __forceinline__ Finish finish(const AttentionParams& p, int head, float m, float l, float unit) {
    float share = 1.0f;
    if (p.sinks) {
        const float sink = p.sinks[head] * kLog2e;
        const float top = fmaxf(m, sink);
        share = exp2_approx(m - top);
        l = l * share + exp2_approx(sink - top);
        m = top;
    }
    // l == 0: nothing was seen (m is kNoScore or the sink is -inf)
    return Finish{l == 0.0f ? 0.0f : unit * share / l, l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2};
}

// Four elements of an output row from their sums relative to 2^m; unit: what the
// sums are to be multiplied by.
template <int D>
__device__ __forceinline__ void put_row(const AttentionParams& p, int b, int head, int d, float m, float l, float4 sum, float unit) {
    const Finish f = finish(p, head, m, l, unit);
    const size_t row = (size_t)b * p.q_heads + head;
    *reinterpret_cast<uint2*>(p.out + row * D + d) =
        make_uint2(pack_bf16(sum.x * f.factor, sum.y * f.factor), pack_bf16(sum.z * f.factor, sum.w * f.factor));
    if (p.lse && d == 0) p.lse[row] = f.lse;
}

// A head unit that several CTAs, first to last, have parts of.
struct Part {
    int b, head0, heads, first, last;
};

// Joins a unit's parts in their order: the first one's from the parts that begin
// in a CTA, the others' from those that go on in one, kAhead of them in flight.
template <int D, int HEADS>
__device__ __forceinline__ void join_parts(const AttentionParams& p, const Part& x, float unit) {
    constexpr int kItems = (HEADS * D / 4 + kThreads - 1) / kThreads;  // quarters of rows a thread
    constexpr int kAhead = kItems > 4 ? 2 : kItems > 1 ? 4 : 8;
    const int quarters = x.heads * (D / 4);
    float m[kItems], l[kItems];
    float4 sum[kItems];
    const float2* ml[kItems];
    const float4* acc[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const int j = min((int)threadIdx.x + k * kThreads, quarters - 1);
        const size_t begin = (size_t)(p.max_ctas + x.first) * HEADS, on = (size_t)(x.first + 1) * HEADS;
        const float2 one = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + begin + j / (D / 4));
        sum[k] = __ldcg(reinterpret_cast<const float4*>(p.part_acc + begin * D) + j);
        m[k] = one.x, l[k] = one.y;
        ml[k] = reinterpret_cast<const float2*>(p.part_ml) + on + j / (D / 4);
        acc[k] = reinterpret_cast<const float4*>(p.part_acc + on * D) + j;
    }
    for (int left = x.last - x.first; left > 0; left -= kAhead) {
        float2 a[kItems][kAhead];
        float4 v[kItems][kAhead];
#pragma unroll
        for (int k = 0; k < kItems; ++k)
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                a[k][i] = make_float2(kNoScore, 0.0f);
                v[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < left) {
                    a[k][i] = __ldcg(ml[k] + i * HEADS);
                    v[k][i] = __ldcg(acc[k] + i * (HEADS * D / 4));
                }
            }
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            ml[k] += kAhead * HEADS, acc[k] += kAhead * (HEADS * D / 4);
            float top = m[k];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) top = fmaxf(top, a[k][i].x);
            const float old = exp2_approx(m[k] - top);
            sum[k].x *= old, sum[k].y *= old, sum[k].z *= old, sum[k].w *= old, l[k] *= old;
            m[k] = top;
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const float add = exp2_approx(a[k][i].x - top);
                sum[k].x += v[k][i].x * add, sum[k].y += v[k][i].y * add, sum[k].z += v[k][i].z * add, sum[k].w += v[k][i].w * add;
                l[k] += a[k][i].y * add;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const int j = (int)threadIdx.x + k * kThreads, h = j / (D / 4);
        if (j < quarters) put_row<D>(p, x.b, x.head0 + h, 4 * (j - h * (D / 4)), m[k], l[k], sum[k], unit);
    }
}

// RUN: a part's keys lie in runs of RUN rows, all CK of them, 16 or one.
template <int KIND, int D, int NT, int RUN>
__global__ void __launch_bounds__(kThreads) decode_attention_kernel(const __grid_constant__ AttentionParams p) {
    using C = Cfg<KIND, D, NT>;
    constexpr int TK = C::TK, CK = C::CK, KT = C::KT, PARTS = C::PARTS, RB = C::RB, SB = C::SB, MT = D / 16, HEADS = C::HEADS;
    constexpr bool kBf16 = KIND == kKvBf16;
    constexpr float kUnit = KIND == kKvNvfp4 ? kScaleUnit : 1.0f;  // of the decoded values
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int s_total[kWarps], s_most[kWarps], s_pre, s_b;
    __shared__ float s_m[kWarps][HEADS], s_l[kWarps][HEADS];
    __shared__ Part s_part[2];
    __shared__ int s_last[2];

    chain();
    // the shuffle tells the compiler that a warp has one of it: branches on what follows from it are uniform
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int units = p.cache.kv_heads * p.group_tiles;

    // ---- the batch's rounds: their number, and the prefix sums of the chunk at hand
    int total = 0, most = 0, mine = 0, before = 0;
    auto scan = [&](int base) {
        const int b = base + tid;
        const int rounds = b < p.batch ? span_of<TK, C::ROUND>(p, b).rounds : 0;
        mine = rounds > 0 ? (rounds + C::SEGMENT) * units : 0;
        int sum = mine, top = rounds;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += other;
        }
        top = __reduce_max_sync(0xffffffffu, top);
        __syncthreads();
        if (lane == 31) s_total[warp] = sum, s_most[warp] = top;
        __syncthreads();
        before = total + sum - mine;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += s_total[w];
            total += s_total[w];
            most = max(most, s_most[w]);
        }
    };
    for (int base = 0; base < p.batch; base += kThreads) scan(base);
    // A round takes about 0.4 us while the GPU is idle, counting and joining P
    // parts about 4 us and 0.06 us a part.  So units of up to 8 rounds (of CK keys a
    // warp) are not split at all (each goes whole to the CTA in whose share it
    // starts), and for longer ones a CTA takes at least the rounds that balance the
    // last two terms.  (5 x 1500 keys of nvfp4, D = 64: 12.4 us whole, 8.5 split;
    // 33 x 500 of fp8, D = 128: 13.7 whole, 16.7 split.)
    const bool split = most > C::WHOLE;
    const int least = split ? max(1, (int)sqrtf((float)most * (1.0f / (7 * PARTS)))) : 1;
    const int ctas = min((int)gridDim.x, max(total / least, min(total, 1)));
    if ((int)blockIdx.x < ctas) {
        // CTA c's share starts at c * each + min(c, extra)
        const int each = total / ctas, extra = total - each * ctas;
        int u = (int)blockIdx.x * each + min((int)blockIdx.x, extra);
        const int u1 = u + each + ((int)blockIdx.x < extra ? 1 : 0);
        auto owner = [&](int x) {
            const int cut = extra * (each + 1);
            return x < cut ? x / (each + 1) : extra + (x - cut) / each;
        };
        if (p.batch > kThreads) {  // the sums at hand are the last chunk's: go over them again
            total = 0;
            for (int base = 0; base < p.batch && total <= u; base += kThreads) {
                scan(base);
                if (before <= u && u < before + mine) s_b = base + tid, s_pre = before;
            }
        } else if (before <= u && u < before + mine) {
            s_b = tid, s_pre = before;
        }
        if (tid < 2) s_part[tid].b = -1;
        __syncthreads();
        int b = s_b, pre = s_pre;  // the sequence at hand and the rounds before it

        uint8_t* ring = smem + warp * C::RING;
        const uint32_t ring_addr = ptx::smem_u32(ring);
        const int my_key = lane & (CK - 1);

        // ---- a segment: rounds [r0, r1) of one head unit, and the stream of this warp's steps of it
        Span span{};
        int unit = 0, unit_start = 0, r0 = 0, r1 = 0, kv_head = 0, head0 = 0, live_heads = 0, step0 = 0, steps = 0, rows = -1;
        int full0 = 0, full1 = 0;  // steps [full0, full1) have all their keys
        int next_page[PARTS];
#pragma unroll
        for (int h = 0; h < PARTS; ++h) next_page[h] = -2;
        uint2 qw[NT][MT];  // the queries as they are read, see below
        const int* table = nullptr;
        // Where the rows of the runs lie: lane i holds the first row (-1: none to read) of
        // run 32 n + i and the page of run 32 (n + 1) + i is on its way.  Without runs
        // the pages of the lane's keys of the next step are.
        constexpr int RUNS = RUN > 1 ? TK / RUN : 1;  // of a step
        auto page_of = [&](int s, int key) {  // page of step s's key (or run from it on); -2 if masked
            return s < steps && key + RUN > span.first && key < span.len ? max(table[key >> p.page_shift], -1) : -2;
        };
        auto run_key = [&](int s) { return step0 + (s + lane / RUNS) * C::ROUND + lane % RUNS * RUN; };
        auto row_of = [&](int page, int key) {
            if (page >= 0 && page < p.cache.num_pages)
                return (page * p.cache.kv_heads + kv_head) * p.cache.page_size + (key & (p.cache.page_size - 1));
            if (page != -2) report(p.err, kErrPageRange);
            return -1;
        };
        constexpr int LR = RB / 16, PER = 32 / LR;  // lanes a row, rows an instruction
        const int sub = lane / LR, c = lane % LR;
        // what a lane adds to its row: an instruction's rows are one run
        const int lane_at = 16 * (RUN > 1 ? lane : c), scale_at = (my_key & (RUN - 1)) * SB;
        const uint8_t* const k_lane = static_cast<const uint8_t*>(p.cache.k) + lane_at;
        const uint8_t* const v_lane = static_cast<const uint8_t*>(p.cache.v) + lane_at;
        const uint8_t* const ks_lane = static_cast<const uint8_t*>(p.cache.k_scale) + scale_at;
        const uint8_t* const vs_lane = static_cast<const uint8_t*>(p.cache.v_scale) + scale_at;
        auto copy_scales = [&](uint32_t part, int row, bool live) {
            if constexpr (SB > 0) {
                const uint32_t to = part + 2 * CK * RB + my_key * SB;
                if (CK == 32 || lane < 16) copy_async<SB>(to, ks_lane + (size_t)row * SB, live);
                if (CK == 32 || lane >= 16) copy_async<SB>(to + CK * SB, vs_lane + (size_t)row * SB, live);
            }
        };
        auto issue_runs = [&](int s, uint32_t dst) {
            constexpr int PER_PART = RUN > 1 ? CK / RUN : 1;
            if ((s * RUNS & 31) == 0) {
                rows = row_of(next_page[0], run_key(s));
                next_page[0] = page_of(s + 32 / RUNS + lane / RUNS, run_key(s + 32 / RUNS));
            }
            int row[RUNS];
            bool full = s >= full0 && s < full1;
#pragma unroll
            for (int n = 0; n < RUNS; ++n) {
                row[n] = __shfl_sync(0xffffffffu, rows, (s * RUNS + n) & 31);
                full = full && row[n] >= 0;
            }
#pragma unroll
            for (int h = 0; h < PARTS; ++h) {
                const uint32_t part = dst + h * C::PART;
                const int key0 = step0 + s * C::ROUND + h * CK;
                // the lane's key's row, for its scales
                const int from = PER_PART > 1 && lane >= 16 ? row[h * PER_PART + PER_PART - 1] : row[h * PER_PART];
                if (full) {
#pragma unroll
                    for (int i = 0; i < CK / PER; ++i) {
                        const int r = i * PER + sub;
                        const size_t at = (size_t)row[h * PER_PART + i * PER / RUN] * RB + i * PER % RUN * RB;
                        copy_async<16>(part + k_offset<RB>(r, c), k_lane + at, true);
                        copy_async<16>(part + CK * RB + v_offset<RB>(r, c), v_lane + at, true);
                    }
                    copy_scales(part, from, true);
                } else {
                    // keys from lo up and below hi are read, the others zero-filled
                    const int lo = span.first - key0, hi = span.len - key0;
#pragma unroll
                    for (int i = 0; i < CK / PER; ++i) {
                        const int r = i * PER + sub, first = row[h * PER_PART + i * PER / RUN];
                        const size_t at = (size_t)max(first, 0) * RB + i * PER % RUN * RB;
                        const bool live = first >= 0 && r >= lo && r < hi;
                        copy_async<16>(part + k_offset<RB>(r, c), k_lane + at, live);
                        copy_async<16>(part + CK * RB + v_offset<RB>(r, c), v_lane + at, live);
                    }
                    copy_scales(part, max(from, 0), from >= 0 && my_key >= lo && my_key < hi);
                }
            }
        };
        auto issue = [&](int s) {
            if (s < steps) {
                const uint32_t dst = ring_addr + (s % C::STAGES) * C::STAGE;
                if constexpr (RUN > 1) {
                    issue_runs(s, dst);
                } else {
#pragma unroll
                    for (int h = 0; h < PARTS; ++h) {
                        const uint32_t part = dst + h * C::PART;
                        const int key = step0 + s * C::ROUND + h * CK + my_key, row = row_of(next_page[h], key);
                        next_page[h] = page_of(s + 1, key + C::ROUND);
#pragma unroll
                        for (int i = 0; i < CK / PER; ++i) {
                            const int r = i * PER + sub, from = __shfl_sync(0xffffffffu, row, r);
                            const size_t at = (size_t)max(from, 0) * RB;
                            copy_async<16>(part + k_offset<RB>(r, c), k_lane + at, from >= 0);
                            copy_async<16>(part + CK * RB + v_offset<RB>(r, c), v_lane + at, from >= 0);
                        }
                        copy_scales(part, max(row, 0), row >= 0);
                    }
                }
            }
            copy_commit();
        };
        // Makes the rounds from u on the segment at hand and starts its stream; false at the share's end.
        auto open = [&]() {
            if (u >= u1) return false;
            for (;;) {
                span = span_of<TK, C::ROUND>(p, b);
                const int length = span.rounds > 0 ? span.rounds + C::SEGMENT : 0;  // of a unit
                if (u < pre + length * units) {
                    const int local = u - pre;
                    unit = local / length;
                    r0 = local - unit * length;
                    unit_start = pre + unit * length;
                    if (split ? r0 < span.rounds : r0 == 0) break;
                    u = unit_start + length;  // no rounds of this unit are this CTA's
                    if (u >= u1) return false;
                } else {
                    pre += length * units;
                    if (++b >= p.batch) return false;
                }
            }
            r1 = split ? min(span.rounds, r0 + (u1 - u)) : span.rounds;
            kv_head = unit / p.group_tiles;
            const int in_group = (unit - kv_head * p.group_tiles) * HEADS;
            head0 = kv_head * p.group + in_group, live_heads = min(HEADS, p.group - in_group);
            table = p.table + (size_t)b * p.table_stride;
            step0 = span.start + (r0 * kWarps + warp) * TK;  // first key of step 0; steps are ROUND keys apart
            steps = r1 - r0;
            if (step0 + (steps - 1) * C::ROUND >= span.len) --steps;
            full0 = step0 < span.first, full1 = span.len - step0 < TK ? 0 : (span.len - step0 - TK) / C::ROUND + 1;
#pragma unroll
            for (int h = 0; h < PARTS; ++h) next_page[h] = RUN > 1 ? page_of(lane / RUNS, run_key(0)) : page_of(0, step0 + h * CK + my_key);
#pragma unroll
            for (int s = 0; s < C::STAGES - 1; ++s) issue(s);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int n = 8 * nt + g;
                const uint16_t* row = p.q + (size_t)b * p.q_sb + (size_t)(head0 + (n < live_heads ? n : 0)) * p.q_sh;
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    const int d = 4 * C::EK * (j / (C::EK / 4)) + C::EK * t + 4 * (j % (C::EK / 4));
                    qw[nt][j] = n < live_heads ? *reinterpret_cast<const uint2*>(row + d) : make_uint2(0u, 0u);
                }
            }
            return true;
        };

        bool more = open();
        while (more) {
            // ---- queries: column g of head tile nt, element 4 EK (j / (EK/4)) + EK t + 4 (j % (EK/4)) of k-step j
            uint32_t qf[NT][MT][2];
            float f0[NT], f1[NT];  // score factors of heads 2t, 2t + 1
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint2 (&w)[MT] = qw[nt];
                float factor = p.scale2;
                if constexpr (kBf16) {
#pragma unroll
                    for (int j = 0; j < MT; ++j) qf[nt][j][0] = w[j].x, qf[nt][j][1] = w[j].y;
                } else {
                    uint32_t top = 0;  // largest magnitude's bits
#pragma unroll
                    for (int j = 0; j < MT; ++j) {
                        top = max(top, max((w[j].x & 0x7FFFu) << 16, w[j].x & 0x7FFF0000u));
                        top = max(top, max((w[j].y & 0x7FFFu) << 16, w[j].y & 0x7FFF0000u));
                    }
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const int k = min(max(141 - (int)(top >> 23), -126), 126);
                    const float up = __int_as_float((127 + k) << 23);
#pragma unroll
                    for (int j = 0; j < MT; ++j) {
                        qf[nt][j][0] = pack_f16(bf16_lo(w[j].x) * up, bf16_hi(w[j].x) * up);
                        qf[nt][j][1] = pack_f16(bf16_lo(w[j].y) * up, bf16_hi(w[j].y) * up);
                    }
                    factor *= __int_as_float((127 - k) << 23);
                    if (KIND == kKvNvfp4) factor *= kScaleUnit;
                }
                f0[nt] = __shfl_sync(0xffffffffu, factor, 8 * t);
                f1[nt] = __shfl_sync(0xffffffffu, factor, 8 * t + 4);
            }

            float acc[NT][MT][4];
            float neg0[NT], neg1[NT], l0[NT], l1[NT];  // the references negated, the sums
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                neg0[nt] = neg1[nt] = -kNoScore;
                l0[nt] = l1[nt] = 0.0f;
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[nt][m][i] = 0.0f;
            }

            for (int s = 0; s < steps; ++s) {
                copy_wait<C::STAGES - 2>();
                __syncwarp();
                issue(s + C::STAGES - 1);
#pragma unroll (RB <= 32 ? 2 : 1)
                for (int h = 0; h < PARTS; ++h) {
                    const uint8_t* sk = ring + (s % C::STAGES) * C::STAGE + h * C::PART;
                    const uint8_t* sv = sk + CK * RB;
                    const uint8_t* ss = sv + CK * RB;

                    // ---- scores
                    float sc[NT][KT][4];
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) sc[nt][kt][i] = 0.0f;
                        const int ra = 16 * kt + g, rb = ra + 8;
                        if constexpr (kBf16) {
#pragma unroll
                            for (int i = 0; i < D / 32; ++i) {
                                const uint4 a = lds128(sk + k_offset<RB>(ra, 4 * i + t)), c = lds128(sk + k_offset<RB>(rb, 4 * i + t));
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    mma<true>(sc[nt][kt], a.x, c.x, a.y, c.y, qf[nt][2 * i][0], qf[nt][2 * i][1]);
                                    mma<true>(sc[nt][kt], a.z, c.z, a.w, c.w, qf[nt][2 * i + 1][0], qf[nt][2 * i + 1][1]);
                                }
                            }
                        } else if constexpr (KIND == kKvFp8) {
#pragma unroll
                            for (int i = 0; i < D / 64; ++i) {
                                const uint4 a = lds128(sk + k_offset<RB>(ra, 4 * i + t)), c = lds128(sk + k_offset<RB>(rb, 4 * i + t));
                                const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, cw[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                                for (int q = 0; q < 4; ++q) {
                                    uint32_t ha[2], hc[2];
                                    e4m3x4_to_f16(aw[q], ha);
                                    e4m3x4_to_f16(cw[q], hc);
#pragma unroll
                                    for (int nt = 0; nt < NT; ++nt) mma<false>(sc[nt][kt], ha[0], hc[0], ha[1], hc[1], qf[nt][4 * i + q][0], qf[nt][4 * i + q][1]);
                                }
                            }
                        } else {
                            constexpr int WORDS = C::EK / 8, PIECES = D / (4 * C::EK);
#pragma unroll
                            for (int i = 0; i < PIECES; ++i) {
                                uint32_t aw[WORDS], cw[WORDS];
                                if constexpr (WORDS == 2) {
                                    const uint2 a = lds64(sk + k_offset<RB>(ra, 0) + 8 * t), c = lds64(sk + k_offset<RB>(rb, 0) + 8 * t);
                                    aw[0] = a.x, aw[1] = a.y, cw[0] = c.x, cw[1] = c.y;
                                } else {
                                    const uint4 a = lds128(sk + k_offset<RB>(ra, 4 * i + t)), c = lds128(sk + k_offset<RB>(rb, 4 * i + t));
                                    aw[0] = a.x, aw[1] = a.y, aw[2] = a.z, aw[3] = a.w, cw[0] = c.x, cw[1] = c.y, cw[2] = c.z, cw[3] = c.w;
                                }
#pragma unroll
                                for (int q = 0; q < WORDS; ++q) {
                                    const int block = (C::EK / 16) * (4 * i + t) + q / 2;
                                    const uint32_t s_a = ue4m3x2_to_f16(ss[ra * SB + block] * 0x10001u), s_c = ue4m3x2_to_f16(ss[rb * SB + block] * 0x10001u);
                                    uint32_t ha[4], hc[4];
                                    e2m1x8_to_f16(aw[q], ha);
                                    e2m1x8_to_f16(cw[q], hc);
#pragma unroll
                                    for (int e = 0; e < 4; ++e) ha[e] = mul_f16x2(ha[e], s_a), hc[e] = mul_f16x2(hc[e], s_c);
                                    const int j = (C::EK / 4) * i + 2 * q;
#pragma unroll
                                    for (int nt = 0; nt < NT; ++nt) {
                                        mma<false>(sc[nt][kt], ha[0], hc[0], ha[1], hc[1], qf[nt][j][0], qf[nt][j][1]);
                                        mma<false>(sc[nt][kt], ha[2], hc[2], ha[3], hc[3], qf[nt][j + 1][0], qf[nt][j + 1][1]);
                                    }
                                }
                            }
                        }
                    }

                    // ---- x = score in base 2 less the reference; the row scales of fp8
                    float va[KT], vb[KT], la[KT], lb[KT];  // value scales of the keys and their logarithms
                    if constexpr (KIND == kKvFp8) {
                        const float* fs = reinterpret_cast<const float*>(ss);
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt) {
                            const int ra = 16 * kt + g, rb = ra + 8;
                            const float ka = fs[ra], kb = fs[rb];
                            va[kt] = fs[CK + ra], vb[kt] = fs[CK + rb];
                            la[kt] = fmaxf(log2_approx(va[kt]), -80.0f), lb[kt] = fmaxf(log2_approx(vb[kt]), -80.0f);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                sc[nt][kt][0] *= ka, sc[nt][kt][1] *= ka;
                                sc[nt][kt][2] *= kb, sc[nt][kt][3] *= kb;
                            }
                        }
                    }
                    float x[NT][KT][4];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                            for (int i = 0; i < 4; i += 2) {
                                const unsigned long long both = fma2(pair_of(sc[nt][kt][i], sc[nt][kt][i + 1]), pair_of(f0[nt], f1[nt]), pair_of(neg0[nt], neg1[nt]));
                                x[nt][kt][i] = first_of(both), x[nt][kt][i + 1] = second_of(both);
                            }
                    if (s < full0 || s >= full1) {
                        const int key0 = step0 + s * C::ROUND + h * CK;
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt) {
                            const int ka = key0 + 16 * kt + g, kb = ka + 8;
                            const bool oa = ka >= span.first && ka < span.len, ob = kb >= span.first && kb < span.len;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                if (!oa) x[nt][kt][0] = x[nt][kt][1] = -INFINITY;
                                if (!ob) x[nt][kt][2] = x[nt][kt][3] = -INFINITY;
                            }
                        }
                    }
                    float most_x = -INFINITY;  // over the headroom anywhere?  (for fp8 with the value scale's share)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt) {
                            const float ta = fmaxf(x[nt][kt][0], x[nt][kt][1]), tb = fmaxf(x[nt][kt][2], x[nt][kt][3]);
                            most_x = fmaxf(most_x, KIND == kKvFp8 ? fmaxf(ta + la[kt], tb + lb[kt]) : fmaxf(ta, tb));
                        }
                    if (__any_sync(0xffffffffu, most_x > kHeadroom)) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            // from the scores themselves (the first reference is too far off to go by x)
                            float full[KT][4], t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
                            for (int kt = 0; kt < KT; ++kt) {
                                const float xa = KIND == kKvFp8 ? la[kt] : 0.0f, xb = KIND == kKvFp8 ? lb[kt] : 0.0f;
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    full[kt][i] = x[nt][kt][i] == -INFINITY ? -INFINITY : sc[nt][kt][i] * (i & 1 ? f1[nt] : f0[nt]);
                                t0 = fmaxf(t0, fmaxf(full[kt][0] + xa, full[kt][2] + xb));
                                t1 = fmaxf(t1, fmaxf(full[kt][1] + xa, full[kt][3] + xb));
                            }
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) {
                                t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, o));
                                t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, o));
                            }
                            const float n0 = fmaxf(-neg0[nt], t0 - kBelowMax), n1 = fmaxf(-neg1[nt], t1 - kBelowMax);
                            const float c0 = exp2_approx(-neg0[nt] - n0), c1 = exp2_approx(-neg1[nt] - n1);
                            neg0[nt] = -n0, neg1[nt] = -n1;
                            l0[nt] *= c0, l1[nt] *= c1;
#pragma unroll
                            for (int m = 0; m < MT; ++m) {
                                acc[nt][m][0] *= c0, acc[nt][m][1] *= c1;
                                acc[nt][m][2] *= c0, acc[nt][m][3] *= c1;
                            }
#pragma unroll
                            for (int kt = 0; kt < KT; ++kt) {
                                x[nt][kt][0] = full[kt][0] - n0, x[nt][kt][1] = full[kt][1] - n1;
                                x[nt][kt][2] = full[kt][2] - n0, x[nt][kt][3] = full[kt][3] - n1;
                            }
                        }
                    }

                    // ---- weights as P^T fragments
                    uint32_t pf[NT][KT][2], pl[NT][KT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int kt = 0; kt < KT; ++kt) {
                            float w[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) w[i] = exp2_approx(x[nt][kt][i]);
                            const unsigned long long sum = add2(pair_of(l0[nt], l1[nt]), add2(pair_of(w[0], w[1]), pair_of(w[2], w[3])));
                            l0[nt] = first_of(sum), l1[nt] = second_of(sum);
                            if constexpr (KIND == kKvFp8) {
                                // a masked key's zero-filled scale keeps its weight zero
                                w[0] *= va[kt], w[1] *= va[kt], w[2] *= vb[kt], w[3] *= vb[kt];
                            }
                            // (pf: the weights rounded, pl: what that left of them)
                            if constexpr (kBf16) {
                                const uint32_t hi0 = pack_bf16(w[0], w[1]), hi1 = pack_bf16(w[2], w[3]);
                                pf[nt][kt][0] = transpose8x8(hi0), pf[nt][kt][1] = transpose8x8(hi1);
                                pl[nt][kt][0] = transpose8x8(pack_bf16(w[0] - bf16_lo(hi0), w[1] - bf16_hi(hi0)));
                                pl[nt][kt][1] = transpose8x8(pack_bf16(w[2] - bf16_lo(hi1), w[3] - bf16_hi(hi1)));
                            } else {
                                const uint32_t hi0 = pack_f16(w[0], w[1]), hi1 = pack_f16(w[2], w[3]);
                                const float2 back0 = f16x2_to_float2(hi0), back1 = f16x2_to_float2(hi1);
                                pf[nt][kt][0] = transpose8x8(hi0), pf[nt][kt][1] = transpose8x8(hi1);
                                pl[nt][kt][0] = transpose8x8(pack_f16(w[0] - back0.x, w[1] - back0.y));
                                pl[nt][kt][1] = transpose8x8(pack_f16(w[2] - back1.x, w[3] - back1.y));
                            }
                        }

                    // ---- values: the lane's keys are 2t, 2t + 1, 2t + 8, 2t + 9 of each 16, its elements run g of each row
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) {
                        const int r = 16 * kt + 2 * t;
                        constexpr int WORDS = C::EV * RB / D / 4, PIECES = D / (8 * C::EV);  // words of a run, runs of a row
#pragma unroll
                        for (int i = 0; i < PIECES; ++i) {
                            uint32_t v[4][WORDS];
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                const int row = r + (x & 1) + 8 * (x >> 1);
                                if constexpr (WORDS == 4) {
                                    const uint4 w = lds128(sv + v_offset<RB>(row, 8 * i + g));
                                    v[x][0] = w.x, v[x][1] = w.y, v[x][2] = w.z, v[x][3] = w.w;
                                } else if constexpr (WORDS == 2) {
                                    const uint2 w = lds64(sv + v_offset<RB>(row, g >> 1) + 8 * (g & 1));
                                    v[x][0] = w.x, v[x][1] = w.y;
                                } else {
                                    v[x][0] = lds32(sv + v_offset<RB>(row, g >> 2) + 4 * (g & 3));
                                }
                            }
                            // A operands: [m-tile][keys 2t, 2t + 1 / 2t + 8, 2t + 9][element 2e / 2e + 1 of the run]
                            constexpr int PAIRS = C::EV / 2;
                            uint32_t h[PAIRS][2][2];
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                if constexpr (kBf16) {
#pragma unroll
                                    for (int e = 0; e < PAIRS; ++e) {
                                        h[e][y][0] = __byte_perm(v[2 * y][e], v[2 * y + 1][e], 0x5410);
                                        h[e][y][1] = __byte_perm(v[2 * y][e], v[2 * y + 1][e], 0x7632);
                                    }
                                } else if constexpr (KIND == kKvFp8) {
                                    // the two keys' bytes side by side, then decoded
#pragma unroll
                                    for (int q = 0; q < WORDS; ++q) {
                                        uint32_t lo[2], hi[2];
                                        e4m3x4_to_f16(__byte_perm(v[2 * y][q], v[2 * y + 1][q], 0x5140), lo);
                                        e4m3x4_to_f16(__byte_perm(v[2 * y][q], v[2 * y + 1][q], 0x7362), hi);
                                        h[2 * q][y][0] = lo[0], h[2 * q][y][1] = lo[1];
                                        h[2 * q + 1][y][0] = hi[0], h[2 * q + 1][y][1] = hi[1];
                                    }
                                } else {
                                    // the two keys' codes side by side in each byte, then decoded
                                    const uint8_t* s_row = ss + CK * SB + (r + 8 * y) * SB;
#pragma unroll
                                    for (int q = 0; q < WORDS; ++q) {
                                        const int block = D == 64 ? g >> 1 : D == 128 ? g : 2 * g + q / 2;
                                        const uint32_t s_v = ue4m3x2_to_f16(s_row[block] + 0x10000u * s_row[SB + block]);
                                        const uint32_t a = v[2 * y][q], c = v[2 * y + 1][q];
                                        uint32_t even[4], odd[4];
                                        e2m1x8_to_f16((a & 0x0F0F0F0Fu) | ((c << 4) & 0xF0F0F0F0u), even);
                                        e2m1x8_to_f16(((a >> 4) & 0x0F0F0F0Fu) | (c & 0xF0F0F0F0u), odd);
#pragma unroll
                                        for (int e = 0; e < 4; ++e) {
                                            h[4 * q + e][y][0] = mul_f16x2(even[e], s_v);
                                            h[4 * q + e][y][1] = mul_f16x2(odd[e], s_v);
                                        }
                                    }
                                }
                            }
#pragma unroll
                            for (int e = 0; e < PAIRS; ++e) {
                                const int m = i * PAIRS + e;
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    mma<kBf16>(acc[nt][m], h[e][0][0], h[e][0][1], h[e][1][0], h[e][1][1], pf[nt][kt][0], pf[nt][kt][1]);
                                    mma<kBf16>(acc[nt][m], h[e][0][0], h[e][0][1], h[e][1][0], h[e][1][1], pl[nt][kt][0], pl[nt][kt][1]);
                                }
                            }
                        }
                    }
                }
            }
            // ---- the warps' results, joined in shared memory; the next segment's stream starts before
            const int seg_b = b, seg_first = unit_start, seg_rounds = span.rounds, seg_r0 = r0, seg_r1 = r1, seg_head0 = head0, seg_heads = live_heads;
            u += r1 - r0;
            __syncwarp();
            if constexpr (C::APART) more = open();
            float* merge = reinterpret_cast<float*>(smem + (C::APART ? kWarps * C::RING : 0));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    l0[nt] += __shfl_xor_sync(0xffffffffu, l0[nt], o);
                    l1[nt] += __shfl_xor_sync(0xffffffffu, l1[nt], o);
                }
            __syncthreads();  // the merge area (the rings, where it lies over them) is idle
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int h0 = 8 * nt + 2 * t;
                if (g == 0) {
                    s_m[warp][h0] = -neg0[nt], s_m[warp][h0 + 1] = -neg1[nt];
                    s_l[warp][h0] = l0[nt], s_l[warp][h0 + 1] = l1[nt];
                }
                float* to = merge + (warp * HEADS + h0) * C::LD;
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const int e = 2 * m, d = 8 * C::EV * (e / C::EV) + C::EV * g + e % C::EV;
                    *reinterpret_cast<float2*>(to + d) = make_float2(acc[nt][m][0], acc[nt][m][2]);
                    *reinterpret_cast<float2*>(to + C::LD + d) = make_float2(acc[nt][m][1], acc[nt][m][3]);
                }
            }
            __syncthreads();

            const bool whole = seg_r0 == 0 && seg_r1 == seg_rounds;
            const int which = seg_r0 == 0 ? 1 : 0, slot = which * p.max_ctas + blockIdx.x;
            for (int i = tid; i < seg_heads * (D / 4); i += kThreads) {
                const int h = i / (D / 4), d = 4 * (i - h * (D / 4));
                float m = kNoScore, l = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_m[w][h]);
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float4 x = *reinterpret_cast<const float4*>(merge + (w * HEADS + h) * C::LD + d);
                    const float c = exp2_approx(s_m[w][h] - m);
                    sum.x += x.x * c, sum.y += x.y * c, sum.z += x.z * c, sum.w += x.w * c;
                    l += s_l[w][h] * c;
                }
                if (whole) {
                    put_row<D>(p, seg_b, seg_head0 + h, d, m, l, sum, kUnit);
                } else {
                    __stcg(reinterpret_cast<float4*>(p.part_acc + ((size_t)slot * HEADS + h) * D + d), sum);
                    if (d == 0) __stcg(reinterpret_cast<float2*>(p.part_ml + ((size_t)slot * HEADS + h) * 2), make_float2(m, l));
                }
            }
            if (!whole && tid == 0)
                s_part[which] = Part{seg_b, seg_head0, seg_heads, owner(seg_first), owner(seg_first + seg_rounds - 1)};
            if constexpr (!C::APART) {
                __syncthreads();  // the merge area is the rings again
                more = open();
            }
        }

        // ---- the units of which this CTA has a part: counted at their first CTA, joined by the last to arrive
        __syncthreads();
        if (s_part[0].b >= 0 || s_part[1].b >= 0) {
            if (tid < 2) {
                // The barrier before put all the CTA's parts behind this thread, the
                // count's release puts them before it, its acquire the others' after.
                const Part& x = s_part[tid];
                uint32_t count = 0;
                if (x.b >= 0)
                    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(count) : "l"(p.counters + x.first) : "memory");
                s_last[tid] = x.b >= 0 && count == (uint32_t)(x.last - x.first);
                if (s_last[tid]) p.counters[x.first] = 0u;  // as it was found
            }
            __syncthreads();
#pragma unroll 1
            for (int i = 0; i < 2; ++i)
                if (s_last[i]) join_parts<D, HEADS>(p, s_part[i], kUnit);
        }
    }

    // ---- sequences without keys: zeros, and the sink's share alone
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
        if (span_of<TK, C::ROUND>(p, b).rounds > 0) continue;
        for (int i = tid; i < p.q_heads * (D / 4); i += kThreads) {
            const int h = i / (D / 4);
            put_row<D>(p, b, h, 4 * (i - h * (D / 4)), kNoScore, 0.0f, make_float4(0.f, 0.f, 0.f, 0.f), 1.0f);
        }
    }
}

constexpr int kMaxDevices = 64;

int sm_count() {
    static int counts[kMaxDevices];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return -1;
    if (!counts[dev] && cudaDeviceGetAttribute(&counts[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -1;
    return counts[dev];
}

// Workspace: counters, then the parts' (maximum, sum) and accumulators.
struct Layout {
    long slots, ml, acc, bytes;
};
Layout layout_of(int sms, int heads, int d) {
    Layout w;
    const long ctas = (long)sms * kMaxCtasPerSm;
    w.slots = 2 * ctas;
    w.ml = FP4B_DECODE_COUNTER_BYTES;
    w.acc = w.ml + w.slots * heads * 8;
    w.bytes = w.acc + w.slots * heads * d * 4;
    return w;
}

int unit_heads(int group) { return group <= 8 ? 8 : 16; }

template <int KIND, int D, int NT, int RUN>
cudaError_t launch(AttentionParams& p, uint8_t* workspace, cudaStream_t st) {
    using C = Cfg<KIND, D, NT>;
    static std::mutex mu;
    static int resident[kMaxDevices];  // CTAs that fit on the device at once
    auto* kernel = decode_attention_kernel<KIND, D, NT, RUN>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const int sms = sm_count();
    if (sms <= 0 || sms * kMaxCtasPerSm * 4 > FP4B_DECODE_COUNTER_BYTES || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (!resident[dev]) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
            int per = 0;
            if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, kThreads, C::SMEM);
            if (e != cudaSuccess) return e;
            resident[dev] = sms * std::max(1, std::min(per, kMaxCtasPerSm));
        }
    }
    p.group_tiles = (p.group + C::HEADS - 1) / C::HEADS;
    const Layout w = layout_of(sms, C::HEADS, D);
    p.max_ctas = sms * kMaxCtasPerSm;
    p.counters = reinterpret_cast<uint32_t*>(workspace);
    p.part_ml = reinterpret_cast<float*>(workspace + w.ml);
    p.part_acc = reinterpret_cast<float*>(workspace + w.acc);
    // No more CTAs than the page table has rounds for (and one for each empty sequence's row).
    const long keys = (long)p.table_width << p.page_shift;
    const long most = (long)p.batch * std::max(1l, (keys + C::ROUND - 1) / C::ROUND * p.cache.kv_heads * p.group_tiles);
    return launch_chained(kernel, dim3((unsigned)std::min<long>(resident[dev], most)), kThreads, C::SMEM, st, p);
}

// Pages of 16 where 32 keys are worked on at once have a form of their own: 3 x
// 131072 keys of nvfp4, D = 64: 60.1 us, where pages of 64 by whole parts take 58.3 and
// pages of 8 key by key 63.2 (one kernel with all three cost each of them 1.3 us more,
// in registers).
template <int KIND, int D, int NT>
cudaError_t launch_run(AttentionParams& p, uint8_t* workspace, cudaStream_t st) {
    constexpr int CK = Cfg<KIND, D, NT>::CK;
    if (p.cache.page_size >= CK) return launch<KIND, D, NT, CK>(p, workspace, st);
    if constexpr (CK > 16)
        if (p.cache.page_size >= 16) return launch<KIND, D, NT, 16>(p, workspace, st);
    return launch<KIND, D, NT, 1>(p, workspace, st);
}

template <int KIND, int D>
cudaError_t launch_heads(AttentionParams& p, uint8_t* workspace, cudaStream_t st) {
    return unit_heads(p.group) == 8 ? launch_run<KIND, D, 1>(p, workspace, st) : launch_run<KIND, D, 2>(p, workspace, st);
}

template <int KIND>
cudaError_t launch_dim(AttentionParams& p, uint8_t* workspace, cudaStream_t st) {
    return p.cache.head_dim == 64    ? launch_heads<KIND, 64>(p, workspace, st)
           : p.cache.head_dim == 128 ? launch_heads<KIND, 128>(p, workspace, st)
                                     : launch_heads<KIND, 256>(p, workspace, st);
}

}  // namespace
}  // namespace fp4b

using namespace fp4b;

FP4B_EXPORT long fp4b_decode_attention_workspace(int q_heads, int kv_heads, int head_dim) {
    if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || head_dim <= 0) {
        set_last_error("fp4b_decode_attention_workspace: bad head counts");
        return -1;
    }
    const int sms = sm_count();
    if (sms <= 0) {
        cudaGetLastError();
        set_last_error("fp4b_decode_attention_workspace: no device");
        return -1;
    }
    return layout_of(sms, unit_heads(q_heads / kv_heads), head_dim).bytes;
}

FP4B_EXPORT int fp4b_decode_attention(const fp4b_decode* call, void* stream) {
    if (!call) {
        set_last_error("fp4b_decode_attention: null arguments");
        return -1;
    }
    const fp4b_decode& c = *call;
    const fp4b_kv_cache* cache = c.cache;
    const char* why = kv_cache_check(cache);
    if (!why && (c.batch < 0 || c.q_heads <= 0 || c.q_heads % cache->kv_heads))
        why = "query heads must be a multiple of the cache's heads";
    if (!why && c.batch > 0 && (!c.q || !c.out || !c.seq_lens || (c.table_width > 0 && !c.page_table))) why = "null tensor";
    if (!why && (c.table_width < 0 || c.table_stride < c.table_width)) why = "bad page table";
    if (!why && (long)c.table_width * cache->page_size > 0x7fff0000L) why = "more than 2^31 keys in one sequence";
    if (!why && (long)c.batch * c.q_heads > 0x7fffffffL) why = "more than 2^31 output rows";
    if (!why && (((long)c.table_width * cache->page_size + 63) / 64 + kSegmentRounds) * c.q_heads > 0x7fffffffL / std::max(c.batch, 1))
        why = "more than 2^31 tiles of 64 keys in one call";
    if (!why && (c.window < 0 || !std::isfinite(c.scale))) why = "window must not be negative, scale finite";
    if (!why && ((reinterpret_cast<uintptr_t>(c.q) & 7) || c.q_sb % 4 || c.q_sh % 4 || (reinterpret_cast<uintptr_t>(c.out) & 15)))
        why = "queries must be 8-byte aligned rows, the output 16-byte aligned";
    if (!why && c.batch > 0 &&
        (!c.workspace || (reinterpret_cast<uintptr_t>(c.workspace) & 15) ||
         c.workspace_bytes < fp4b_decode_attention_workspace(c.q_heads, cache->kv_heads, cache->head_dim)))
        why = "workspace too small or misaligned";
    if (why) {
        set_last_error("fp4b_decode_attention: %s", why);
        return -1;
    }
    if (c.batch == 0) return 0;
    AttentionParams p{};
    p.q = static_cast<const uint16_t*>(c.q), p.q_sb = c.q_sb, p.q_sh = c.q_sh;
    p.batch = c.batch, p.q_heads = c.q_heads, p.group = c.q_heads / cache->kv_heads;
    p.cache = *cache;
    while ((1 << p.page_shift) < cache->page_size) ++p.page_shift;
    p.table = c.page_table, p.table_stride = c.table_stride, p.table_width = c.table_width;
    p.lens = c.seq_lens, p.scale2 = c.scale * kLog2e, p.window = c.window, p.sinks = c.sinks;
    p.out = static_cast<uint16_t*>(c.out), p.lse = c.lse, p.err = device_error_word();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint8_t* ws = static_cast<uint8_t*>(c.workspace);
    const cudaError_t e = cache->kind == kKvBf16 ? launch_dim<kKvBf16>(p, ws, st)
                          : cache->kind == kKvFp8 ? launch_dim<kKvFp8>(p, ws, st)
                                                  : launch_dim<kKvNvfp4>(p, ws, st);
    return launch_status(e, "fp4b_decode_attention");
}
