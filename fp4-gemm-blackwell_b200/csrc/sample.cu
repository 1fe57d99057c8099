// sample.cu -- the next token of each row of logits, by temperature, top-k,
// top-p and min-p, from a given uniform number.
//
// The tokens of a row are taken in the order of their logits, largest first,
// equal ones by index (-inf and NaN are no candidates), with the weights
//   w_i = exp((l_i - max) / T).
// Kept are: the first k of them; of those, with W their weights' sum, the ones
// before which less than p * W lies (always the first); and of those the ones
// with w_i >= min_p.  Each is a prefix of the order, so what is kept is a prefix
// too, and has a mass; the token is the first whose weights' sum, up to it and
// with it, is more than u times that mass.  T = 0: the first token.
//
// So every question is the same: where in the order does a running count, or a
// running sum of weights, pass a number.  It is answered without sorting, by a
// histogram of the logits' leading bits in the order's own direction: a bin has
// a count and a mass.  Where the leading bits are all the bits (BF16), a bin is
// one logit: its mass is its count times one weight, no element needs an
// exponential, and a place in it is a place among equal logits, found by
// counting.  Where a bin has more bits (FP16, FP32, and the logits nearest to
// zero), elements add their weights to it, and the bin at hand is looked into: up to 512
// candidates are listed and ranked one by one, more are split 8 bits at a time,
// until they are few or all one logit.
//
// Bins.  bits 16 up of the logit as FP32: sign, exponent, 7 bits.  The weights
// that matter lie within 46 of the maximum (e^-46 * 2^32 is below 2^-33, and u
// is at most 1 - 2^-24), so exponents from the largest of that range down are
// 16 octaves x 128 bins for each sign; smaller magnitudes are one bin between
// them, and what lies below the range is in none.
//
// Sums.  Which token it is turns on sums over the whole row that lie next to a
// border, so they are exact: a weight is an exponential in FP64 (to about 1e-14),
// rounded once to a whole multiple of 2^-bits, bits the most that cannot overflow
// 64 (44 at 2^18 tokens), and sums of these do not depend on their order.
//
// A row belongs to a cluster of 1 to 8 CTAs, as many as give all rows' CTAs a
// place on the GPU at once; each counts a slice, then merges its share of the
// bins over distributed shared memory into the first CTA's, which walks them.
// (Twice as many CTAs as fit at once: 64 x 131072 49 us where one wave takes 33.)
//
// Measured on B200, BF16: 256 x 131072 90 us, of which the bytes would take 10. The
// row's phases follow one another in all CTAs alike: the maximum 5 us, the counting
// 26 (42 instructions for 32 logits in all, half the issue slots in use, waits for
// instructions among the rest), the token's place by another reading 9; what the 4097
// weights in FP64, the scans and the questions take of the rest was not measured apart.
// 64 x 131072 33 us, 1 x 32768 15 (eight CTAs, five meetings of the cluster of 0.5 us,
// three questions); FP32 with all filters, 7 x 100003, 42 us (an exponential and three
// atomics an element, three lists). 256 x 131072 of FP16 194 us, of FP32 223.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <mutex>

#include "decode_core.cuh"
#include "fp4b_internal.h"

#define FP4B_EXPORT extern "C" __attribute__((visibility("default")))

namespace fp4b {
namespace {

using namespace decode;
namespace cg = cooperative_groups;
typedef unsigned long long u64;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kOctaves = 16;
constexpr int kSide = kOctaves * 128;      // bins of a sign
constexpr int kBins = 2 * kSide + 1;       // the one between them is bin kSide
constexpr int kPer = (kBins + kThreads - 1) / kThreads;  // bins a thread walks
constexpr float kReach = 46.0f;
constexpr int kMaxCluster = 8;
constexpr int kBatch = 4;
constexpr int kList = kThreads;  // candidates of a run that are ranked one by one
constexpr int kMaxDevices = 64;

struct SampleParams {
    const void* logits;
    long stride;
    const float* u;
    const float* temperature;  // null: temperature1, and so on
    const int* top_k;
    const float* top_p;
    const float* min_p;
    float temperature1, top_p1, min_p1;
    int top_k1;
    long long* tokens;
    float* probs;
    int vocab, slice;  // slice: elements a CTA, a multiple of 8
    int bits;          // of a weight behind the point
};

enum LogitType { kBf16 = FP4B_LOGITS_BF16, kFp16 = FP4B_LOGITS_FP16, kFp32 = FP4B_LOGITS_FP32 };

template <int TYPE>
struct Traits {
    using T = uint16_t;
    static constexpr int PER = 8;                            // elements of 16 bytes
    static constexpr int FREE = TYPE == kBf16 ? 16 : 13;     // low bits of the FP32 form that are zero
    static constexpr uint32_t NONE = TYPE == kBf16 ? 0xFF80u : 0xFC00u;  // -inf
};
template <>
struct Traits<kFp32> {
    using T = uint32_t;
    static constexpr int PER = 4;
    static constexpr int FREE = 0;
    static constexpr uint32_t NONE = 0xFF800000u;
};

// FP32 bits of a logit; what is no candidate (NaN) becomes -inf, -0 becomes +0.
__device__ __forceinline__ uint32_t tidy(uint32_t b) {
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 0xFF800000u;
    return b == 0x80000000u ? 0u : b;
}
template <int TYPE>
__device__ __forceinline__ uint32_t bits_of(typename Traits<TYPE>::T raw) {
    if constexpr (TYPE == kBf16) return tidy((uint32_t)raw << 16);
    else if constexpr (TYPE == kFp16) return tidy(__float_as_uint(__half2float(__ushort_as_half(raw))));
    else return tidy(raw);
}

// Keys grow with the logits.
__device__ __forceinline__ uint32_t key_of(uint32_t b) { return b & 0x80000000u ? ~b : b | 0x80000000u; }
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }
constexpr uint32_t kMinusInf = 0x007FFFFFu;  // key of -inf

// A run of keys [first, first + 2^size): all the logits of one bin.
struct Run {
    uint32_t first;
    int size;
    // the logit of a run of one (of BF16's or FP16's: whose other bits are zero)
    __device__ __forceinline__ float logit() const { return logit_of(first & 0x80000000u ? first : first + ((1u << size) - 1u)); }
};

struct Row {
    float max;
    double inv;        // 1 / T
    int lo;            // leading bits of the smallest magnitude with a bin of its own
    double one;        // 2^bits
    const double* powers;  // 2^(i / 32), i < 32, in shared memory
    // Weights: of the largest 1, by a table-driven exponential (Tang's method).  exp(x) = 2^(n / 32) exp(y), n the nearest whole number
    // to 32 x / ln 2, |y| <= ln 2 / 64, exp(y) by its series up to y^5 (the next term is
    // below 3e-15): to within about 1e-14, with a third of the library's instructions.
    __device__ __forceinline__ double share(float l) const {
        const double x = l == max ? 0.0 : fmax(((double)l - (double)max) * inv, -700.0);  // (-inf counts as that, whose weight is 0)
        const double shifted = fma(x, 46.166241308446828384, 6755399441055744.0);  // 32 / ln 2; 1.5 * 2^52 leaves a whole number in the low bits
        const int n = __double2loint(shifted);
        const double y = fma(shifted - 6755399441055744.0, -0.021660849392498290195, x);  // ln 2 / 32
        double e = fma(y, 1.0 / 120.0, 1.0 / 24.0);
        e = fma(e, y, 1.0 / 6.0);
        e = fma(e, y, 0.5);
        e = fma(e, y, 1.0);
        e = fma(e, y, 1.0) * powers[n & 31];
        return __hiloint2double(__double2hiint(e) + ((n >> 5) << 20), __double2loint(e));
    }
    __device__ __forceinline__ u64 whole(double w) const { return (u64)__double2ll_rn(w * one); }
    __device__ __forceinline__ u64 weight(float l) const { return whole(share(l)); }
    // Bin of a candidate's bits, -1 for none.
    __device__ __forceinline__ int bin(uint32_t b) const {
        const int i = (int)((b >> 16) & 0x7FFFu) - lo;
        if (i < 0) return kSide;
        if (i >= kSide) return b & 0x80000000u ? -1 : 0;
        return b & 0x80000000u ? kSide + 1 + i : kSide - 1 - i;
    }
    __device__ __forceinline__ Run run(int bin) const {
        if (bin == kSide) {
            // keys 2^31 - n up to 2^31 + n - 1, n = lo * 2^16
            const uint32_t n = (uint32_t)lo << 16;
            return Run{0x80000000u - n, n ? 33 - __clz(n - 1u) : 0};  // 2^size >= 2 n
        }
        if (bin < kSide) return Run{0x80000000u + ((uint32_t)(lo + kSide - 1 - bin) << 16), 16};
        return Run{0x80000000u - ((uint32_t)(lo + bin - kSide) << 16), 16};
    }
};

struct Place {  // of a crossing: a bin or a part of one, and what lies before it
    int bin;
    uint32_t before, count;
    u64 mass_before;
};

// What the first CTA tells the others to do next.
struct Command {
    int what;  // 0: done, 1: split a run, 2: find the token, 3: list a run
    Run run;
    int cta;
    uint32_t rank;
    float prob;
};

struct Shared {
    uint32_t hist[kBins];
    uint32_t sub_count[256];
    u64 sub_mass[256];
    double powers[32];
    float max[kMaxCluster], warp_max[kWarps];
    u64 near_mass;  // of the bin between, where the others have one logit each
    uint32_t warp_count[kWarps];
    u64 warp_mass[kWarps];
    u64 least_mass;  // of the row's candidates with w >= min_p
    u64 list[kList];  // key and what the index lacks of 2^32 - 1: larger ones come first
    u64 list_weight[kList];
    uint32_t listed;
    u64 answer_mass, answer_weight;
    int answer_token;
    Place place;
    Command command;
    int token;
};

// Sums of the threads before this one (exclusive), over the CTA.
__device__ __forceinline__ void scan(Shared& s, uint32_t& count, u64& mass) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t c0 = count;
    const u64 m0 = mass;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t c = __shfl_up_sync(0xffffffffu, count, o);
        const u64 m = __shfl_up_sync(0xffffffffu, mass, o);
        if (lane >= o) count += c, mass += m;
    }
    __syncthreads();
    if (lane == 31) s.warp_count[warp] = count, s.warp_mass[warp] = mass;
    __syncthreads();
    for (int w = 0; w < warp; ++w) count += s.warp_count[w], mass += s.warp_mass[w];
    count -= c0, mass -= m0;
}

// Adds to a sum in shared memory by its halves: where many threads meet at one sum (equal
// logits, zeros of a mask or of a padded vocabulary) an addition of 64 bits, which is a loop
// of comparisons and exchanges, goes round once for each of them.  (256 x 131072, all logits
// equal: FP32 16.7 ms so, 0.94 by halves; half of BF16 logits zeros 8.2 and 0.40.)
__device__ __forceinline__ void add_mass(u64* at, u64 m) {
    uint32_t* const half = reinterpret_cast<uint32_t*>(at);
    const uint32_t low = (uint32_t)m, old = atomicAdd(half, low);
    const uint32_t high = (uint32_t)(m >> 32) + (old + low < low ? 1u : 0u);
    if (high) atomicAdd(half + 1, high);
}

enum Kind { kByCount, kByMassBefore, kByMassWith };

// The question of one crossing.  kByCount: the last of the first k.
// kByMassBefore: the last before which less than `target` lies.  kByMassWith:
// the first with which more than `target` lies.
struct Question {
    Kind kind;
    uint32_t k;
    double target;
    // Does it lie in a bin with `count` and `mass`, `before` and `mass_before` before it?
    __device__ __forceinline__ bool in(uint32_t before, u64 mass_before, uint32_t count, u64 mass) const {
        if (count == 0) return false;
        if (kind == kByCount) return before < k && k <= before + count;
        if (kind == kByMassBefore) {
            // the last bin before which less than the target lies: its mass reaches it
            return (double)mass_before < target && (double)(mass_before + mass) >= target;
        }
        return (double)mass_before <= target && (double)(mass_before + mass) > target;
    }
    // How many of `count` elements of weight w lie up to and with it.
    __device__ __forceinline__ uint32_t part(uint32_t before, u64 mass_before, uint32_t count, u64 w) const {
        if (kind == kByCount) return k - before;
        if (w == 0) return 1;
        const double d = floor((target - (double)mass_before) / (double)w);
        uint32_t n = d < 1.0 ? 1u : d >= (double)count ? count : (uint32_t)d;
        if (kind == kByMassBefore) {
            while (n < count && (double)(mass_before + (u64)n * w) < target) ++n;
            while (n > 1 && (double)(mass_before + (u64)(n - 1) * w) >= target) --n;
        } else {
            while (n < count && (double)(mass_before + (u64)n * w) <= target) ++n;
            while (n > 1 && (double)(mass_before + (u64)(n - 1) * w) > target) --n;
        }
        return n;
    }
};

// Sums of one bin's or part's entry over the cluster's CTAs, read side by side.
template <typename T>
__device__ __forceinline__ T over_cluster(cg::cluster_group& cluster, T* at, int ctas) {
    T v[kMaxCluster], sum = 0;
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) v[c] = c < ctas ? *cluster.map_shared_rank(at, c) : T(0);
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) sum += v[c];
    return sum;
}

template <int TYPE>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleParams p) {
    using T = typename Traits<TYPE>::T;
    constexpr int PER = Traits<TYPE>::PER, FREE = Traits<TYPE>::FREE;
    constexpr bool kMasses = FREE < 16;  // bins of more than one logit
    extern __shared__ __align__(16) uint8_t dynamic[];
    // With masses: this CTA's [kBins]; in a cluster: what the first CTA has of all of them, masses and counts.
    u64* const my_mass = reinterpret_cast<u64*>(dynamic);
    u64* const all_mass = my_mass + (kMasses ? kBins : 0);
    uint32_t* const all_count = reinterpret_cast<uint32_t*>(all_mass + (kMasses ? kBins : 0));
    __shared__ Shared s;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), me = (int)cluster.block_rank();
    const long row = blockIdx.x / ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    if (ctas > 1) ptx::cluster_start_arrive();
    chain();

    // ---- this CTA's slice; a warp goes over a run of its own, 16 bytes a lane, in the order of the indices
    const int first = min(me * p.slice, p.vocab), last = min(first + p.slice, p.vocab);
    const T* const logits = static_cast<const T*>(p.logits) + row * p.stride;
    // pieces of 16 aligned bytes: piece i holds elements [i * PER - shift, + PER) of the slice
    const int shift = (int)((reinterpret_cast<uintptr_t>(logits + first) & 15) / sizeof(T));
    const int pieces = last > first ? (last - first + shift + PER - 1) / PER : 0;
    const int warp_pieces = ((pieces + kWarps - 1) / kWarps + 31) / 32 * 32;
    const int piece0 = min(warp * warp_pieces, pieces), piece1 = min(piece0 + warp_pieces, pieces);
    // Piece i as it lies there, what is outside the slice as -inf.
    auto load = [&](int i) {
        const int at = first + i * PER - shift;
        if (at >= first && at + PER <= last) return __ldg(reinterpret_cast<const uint4*>(logits + at));
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const uint32_t v = at + e >= first && at + e < last ? (uint32_t)logits[at + e] : Traits<TYPE>::NONE;
            if constexpr (PER == 4) w[e] = v;
            else w[e / 2] |= v << (e & 1) * 16;
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    auto bits = [&](const uint4& v, int e) {  // of its element e, as FP32
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if constexpr (PER == 4) return bits_of<TYPE>(w[e]);
        else return bits_of<TYPE>((uint16_t)(e & 1 ? w[e / 2] >> 16 : w[e / 2]));
    };

    // f of all pieces, kBatch of them on their way at once.
    auto over_pieces = [&](auto f) {
        uint4 next[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
            if (piece0 + lane + 32 * k < piece1) next[k] = load(piece0 + lane + 32 * k);
        for (int i = piece0 + lane; i < piece1; i += 32 * kBatch) {
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                if (i + 32 * k >= piece1) break;
                const uint4 v = next[k];
                if (i + 32 * (k + kBatch) < piece1) next[k] = load(i + 32 * (k + kBatch));
                f(v);
            }
        }
    };

    // ---- the maximum
    float most = -INFINITY;
    if constexpr (TYPE == kBf16) {
        __nv_bfloat162 top = __floats2bfloat162_rn(-INFINITY, -INFINITY);
#pragma unroll 4
        for (int i = piece0 + lane; i < piece1; i += 32) {
            const uint4 v = load(i);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) top = __hmax2(top, *reinterpret_cast<const __nv_bfloat162*>(&w[k]));  // (not a NaN)
        }
        most = fmaxf(__low2float(top), __high2float(top));
    } else {
#pragma unroll 4
        for (int i = piece0 + lane; i < piece1; i += 32) {
            const uint4 v = load(i);
#pragma unroll
            for (int e = 0; e < PER; ++e) most = fmaxf(most, __uint_as_float(bits(v, e)));
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    for (int i = tid; i < kBins; i += kThreads) {
        s.hist[i] = 0;
        if (kMasses) my_mass[i] = 0;
    }
    if (tid == 0) s.near_mass = 0, s.least_mass = 0, s.token = 0x7fffffff;
    if (lane == 0) s.warp_max[warp] = most;
    if (tid < 32) s.powers[tid] = exp2((double)tid / 32.0);
    __syncthreads();
    if (ctas > 1) ptx::cluster_start_wait();  // the others have started: their shared memory is there
    if (warp == 0) {
        most = lane < kWarps ? s.warp_max[lane] : -INFINITY;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        if (lane < ctas) cluster.map_shared_rank(s.max, lane)[me] = most;
    }
    cluster.sync();
    most = s.max[0];
    for (int c = 1; c < ctas; ++c) most = fmaxf(most, s.max[c]);

    const float t = p.temperature ? p.temperature[row] : p.temperature1;
    const bool greedy = !(t > 0.0f);
    if (most == -INFINITY) {  // no candidates
        if (me == 0 && tid == 0) {
            p.tokens[row] = -1;
            if (p.probs) p.probs[row] = 0.0f;
        }
        return;
    }
    Row r;
    r.max = most == 0.0f ? 0.0f : most;                // (+0)
    r.inv = fmax(1.0 / (double)t, 0x1p-1000);          // (an infinite T: all alike)
    r.one = (double)(1ull << p.bits), r.powers = s.powers;
    {
        const uint32_t far = __float_as_uint(fmaf(-kReach, t, most)) & 0x7FFFFFFFu, top = __float_as_uint(most) & 0x7FFFFFFFu;
        const int octave = (int)(max(min(far, 0x7F800000u), top) >> 23);
        // (an octave at least: zeros of both signs are in the bin between, as one)
        r.lo = max(octave - (kOctaves - 1), 1) << 7;
    }
    const float least = p.min_p ? p.min_p[row] : p.min_p1;
    const bool has_least = least > 0.0f;

    // ---- the token of a run of equal logits: the rank-th of them, in this CTA's slice
    auto find = [&](Run run, uint32_t rank, float prob) {
        const uint32_t exact = (__float_as_uint(run.logit()) >> 16) * 0x10001u;  // BF16, twice
        auto hits = [&](int i) {  // of piece i, as bits
            uint32_t mask = 0;
            if (i >= piece1) return mask;
            const uint4 v = load(i);
            if constexpr (TYPE == kBf16) {
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t same = __vcmpeq2(w[k], exact);
                    if (exact == 0u) same |= __vcmpeq2(w[k], 0x80008000u);
                    mask |= ((same & 1u) | ((same >> 15) & 2u)) << 2 * k;
                }
            } else {
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    const uint32_t key = key_of(bits(v, e));
                    if (key > kMinusInf && key >= run.first && ((key - run.first) >> run.size) == 0) mask |= 1u << e;
                }
            }
            return mask;
        };
        uint32_t mine = 0;
#pragma unroll 4
        for (int i = piece0 + lane; i < piece1; i += 32) mine += __popc(hits(i));
        const uint32_t all = __reduce_add_sync(0xffffffffu, mine);
        __syncthreads();
        if (lane == 0) s.warp_count[warp] = all;
        __syncthreads();
        uint32_t before = 0;
        for (int w = 0; w < warp; ++w) before += s.warp_count[w];
        if (rank < before || rank >= before + all) return;
        rank -= before;
        for (int i = piece0; i < piece1; i += 32) {
            uint32_t mask = hits(i + lane);
            const uint32_t here = __popc(mask);
            uint32_t upto = here;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t other = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += other;
            }
            if (rank < upto && rank >= upto - here) {
                for (uint32_t k = rank - (upto - here); k > 0; --k) mask &= mask - 1;
                p.tokens[row] = first + (i + lane) * PER - shift + (__ffs(mask) - 1);
                if (p.probs) p.probs[row] = prob;
            }
            const uint32_t tile = __shfl_sync(0xffffffffu, upto, 31);
            if (rank < tile) return;
            rank -= tile;
        }
    };

    if (greedy) {  // the first of the largest: the least index
        int at = 0x7fffffff;
        for (int i = piece0 + lane; i < piece1 && at == 0x7fffffff; i += 32) {
            const uint4 v = load(i);
#pragma unroll
            for (int e = PER - 1; e >= 0; --e)
                if (__uint_as_float(bits(v, e)) == most) at = first + i * PER - shift + e;
        }
        at = __reduce_min_sync(0xffffffffu, at);
        Shared* home = cluster.map_shared_rank(&s, 0);
        if (lane == 0 && at != 0x7fffffff) atomicMin(&home->token, at);
        cluster.sync();
        if (me == 0 && tid == 0) {
            p.tokens[row] = s.token;
            if (p.probs) p.probs[row] = 1.0f;
        }
        return;
    }

    // ---- counts (and masses) of the slice's bins
    u64 kept_mass = 0, near_mass = 0;
    uint32_t near_count = 0, zeros = 0;  // (zeros, which a mask or a padded vocabulary has many of, share one weight)
    auto heavy = [&](int bin, float l) {  // of a bin of more than one logit
        const double w = r.share(l);
        const u64 m = r.whole(w);
        if (kMasses) add_mass(&my_mass[bin], m);
        else near_mass += m, ++near_count;
        if (has_least && w >= (double)least) kept_mass += m;
    };
    if constexpr (TYPE == kBf16) {
        // infinities and NaN lie above these
        const int most_plus = min(kSide, 0x7F81 - r.lo), most_minus = min(kSide, 0x7F80 - r.lo);
        over_pieces([&](const uint4& v) {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const int h = (int)(e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu), k = (h & 0x7FFF) - r.lo;
                const bool minus = h & 0x8000;
                if (k >= 0) {
                    if (k < (minus ? most_minus : most_plus)) atomicAdd(&s.hist[minus ? kSide + 1 + k : kSide - 1 - k], 1u);
                } else if ((h & 0x7FFF) == 0) {
                    ++zeros;
                } else {
                    heavy(kSide, __uint_as_float((uint32_t)h << 16));
                }
            }
        });
    } else {
        over_pieces([&](const uint4& v) {
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const uint32_t b = bits(v, e);
                if (b == 0xFF800000u) continue;
                if (b == 0u) {
                    ++zeros;
                    continue;
                }
                const int bin = r.bin(b);
                if (bin < 0) continue;
                atomicAdd(&s.hist[bin], 1u);
                heavy(bin, __uint_as_float(b));
            }
        });
    }
    if (zeros + near_count) {
        const double w = r.share(0.0f);
        const u64 m = r.whole(w) * zeros;
        if (has_least && w >= (double)least) kept_mass += m;
        atomicAdd(&s.hist[kSide], zeros + near_count);
        add_mass(kMasses ? &my_mass[kSide] : &s.near_mass, near_mass + m);
    }
    if (ctas > 1) cluster.sync();
    else __syncthreads();

    // ---- in a cluster: this CTA's share of the bins over all slices, into the first CTA's
    if (ctas > 1) {
        uint32_t* to_count = cluster.map_shared_rank(all_count, 0);
        u64* to_mass = cluster.map_shared_rank(all_mass, 0);
        for (int i = me * kThreads + tid; i < kBins; i += ctas * kThreads) {
            to_count[i] = over_cluster(cluster, &s.hist[i], ctas);
            if (kMasses) to_mass[i] = over_cluster(cluster, &my_mass[i], ctas);
        }
        Shared* home = cluster.map_shared_rank(&s, 0);
        if (!kMasses && me != 0 && tid == 0 && s.near_mass) atomicAdd(&home->near_mass, s.near_mass);
        if (me != 0) {
            if (has_least) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) kept_mass += __shfl_xor_sync(0xffffffffu, kept_mass, o);
                if (lane == 0 && kept_mass) atomicAdd(&home->least_mass, kept_mass);
            }
            kept_mass = 0;
        }
        cluster.sync();
    }
    const uint32_t* const count = ctas > 1 ? all_count : s.hist;
    const u64* const mass = ctas > 1 ? all_mass : my_mass;

    // ---- the first CTA asks; a run of more than one logit is split by all of them
    auto split = [&](Run run) {  // all CTAs: counts and masses of the run's 256 parts, ascending
        for (int i = tid; i < 256; i += kThreads) s.sub_count[i] = 0, s.sub_mass[i] = 0;
        __syncthreads();
        const int down = max(run.size - 8, 0);
        over_pieces([&](const uint4& v) {
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const uint32_t b = bits(v, e), key = key_of(b);
                if (key <= kMinusInf || key < run.first || (run.size < 32 && ((key - run.first) >> run.size) != 0)) continue;
                const uint32_t part = (key - run.first) >> down;
                if (part > 255) continue;
                if (run.size > 16 && r.bin(b) != kSide) continue;  // (the bin between is less than its power of two)
                atomicAdd(&s.sub_count[part], 1u);
                add_mass(&s.sub_mass[part], r.weight(__uint_as_float(b)));
            }
        });
        cluster.sync();
    };

    auto list = [&](Run run) {  // all CTAs: the run's candidates into the first CTA's list
        Shared* home = cluster.map_shared_rank(&s, 0);
        for (int i = piece0 + lane; i < piece1; i += 32) {
            const uint4 v = load(i);
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const uint32_t b = bits(v, e), key = key_of(b);
                if (key > kMinusInf && key - run.first < (1u << run.size) && (run.size <= 16 || r.bin(b) == kSide)) {
                    const uint32_t at = atomicAdd(&home->listed, 1u);
                    if (at < kList) home->list[at] = (u64)key << 32 | (0xFFFFFFFFu - (uint32_t)(first + i * PER - shift + e));
                }
            }
        }
        cluster.sync();
    };

    if (me != 0) {
        for (;;) {
            cluster.sync();  // a command is there
            const Command c = s.command;
            if (c.what == 3) {
                list(c.run);
            } else if (c.what == 1) {
                split(c.run);
                cluster.sync();  // the parts were read
            } else {
                if (c.what == 2 && c.cta == me) find(c.run, c.rank, c.prob);
                return;
            }
        }
    }
    auto tell = [&](const Command& c) {
        if (tid < ctas) cluster.map_shared_rank(&s, tid)->command = c;
        cluster.sync();
    };

    // ---- a thread's bins, kPer of them: what lies before them, and in them
    uint32_t my_before = 0, my_count = 0;
    u64 my_mass_before = 0, my_total = 0;
    // (all weights side by side: their exponentials have long chains)
    u64 bin_mass[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int i = min(tid * kPer + k, kBins - 1);
        const bool there = tid * kPer + k < kBins;
        const uint32_t n = there ? count[i] : 0u;
        if constexpr (kMasses) {
            bin_mass[k] = there ? mass[i] : 0;
        } else {
            const double w = r.share(r.run(i).logit());
            bin_mass[k] = i == kSide ? (there ? s.near_mass : 0) : r.whole(w) * n;
            if (has_least && i != kSide && w >= (double)least) kept_mass += bin_mass[k];
        }
        my_count += n, my_total += bin_mass[k];
    }
    my_before = my_count, my_mass_before = my_total;
    scan(s, my_before, my_mass_before);
    if (has_least) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) kept_mass += __shfl_xor_sync(0xffffffffu, kept_mass, o);
        if (lane == 0 && kept_mass) atomicAdd(&s.least_mass, kept_mass);
    }
    if (tid == kThreads - 1) s.place.before = my_before + my_count, s.place.mass_before = my_mass_before + my_total;
    __syncthreads();
    u64 total = s.place.mass_before;
    const uint32_t candidates = s.place.before;
    const u64 least_mass = s.least_mass;
    __syncthreads();

    struct Answer {
        u64 mass;       // up to the place, with it
        Run run;        // of its logit
        uint32_t rank;  // among equal ones
        int bin;        // >= 0: counts are the bins', else the parts'
        u64 weight;
        int token;      // >= 0: it is known
    };
    // (a question's place is among the candidates)
    auto ask = [&](const Question& q) {
        if (q.in(my_before, my_mass_before, my_count, my_total)) {
            uint32_t n = my_before;
            u64 m = my_mass_before;
#pragma unroll
            for (int k = 0; k < kPer; ++k) {
                const int i = tid * kPer + k;
                const uint32_t here = i < kBins ? count[i] : 0;
                if (q.in(n, m, here, bin_mass[k])) s.place = Place{i, n, here, m};
                n += here, m += bin_mass[k];
            }
        }
        __syncthreads();
        Place x = s.place;
        Run run = r.run(x.bin);
        int bin = x.bin;
        while (run.size > FREE) {
            Command c{};
            c.what = 1, c.run = run;
            if (x.count <= kList && run.size <= 24) {
                // few: each is ranked among all of them
                c.what = 3;
                if (tid == 0) s.listed = 0;
                tell(c);
                list(run);
                const int n = (int)min(s.listed, (uint32_t)kList);
                const u64 mine = tid < n ? s.list[tid] : 0;
                const u64 w = tid < n ? r.weight(logit_of((uint32_t)(mine >> 32))) : 0;
                s.list_weight[tid] = w;
                __syncthreads();
                if (tid < n) {
                    uint32_t before = x.before;
                    u64 m = x.mass_before;
#pragma unroll 4
                    for (int j = 0; j < n; ++j)
                        if (s.list[j] > mine) ++before, m += s.list_weight[j];
                    if (q.in(before, m, 1, w)) s.answer_mass = m + w, s.answer_weight = w, s.answer_token = (int)(0xFFFFFFFFu - (uint32_t)mine);
                }
                __syncthreads();
                return Answer{s.answer_mass, run, 0, -1, s.answer_weight, s.answer_token};
            }
            tell(c);
            split(run);
            // parts from the last (the largest logits) down, one a thread
            const int i = 255 - tid;
            uint32_t n = 0;
            u64 m = 0;
            if (i >= 0) n = over_cluster(cluster, &s.sub_count[i], ctas), m = over_cluster(cluster, &s.sub_mass[i], ctas);
            const uint32_t part_count = n;
            const u64 part_mass = m;
            scan(s, n, m);
            n += x.before, m += x.mass_before;
            if (i >= 0 && q.in(n, m, part_count, part_mass)) s.place = Place{i, n, part_count, m};
            cluster.sync();
            x = s.place;
            const int down = max(run.size - 8, 0);
            run = Run{run.first + ((uint32_t)x.bin << down), down};
            bin = -1;
        }
        Answer a;
        a.weight = r.weight(run.logit());
        const uint32_t part = q.part(x.before, x.mass_before, x.count, a.weight);
        a.mass = x.mass_before + (u64)part * a.weight;
        a.run = run, a.rank = part - 1, a.bin = bin, a.token = -1;
        __syncthreads();
        return a;
    };

    // ---- what is kept: the sum of its weights
    {
        const int k = p.top_k ? p.top_k[row] : p.top_k1;
        if (k > 0 && (uint32_t)k < candidates) total = ask(Question{kByCount, (uint32_t)k, 0.0}).mass;
        const float nucleus = p.top_p ? p.top_p[row] : p.top_p1;
        u64 smaller = total;
        // (at least the first token: a target of nothing is less than the least weight)
        if (nucleus < 1.0f) smaller = min(smaller, ask(Question{kByMassBefore, 0, fmax((double)nucleus * (double)total, 0.5)}).mass);
        if (has_least) smaller = min(smaller, least_mass ? least_mass : (u64)r.one);
        total = smaller;
    }
    const float given = p.u[row];
    const double u = given > 0.0f ? fmin((double)given, 1.0 - 0x1p-24) : 0.0;
    const Answer a = ask(Question{kByMassWith, 0, u * (double)total});
    Command c{};
    c.what = 2, c.run = a.run, c.prob = (float)((double)a.weight / (double)total);
    if (a.token >= 0) {
        if (tid == 0) {
            p.tokens[row] = a.token;
            if (p.probs) p.probs[row] = c.prob;
        }
        c.what = 0;
        if (ctas > 1) tell(c);
        return;
    }
    // which CTA has it: the slices' counts of its logit, in order
    c.rank = a.rank;
    for (; c.cta < ctas - 1; ++c.cta) {
        const uint32_t n = a.bin >= 0 ? cluster.map_shared_rank(s.hist, c.cta)[a.bin] : cluster.map_shared_rank(s.sub_count, c.cta)[s.place.bin];
        if (c.rank < n) break;
        c.rank -= n;
    }
    if (ctas > 1) tell(c);
    if (c.cta == 0) find(c.run, c.rank, c.prob);
}

template <int TYPE>
cudaError_t launch(SampleParams& p, int rows, cudaStream_t st) {
    constexpr int kOne = Traits<TYPE>::FREE < 16 ? kBins * 8 : 0, kMore = kOne + kBins * 4;  // of a CTA, of one in a cluster
    auto* kernel = sample_kernel<TYPE>;
    static std::mutex mu;
    static int resident[kMaxDevices];  // CTAs that fit on the device at once
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const int sms = device_sm_count();
    if (sms <= 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
    {
        std::lock_guard<std::mutex> lk(mu);
        if (!resident[dev]) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kOne + kMore);
            int per = 0;
            if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, kThreads, kOne + kMore);
            if (e != cudaSuccess) return e;
            resident[dev] = sms * std::max(1, per);
        }
    }
    int ctas = 1;
    while (ctas < kMaxCluster && (long)rows * ctas * 2 <= resident[dev] && p.vocab / (ctas * 2) >= 2048) ctas *= 2;
    p.slice = ((p.vocab + ctas - 1) / ctas + 7) / 8 * 8;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)rows * (unsigned)ctas);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = kOne + (ctas > 1 ? kMore : 0);
    config.stream = st;
    cudaLaunchAttribute attributes[2]{};
    attributes[0].id = cudaLaunchAttributeClusterDimension;
    attributes[0].val.clusterDim.x = (unsigned)ctas, attributes[0].val.clusterDim.y = 1, attributes[0].val.clusterDim.z = 1;
    attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attributes;
    config.numAttrs = 2;  // (a cluster of one, too)
    return cudaLaunchKernelEx(&config, kernel, p);
}

}  // namespace
}  // namespace fp4b

using namespace fp4b;

FP4B_EXPORT int fp4b_sample(const fp4b_sampling* call, void* stream) {
    const char* why = nullptr;
    if (!call) {
        why = "null arguments";
    } else {
        const fp4b_sampling& c = *call;
        const int size = c.type == FP4B_LOGITS_FP32 ? 4 : 2;
        if (c.type != FP4B_LOGITS_BF16 && c.type != FP4B_LOGITS_FP16 && c.type != FP4B_LOGITS_FP32) why = "logits must be BF16, FP16 or FP32";
        else if (c.rows < 0 || c.rows > (1 << 27)) why = "rows must be 0 to 2^27";
        else if (c.vocab <= 0 || c.vocab > (1 << 30)) why = "the vocabulary must be 1 to 2^30 tokens";
        else if (c.rows > 0 && (!c.logits || !c.u || !c.tokens)) why = "null tensor";
        else if (reinterpret_cast<uintptr_t>(c.logits) % size) why = "misaligned logits";
        else if (!c.temperature && !(c.temperature1 >= 0.0f)) why = "the temperature must not be negative";
    }
    if (why) {
        set_last_error("fp4b_sample: %s", why);
        return -1;
    }
    const fp4b_sampling& c = *call;
    if (c.rows == 0) return 0;
    SampleParams p{};
    p.logits = c.logits, p.stride = c.stride, p.u = c.u;
    p.temperature = c.temperature, p.top_k = c.top_k, p.top_p = c.top_p, p.min_p = c.min_p;
    p.temperature1 = c.temperature1, p.top_k1 = c.top_k1, p.top_p1 = c.top_p1, p.min_p1 = c.min_p1;
    p.tokens = c.tokens, p.probs = c.probs, p.vocab = c.vocab;
    p.bits = 62;
    while (p.bits > 0 && ((long long)1 << (62 - p.bits)) < c.vocab) --p.bits;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = c.type == FP4B_LOGITS_BF16   ? launch<kBf16>(p, c.rows, st)
                          : c.type == FP4B_LOGITS_FP16 ? launch<kFp16>(p, c.rows, st)
                                                       : launch<kFp32>(p, c.rows, st);
    return launch_status(e, "fp4b_sample");
}
