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
// once and stays in its threads' registers over both means.
// A row is a CTA's, of as many warps as it takes (up to 16384, or 5120, elements), or
// (wide rows, and rows so few that they leave SMs idle) a cluster's, which sums
// over distributed shared memory.  One wave of CTAs goes over the rows; the next
// row's loads start as soon as this one's registers are free, before its second
// sum.  A thread has two pieces of 8 elements (16 bytes of BF16), or, where the
// rows do not start on 16 bytes or the width is not a multiple of 8, four of two or
// eight single ones.
//
// Measured on B200 (copy bandwidth 6.57 TB/s): 8192 x 2880 with both norms 31.1 us =
// 6.1 TB/s (each row by a CTA of its own, loads not ahead: 37.6; rows through a ring
// of bulk copies in shared memory: 49), 1024 x 16384 27.9, 1021 x 5003 in single
// elements 20 us = 3.6 TB/s, bound by their instructions (1021 x 5004 in pairs 13.9),
// 33 x 16384 4.1 and 1 x 2880 1.8, launches and a chain of waits.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>

#include "decode_core.cuh"
#include "fp4b_internal.h"

#define FP4B_EXPORT extern "C" __attribute__((visibility("default")))

namespace fp4b {
namespace {

using namespace decode;
namespace cg = cooperative_groups;

constexpr int kMaxWidth = 32768;
constexpr int kMaxCtasPerSm = 32;
constexpr int kMaxCluster = 8;
constexpr int kLeastWidth = 2048;  // of a CTA of a cluster that is there to fill the GPU

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

template <int VEC>
struct Shape {
    static constexpr int ITEMS = VEC == 8 ? 2 : 8 / VEC;    // pieces a thread
    static constexpr int RESIDENT = VEC == 8 ? 1024 : 1280;  // threads of an SM, by their registers
    static constexpr int THREADS = VEC == 8 ? 1024 : 640;    // of a CTA at most
};

typedef unsigned long long pair;  // of fp32 values, see decode_core.cuh

// Loads and stores of what lies below `end`, without a branch: zeros beyond it.
__device__ __forceinline__ uint4 load_below(const uint4* p, int i, int end) {
    uint4 v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.s32 p, %5, %6;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
                 "@p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
                 : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "l"(p), "r"(i), "r"(end) : "memory");
    return v;
}
__device__ __forceinline__ uint2 load_below(const uint2* p, int i, int end) {
    uint2 v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.s32 p, %3, %4;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\t@p ld.global.v2.b32 {%0, %1}, [%2];\n\t}"
                 : "=&r"(v.x), "=&r"(v.y) : "l"(p), "r"(i), "r"(end) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t load_below(const uint32_t* p, int i, int end) {
    uint32_t v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.s32 p, %2, %3;\n\tmov.b32 %0, 0;\n\t@p ld.global.b32 %0, [%1];\n\t}"
                 : "=&r"(v) : "l"(p), "r"(i), "r"(end) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t load_below(const uint16_t* p, int i, int end) {
    uint16_t v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.s32 p, %2, %3;\n\tmov.b16 %0, 0;\n\t@p ld.global.b16 %0, [%1];\n\t}"
                 : "=&h"(v) : "l"(p), "r"(i), "r"(end) : "memory");
    return v;
}
__device__ __forceinline__ float load_below(const float* p, int i, int end) {
    float v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.s32 p, %2, %3;\n\tmov.f32 %0, 0f00000000;\n\t@p ld.global.f32 %0, [%1];\n\t}"
                 : "=&f"(v) : "l"(p), "r"(i), "r"(end) : "memory");
    return v;
}
__device__ __forceinline__ void store_below(uint4* p, uint4 v, int i, int end) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.s32 p, %5, %6;\n\t@p st.global.v4.b32 [%0], {%1, %2, %3, %4};\n\t}"
                 ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "r"(i), "r"(end) : "memory");
}
__device__ __forceinline__ void store_below(uint2* p, uint2 v, int i, int end) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.s32 p, %3, %4;\n\t@p st.global.v2.b32 [%0], {%1, %2};\n\t}"
                 ::"l"(p), "r"(v.x), "r"(v.y), "r"(i), "r"(end) : "memory");
}
__device__ __forceinline__ void store_below(uint32_t* p, uint32_t v, int i, int end) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.s32 p, %2, %3;\n\t@p st.global.b32 [%0], %1;\n\t}" ::"l"(p), "r"(v), "r"(i), "r"(end) : "memory");
}
__device__ __forceinline__ void store_below(uint16_t* p, uint32_t v, int i, int end) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.s32 p, %2, %3;\n\t@p st.global.b16 [%0], %1;\n\t}" ::"l"(p), "h"((uint16_t)v), "r"(i), "r"(end) : "memory");
}
__device__ __forceinline__ void store_below(float* p, float v, int i, int end) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.s32 p, %2, %3;\n\t@p st.global.f32 [%0], %1;\n\t}" ::"l"(p), "f"(v), "r"(i), "r"(end) : "memory");
}

// A thread's pieces of a BF16 row or weight, two elements a register.  A warp's
// pieces are one run; `at` is the thread's first element, the next piece's is the
// 32nd piece on.
template <int VEC>
struct Pieces {
    static constexpr int ITEMS = Shape<VEC>::ITEMS, WORDS = VEC * ITEMS / 2;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const uint16_t* p, int at, int width) {
        p += at;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            if constexpr (VEC == 8) {
                const uint4 v = load_below(reinterpret_cast<const uint4*>(p) + 32 * k, at + 256 * k, width);
                w[4 * k] = v.x, w[4 * k + 1] = v.y, w[4 * k + 2] = v.z, w[4 * k + 3] = v.w;
            } else if constexpr (VEC == 2) {
                w[k] = load_below(reinterpret_cast<const uint32_t*>(p) + 32 * k, at + 64 * k, width);
            } else {
                const uint32_t v = load_below(p + 32 * k, at + 32 * k, width);
                w[k / 2] = k & 1 ? __byte_perm(w[k / 2], v, 0x5410) : v;
            }
        }
    }
    __device__ __forceinline__ pair get(int i) const { return pair_of(bf16_lo(w[i]), bf16_hi(w[i])); }
};
template <int VEC>
struct Values {
    static constexpr int ITEMS = Shape<VEC>::ITEMS, WORDS = VEC * ITEMS / 2;
    pair v[WORDS];
    __device__ __forceinline__ void load(const float* p, int at, int width) {
        p += at;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            if constexpr (VEC == 8) {
                const uint4 a = load_below(reinterpret_cast<const uint4*>(p) + 64 * k, at + 256 * k, width);
                const uint4 b = load_below(reinterpret_cast<const uint4*>(p) + 64 * k + 1, at + 256 * k, width);
                v[4 * k] = words(a.x, a.y), v[4 * k + 1] = words(a.z, a.w), v[4 * k + 2] = words(b.x, b.y), v[4 * k + 3] = words(b.z, b.w);
            } else if constexpr (VEC == 2) {
                const uint2 a = load_below(reinterpret_cast<const uint2*>(p) + 32 * k, at + 64 * k, width);
                v[k] = words(a.x, a.y);
            } else {
                const float f = load_below(p + 32 * k, at + 32 * k, width);
                v[k / 2] = k & 1 ? pair_of(first_of(v[k / 2]), f) : pair_of(f, 0.0f);
            }
        }
    }
    __device__ __forceinline__ void store(uint16_t* p, int at, int width) const {
        p += at;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            if constexpr (VEC == 8)
                store_below(reinterpret_cast<uint4*>(p) + 32 * k, make_uint4(pack(4 * k), pack(4 * k + 1), pack(4 * k + 2), pack(4 * k + 3)), at + 256 * k, width);
            else if constexpr (VEC == 2)
                store_below(reinterpret_cast<uint32_t*>(p) + 32 * k, pack(k), at + 64 * k, width);
            else
                store_below(p + 32 * k, k & 1 ? pack(k / 2) >> 16 : pack(k / 2), at + 32 * k, width);
        }
    }
    __device__ __forceinline__ void store(float* p, int at, int width) const {
        p += at;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            if constexpr (VEC == 8) {
                store_below(reinterpret_cast<uint4*>(p) + 64 * k, make_uint4(lo(4 * k), hi(4 * k), lo(4 * k + 1), hi(4 * k + 1)), at + 256 * k, width);
                store_below(reinterpret_cast<uint4*>(p) + 64 * k + 1, make_uint4(lo(4 * k + 2), hi(4 * k + 2), lo(4 * k + 3), hi(4 * k + 3)), at + 256 * k, width);
            } else if constexpr (VEC == 2) {
                store_below(reinterpret_cast<uint2*>(p) + 32 * k, make_uint2(lo(k), hi(k)), at + 64 * k, width);
            } else {
                store_below(p + 32 * k, k & 1 ? second_of(v[k / 2]) : first_of(v[k / 2]), at + 32 * k, width);
            }
        }
    }
    __device__ __forceinline__ pair get(int i) const { return v[i]; }
    __device__ __forceinline__ uint32_t pack(int i) const { return pack_bf16(first_of(v[i]), second_of(v[i])); }
    static __device__ __forceinline__ pair words(uint32_t a, uint32_t b) { return ((pair)b << 32) | a; }
    __device__ __forceinline__ uint32_t lo(int i) const { return (uint32_t)v[i]; }
    __device__ __forceinline__ uint32_t hi(int i) const { return (uint32_t)(v[i] >> 32); }
};
__device__ __forceinline__ pair both(float f) { return pair_of(f, f); }

// Sums over a row's threads, in one order for all of them.  They take two sets
// of slots in turn: one is written again behind the barrier of the other.
struct Slots {
    float warp[2][32], cta[2][kMaxCluster];
};
__device__ __forceinline__ float row_sum(float v, Slots& s, int& turn, int ctas) {
    v = group_sum<32>(v);
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warps > 1) {
        if (lane == 0) s.warp[turn][warp] = v;
        __syncthreads();
        v = group_sum<32>(lane < warps ? s.warp[turn][lane] : 0.0f);
    }
    if (ctas > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        if ((int)threadIdx.x < ctas) cluster.map_shared_rank(s.cta[turn], threadIdx.x)[cluster.block_rank()] = v;
        cluster.sync();
        v = group_sum<kMaxCluster>(lane % kMaxCluster < ctas ? s.cta[turn][lane % kMaxCluster] : 0.0f);
    }
    turn ^= 1;
    return v;
}

// The arithmetic of a row, in three steps between which its threads meet.
template <int VEC>
__device__ __forceinline__ float squares(const Pieces<VEC>& x) {
    pair sum = both(0.0f);
#pragma unroll
    for (int i = 0; i < Pieces<VEC>::WORDS; ++i) sum = fma2(x.get(i), x.get(i), sum);
    return first_of(sum) + second_of(sum);
}
// r, the residual, becomes r'; returns its squares' sum.
template <int VEC, bool POST, bool GATE>
__device__ __forceinline__ float block_end(Values<VEC>& r, const Pieces<VEC>& x, const Pieces<VEC>& post_weight, const Pieces<VEC>& gate, float factor) {
    pair sum = both(0.0f);
#pragma unroll
    for (int i = 0; i < Pieces<VEC>::WORDS; ++i) {
        pair f = both(factor);
        if constexpr (POST) f = mul2(f, post_weight.get(i));
        if constexpr (GATE) f = mul2(f, gate.get(i));
        r.v[i] = fma2(x.get(i), f, r.v[i]);
        sum = fma2(r.v[i], r.v[i], sum);
    }
    return first_of(sum) + second_of(sum);
}
template <int VEC>
__device__ __forceinline__ void norm_begin(Values<VEC>& r, const Pieces<VEC>& weight, float factor) {
#pragma unroll
    for (int i = 0; i < Pieces<VEC>::WORDS; ++i) r.v[i] = mul2(mul2(r.v[i], both(factor)), weight.get(i));
}

template <int VEC, typename R, bool POST, bool GATE>
__global__ void __launch_bounds__(Shape<VEC>::THREADS, Shape<VEC>::RESIDENT / Shape<VEC>::THREADS) block_norm_kernel(const __grid_constant__ NormParams p) {
    __shared__ Slots slots;
    const int ctas = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
    if (ctas > 1) ptx::cluster_start_arrive();
    chain();
    const int warp = rank * (int)(blockDim.x >> 5) + (int)(threadIdx.x >> 5);
    const int at = (warp * 32 * Shape<VEC>::ITEMS + (int)(threadIdx.x & 31)) * VEC;  // the thread's first element
    const int each = (int)gridDim.x / ctas;  // rows at once
    int turn = 0;
    Pieces<VEC> x, gate;
    typename std::conditional<sizeof(R) == 2, Pieces<VEC>, Values<VEC>>::type residual;
#pragma unroll
    for (int i = 0; i < Pieces<VEC>::WORDS; ++i) x.w[i] = 0u;
    auto load = [&](long row) {
        if (p.x) x.load(p.x + row * p.x_stride, at, p.width);
        residual.load(static_cast<const R*>(p.residual) + row * p.residual_stride, at, p.width);
        if constexpr (GATE) gate.load(p.gate + row * p.gate_stride, at, p.width);
    };
    long row = blockIdx.x / ctas;
    load(row);
    if (ctas > 1) ptx::cluster_start_wait();  // before the first sum goes to the other CTAs, behind the loads' starts
    for (; row < p.rows; row += each) {
        float factor = p.scale;  // what x is multiplied by besides the weights
        Pieces<VEC> weight;
        if constexpr (POST) {
            weight.load(p.post_weight, at, p.width);
            factor *= rsqrtf(fmaf(row_sum(squares<VEC>(x), slots, turn, ctas), p.inv_width, p.eps));
        }
        Values<VEC> r;
#pragma unroll
        for (int i = 0; i < Pieces<VEC>::WORDS; ++i) r.v[i] = residual.get(i);
        const float sum = block_end<VEC, POST, GATE>(r, x, weight, gate, factor);
        if (row + each < p.rows) load(row + each);
        weight.load(p.weight, at, p.width);
        if (p.x) r.store(static_cast<R*>(p.residual_out) + row * p.width, at, p.width);
        norm_begin<VEC>(r, weight, rsqrtf(fmaf(row_sum(sum, slots, turn, ctas), p.inv_width, p.eps)));
        r.store(p.normed + row * p.width, at, p.width);
    }
}

template <int VEC, typename R, bool POST, bool GATE>
cudaError_t launch(const NormParams& p, cudaStream_t st) {
    using S = Shape<VEC>;
    const int pieces = (p.width + VEC - 1) / VEC, sms = device_sm_count();
    if (sms <= 0) return cudaErrorInvalidDevice;
    int ctas = 1;
    while (pieces > ctas * S::ITEMS * S::THREADS || (ctas < kMaxCluster && (long)p.rows * ctas * 2 <= sms && p.width >= ctas * 2 * kLeastWidth)) ctas *= 2;
    const int threads = ((pieces + ctas * S::ITEMS - 1) / (ctas * S::ITEMS) + 31) / 32 * 32;
    const int resident = std::min(kMaxCtasPerSm, S::RESIDENT / threads);
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)std::min(p.rows, sms * resident / ctas) * (unsigned)ctas);
    config.blockDim = dim3(threads);
    config.stream = st;
    cudaLaunchAttribute attributes[2]{};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = (unsigned)ctas, attributes[1].val.clusterDim.y = 1, attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = ctas > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&config, block_norm_kernel<VEC, R, POST, GATE>, p);
}

template <int VEC, typename R>
cudaError_t launch_parts(const NormParams& p, cudaStream_t st) {
    return p.post_weight ? (p.gate ? launch<VEC, R, true, true>(p, st) : launch<VEC, R, true, false>(p, st))
                         : (p.gate ? launch<VEC, R, false, true>(p, st) : launch<VEC, R, false, false>(p, st));
}
template <typename R>
cudaError_t launch_width(const NormParams& p, int piece, cudaStream_t st) {
    return piece == 8 ? launch_parts<8, R>(p, st) : piece == 2 ? launch_parts<2, R>(p, st) : launch_parts<1, R>(p, st);
}

bool whole(const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }
// Are all rows aligned to pieces of `piece` elements?
bool aligned(const void* p, long stride, int size, int piece) { return whole(p, piece * 2) && stride % piece == 0 && (size == 2 || whole(p, std::min(piece * 4, 16))); }

}  // namespace
}  // namespace fp4b

using namespace fp4b;

FP4B_EXPORT int fp4b_block_norm(const fp4b_norm* call, void* stream) {
    const char* why = nullptr;
    if (!call) {
        why = "null arguments";
    } else {
        const fp4b_norm& c = *call;
        if (c.rows < 0 || c.rows > (1 << 28)) why = "rows must be 0 to 2^28";
        else if (c.width <= 0 || c.width > kMaxWidth) why = "the width must be 1 to 32768";
        else if (c.rows > 0 && (!c.residual || !c.weight || !c.normed || (c.x && !c.residual_out))) why = "null tensor";
        else if (c.x && c.residual_out == c.residual && c.rows > 1 && c.residual_stride != c.width)
            why = "a residual that is updated in place must have its rows one after another";  // (a row's r' would lie over another's r)
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
    int piece = 8;
    auto fits = [&](int n) {
        return c.width % n == 0 && aligned(c.x, c.x_stride, 2, n) && aligned(c.residual, c.residual_stride, size, n) && aligned(c.gate, c.gate_stride, 2, n) &&
               aligned(c.weight, 0, 2, n) && aligned(c.post_weight, 0, 2, n) && aligned(c.normed, 0, 2, n) && aligned(c.residual_out, 0, size, n);
    };
    while (!fits(piece)) piece = piece == 8 ? 2 : 1;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return launch_status(c.residual_fp32 ? launch_width<float>(p, piece, st) : launch_width<uint16_t>(p, piece, st), "fp4b_block_norm");
}
