// decode_core.cuh -- device code shared by the decode-side operators: the
// paged key-value cache's formats, warp reductions, the error word.
//
// Cache layout (fp4b_kv_cache in fp4gemm.h): pages [num_pages, kv_heads,
// page_size, head_dim], so that the keys of one head in one page are one
// contiguous run.  A "row" is one (page, head, slot): head_dim elements, with
//   bf16   2 * D bytes;
//   fp8    D bytes of E4M3 and one fp32 scale;
//   nvfp4  D / 2 bytes of E2M1 (even element in the low nibble) and D / 16
//          UE4M3 scale bytes, the codec of the weight quantizer.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "fp4gemm.h"
#include "nvfp4_codec.cuh"
#include "ptx_sm100.cuh"

namespace fp4b {

enum KvKind : int { kKvBf16 = FP4B_KV_BF16, kKvFp8 = FP4B_KV_FP8, kKvNvfp4 = FP4B_KV_NVFP4, kKvNone = -1 };

// Codes in the device error word (fp4b_device_error) of indices that the
// kernels found out of range; the access is left out.
constexpr int kErrSlotRange = 11;
constexpr int kErrPositionRange = 12;
constexpr int kErrPageRange = 13;

// |x|max below which a block takes the arithmetic rounding; larger, infinite
// and NaN blocks take the codec's literal scan (as in the weight quantizer).
constexpr uint32_t kFastAbsmaxF32Limit = kFastAbsmaxBf16Limit << 16;

constexpr float kFp8Max = 448.0f;
// Smallest absmax an fp8 row's scale stands for (2^-100): 448 / absmax and
// absmax / 448 both stay normal, and a row of zeros needs no case of its own.
constexpr float kFp8AbsmaxFloor = 7.888609052210118e-31f;

namespace decode {

__device__ __forceinline__ void report(int* err, int code) {
    if (err) atomicCAS(err, 0, code);
}

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

// Eight E2M1 codes -> four FP16 pairs, exact; pair i from byte i, the low
// nibble in the low half.
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t (&pair)[4]) {
    asm("{\n"
        ".reg .b8 b0, b1, b2, b3;\n"
        "mov.b32 {b0, b1, b2, b3}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n"
        "}"
        : "=r"(pair[0]), "=r"(pair[1]), "=r"(pair[2]), "=r"(pair[3])
        : "r"(w));
}

// Four E4M3 codes -> two FP16 pairs, exact.
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t w, uint32_t (&pair)[2]) {
    asm("{\n"
        ".reg .b16 h0, h1;\n"
        "mov.b32 {h0, h1}, %2;\n"
        "cvt.rn.f16x2.e4m3x2 %0, h0;\n"
        "cvt.rn.f16x2.e4m3x2 %1, h1;\n"
        "}"
        : "=r"(pair[0]), "=r"(pair[1])
        : "r"(w));
}

__device__ __forceinline__ float2 f16x2_to_float2(uint32_t h) { return __half22float2(*reinterpret_cast<__half2*>(&h)); }

// x * inv -> the fp32 stand-in whose hardware conversion to E2M1 (nearest even)
// equals the codec's rule (ties to the lower magnitude, no sign on a zero): the
// odd-bit float at or one ulp below the product's magnitude.  Adding +0 turns a
// product of -0 into +0, whose bits count as 1.  The product must be finite.
__device__ __forceinline__ float e2m1_stand_in(float x, float inv) {
    const uint32_t b = __float_as_uint(__fmaf_rn(x, inv, 0.0f));
    return __uint_as_float((max(b, 1u) - 1u) | 1u);
}

// Four values times inv -> four E2M1 codes, the first in the lowest nibble.
__device__ __forceinline__ uint32_t e2m1x4(float a, float b, float c, float d, float inv) {
    uint16_t r;
    asm("{\n"
        ".reg .b8 b0, b1;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
        "mov.b16 %0, {b0, b1};\n"
        "}"
        : "=h"(r)
        : "f"(e2m1_stand_in(a, inv)), "f"(e2m1_stand_in(b, inv)), "f"(e2m1_stand_in(c, inv)), "f"(e2m1_stand_in(d, inv)));
    return r;
}

// Four fp32 values -> four E4M3 codes (nearest even, saturating).
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(lo) : "f"(a), "f"(b));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(hi) : "f"(c), "f"(d));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Per half: the larger magnitude of two BF16 pairs, NaN if either is; the sign
// bits of the result mean nothing.
__device__ __forceinline__ uint32_t max_abs_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

template <int WIDTH>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = WIDTH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <int WIDTH>
__device__ __forceinline__ uint32_t group_umax(uint32_t v) {
#pragma unroll
    for (int o = WIDTH / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Index `i` of an int32 or int64 array.
__device__ __forceinline__ long load_index(const void* p, long i, int is64) {
    return is64 ? (long)static_cast<const int64_t*>(p)[i] : (long)static_cast<const int32_t*>(p)[i];
}

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool live) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(live ? BYTES : 0)
                     : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint4 lds128(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ uint2 lds64(const uint8_t* p) { return *reinterpret_cast<const uint2*>(p); }
__device__ __forceinline__ uint32_t lds32(const uint8_t* p) { return *reinterpret_cast<const uint32_t*>(p); }

// 2^x and log2(x); subnormal results and arguments count as zero, which no sum of
// softmax weights notices and which saves three instructions each.
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float log2_approx(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 values an instruction.
__device__ __forceinline__ unsigned long long pair_of(float lo, float hi) {
    return ((unsigned long long)__float_as_uint(hi) << 32) | __float_as_uint(lo);
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float first_of(unsigned long long a) { return __uint_as_float((uint32_t)a); }
__device__ __forceinline__ float second_of(unsigned long long a) { return __uint_as_float((uint32_t)(a >> 32)); }

template <bool BF16>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}

// UE4M3 bytes in bits 0-7 and 16-23 as FP16 pair of 2^-8 of their values: the
// byte's exponent and mantissa moved into FP16's (exact, subnormals too).
__device__ __forceinline__ uint32_t ue4m3x2_to_f16(uint32_t bytes) { return bytes << 7; }
constexpr float kScaleUnit = 256.0f;

// Every kernel of the decode side starts with this: it was launched while the
// kernel before it in the stream may still run, waits here until that one has
// completed, and lets the next one come the same way.  Nothing in global memory
// is touched before.  In a chain of such kernels this hides the launch of each
// behind the one before (about 2 us a kernel on B200).
__device__ __forceinline__ void chain() {
    ptx::grid_dependency_wait();
    ptx::launch_dependents();
}

template <typename Params>
cudaError_t launch_chained(void (*kernel)(Params), dim3 grid, int threads, int smem, cudaStream_t stream, const Params& p) {
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, p);
}

}  // namespace decode

// Host side: why a cache description cannot be used (nullptr if it can).
const char* kv_cache_check(const fp4b_kv_cache* c);

}  // namespace fp4b
