// decode_attention.cu -- the C entry points of decode_attention.cuh.
#include "decode_attention.cuh"

#define FP4B_EXPORT extern "C" __attribute__((visibility("default")))

using namespace fp4b;

FP4B_EXPORT long fp4b_decode_attention_workspace(int q_heads, int kv_heads, int head_dim) {
    if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || head_dim <= 0) {
        set_last_error("fp4b_decode_attention_workspace: bad head counts");
        return -1;
    }
    const int sms = device_sm_count();
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
    const long need = c.batch > 0 && cache && cache->kv_heads > 0 ? fp4b_decode_attention_workspace(c.q_heads, cache->kv_heads, cache->head_dim) : 0;
    const char* why = decode_check(c, need);
    if (why) {
        set_last_error("fp4b_decode_attention: %s", why);
        return -1;
    }
    if (c.batch == 0) return 0;
    AttentionParams p = params_of(c);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint8_t* ws = static_cast<uint8_t*>(c.workspace);
    const cudaError_t e = cache->kind == kKvBf16 ? launch_dim<kKvBf16, false>(p, ws, st)
                          : cache->kind == kKvFp8 ? launch_dim<kKvFp8, false>(p, ws, st)
                                                  : launch_dim<kKvNvfp4, false>(p, ws, st);
    return launch_status(e, "fp4b_decode_attention");
}
