// 4-bit K/V attention for fp16 queries (kv4_attention.cuh).
#define KV4_ATTENTION_KERNELS
#include "kv4_attention.cuh"

namespace msb {

cudaError_t launch_kv4_attention_f16(const Kv4Pool& pool, const Kv4Attention& a, const AttSplit& sp, cudaStream_t s) {
    return launch_type<__half>(pool, a, sp, s);
}

}  // namespace msb
