// 4-bit K/V attention of the batched decoder step (kv4_attention.cuh).
#define KV4_ATTENTION_KERNELS
#include "kv4_attention.cuh"

namespace msb {

cudaError_t launch_kv4_attention_step(const Kv4Pool& pool, const Kv4Attention& a, const AttSplit& sp, cudaStream_t s) {
    return a.lo_off ? launch_type<StepSplit>(pool, a, sp, s) : launch_type<Step>(pool, a, sp, s);
}

}  // namespace msb
