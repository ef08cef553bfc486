// The batched decoder step's form of the attention over 4-bit pages (KV4_STEP: fp32 queries, bf16
// planes out) for a test: plain arguments onto the launcher that the engine calls.
#include "kernels.h"

extern "C" int64_t step_attention(void* base, int pages, int kv_heads, int head_dim, int page_size, const void* q,
                                  void* out, int heads, int rows, const int* table, int width, const int* lens,
                                  float scale, int64_t lo_off, void* workspace, unsigned* status, void* stream) {
    msb::Kv4Pool pool;
    pool.base = base;
    pool.pages = pages;
    pool.kv_heads = kv_heads;
    pool.head_dim = head_dim;
    pool.page_size = page_size;
    pool.head_stride = (long long)page_size * (head_dim + 8 * ((head_dim + 63) / 64));
    pool.page_stride = pool.head_stride * kv_heads;
    msb::Kv4Attention a;
    a.q = q;
    a.out = out;
    a.dtype = msb::KV4_STEP;
    a.heads = heads;
    a.q_tokens = a.rows = rows;
    a.q_token_stride = a.out_token_stride = (long long)heads * head_dim;
    a.q_head_stride = a.out_head_stride = head_dim;
    a.table = table;
    a.table_stride = a.width = width;
    a.lens = lens;
    a.scale = scale;
    a.lo_off = (size_t)lo_off;
    a.status = status;
    if (!workspace) return (int64_t)msb::kv4_attention_workspace(pool, a);
    return msb::launch_kv4_attention(pool, a, workspace, (cudaStream_t)stream);
}
