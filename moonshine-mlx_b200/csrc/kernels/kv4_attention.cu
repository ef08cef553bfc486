// How attention over the 4-bit K/V pages is cut into CTAs (kernels: kv4_attention.cuh).
#include "kv4_attention.cuh"

namespace msb {
namespace {

AttSplit split_of(const Kv4Pool& pool, const Kv4Attention& a) {
    AttSplit sp;
    // rows per CTA: as many as one K/V head has, up to what the registers hold
    const long long rows = (long long)a.max_q * (a.heads / pool.kv_heads);
    const int most = kv4_groups(pool.head_dim) == 1 && a.dtype != KV4_F32 ? 32 : 16;
    sp.rows = rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 || most == 16 ? 16 : 32;
    const long long ctas = (rows + sp.rows - 1) / sp.rows * pool.kv_heads * a.rows;
    const long long width = (long long)a.width * pool.page_size;
    // positions per CTA: the whole work over about four CTAs per SM, in steps of the four
    // warps' 256 positions, at least 1024 (a shorter chunk costs more in joining than it
    // saves) and at most 4096 (a long row beside short ones still spreads)
    long long chunk = (ctas * width + 4 * 148 - 1) / (4 * 148);
    chunk = std::min(4096ll, std::max(1024ll, (chunk + 255) / 256 * 256));
    sp.chunk = (int)chunk;
    sp.splits = (int)std::max(1ll, (width + chunk - 1) / chunk);
    sp.warps = 4;
    const int tpp = pool.page_size / KV4_TILE;
    if ((tpp & (tpp - 1)) == 0)
        while (1 << (sp.page_shift + 1) <= tpp) ++sp.page_shift;
    return sp;
}

}  // namespace

size_t kv4_attention_workspace(const Kv4Pool& pool, const Kv4Attention& a) {
    if (a.rows == 0 || a.q_tokens == 0 || a.max_q == 0) return 0;
    const AttSplit sp = split_of(pool, a);
    return sp.splits == 1 ? 0 : (size_t)sp.splits * a.q_tokens * a.heads * (pool.head_dim + 2) * 4;
}

cudaError_t launch_kv4_attention(const Kv4Pool& pool, const Kv4Attention& a, void* workspace, cudaStream_t s) {
    AttSplit sp = split_of(pool, a);
    sp.part = reinterpret_cast<float*>(workspace);
    if (a.dtype == KV4_F32) return launch_kv4_attention_f32(pool, a, sp, s);
    if (a.dtype == KV4_F16) return launch_kv4_attention_f16(pool, a, sp, s);
    return launch_kv4_attention_bf16(pool, a, sp, s);
}

}  // namespace msb
