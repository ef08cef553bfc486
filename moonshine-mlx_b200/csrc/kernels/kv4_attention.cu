// How attention over the 4-bit K/V pages is cut into CTAs (kernels: kv4_attention.cuh).
#include <climits>

#include "kv4_attention.cuh"

namespace msb {
namespace {

// Rows per CTA: as many as one K/V head has, up to 16, or 128 in the wide kernel.
int rows_per_cta(const Kv4Attention& a, int kv_heads, int head_dim) {
    // A stage of the wide kernel takes as long for 20 rows as for 128.  Against the other, us for
    // ragged requests of 4 K/V heads, (33 of 1000 .. 8000 positions; 64 of 190 .. 1500):
    //   bf16, heads of 64   20 rows (81; 38) and (67; 37), 32 (73; 39) and (67; 38), 35 (81; 43) and (90; 52)
    //   bf16, heads of 128  20 rows (113; 53) and (99; 50), 32 (116; 55) and (110; 55), 35 (112; 56) and (135; 67)
    //   fp16, heads of 64   35 rows (114; 53) and (105; 51), 48 (107; 54) and (105; 55), 64 (118; 55) and (144; 69)
    //   fp16, heads of 128  48 rows (200; 101) and (150; 80), 64 (226; 104) and (200; 99)
    // (fp16 takes the codes exactly, so its softmax does more.  fp32 has no wide kernel: its
    // products need more planes.)
    const long long rows = (long long)a.max_q * (a.heads / kv_heads);
    if (rows > 32 && a.dtype == KV4_BF16) return 128;
    if (rows > 32 + 16 * kv4_groups(head_dim) && a.dtype == KV4_F16) return 128;
    return rows <= 4 ? 4 : rows <= 8 ? 8 : 16;
}

AttSplit split_of(const Kv4Pool& pool, const Kv4Attention& a) {
    AttSplit sp;
    sp.rows = rows_per_cta(a, pool.kv_heads, pool.head_dim);
    const bool wide = sp.rows == 128;
    const long long rows = (long long)a.max_q * (a.heads / pool.kv_heads);
    const long long per_row = (rows + sp.rows - 1) / sp.rows * pool.kv_heads, pairs = per_row * a.rows;
    sp.per_row = (int)per_row;
    const long long width = (long long)a.width * pool.page_size;
    // eight warps per CTA when there are fewer CTAs than half the GPU holds, two when there are
    // several waves of them (less to join and to wait for)
    sp.warps = pairs < 148 && sp.rows <= 8 ? 8 : pairs > 2 * 592 && sp.rows <= 8 ? 2 : 4;
    // What one CTA would read of a row is cut where the rows are too few to fill the GPU (16
    // warps per SM): a few pairs into one wave of equal pieces, by the lengths on the device;
    // more pairs into chunks of 2048, a full GPU's of 4096, for long rows among short ones.  A
    // CTA costs about 4 us before its first product, so smaller pieces lose (and one 30 s
    // utterance's 1500 frames are better left whole: 15.4 us cut in 3, 14.3 in one).
    const int slots = wide ? 148 * 2 : 148 * 16 / sp.warps;
    const bool few = pairs * 8 < slots;
    sp.ctas = few ? (int)(slots - pairs) : 0;
    sp.chunk = few ? (width <= 1536 ? 1536 : 512) : pairs < slots ? 2048 : 4096;
    sp.splits = (int)std::max(1ll, (width + sp.chunk - 1) / sp.chunk);
    if (few) sp.splits = (int)std::min((long long)sp.splits, sp.ctas / per_row + 1);
    // At most 256 MB of parts (prompts of thousands of tokens fill the GPU without them).
    const long long each = a.q_tokens * a.heads * (pool.head_dim + 2) * 4;
    const long long most = std::min(65535ll, std::max(1ll, (256ll << 20) / each));
    if (sp.splits > most) {
        sp.splits = (int)most;
        sp.chunk = (int)std::max((long long)sp.chunk, (width + most - 1) / most);
    }
    const int tpp = pool.page_size / KV4_TILE;
    if ((tpp & (tpp - 1)) == 0)
        while (1 << (sp.page_shift + 1) <= tpp) ++sp.page_shift;
    return sp;
}

}  // namespace

bool kv4_head_dim_ok(int hd) { return hd >= 8 && hd <= 128 && hd % 8 == 0; }

size_t kv4_attention_workspace(const Kv4Pool& pool, const Kv4Attention& a) {
    if (a.rows == 0 || a.q_tokens == 0 || a.max_q == 0) return 0;
    const AttSplit sp = split_of(pool, a);
    return sp.splits == 1 ? 0 : (size_t)sp.splits * a.q_tokens * a.heads * (pool.head_dim + 2) * 4;
}

cudaError_t launch_kv4_attention(const Kv4Pool& pool, const Kv4Attention& a, void* workspace, cudaStream_t s) {
    AttSplit sp = split_of(pool, a);
    sp.part = reinterpret_cast<float*>(workspace);
    if (sp.rows == 128) return launch_kv4_attention_wide(pool, a, sp, s);
    if (a.dtype == KV4_F32) return launch_kv4_attention_f32(pool, a, sp, s);
    if (a.dtype == KV4_F16) return launch_kv4_attention_f16(pool, a, sp, s);
    if (a.dtype == KV4_STEP) return launch_kv4_attention_step(pool, a, sp, s);
    return launch_kv4_attention_bf16(pool, a, sp, s);
}

}  // namespace msb
