// Attention over the 4-bit K/V pages.
//
// One query head of one token per CTA; its four warps take the tiles of 16 positions in turn,
// each with a running maximum and sum of the softmax (fp32), and join their states at the end.
#include "kv4.cuh"

namespace msb {
namespace {

constexpr int ATT_WARPS = 4;

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float half_lo(uint32_t m) { return __half2float(__ushort_as_half((unsigned short)(m & 0xffff))); }
__device__ __forceinline__ float half_hi(uint32_t m) { return __half2float(__ushort_as_half((unsigned short)(m >> 16))); }

template <class T>
__global__ void __launch_bounds__(32 * ATT_WARPS) kv4_attention_kernel(const Kv4Pool pool, const Kv4Attention a) {
    __shared__ float q[128];
    __shared__ float wm[ATT_WARPS], wl[ATT_WARPS], wo[ATT_WARPS][128];
    pdl_wait();
    const int b = blockIdx.z, h = blockIdx.y, i = blockIdx.x;
    const int hd = pool.head_dim, nw = kv4_words(hd), P = pool.page_size;
    const int kvh = h / (a.heads / pool.kv_heads);
    const int q0 = a.cu_q ? max(0, a.cu_q[b]) : b, q1 = a.cu_q ? min((long long)a.cu_q[b + 1], a.q_tokens) : b + 1;
    if (i >= q1 - q0) return;
    const long long tok = q0 + i;
    const int len = (int)min((long long)max(0, a.lens[b]), (long long)a.width * P);
    const int end = a.causal ? max(0, min(len, len - (q1 - q0) + i + 1)) : len;  // positions < end are seen
    const T* qp = reinterpret_cast<const T*>(a.q) + tok * a.q_token_stride + h * a.q_head_stride;
    for (int d = threadIdx.x; d < hd; d += blockDim.x) q[d] = to_f32<T>(qp[d]) * a.scale;
    __syncthreads();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, r = lane & 15, half = lane >> 4;
    float m = -INFINITY, l = 0.f, o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = 0.f;
    for (int t0 = wid * KV4_TILE; t0 < end; t0 += ATT_WARPS * KV4_TILE) {
        const int page = a.table[b * a.table_stride + t0 / P];
        if (page < 0 || page >= pool.pages) continue;  // no page: positions that are not there
        const uint32_t* tile = reinterpret_cast<const uint32_t*>(reinterpret_cast<const char*>(pool.base) +
                                                                 (long long)page * pool.page_stride +
                                                                 kvh * pool.head_stride) +
                               (long long)(t0 % P / KV4_TILE) * kv4_tile_words(hd);
        // score of position r: the two half warps take every other word
        float s = 0.f;
        for (int w = half; w < nw; w += 2) {
            const uint32_t word = tile[kv4_k_word(nw, w, r)], meta = tile[kv4_meta_word(nw, w >> 3, r, 0)];
            const float sc = half_lo(meta), bi = half_hi(meta);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(q[8 * w + e], fmaf(sc, (float)((word >> (4 * e)) & 15u), bi), s);
        }
        s += __shfl_xor_sync(FULL, s, 16);
        if (t0 + r >= end) s = -INFINITY;
        const float mn = fmaxf(m, warp_max(s));
        const float base = mn == -INFINITY ? 0.f : mn;
        const float p = t0 + r < end ? expf(s - base) : 0.f;
        const float corr = m == -INFINITY ? 0.f : expf(m - base);
        l = l * corr + warp_sum(half ? 0.f : p);
        m = mn;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] *= corr;
        // word r of V for the positions of this half of the tile
        for (int u = 0; u < 8; ++u) {
            const int rr = 8 * half + u;
            const float pu = __shfl_sync(FULL, p, rr);
            if (r >= nw || t0 + rr >= end) continue;
            const uint32_t word = tile[kv4_v_word(nw, r, rr)], meta = tile[kv4_meta_word(nw, r >> 3, rr, 1)];
            const float sc = half_lo(meta), bi = half_hi(meta);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = fmaf(pu, fmaf(sc, (float)((word >> (4 * e)) & 15u), bi), o[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] += __shfl_xor_sync(FULL, o[e], 16);
    if (lane == 0) {
        wm[wid] = m;
        wl[wid] = l;
    }
    if (!half && r < nw)
#pragma unroll
        for (int e = 0; e < 8; ++e) wo[wid][8 * r + e] = o[e];
    __syncthreads();
    T* op = reinterpret_cast<T*>(a.out) + tok * a.out_token_stride + h * a.out_head_stride;
    for (int d = threadIdx.x; d < hd; d += blockDim.x) {
        float mx = -INFINITY, ls = 0.f, ov = 0.f;
        bool nan = false;
        for (int w = 0; w < ATT_WARPS; ++w) {
            mx = fmaxf(mx, wm[w]);
            nan |= wl[w] != wl[w];
        }
        if (mx == -INFINITY) mx = 0.f;
        for (int w = 0; w < ATT_WARPS; ++w) {
            const float f = wm[w] == -INFINITY ? 0.f : expf(wm[w] - mx);
            ls = fmaf(wl[w], f, ls);
            ov = fmaf(wo[w][d], f, ov);
        }
        op[d] = from_f32<T>(nan ? NAN : ls == 0.f ? 0.f : ov / ls);  // nothing seen: zeros
    }
}

}  // namespace

size_t kv4_attention_workspace(const Kv4Pool&, const Kv4Attention&) { return 0; }

cudaError_t launch_kv4_attention(const Kv4Pool& pool, const Kv4Attention& a, void*, cudaStream_t s) {
    const dim3 grid(a.max_q, a.heads, a.rows);
    ++launch_counter();
    if (a.dtype == KV4_F32) return launch_kernel(kv4_attention_kernel<float>, grid, dim3(32 * ATT_WARPS), 0, s, pool, a);
    if (a.dtype == KV4_F16) return launch_kernel(kv4_attention_kernel<__half>, grid, dim3(32 * ATT_WARPS), 0, s, pool, a);
    return launch_kernel(kv4_attention_kernel<__nv_bfloat16>, grid, dim3(32 * ATT_WARPS), 0, s, pool, a);
}

}  // namespace msb
