// Keys and values into the 4-bit cache pages, and back.
//
// Per group of 64 dims (kv4.cuh): b = fp16(min x), s = fp16(fp32((max x - min x) / 15)), and the
// code of x is how many of the borders b + (k + 1/2) s, k = 0 .. 14, are <= x, in exact
// arithmetic: an fp32 quotient decides unless it lies next to a border, where b, s and x in fp64
// do (b and (k + 1/2) s have 42 bits together).  So the codes do not depend on how the quotient
// is rounded.
#include <type_traits>

#include "kv4.cuh"

namespace msb {
namespace {

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 8 elements as they lie in memory
template <class T>
struct Raw {
    uint4 v[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p, bool wide) {
        if (wide) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
        } else {
            T* e = reinterpret_cast<T*>(v);
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = p[i];
        }
    }
    __device__ __forceinline__ void store(T* p, bool wide) const {
        if (wide) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, v[i]);
        } else {
            const T* e = reinterpret_cast<const T*>(v);
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = e[i];
        }
    }
    __device__ __forceinline__ float get(int i) const { return to_f32<T>(reinterpret_cast<const T*>(v)[i]); }
    __device__ __forceinline__ void set(int i, float x) { reinterpret_cast<T*>(v)[i] = from_f32<T>(x); }
};

// minimum and maximum that are NaN if either is
__device__ __forceinline__ float min_nan(float a, float b) {
    float c;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}

// fp32((hi - lo) / 15), the difference and the quotient each corrected by what its rounding left
__device__ __forceinline__ float fifteenth(float hi, float lo) {
    const float d = hi - lo, z = d - hi;
    const float e = (hi - (d - z)) + (-lo - z);  // hi - lo = d + e exactly (Knuth's two-sum)
    const float q = __fdiv_rn(d, 15.f);
    return fmaf(fmaf(-q, 15.f, d) + e, 1.f / 15.f, q);
}

// Adds the code of x under scale s (1 / s = inv) and bias b to `word` in 4 bits from the top.
// The quotient is off by three roundings of a value below 17, so by 2^-18: only one within 2^-12
// of a border needs the exact comparison.
__device__ __forceinline__ void add_code(uint32_t& word, float x, float s, float b, float inv) {
    const float f = fminf(fmaxf((x - b) * inv, 0.f), 15.f);
    float n = f + 12582912.f;  // rounds f to a whole number, in the low bits
    const float off = f - (n - 12582912.f);
    if (fabsf(off) > 0.499755859375f) {
        const float below = floorf(f);
        n = 12582912.f + below + ((double)x >= (double)b + ((double)below + 0.5) * (double)s ? 1.f : 0.f);
    }
    word = (word >> 4) + (__float_as_uint(n) << 28);
}

// Where a slot lies: tile word pointer of the head and position in the tile
__device__ __forceinline__ uint32_t* tile_at(const Kv4Pool& pool, int page_shift, long long slot, int h, int& r) {
    const long long page = page_shift >= 0 ? slot >> page_shift : slot / pool.page_size;
    const int at = (int)(slot - page * pool.page_size);
    r = at & (KV4_TILE - 1);
    return reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(pool.base) + page * pool.page_stride + h * pool.head_stride) +
           (long long)(at / KV4_TILE) * kv4_tile_words(pool.head_dim);
}

constexpr int STORE_WARPS = 4;
constexpr int STORE_TILE = 32 * 16 + 64;  // words of the largest tile (head size 128)

// The 16 tokens of a warp, one head.  Lane r (and r + 16) holds token r's slot; `whole` if they
// are one tile of the cache in order.
struct Tokens {
    long long slot;
    bool whole;
    __device__ Tokens(const Kv4Pool& pool, const long long* slots, long long first, long long tokens) {
        const int r = threadIdx.x & 15;
        const long long total = (long long)pool.pages * pool.page_size;
        slot = first + r < tokens ? slots[first + r] : -1;
        if (slot < 0 || slot >= total) slot = -1;
        const long long s0 = __shfl_sync(FULL, slot, 0);
        whole = __all_sync(FULL, s0 >= 0 && (s0 & (KV4_TILE - 1)) == 0 && slot == s0 + r);
    }
};

// One warp per (16 tokens, head): 8 dims per lane, 8 lanes per group of 64, 4 tokens at a time,
// all loads first.  Bound by HBM for prompts: about 14 operations per element against 13 that
// the issue rate allows at copy bandwidth.  A whole tile goes out through shared memory in
// 16-byte stores; tokens that lie elsewhere (a decode step's) word by word.
template <class T>
__global__ void __launch_bounds__(32 * STORE_WARPS) kv4_append_kernel(const Kv4Pool pool, const T* __restrict__ k,
                                                                      const T* __restrict__ v, long long kst,
                                                                      long long ksh, long long vst, long long vsh,
                                                                      long long tokens,
                                                                      const long long* __restrict__ slots, int wide,
                                                                      int page_shift) {
    __shared__ __align__(16) uint32_t s_tile[STORE_WARPS][STORE_TILE];
    pdl_wait();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, sub = lane & 7, of4 = lane >> 3;
    const int hd = pool.head_dim, nw = kv4_words(hd), ng = kv4_groups(hd), H = pool.kv_heads;
    const long long unit = (long long)blockIdx.x * STORE_WARPS + wid, block = unit / H;
    const int h = (int)(unit - block * H);
    const long long first = block * KV4_TILE;
    if (first >= tokens) return;
    const Tokens t(pool, slots, first, tokens);
    uint32_t* out = s_tile[wid];
    for (int n = 0; n < ng; ++n) {
        const int w = 8 * n + sub;
        Raw<T> raw[2][4];
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const long long tok = first + 4 * i + of4;
                const bool mine = tok < tokens && w < nw;
                if (mine) raw[kv][i].load((kv ? v + tok * vst + h * vsh : k + tok * kst + h * ksh) + 8 * w, wide != 0);
            }
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = 4 * i + of4;
                const bool mine = first + at < tokens && w < nw;
                float lo = INFINITY, hi = -INFINITY;
                if (mine) {
                    lo = hi = raw[kv][i].get(0);
#pragma unroll
                    for (int e = 1; e < 8; ++e) {
                        lo = min_nan(lo, raw[kv][i].get(e));
                        hi = max_nan(hi, raw[kv][i].get(e));
                    }
                }
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) {
                    lo = min_nan(lo, __shfl_xor_sync(FULL, lo, o));
                    hi = max_nan(hi, __shfl_xor_sync(FULL, hi, o));
                }
                const bool nan = lo != lo;
                lo = fminf(fmaxf(lo, -65504.f), 65504.f);
                hi = fminf(fmaxf(hi, -65504.f), 65504.f);
                const __half sh = __float2half_rn(fifteenth(hi, lo));
                const __half bh = nan ? __ushort_as_half(0x7fff) : __float2half_rn(lo);
                const float s = __half2float(sh), b = __half2float(bh);
                uint32_t word = 0;
                if (mine && s > 0.f && !nan) {
                    const float inv = 1.f / s;
#pragma unroll
                    for (int e = 0; e < 8; ++e) add_code(word, raw[kv][i].get(e), s, b, inv);
                }
                const uint32_t meta = (uint32_t)__half_as_ushort(sh) | (uint32_t)__half_as_ushort(bh) << 16;
                if (t.whole) {
                    if (w < nw) out[kv ? kv4_v_word(nw, w, at) : kv4_k_word(nw, w, at)] = word;
                    if (sub == 0) out[kv4_meta_word(nw, n, at, kv)] = meta;
                } else {
                    const long long slot = __shfl_sync(FULL, t.slot, at);
                    if (slot >= 0) {
                        int r;
                        uint32_t* tile = tile_at(pool, page_shift, slot, h, r);
                        if (w < nw) tile[kv ? kv4_v_word(nw, w, r) : kv4_k_word(nw, w, r)] = word;
                        if (sub == 0) tile[kv4_meta_word(nw, n, r, kv)] = meta;
                    }
                }
            }
    }
    if (!t.whole) return;
    __syncwarp();
    int r;
    uint4* tile = reinterpret_cast<uint4*>(tile_at(pool, page_shift, __shfl_sync(FULL, t.slot, 0), h, r));
    for (int i = lane; i < kv4_tile_words(hd) / 4; i += 32) tile[i] = reinterpret_cast<const uint4*>(out)[i];
}

// The reverse: a whole tile comes in by 16-byte loads.
template <class T>
__global__ void __launch_bounds__(32 * STORE_WARPS) kv4_read_kernel(const Kv4Pool pool, T* __restrict__ k,
                                                                    T* __restrict__ v, long long kst, long long ksh,
                                                                    long long vst, long long vsh, long long tokens,
                                                                    const long long* __restrict__ slots, int wide,
                                                                    int page_shift) {
    __shared__ __align__(16) uint32_t s_tile[STORE_WARPS][STORE_TILE];
    pdl_wait();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, sub = lane & 7, of4 = lane >> 3;
    const int hd = pool.head_dim, nw = kv4_words(hd), ng = kv4_groups(hd), H = pool.kv_heads;
    const long long unit = (long long)blockIdx.x * STORE_WARPS + wid, block = unit / H;
    const int h = (int)(unit - block * H);
    const long long first = block * KV4_TILE;
    if (first >= tokens) return;
    const Tokens t(pool, slots, first, tokens);
    uint32_t* in = s_tile[wid];
    if (t.whole) {
        int r;
        const uint4* tile =
            reinterpret_cast<const uint4*>(tile_at(pool, page_shift, __shfl_sync(FULL, t.slot, 0), h, r));
        for (int i = lane; i < kv4_tile_words(hd) / 4; i += 32) reinterpret_cast<uint4*>(in)[i] = __ldcs(tile + i);
        __syncwarp();
    }
    for (int n = 0; n < ng; ++n) {
        const int w = 8 * n + sub;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = 4 * i + of4;
                const long long tok = first + at, slot = __shfl_sync(FULL, t.slot, at);
                if (tok >= tokens || w >= nw) continue;
                uint32_t word = 0, meta = 0;
                if (t.whole) {
                    word = in[kv ? kv4_v_word(nw, w, at) : kv4_k_word(nw, w, at)];
                    meta = in[kv4_meta_word(nw, n, at, kv)];
                } else if (slot >= 0) {
                    int r;
                    const uint32_t* tile = tile_at(pool, page_shift, slot, h, r);
                    word = tile[kv ? kv4_v_word(nw, w, r) : kv4_k_word(nw, w, r)];
                    meta = tile[kv4_meta_word(nw, n, r, kv)];
                }
                const float2 sb = __half22float2(*reinterpret_cast<const __half2*>(&meta));
                Raw<T> raw;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    // 2^23 + c by its bits, less 2^23
                    const float c = __uint_as_float(((word >> (4 * e)) & 15u) | 0x4b000000u) - 8388608.f;
                    raw.set(e, fmaf(sb.x, c, sb.y));
                }
                raw.store((kv ? v + tok * vst + h * vsh : k + tok * kst + h * ksh) + 8 * w, wide != 0);
            }
    }
}

bool wide_ok(const void* p, long long st, long long sh, int esize) {
    return !((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(st * esize) | (uintptr_t)(sh * esize)) & 15);
}

}  // namespace

namespace {
// log2 of the page size, -1 if it is no power of two
int shift_of(int page) {
    int n = 0;
    while (1 << n < page) ++n;
    return 1 << n == page ? n : -1;
}

template <class Kernel, class P>
cudaError_t launch_store(Kernel kernel, const Kv4Pool& pool, P* k, P* v, long long tokens, long long kst, long long ksh,
                         long long vst, long long vsh, const long long* slots, cudaStream_t s) {
    const int es = (int)sizeof(P);
    const int wide = wide_ok(k, kst, ksh, es) && wide_ok(v, vst, vsh, es);
    const long long units = (tokens + KV4_TILE - 1) / KV4_TILE * pool.kv_heads;
    const long long grid = (units + STORE_WARPS - 1) / STORE_WARPS;
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    ++launch_counter();
    return launch_kernel(kernel, dim3((unsigned)grid), dim3(32 * STORE_WARPS), 0, s, pool, k, v, kst, ksh, vst, vsh,
                         tokens, slots, wide, shift_of(pool.page_size));
}
}  // namespace

cudaError_t launch_kv4_append(const Kv4Pool& pool, const void* k, const void* v, int dtype, long long tokens,
                              long long kst, long long ksh, long long vst, long long vsh, const long long* slots,
                              cudaStream_t s) {
    auto go = [&](auto kernel, auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        return launch_store(kernel, pool, (const T*)k, (const T*)v, tokens, kst, ksh, vst, vsh, slots, s);
    };
    if (dtype == KV4_F32) return go(kv4_append_kernel<float>, (float*)nullptr);
    if (dtype == KV4_F16) return go(kv4_append_kernel<__half>, (__half*)nullptr);
    return go(kv4_append_kernel<__nv_bfloat16>, (__nv_bfloat16*)nullptr);
}

cudaError_t launch_kv4_read(const Kv4Pool& pool, void* k, void* v, int dtype, long long tokens, long long kst,
                            long long ksh, long long vst, long long vsh, const long long* slots, cudaStream_t s) {
    auto go = [&](auto kernel, auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        return launch_store(kernel, pool, (T*)k, (T*)v, tokens, kst, ksh, vst, vsh, slots, s);
    };
    if (dtype == KV4_F32) return go(kv4_read_kernel<float>, (float*)nullptr);
    if (dtype == KV4_F16) return go(kv4_read_kernel<__half>, (__half*)nullptr);
    return go(kv4_read_kernel<__nv_bfloat16>, (__nv_bfloat16*)nullptr);
}

}  // namespace msb
