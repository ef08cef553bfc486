// Keys and values into the 4-bit cache pages, and back.
//
// Per group of 64 dims (kv4.cuh): b = fp16(min x), s = fp16(fp32((max x - min x) / 15)), and the
// code of x is how many of the borders b + (k + 1/2) s, k = 0 .. 14, are <= x, in exact
// arithmetic: an fp32 quotient decides unless it lies next to a border, where the difference of
// x and the border does, formed without rounding.  So the codes do not depend on how the
// quotient is rounded.
//
// A warp takes 16 tokens of one head, one tile of the cache when they lie in order: it is put
// together in shared memory and leaves (or comes) in whole 16-byte accesses.  Bound: HBM for
// reading back (1.4 GB, 262144 tokens of 8 x 128 bf16, in 223 us, 97 % of copy bandwidth), half
// HBM and half issue for storing (360 us, 60 %: about 10 operations per value).  32001 tokens
// of 8 x 40 in fp32, stored and read back: 54 us against 29 at copy bandwidth.
#include <type_traits>

#include "kv4.cuh"

namespace msb {
namespace {

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// 8 elements as they lie in memory: one 16-byte or, for fp32, 32-byte access
template <class T>
struct Raw {
    uint4 v[sizeof(T) / 2];
    template <bool WIDE>
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (WIDE && sizeof(T) == 4) {
            asm volatile("ld.global.cs.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(v[0].x), "=r"(v[0].y), "=r"(v[0].z), "=r"(v[0].w), "=r"(v[1].x), "=r"(v[1].y), "=r"(v[1].z),
                           "=r"(v[1].w)
                         : "l"(p));
        } else if constexpr (WIDE) {
            v[0] = __ldcs(reinterpret_cast<const uint4*>(p));
        } else {
            T* e = reinterpret_cast<T*>(v);
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = p[i];
        }
    }
    template <bool WIDE>
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (WIDE && sizeof(T) == 4) {
            asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0].x), "r"(v[0].y),
                         "r"(v[0].z), "r"(v[0].w), "r"(v[1].x), "r"(v[1].y), "r"(v[1].z), "r"(v[1].w)
                         : "memory");
        } else if constexpr (WIDE) {
            __stcs(reinterpret_cast<uint4*>(p), v[0]);
        } else {
            const T* e = reinterpret_cast<const T*>(v);
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = e[i];
        }
    }
    __device__ __forceinline__ void clamp() {  // fp32: to fp16's largest (below -65504 is code 0 either way)
        float* e = reinterpret_cast<float*>(v);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = fminf(e[i], 65504.f);
    }
    __device__ __forceinline__ float get(int i) const { return to_f32<T>(reinterpret_cast<const T*>(v)[i]); }
    __device__ __forceinline__ void set2(int i, float x, float y) {  // elements i (even) and i + 1
        if constexpr (std::is_same<T, float>::value) {
            reinterpret_cast<float2*>(v)[i / 2] = make_float2(x, y);
        } else if constexpr (std::is_same<T, __half>::value) {
            reinterpret_cast<__half2*>(v)[i / 2] = __floats2half2_rn(x, y);
        } else {
            reinterpret_cast<__nv_bfloat162*>(v)[i / 2] = __floats2bfloat162_rn(x, y);
        }
    }
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
// those of 8 elements, two at a time where a register holds two
__device__ __forceinline__ void range_of(const Raw<float>& r, float& lo, float& hi) {
    lo = hi = r.get(0);
#pragma unroll
    for (int e = 1; e < 8; ++e) {
        lo = min_nan(lo, r.get(e));
        hi = max_nan(hi, r.get(e));
    }
}
template <class T>
__device__ __forceinline__ void range_of(const Raw<T>& r, float& lo, float& hi) {
    using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
    const T2* p = reinterpret_cast<const T2*>(r.v);
    const T2 l = __hmin2_nan(__hmin2_nan(p[0], p[1]), __hmin2_nan(p[2], p[3]));
    const T2 h = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3]));
    lo = min_nan(to_f32<T>(l.x), to_f32<T>(l.y));
    hi = max_nan(to_f32<T>(h.x), to_f32<T>(h.y));
}

// fp32((hi - lo) / 15), the difference and the quotient each corrected by what its rounding left
__device__ __forceinline__ float fifteenth(float hi, float lo) {
    const float d = hi - lo, z = d - hi;
    const float e = (hi - (d - z)) + (-lo - z);  // hi - lo = d + e exactly (Knuth's two-sum)
    const float q = d * (1.f / 15.f);
    return fmaf(fmaf(-q, 15.f, d) + e, 1.f / 15.f, q);
}

// The code of x next to a border, by its definition: f estimates the quotient, so the border in
// question is b + (floor(f) + 1/2) s.  x - b is d + e exactly (Knuth's two-sum), the border's
// distance t from b is exact (16 bits), and so is d - t (d and t are within a factor of two), so
// the last sum has the sign of x - b - t.
__device__ __forceinline__ uint32_t exact_code(float x, float f, float s, float b) {
    const float k = floorf(f), t = (k + 0.5f) * s;
    const float d = x - b, z = d - x, e = (x - (d - z)) + (-b - z);
    return (uint32_t)fminf((d - t) + e >= 0.f ? k + 1.f : k, 15.f);
}
// The codes of 8 values, of which some lie next to a border.  Out of line: bf16 values meet
// borders exactly, one word in 170.
__device__ __noinline__ uint32_t exact_codes(uint32_t word, float x0, float x1, float x2, float x3, float x4, float x5,
                                             float x6, float x7, float s, float b, float inv) {
    const float x[8] = {x0, x1, x2, x3, x4, x5, x6, x7};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float f = __saturatef((x[e] - b) * inv) * 15.f, n = f + 12582912.f;
        if (fabsf(f - (n - 12582912.f)) > 0.49997f)
            word = (word & ~(15u << (4 * e))) | exact_code(x[e], f, s, b) << (4 * e);
    }
    return word;
}

// The codes of 8 values.  The quotient, as a part of 15 so that its clamp is the multiply's
// saturation, is off by five roundings of a value up to 15, so by 2^-17: only when one of the 8
// lies within 2^-16 of a border does the exact comparison decide.
template <class T>
__device__ __forceinline__ uint32_t codes_of(const Raw<T>& r, float s, float b, float inv) {
    float x[8], off = 0.f;
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = r.get(e);
        const float y = __saturatef((x[e] - b) * inv);
        const float n = fmaf(y, 15.f, 12582912.f);  // 1.5 2^23 and the nearest whole number
        off = fmaxf(off, fabsf(fmaf(y, 15.f, 12582912.f - n)));
        word += __float_as_uint(n) << (4 * e);
    }
    word -= 0x4b400000u + 0xb4000000u + 0x40000000u;  // the bits of 1.5 2^23, shifted as they were added
    if (off > 0.499984741f) word = exact_codes(word, x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7], s, b, inv);
    return word;
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

// One warp per (16 tokens, head): two words (16 dims) per lane, 4 lanes per group of 64, 8 tokens
// at a time; the lanes of a vector take neighbouring words, so that an access fills whole
// sectors.  A whole tile goes out through shared memory in 16-byte stores; tokens that lie
// elsewhere (a decode step's) word by word.
template <class T, bool WIDE>
__global__ void __launch_bounds__(32 * STORE_WARPS) kv4_append_kernel(const Kv4Pool pool, const T* __restrict__ k,
                                                                      const T* __restrict__ v, long long kst,
                                                                      long long ksh, long long vst, long long vsh,
                                                                      long long tokens,
                                                                      const long long* __restrict__ slots,
                                                                      int page_shift) {
    __shared__ __align__(16) uint32_t s_tile[STORE_WARPS][STORE_TILE];
    pdl_wait();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, sub = lane & 3, of8 = lane >> 2;
    const int hd = pool.head_dim, nw = kv4_words(hd), ng = kv4_groups(hd), H = pool.kv_heads;
    const long long unit = (long long)blockIdx.x * STORE_WARPS + wid, block = unit / H;
    const int h = (int)(unit - block * H);
    const long long first = block * KV4_TILE;
    if (first >= tokens) return;
    const Tokens t(pool, slots, first, tokens);
    uint32_t* out = s_tile[wid];
    // (whole tile, part): K or V of one group
    auto work = [&](auto whole, int part) {
        constexpr bool WHOLE = decltype(whole)::value;
        const int kv = part & 1, n = part >> 1, w = 8 * n + sub, have = nw > w ? nw > w + 4 ? 2 : 1 : 0;  // words w and w + 4
        const long long step = kv ? vst : kst;
        const T* src = (kv ? v + h * vsh : k + h * ksh) + 8 * w + (first + of8) * step;
        const int left = (int)min(tokens - first, (long long)KV4_TILE) - of8;  // tokens from this lane's on
        // tile words of position of8; 8 positions on they are 1 (K, scales) or 2 (V) further
        const int at0 = kv ? kv4_v_word(nw, w, of8) : kv4_k_word(nw, w, of8);
        const int at1 = kv ? at0 + 64 : kv4_k_word(nw, w + 4, of8), at_meta = kv4_meta_word(nw, n, of8, kv);
        Raw<T> raw[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if ((WHOLE || left > 8 * i) && j < have) raw[i][j].template load<WIDE>(src + 8 * i * step + 32 * j);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool mine = WHOLE || left > 8 * i;
            float lo = INFINITY, hi = -INFINITY;
            if (mine && have > 0) range_of(raw[i][0], lo, hi);
            if (mine && have > 1) {
                float l, m;
                range_of(raw[i][1], l, m);
                lo = min_nan(lo, l);
                hi = max_nan(hi, m);
            }
#pragma unroll
            for (int o = 2; o > 0; o >>= 1) {
                lo = min_nan(lo, __shfl_xor_sync(FULL, lo, o));
                hi = max_nan(hi, __shfl_xor_sync(FULL, hi, o));
            }
            const bool nan = lo != lo;
            // The values are clamped as their range is.  Of 16-bit values that changes no code: b is
            // their minimum exactly, so 65504 has code 15 already.  Of fp32 ones within 500 of 65504, b
            // can be 16 off, more than a step.
            if constexpr (sizeof(T) == 4) {
                if (hi > 65504.f) {
                    raw[i][0].clamp();
                    raw[i][1].clamp();
                }
            }
            lo = fminf(fmaxf(lo, -65504.f), 65504.f);
            hi = fminf(fmaxf(hi, -65504.f), 65504.f);
            const __half sh = __float2half_rn(fifteenth(hi, lo));
            const __half bh = nan ? __ushort_as_half(0x7fff) : __float2half_rn(lo);
            const float s = __half2float(sh), b = __half2float(bh);
            float inv;  // of 15 s, to 2^-23
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(15.f * s));
            uint32_t word[2] = {0, 0};
            if (mine && s > 0.f && !nan) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (j < have) word[j] = codes_of(raw[i][j], s, b, inv);
            }
            const uint32_t meta = (uint32_t)__half_as_ushort(sh) | (uint32_t)__half_as_ushort(bh) << 16;
            if constexpr (WHOLE) {
                if (have > 0) out[at0 + (1 + kv) * i] = word[0];
                if (have > 1) out[at1 + (1 + kv) * i] = word[1];
                if (sub == 0) out[at_meta + i] = meta;
            } else {
                const long long slot = __shfl_sync(FULL, t.slot, of8 + 8 * i);
                if (slot < 0) continue;
                int r;
                uint32_t* to = tile_at(pool, page_shift, slot, h, r);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (j < have) to[kv ? kv4_v_word(nw, w + 4 * j, r) : kv4_k_word(nw, w + 4 * j, r)] = word[j];
                if (sub == 0) to[kv4_meta_word(nw, n, r, kv)] = meta;
            }
        }
    };
    if (!t.whole) {
#pragma unroll 1
        for (int part = 0; part < 2 * ng; ++part) work(std::false_type{}, part);
        return;
    }
#pragma unroll 1
    for (int part = 0; part < 2 * ng; ++part) work(std::true_type{}, part);
    __syncwarp();
    int r;
    uint4* tile = reinterpret_cast<uint4*>(tile_at(pool, page_shift, __shfl_sync(FULL, t.slot, 0), h, r));
    for (int i = lane; i < kv4_tile_words(hd) / 4; i += 32) tile[i] = reinterpret_cast<const uint4*>(out)[i];
}

// The reverse: a whole tile comes in by 16-byte loads.
template <class T, bool WIDE>
__global__ void __launch_bounds__(32 * STORE_WARPS) kv4_read_kernel(const Kv4Pool pool, T* __restrict__ k,
                                                                    T* __restrict__ v, long long kst, long long ksh,
                                                                    long long vst, long long vsh, long long tokens,
                                                                    const long long* __restrict__ slots,
                                                                    int page_shift) {
    __shared__ __align__(16) uint32_t s_tile[STORE_WARPS][STORE_TILE];
    pdl_wait();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, sub = lane & 3, of8 = lane >> 2;
    const int hd = pool.head_dim, nw = kv4_words(hd), ng = kv4_groups(hd), H = pool.kv_heads;
    const long long unit = (long long)blockIdx.x * STORE_WARPS + wid, block = unit / H;
    const int h = (int)(unit - block * H);
    const long long first = block * KV4_TILE;
    if (first >= tokens) return;
    const Tokens t(pool, slots, first, tokens);
    uint32_t* in = s_tile[wid];
    auto work = [&](auto whole, int part) {
        constexpr bool WHOLE = decltype(whole)::value;
        const int kv = part & 1, n = part >> 1, w = 8 * n + sub, have = nw > w ? nw > w + 4 ? 2 : 1 : 0;
        const long long step = kv ? vst : kst;
        T* dst = (kv ? v + h * vsh : k + h * ksh) + 8 * w + (first + of8) * step;
        const int left = (int)min(tokens - first, (long long)KV4_TILE) - of8;
        // tile words of position of8; 8 positions on they are 1 (K, scales) or 2 (V) further
        const int at0 = kv ? kv4_v_word(nw, w, of8) : kv4_k_word(nw, w, of8);
        const int at1 = kv ? at0 + 64 : kv4_k_word(nw, w + 4, of8), at_meta = kv4_meta_word(nw, n, of8, kv);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t meta = 0, words[2] = {0, 0};
            if constexpr (WHOLE) {
                meta = in[at_meta + i];
                words[0] = in[at0 + (1 + kv) * i];  // lanes past the vector read what lies behind
                words[1] = in[at1 + (1 + kv) * i];
            } else {
                const long long slot = __shfl_sync(FULL, t.slot, of8 + 8 * i);
                if (left <= 8 * i) continue;
                if (slot >= 0) {
                    int r;
                    const uint32_t* from = tile_at(pool, page_shift, slot, h, r);
                    meta = from[kv4_meta_word(nw, n, r, kv)];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        if (j < have) words[j] = from[kv ? kv4_v_word(nw, w + 4 * j, r) : kv4_k_word(nw, w + 4 * j, r)];
                }
            }
            const float2 sb = __half22float2(*reinterpret_cast<const __half2*>(&meta));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (j >= have) continue;
                const uint32_t word = words[j];
                Raw<T> raw;
                float x[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // codes e and e + 4 as fp16: in the mantissa of 1024, less 1024
                    uint32_t c;
                    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(c) : "r"(word >> (4 * e)), "r"(0x000f000fu), "r"(0x64006400u));
                    const float2 f = __half22float2(__hsub2(*reinterpret_cast<const __half2*>(&c), __float2half2_rn(1024.f)));
                    x[e] = fmaf(sb.x, f.x, sb.y);
                    x[e + 4] = fmaf(sb.x, f.y, sb.y);
                }
#pragma unroll
                for (int e = 0; e < 8; e += 2) raw.set2(e, x[e], x[e + 1]);
                raw.template store<WIDE>(dst + 8 * i * step + 32 * j);
            }
        }
    };
    if (!t.whole) {
#pragma unroll 1
        for (int part = 0; part < 2 * ng; ++part) work(std::false_type{}, part);
        return;
    }
    int r;
    const uint32_t* tile = tile_at(pool, page_shift, __shfl_sync(FULL, t.slot, 0), h, r);
    for (int i = 4 * lane; i < kv4_tile_words(hd); i += 128)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(smem_u32(in + i)), "l"(tile + i) : "memory");
    asm volatile("cp.async.commit_group;\ncp.async.wait_all;\n" ::: "memory");
    __syncwarp();
#pragma unroll 1
    for (int part = 0; part < 2 * ng; ++part) work(std::true_type{}, part);
}

bool wide_ok(const void* p, long long st, long long sh, int esize) {
    return !((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(st * esize) | (uintptr_t)(sh * esize)) & (8 * esize - 1));
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
    const long long units = (tokens + KV4_TILE - 1) / KV4_TILE * pool.kv_heads;
    const long long grid = (units + STORE_WARPS - 1) / STORE_WARPS;
    if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
    ++launch_counter();
    return launch_kernel(kernel, dim3((unsigned)grid), dim3(32 * STORE_WARPS), 0, s, pool, k, v, kst, ksh, vst, vsh,
                         tokens, slots, shift_of(pool.page_size));
}
}  // namespace

cudaError_t launch_kv4_append(const Kv4Pool& pool, const void* k, const void* v, int dtype, long long tokens,
                              long long kst, long long ksh, long long vst, long long vsh, const long long* slots,
                              cudaStream_t s) {
    auto go = [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        const bool wide = wide_ok(k, kst, ksh, sizeof(T)) && wide_ok(v, vst, vsh, sizeof(T));
        return launch_store(wide ? kv4_append_kernel<T, true> : kv4_append_kernel<T, false>, pool, (const T*)k,
                            (const T*)v, tokens, kst, ksh, vst, vsh, slots, s);
    };
    if (dtype == KV4_F32) return go((float*)nullptr);
    if (dtype == KV4_F16) return go((__half*)nullptr);
    return go((__nv_bfloat16*)nullptr);
}

cudaError_t launch_kv4_read(const Kv4Pool& pool, void* k, void* v, int dtype, long long tokens, long long kst,
                            long long ksh, long long vst, long long vsh, const long long* slots, cudaStream_t s) {
    auto go = [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        const bool wide = wide_ok(k, kst, ksh, sizeof(T)) && wide_ok(v, vst, vsh, sizeof(T));
        return launch_store(wide ? kv4_read_kernel<T, true> : kv4_read_kernel<T, false>, pool, (T*)k, (T*)v, tokens,
                            kst, ksh, vst, vsh, slots, s);
    };
    if (dtype == KV4_F32) return go((float*)nullptr);
    if (dtype == KV4_F16) return go((__half*)nullptr);
    return go((__nv_bfloat16*)nullptr);
}

}  // namespace msb
