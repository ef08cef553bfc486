// Keys and values into the 4-bit cache pages, and back.
//
// Per group of 64 dims (kv4.cuh): b = fp16(min x), s = fp16((max x - min x) / 15), and the code
// of x is how many of the borders b + (k + 1/2) s, k = 0 .. 14, are <= x, in exact arithmetic:
// an fp32 estimate decides unless it lies next to a border, where b, s and x in fp64 do (b and
// (k + 1/2) s have 42 bits together).  So the codes do not depend on how the quotient is rounded.
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

template <class T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8], bool wide) {
    if (wide) {
        __align__(16) T v[8];
        if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<uint4*>(v) = __ldg(reinterpret_cast<const uint4*>(p));
        } else {
            *reinterpret_cast<uint4*>(v) = __ldg(reinterpret_cast<const uint4*>(p));
            *reinterpret_cast<uint4*>(v + 4) = __ldg(reinterpret_cast<const uint4*>(p + 4));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32<T>(p[i]);
    }
}

template <class T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8], bool wide) {
    __align__(16) T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = from_f32<T>(x[i]);
    if (wide) {
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
        if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(p + 4) = *reinterpret_cast<const uint4*>(v + 4);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = v[i];
    }
}

// Code of x under scale s > 0 and bias b.  f is (x - b) / s + 1/2 to three roundings of a value
// below 17, so to 2^-18: only an f within 2^-12 of a whole number, a border, needs the exact
// comparison.
__device__ __forceinline__ unsigned code_of(float x, float s, float b, float inv) {
    const float f = fmaf(x - b, inv, 0.5f);
    float c = fminf(fmaxf(floorf(f), 0.f), 15.f);
    const float near = rintf(f);
    if (fabsf(f - near) < 2.44140625e-4f && near >= 1.f && near <= 15.f)
        c = (double)x >= (double)b + ((double)near - 0.5) * (double)s ? near : near - 1.f;
    return (unsigned)c;
}

// One (token, head, K or V, group) per 8 lanes, 8 dims per lane.
template <class T>
__global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4Pool pool, const T* __restrict__ k,
                                                         const T* __restrict__ v, long long kst, long long ksh,
                                                         long long vst, long long vsh, long long tokens,
                                                         const long long* __restrict__ slots, int wide) {
    pdl_wait();
    const int hd = pool.head_dim, nw = kv4_words(hd), ng = kv4_groups(hd), H = pool.kv_heads;
    const long long items = tokens * H * 2 * ng;
    const int sub = threadIdx.x & 7;
    for (long long it0 = ((long long)blockIdx.x * blockDim.x + (threadIdx.x & ~31)) >> 3; it0 < items;
         it0 += (long long)gridDim.x * blockDim.x >> 3) {
        const long long it = it0 + ((threadIdx.x & 31) >> 3);
        long long rest = it < items ? it : items - 1;
        const int n = (int)(rest % ng);
        rest /= ng;
        const int kv = (int)(rest & 1);
        rest >>= 1;
        const int h = (int)(rest % H);
        const long long tok = rest / H;
        const long long slot = slots[tok];
        const int w = n * 8 + sub;
        const bool mine = it < items && w < nw && slot >= 0 && slot < (long long)pool.pages * pool.page_size;
        float x[8];
        float lo = INFINITY, hi = -INFINITY;
        bool nan = false;
        if (mine) {
            load8((kv ? v + tok * vst + h * vsh : k + tok * kst + h * ksh) + 8 * w, x, wide != 0);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                nan |= x[i] != x[i];
                x[i] = fminf(fmaxf(x[i], -65504.f), 65504.f);
                lo = fminf(lo, x[i]);
                hi = fmaxf(hi, x[i]);
            }
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(FULL, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(FULL, hi, o));
            nan |= __shfl_xor_sync(FULL, (int)nan, o) != 0;
        }
        if (!mine) continue;
        const __half sh = __float2half_rn((float)(((double)hi - (double)lo) / 15.0));
        const __half bh = nan ? __ushort_as_half(0x7fff) : __float2half_rn(lo);
        const float s = __half2float(sh), b = __half2float(bh);
        unsigned word = 0;
        if (s > 0.f && !nan) {
            const float inv = 1.f / s;
#pragma unroll
            for (int i = 0; i < 8; ++i) word |= code_of(x[i], s, b, inv) << (4 * i);
        }
        const long long page = slot / pool.page_size;
        const int at = (int)(slot - page * pool.page_size), r = at & (KV4_TILE - 1);
        uint32_t* tile = reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(pool.base) + page * pool.page_stride +
                                                     h * pool.head_stride) +
                         (long long)(at / KV4_TILE) * kv4_tile_words(hd);
        tile[kv ? kv4_v_word(nw, w, r) : kv4_k_word(nw, w, r)] = word;
        if (sub == 0)
            tile[kv4_meta_word(nw, n, r, kv)] =
                (uint32_t)__half_as_ushort(sh) | (uint32_t)__half_as_ushort(bh) << 16;
    }
}

template <class T>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4Pool pool, T* __restrict__ k, T* __restrict__ v,
                                                       long long kst, long long ksh, long long vst, long long vsh,
                                                       long long tokens, const long long* __restrict__ slots,
                                                       int wide) {
    pdl_wait();
    const int hd = pool.head_dim, nw = kv4_words(hd), H = pool.kv_heads;
    const long long items = tokens * H * 2 * nw;
    for (long long it = (long long)blockIdx.x * blockDim.x + threadIdx.x; it < items;
         it += (long long)gridDim.x * blockDim.x) {
        long long rest = it;
        const int w = (int)(rest % nw);
        rest /= nw;
        const int kv = (int)(rest & 1);
        rest >>= 1;
        const int h = (int)(rest % H);
        const long long tok = rest / H;
        const long long slot = slots[tok];
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (slot >= 0 && slot < (long long)pool.pages * pool.page_size) {
            const long long page = slot / pool.page_size;
            const int at = (int)(slot - page * pool.page_size), r = at & (KV4_TILE - 1);
            const uint32_t* tile =
                reinterpret_cast<const uint32_t*>(reinterpret_cast<const char*>(pool.base) + page * pool.page_stride +
                                                  h * pool.head_stride) +
                (long long)(at / KV4_TILE) * kv4_tile_words(hd);
            const uint32_t word = tile[kv ? kv4_v_word(nw, w, r) : kv4_k_word(nw, w, r)];
            const uint32_t meta = tile[kv4_meta_word(nw, w >> 3, r, kv)];
            const float s = __half2float(__ushort_as_half((unsigned short)(meta & 0xffff)));
            const float b = __half2float(__ushort_as_half((unsigned short)(meta >> 16)));
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fmaf(s, (float)((word >> (4 * i)) & 15u), b);
        }
        store8((kv ? v + tok * vst + h * vsh : k + tok * kst + h * ksh) + 8 * w, x, wide != 0);
    }
}

bool wide_ok(const void* p, long long st, long long sh, int esize) {
    return !((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(st * esize) | (uintptr_t)(sh * esize)) & 15);
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4Pool& pool, const void* k, const void* v, int dtype, long long tokens,
                              long long kst, long long ksh, long long vst, long long vsh, const long long* slots,
                              cudaStream_t s) {
    const int es = dtype == KV4_F32 ? 4 : 2;
    const int wide = wide_ok(k, kst, ksh, es) && wide_ok(v, vst, vsh, es);
    const long long items = tokens * pool.kv_heads * 2 * kv4_groups(pool.head_dim);
    const int grid = (int)std::min<long long>((items * 8 + 255) / 256, 148 * 8);
    ++launch_counter();
    if (dtype == KV4_F32)
        return launch_kernel(kv4_append_kernel<float>, dim3(grid), dim3(256), 0, s, pool, (const float*)k,
                             (const float*)v, kst, ksh, vst, vsh, tokens, slots, wide);
    if (dtype == KV4_F16)
        return launch_kernel(kv4_append_kernel<__half>, dim3(grid), dim3(256), 0, s, pool, (const __half*)k,
                             (const __half*)v, kst, ksh, vst, vsh, tokens, slots, wide);
    return launch_kernel(kv4_append_kernel<__nv_bfloat16>, dim3(grid), dim3(256), 0, s, pool,
                         (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, kst, ksh, vst, vsh, tokens, slots, wide);
}

cudaError_t launch_kv4_read(const Kv4Pool& pool, void* k, void* v, int dtype, long long tokens, long long kst,
                            long long ksh, long long vst, long long vsh, const long long* slots, cudaStream_t s) {
    const int es = dtype == KV4_F32 ? 4 : 2;
    const int wide = wide_ok(k, kst, ksh, es) && wide_ok(v, vst, vsh, es);
    const long long items = tokens * pool.kv_heads * 2 * kv4_words(pool.head_dim);
    const int grid = (int)std::min<long long>((items + 255) / 256, 148 * 8);
    ++launch_counter();
    if (dtype == KV4_F32)
        return launch_kernel(kv4_read_kernel<float>, dim3(grid), dim3(256), 0, s, pool, (float*)k, (float*)v, kst,
                             ksh, vst, vsh, tokens, slots, wide);
    if (dtype == KV4_F16)
        return launch_kernel(kv4_read_kernel<__half>, dim3(grid), dim3(256), 0, s, pool, (__half*)k, (__half*)v, kst,
                             ksh, vst, vsh, tokens, slots, wide);
    return launch_kernel(kv4_read_kernel<__nv_bfloat16>, dim3(grid), dim3(256), 0, s, pool, (__nv_bfloat16*)k,
                         (__nv_bfloat16*)v, kst, ksh, vst, vsh, tokens, slots, wide);
}

}  // namespace msb
