// Attention over the 4-bit K/V pages.
//
// With k = s c + b (codes c, one scale and bias per 64 dims and position) and d = c - 8,
//     q . k_t = sum_g s_tg (q_g . d_tg) + (b_tg + 8 s_tg) sum(q_g)
//     sum_t p_t v_t = sum_t (p_t s_tg) d_tg + sum_t p_t (b_tg + 8 s_tg),
// so the matrix instructions take the codes themselves, and the scales multiply the fp32 scores
// and the probabilities.
//
// V's nibbles become fp16 by one AND-OR into the mantissa of 1024 (the odd nibbles in place, as 16
// c) and one packed multiply-add, 9 operations per word, after a byte permute, since its
// fragments want two positions side by side.  (Codes taken as the fp16 subnormals that masked
// nibbles already are cost fewer, but the tensor core aligns its sums by the exponent field, which
// lost 6 to 10 bits, and sums of one-sided codes as much again.)  Probabilities times scales
// are rounded to fp16, as one value for bf16 results (which keep 8 bits), as two otherwise.
//
// Scores of up to 4 query rows are integer products: the codes as bytes (3 operations per word)
// times q as fixed point of 24 bits in three planes of bytes, sums exact.  Rows have two columns of
// the products there, which take two planes at a time; fp32 queries of more rows are three
// products.  (fp32 results start the sums at -8 sum(q), so that they are those of d and s d q and
// b sum(q) do not cancel.)  16-bit queries of more rows are fp16 after a power of two, exact down to 2^-28 of a
// row's largest, and the codes for them made as V's; for up to 4 rows that costs 4 us more of the
// 50 and 91 below.  16-bit fixed point is not enough: one channel 1000 times the others took
// their bits, and scores were off by a hundredth.
//
// S^T = K q^T and O^T = V^T P^T: positions and dims are the 16 rows of the products, queries
// their 8 columns, since one K/V head rarely has more query rows in a decode step; the score
// accumulators become the probability operand by one 8x8 transpose (movmatrix).  The warps of a
// CTA take the runs of SU tiles in turn, each through its own ring of bulk copies, with a running
// maximum and sum of the softmax; their states are joined at the end, and those of the CTAs
// that share a long context by a second kernel.
//
// Bound: issue inside a run (60 to 80 % of the slots), and 4 to 6 us of latency per CTA around
// them (2560 CTAs of one position take 16 us).  bf16, at the cache's bytes: 256 contexts of 187 ..
// 1500 on 10 heads of 64, 50 us (3.2 TB/s, half of copy bandwidth); four of 16K .. 131K on 32 heads
// of 128, 4 per K/V head, 91 us (4.1 TB/s, 64 %); one of 1500 in fp32, 10 us.
#pragma once

#include <climits>
#include <type_traits>

#include "kv4.cuh"

namespace msb {

struct AttSplit {
    int warps = 4;           // per CTA
    int rows = 4;            // (token, head) rows per CTA
    int per_row = 1;         // CTAs of one batch row along its heads and queries
    int splits = 1;          // CTAs along the positions at most
    int chunk = 0;           // positions per CTA at least
    int ctas = 0;            // > 0: CTAs to cut the positions of all rows into
    int page_shift = -1;     // log2 of a page's tiles, -1 if it is no power of two
    float* part = nullptr;   // [splits][tokens * heads][head_dim], then their (max, sum)
};

// One launch per type (kv4_attention_*.cu); `sp` from split_of.
cudaError_t launch_kv4_attention_f32(const Kv4Pool& pool, const Kv4Attention& a, const AttSplit& sp, cudaStream_t s);
cudaError_t launch_kv4_attention_f16(const Kv4Pool& pool, const Kv4Attention& a, const AttSplit& sp, cudaStream_t s);
cudaError_t launch_kv4_attention_bf16(const Kv4Pool& pool, const Kv4Attention& a, const AttSplit& sp, cudaStream_t s);
cudaError_t launch_kv4_attention_wide(const Kv4Pool& pool, const Kv4Attention& a, const AttSplit& sp, cudaStream_t s);
cudaError_t launch_kv4_attention_step(const Kv4Pool& pool, const Kv4Attention& a, const AttSplit& sp, cudaStream_t s);

#ifdef KV4_ATTENTION_KERNELS
#ifndef KV4_WAIT_LIMIT  // polls of a wait for a copy; a test has it run out
#define KV4_WAIT_LIMIT WAIT_LIMIT
#endif
namespace {

constexpr int ATT_WARPS = 8;   // most per CTA
constexpr int ATT_STAGES = 2;   // ring slots per warp
constexpr float LOG2E = 1.4426950408889634f;

// Element types of the batched decoder step: fp32 queries, bf16 planes of a GEMM input out
struct Step { float v; };       // probabilities as for bf16
struct StepSplit { float v; };  // probabilities as for fp32, and the low plane

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<Step>(Step v) { return v.v; }
template <> __device__ __forceinline__ float to_f32<StepSplit>(StepSplit v) { return v.v; }
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class T> constexpr bool is_step = std::is_same<T, Step>::value || std::is_same<T, StepSplit>::value;
template <class T> constexpr bool is_f32 = std::is_same<T, float>::value || std::is_same<T, StepSplit>::value;
template <class T> constexpr bool is_bf16 = std::is_same<T, __nv_bfloat16>::value || std::is_same<T, Step>::value;

// element `at` of the result
template <class T>
__device__ __forceinline__ void put(const Kv4Attention& a, long long at, float v) {
    if constexpr (is_step<T>) st_bf16_split(reinterpret_cast<__nv_bfloat16*>(a.out) + at, v, a.lo_off);
    else reinterpret_cast<T*>(a.out)[at] = from_f32<T>(v);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The probability of what a query does not see: a zero that no exponential gives
constexpr float NOT_SEEN = -0.f;
__device__ __forceinline__ bool not_seen(float p) { return __float_as_uint(p) == 0x80000000u; }
__device__ __forceinline__ float pow2(int n) { return __int_as_float((n + 127) << 23); }  // -126 <= n <= 127
__device__ __forceinline__ float2 half2_of(uint32_t m) {
    return __half22float2(*reinterpret_cast<const __half2*>(&m));
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// codes times bytes of q onto c0 (columns 2 t) and c1 (2 t + 1)
__device__ __forceinline__ void imma16832_on(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                             uint32_t b1, int c0, int c1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c0), "r"(c1));
}
__device__ __forceinline__ void imma16832(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// c = a b without an accumulator
__device__ __forceinline__ void mma16816_new(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// two fp32 operations in one
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\t"
        "mov.b64 {%0, %1}, a;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\t"
        "mov.b64 {%0, %1}, a;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// maximum and sum over the eight lanes that hold one column pair
__device__ __forceinline__ float rows_max(float v) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
    return v;
}
__device__ __forceinline__ float rows_sum(float v) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}

// (x & mask) | 0x6400 in both halves, one operation
__device__ __forceinline__ uint32_t on_1024(uint32_t x, uint32_t mask) {
    uint32_t h;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(h) : "r"(x), "r"(mask), "r"(0x64006400u));
    return h;
}
__device__ __forceinline__ uint32_t hfma2_of(uint32_t x, uint32_t y, uint32_t z) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(x), "r"(y), "r"(z));
    return d;
}
// Codes 0 .. 3 of both halves of x as fp16 pairs: in the mantissa of 1024 a nibble adds c, or
// 16 c one nibble up; every value here is exact in fp16.
__device__ __forceinline__ void codes_minus_8(uint32_t x, uint32_t* d) {
    const uint32_t y = x >> 8;
    d[0] = hfma2_of(on_1024(x, 0x000f000fu), 0x3c003c00u, 0xe408e408u);  // 1, -1032
    d[1] = hfma2_of(on_1024(x, 0x00f000f0u), 0x2c002c00u, 0xd480d480u);  // 1/16, -72
    d[2] = hfma2_of(on_1024(y, 0x000f000fu), 0x3c003c00u, 0xe408e408u);
    d[3] = hfma2_of(on_1024(y, 0x00f000f0u), 0x2c002c00u, 0xd480d480u);
}
// How one row's queries and positions are cut, the same in both kernels.
struct Row {
    int q0, n, len;  // first token, queries, positions
    __device__ Row(const Kv4Pool& pool, const Kv4Attention& a, int b) {
        q0 = b;
        n = 1;
        if (a.cu_q) {
            q0 = max(0, a.cu_q[b]);
            n = (int)max(0ll, min((long long)a.cu_q[b + 1], a.q_tokens) - q0);
        }
        len = (int)min((long long)max(0, a.lens[b]), (long long)a.width * pool.page_size);
    }
    // positions that query i sees
    __device__ int end(const Kv4Attention& a, int i) const {
        return a.causal ? max(0, min(len, len - n + i + 1)) : len;
    }
};
// Positions per CTA.  With sp.ctas the positions of all rows over so many, so that a few long
// rows fill the GPU in one wave of about equal CTAs: the lengths are on the device, and every
// warp sums them up for itself.
__device__ __forceinline__ int chunk_of(const Kv4Pool& pool, const Kv4Attention& a, const AttSplit& sp) {
    if (sp.splits == 1) return INT_MAX;
    if (sp.ctas == 0) return sp.chunk;
    const int most = (int)min((long long)a.width * pool.page_size, (long long)INT_MAX);
    unsigned long long sum = 0;
    for (int b = threadIdx.x & 31; b < a.rows; b += 32) sum += (unsigned)min(max(0, a.lens[b]), most);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
    const unsigned long long each = (sum * sp.per_row + sp.ctas - 1) / sp.ctas;
    return (int)max((unsigned long long)sp.chunk, min(each, 1ull << 30));
}
__device__ __forceinline__ int splits_of(int end, int chunk) { return end <= chunk ? 1 : (end + chunk - 1) / chunk; }
__device__ __forceinline__ int over(int n, int d) { return d == 1 ? n : n / d; }  // d == 1 for most models' heads

// Queries of one K/V head: ROWS (token, head) rows, token major, in NT n-tiles of 8 columns; with
// NC = 1 (up to 4 rows) a row has two columns, for two planes of q at a time in the scores, and only
// the even one after them, which halves the softmax work.
template <class T, int NG, int NT, int NC>
struct AttShape {
    static constexpr int ROWS = 4 * NC * NT;
    static constexpr bool INT = NC == 1 || is_f32<T> || is_step<T>;            // scores as integer products
    static constexpr int QP = INT ? 3 : 2;                                     // planes of q: bytes, or halves of its words
    static constexpr int QM = NC == 1 ? 2 : QP;                                // score products
    static constexpr int PP = is_bf16<T> ? 1 : 2;                              // fp16 planes of the probabilities
    static constexpr int SU = NG == 2 ? 2 : 4;                                 // tiles per ring stage
    static constexpr int QROW = 64 * NG + 8;                                   // bytes per q row, padded
    static size_t ring(int hd, int warps) {  // lanes of a short group read past the last tile; also the join
        const size_t r = (size_t)warps * ATT_STAGES * SU * kv4_tile_words(hd) * 4 + 512;
        return std::max(r, (size_t)warps * ROWS * (hd + 4) * 4);
    }
    static size_t smem(int hd, int warps) { return ring(hd, warps) + (size_t)QP * ROWS * QROW; }
};

// HD: the head size, or 0 to take it from the pool
template <class T, int NG, int NT, int NC, int HD>
__global__ void __launch_bounds__(NT == 1 ? 32 * ATT_WARPS : 128, 2) kv4_attention_kernel(const Kv4Pool pool, const Kv4Attention a,
                                                                       const AttSplit sp, int ring_bytes) {
    using S = AttShape<T, NG, NT, NC>;
    constexpr int ROWS = S::ROWS, QP = S::QP, QM = S::QM, PP = S::PP, SU = S::SU;
    constexpr bool F32 = is_f32<T>, INT = S::INT;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) uint64_t s_bar[ATT_WARPS][ATT_STAGES];
    __shared__ uint32_t s_ok[ATT_WARPS][ATT_STAGES];
    __shared__ float s_f[ROWS], s_qs[ROWS][NG], s_m[ATT_WARPS][ROWS], s_l[ATT_WARPS][ROWS];
    __shared__ int s_end[ROWS], s_from[F32 ? ROWS : 1][NG][QP];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, W = sp.warps;
    const int hd = HD ? HD : pool.head_dim, nw = kv4_words(hd), P = pool.page_size, per = over(a.heads, pool.kv_heads);
    // The parts are the grid's slowest dimension: CTAs of parts that a short row does not have come
    // last.  Between the others they cost 3 to 4 us of a slot each (4 contexts of 82K positions, 8
    // heads of 64: 60 us, now 48; 33 of 8K, 28 heads on 4 of 128, lose 119 -> 123).
    const int b = blockIdx.y, part_nr = blockIdx.z, above = gridDim.x == pool.kv_heads ? 0 : blockIdx.x / pool.kv_heads;
    const int kvh = blockIdx.x - above * pool.kv_heads, row0 = above * ROWS;
    const int tile_words = kv4_tile_words(hd), tpp = P / KV4_TILE;
    const uint32_t tile_bytes = (uint32_t)tile_words * 4;
    unsigned char* ring = smem + (size_t)wid * ATT_STAGES * SU * tile_bytes;
    if (lane < ATT_STAGES) mbar_init(&s_bar[wid][lane], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
    const int* table = a.table + (long long)b * a.table_stride;
    const char* head = reinterpret_cast<const char*>(pool.base) + kvh * pool.head_stride;
    // Run `run` of the tiles tile0 .. tile0 + tiles - 1: lane u stands for tile u of the run; the
    // first tile of the run and of every page copies the tiles that lie behind one another.
    struct Look {
        int page, in_page, len;  // len 0: nothing to copy
    };
    auto look = [&](int tile0, int tiles, int run) {
        const int u0 = run * SU, n = min(SU, tiles - u0);
        const int tile = tile0 + u0 + lane;
        const int nth = sp.page_shift >= 0 ? tile >> sp.page_shift : tile / tpp, in_page = tile - nth * tpp;
        const bool starts = lane < n && (lane == 0 || in_page == 0);
        return Look{starts ? table[nth] : -1, in_page, starts ? min(n - lane, tpp - in_page) : 0};
    };
    auto copy = [&](const Look& k, int slot) {
        const bool there = k.len > 0 && k.page >= 0 && k.page < pool.pages;
        const uint32_t ok = __reduce_or_sync(FULL, there ? ((1u << k.len) - 1) << lane : 0u);
        if (lane == 0) {
            s_ok[wid][slot] = ok;
            mbar_expect_tx(&s_bar[wid][slot], __popc(ok) * tile_bytes);
        }
        __syncwarp();
        if (there)
            bulk_load(ring + (size_t)(slot * SU + lane) * tile_bytes,
                      head + k.page * pool.page_stride + (long long)k.in_page * tile_bytes, k.len * tile_bytes,
                      &s_bar[wid][slot]);
    };
    pdl_wait();
    // A CTA that begins at position 0 asks for its first runs by the table alone, whatever the
    // row's length: one memory latency less (2560 CTAs of one position 18.3 -> 16.4 us; with two
    // groups the registers it holds cost more than that).  Runs behind the length are waited for.
    const int whole_row = NG == 1 && sp.splits == 1 && above == 0 ? a.width * tpp : 0;
    Look ahead[ATT_STAGES];
    if constexpr (NG == 1)
#pragma unroll
        for (int i = 0; i < ATT_STAGES; ++i) ahead[i] = look(0, whole_row, wid + i * W);
    const int chunk = chunk_of(pool, a, sp);
    const Row row(pool, a, b);
    int early = 0;
    if constexpr (NG == 1)
#pragma unroll
        for (int i = 0; i < ATT_STAGES; ++i)
            if ((wid + i * W) * SU < whole_row) {
                copy(ahead[i], i);
                early = i + 1;
            }
    const int rows = min(ROWS, min(row.n, a.max_q) * per - row0);  // this CTA's (token, head) rows
    const int end = rows > 0 ? row.end(a, over(row0 + rows - 1, per)) : 0, all_see = rows > 0 ? row.end(a, over(row0, per)) : 0;
    const int n_split = splits_of(end, chunk);
    if (rows <= 0 || part_nr >= n_split) {
        for (int i = 0; i < early; ++i) mbar_wait(&s_bar[wid][i], 0);
        return;
    }
    // its pieces of equal size, in whole runs
    constexpr int RUN = SU * KV4_TILE;
    const int piece = n_split == 1 ? end : ((end + n_split - 1) / n_split + RUN - 1) / RUN * RUN;
    const int first = min(end, part_nr * piece), last = min(end, first + piece);
    // this warp's runs of SU tiles: wid, wid + W, ... of the piece
    const int tile0 = first / KV4_TILE, tiles = (last - first + KV4_TILE - 1) / KV4_TILE;
    const int runs = (tiles + SU - 1) / SU;
    if (early == 0)
#pragma unroll
        for (int i = 0; i < ATT_STAGES; ++i)
            if (wid + i * W < runs) copy(look(tile0, tiles, wid + i * W), i);

    // q in fragment order; a negative scale goes into it.  Fixed point of 24 bits relative to its row's
    // largest, in planes of signed bytes (dims 0 2 4 6, 1 3 5 7 of a word), or fp16 after a power of
    // two, in planes of a word's dims 0 4 1 5 and 2 6 3 7.  A q that is not finite makes its
    // row NaN by its factor.
    int8_t* qb = reinterpret_cast<int8_t*>(smem + ring_bytes);
    constexpr int MAGIC = 0x4b400000;  // 1.5 2^23 as bits: sums onto it read as floats, exact below 2^22
    for (int r = wid; r < ROWS; r += W) {
        if (r >= rows) {
            for (int k = lane; k < 16 * NG; k += 32)
#pragma unroll
                for (int pl = 0; pl < QP; ++pl) *reinterpret_cast<int*>(qb + (pl * ROWS + r) * S::QROW + 4 * k) = 0;
            if (lane < NG) {
                s_qs[r][lane] = 0.f;
#pragma unroll
                for (int pl = 0; pl < QP; ++pl)
                    if (F32) s_from[r][lane][pl] = MAGIC;
            }
            if (lane == 0) {
                s_f[r] = 1.f;
                s_end[r] = end;
            }
            continue;
        }
        const int qi = over(row0 + r, per), h = kvh * per + (row0 + r - qi * per);
        const T* qp = reinterpret_cast<const T*>(a.q) + (row.q0 + (long long)qi) * a.q_token_stride + h * a.q_head_stride;
        float x[2 * NG], mx = 0.f;
        bool odd = false;
#pragma unroll
        for (int k = 0; k < 2 * NG; ++k) {
            const int d = lane + 32 * k;
            x[k] = d < hd ? to_f32<T>(qp[d]) : 0.f;
            odd |= !(fabsf(x[k]) < INFINITY);
            mx = fmaxf(mx, fabsf(x[k]));
        }
        mx = warp_max(mx);
        odd = __any_sync(FULL, odd);
        if constexpr (!INT) {
            // the exponent of the row's largest; rows below 2^-100 keep less
            const int e2 = mx > 0.f && !odd ? max(-100, (__float_as_int(mx) >> 23) - 127) : 0;
            const float up = a.scale < 0.f ? -pow2(14 - e2) : pow2(14 - e2);
            float sum[NG];
#pragma unroll
            for (int n = 0; n < NG; ++n) sum[n] = 0.f;
#pragma unroll
            for (int k = 0; k < 2 * NG; ++k) {
                const int d = lane + 32 * k, i = d & 7, pl = (i >> 1) & 1, at = (d & ~7) + 4 * (i & 1) + 2 * (i >> 2);
                const __half v = __float2half_rn(odd ? 0.f : x[k] * up);
                *reinterpret_cast<__half*>(qb + (pl * ROWS + r) * S::QROW + at) = v;
                sum[k >> 1] += __half2float(v);
            }
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                sum[n] = warp_sum(sum[n]);
                if (lane == 0) s_qs[r][n] = sum[n];
            }
            if (lane == 0) {
                s_f[r] = odd ? NAN : fmaxf(fabsf(a.scale) * LOG2E * pow2(e2 - 14), 1e-37f);
                s_end[r] = row.end(a, qi);
            }
            continue;
        }
        // the largest integer of three signed bytes, less what rounding may add
        constexpr float top = 8355000.f;
        const float up = mx > 1e-30f && !odd ? (a.scale < 0.f ? -top : top) / mx : 0.f;
        int sum[NG][QP];
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int pl = 0; pl < QP; ++pl) sum[n][pl] = 0;
#pragma unroll
        for (int k = 0; k < 2 * NG; ++k) {
            const int d = lane + 32 * k, i = d & 7, at = (d & ~7) + 4 * (i & 1) + (i >> 1);
            int v = odd ? 0 : __float2int_rn(x[k] * up);
#pragma unroll
            for (int pl = 0; pl < QP; ++pl) {  // plane 0 is the lowest byte
                const int8_t byte = (int8_t)v;
                qb[(pl * ROWS + r) * S::QROW + at] = byte;
                sum[k >> 1][pl] += byte;
                v = (v - byte) >> 8;
            }
        }
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            float all = 0.f;
#pragma unroll
            for (int pl = QP - 1; pl >= 0; --pl) {
                sum[n][pl] = __reduce_add_sync(FULL, sum[n][pl]);
                all = fmaf(all, 256.f, (float)sum[n][pl]);
                if (F32 && lane == 0) s_from[r][n][pl] = MAGIC - 8 * sum[n][pl];
            }
            if (lane == 0) s_qs[r][n] = all;
        }
        if (lane == 0) {
            s_f[r] = odd ? NAN : up == 0.f ? 1.f : fmaxf(fabsf(a.scale) * LOG2E / fabsf(up), 1e-37f);
            s_end[r] = row.end(a, qi);
        }
    }
    __syncthreads();
    pdl_trigger();
    uint32_t qf[QM][NT][2 * NG][2];
    float f[NT][NC], qs[NG][NT][NC];
    int from[NG][QP][NT][NC];  // fp32 only: MAGIC - 8 sum(q)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int m = 0; m < QM; ++m)
#pragma unroll
            for (int j = 0; j < 2 * NG; ++j) {
                const int r = NC == 2 ? nt * 8 + g : nt * 4 + (g >> 1), pl = NC == 2 ? m : min(2, 2 * m + (g & 1));
                uint2 v = *reinterpret_cast<const uint2*>(qb + (pl * ROWS + r) * S::QROW + 8 * (4 * j + t));
                if (NC == 1 && m == 1 && (g & 1)) v = make_uint2(0, 0);
                qf[m][nt][j][0] = v.x;
                qf[m][nt][j][1] = v.y;
            }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int r = NC * (nt * 4 + t) + c;
            f[nt][c] = s_f[r];
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                qs[n][nt][c] = s_qs[r][n];
#pragma unroll
                for (int pl = 0; pl < QP; ++pl) from[n][pl][nt][c] = F32 ? s_from[r][n][pl] : MAGIC;
            }
        }
    }

    // per lane: columns 2 t (and 2 t + 1), c = 0 (1); accumulator element c + 2 i is row g + 8 i.
    // Scores are kept without the factor f: m is the running maximum of those, and probabilities are
    // 2^((score - m) f), since score f - m f would be off by the rounding of m f, which is no longer small
    // where scores pass 2^24.
    float o[NG][4][NT][4], ob[NG][NT][NC], m[NT][NC], l[NT][NC];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            m[nt][c] = -INFINITY;
            l[nt][c] = 0.f;
#pragma unroll
            for (int n = 0; n < NG; ++n) ob[n][nt][c] = 0.f;
        }
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][mt][nt][e] = 0.f;
    // Probabilities times V scales enter the product as fp16: `cv`, a power of two that keeps
    // the largest scale so far below 2^15, holds them at the top of its range, so that
    // those of 2^-27 still have full precision.
    float cv = 274877906944.f;  // 2^38: fp16's smallest scale is 2^14 times it; any larger one lowers it
    // byte offsets of this lane's words in a tile
    uint32_t k_at[2 * NG];
#pragma unroll
    for (int j = 0; j < 2 * NG; ++j) k_at[j] = 4 * (64 * j + 2 * (min(4, max(0, nw - 4 * j)) * g + t));
    const uint32_t v_at = 4 * (16 * nw + 16 * g + 4 * t), m_at = 4 * (32 * nw + 4 * g);
    const uint32_t ring_at = smem_u32(ring);

    // One run.  PLAIN: all its tiles are there and every query sees every position.
    auto work = [&](auto plain, int run, int slot, uint32_t ok) {
        constexpr bool PLAIN = decltype(plain)::value;
        const uint32_t st = ring_at + slot * SU * tile_bytes;
        const int pos0 = (tile0 + run * SU) * KV4_TILE + g;  // this lane's positions: pos0 + 16 u and 8 further
        float s[SU][NT][2 * NC];
        uint32_t vm[SU][NG][2];  // V (s, b) of this lane's positions
        float vmax = 0.f;
#pragma unroll
        for (int u = 0; u < SU; ++u) {
            const uint32_t tile = st + u * tile_bytes;
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                [[maybe_unused]] int acc[QM][NT][4];
                [[maybe_unused]] float dots[NT][4];
#pragma unroll
                for (int jj = 0; jj < 2; ++jj) {
                    const int j = 2 * n + jj;
                    // lanes past the vector's last word read what lies behind; their q is zero
                    const uint2 w = lds64(tile + k_at[j]);
                    if constexpr (!INT) {
                        uint32_t x[4], y[4];
                        codes_minus_8(w.x, x);
                        codes_minus_8(w.y, y);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int m = 0; m < QM; ++m) {
                                const uint32_t* b = qf[m][nt][j];
                                if (jj == 0 && m == 0) mma16816_new(dots[nt], x[0], y[0], x[1], y[1], b[0], b[1]);
                                else mma16816(dots[nt], x[2 * m], y[2 * m], x[2 * m + 1], y[2 * m + 1], b[0], b[1]);
                            }
                        continue;
                    }
                    const uint32_t x0 = w.x & 0x0f0f0f0fu, x1 = (w.x >> 4) & 0x0f0f0f0fu;
                    const uint32_t y0 = w.y & 0x0f0f0f0fu, y1 = (w.y >> 4) & 0x0f0f0f0fu;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int m = 0; m < QM; ++m) {
                            if (jj == 0)
                                imma16832_on(acc[m][nt], x0, y0, x1, y1, qf[m][nt][j][0], qf[m][nt][j][1],
                                             from[n][NC == 1 ? 2 * m : m][nt][0],
                                             NC == 2 ? from[n][m][nt][NC - 1] : m == 0 ? from[n][1][nt][0] : MAGIC);
                            else imma16832(acc[m][nt], x0, y0, x1, y1, qf[m][nt][j][0], qf[m][nt][j][1]);
                        }
                }
                const uint4 meta = lds128(tile + m_at + 128 * n);
                vm[u][n][0] = meta.z;
                vm[u][n][1] = meta.w;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float2 k = half2_of(i ? meta.y : meta.x);
                    const float kb = F32 || !INT ? fmaf(8.f, k.x, k.y) : k.y;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < NC; ++c) {
                            float dot = 0.f;
                            if constexpr (INT) {
#pragma unroll
                                for (int pl = QP - 1; pl >= 0; --pl) {
                                    const int sum = NC == 2 ? acc[pl][nt][2 * i + c] : acc[pl >> 1][nt][2 * i + (pl & 1)];
                                    const float part = __int_as_float(sum) - 12582912.f;
                                    dot = pl == QP - 1 ? part : fmaf(dot, 256.f, part);
                                }
                            } else {
                                dot = dots[nt][2 * i + c];
                            }
                            float& d = s[u][nt][NC * i + c];
                            d = fmaf(kb, qs[n][nt][c], n == 0 ? dot * k.x : fmaf(dot, k.x, d));
                        }
                    const float vs = half2_of(vm[u][n][i]).x;
                    if (PLAIN || (((ok >> u) & 1) && pos0 + 16 * u + 8 * i < last)) vmax = fmaxf(vmax, vs);
                }
            }
            if constexpr (!PLAIN) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2 * NC; ++e) {
                        const int pos = pos0 + 16 * u + 8 * (e / NC);
                        if (!((ok >> u) & 1) || pos >= last || pos >= s_end[NC * (nt * 4 + t) + e % NC])
                            s[u][nt][e] = -INFINITY;
                    }
            }
        }
        // running maxima, and the accumulators when one rose or a scale outgrew `cv`: rare once
        // the first positions are behind, so only then do the lanes of a column compare theirs
        bool rose = vmax * cv > 32768.f;
        float top[NT][NC];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                top[nt][c] = fmaxf(s[0][nt][c], s[0][nt][NC + c]);
#pragma unroll
                for (int u = 1; u < SU; ++u) top[nt][c] = fmaxf(top[nt][c], fmaxf(s[u][nt][c], s[u][nt][NC + c]));
                rose |= top[nt][c] > m[nt][c];
            }
        if (__any_sync(FULL, rose)) {
            vmax = fminf(rows_max(vmax), 65504.f);
            float down = 1.f;
            if (vmax * cv > 32768.f) {
                const float to = pow2(13 - ilogbf(vmax));
                down = to / cv;
                cv = to;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const float mx = fmaxf(m[nt][c], rows_max(top[nt][c]));
                    const float corr = m[nt][c] == -INFINITY ? 0.f : ex2((m[nt][c] - mx) * f[nt][c]), both = corr * down;
                    m[nt][c] = mx;
                    l[nt][c] *= corr;
#pragma unroll
                    for (int n = 0; n < NG; ++n) {
                        ob[n][nt][c] *= corr;
#pragma unroll
                        for (int mt = 0; mt < 4; ++mt) {
                            o[n][mt][nt][c] *= both;
                            o[n][mt][nt][2 + c] *= both;
                        }
                    }
                }
        }
        // probabilities, and their product with V
#pragma unroll
        for (int u = 0; u < SU; ++u)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2 * NC; e += 2) {
                    const float2 x = make_float2(s[u][nt][e], s[u][nt][e + 1]);
                    const float2 y = mul2(add2(x, make_float2(-m[nt][0], -m[nt][NC - 1])), make_float2(f[nt][0], f[nt][NC - 1]));
                    s[u][nt][e] = ex2(y.x);
                    s[u][nt][e + 1] = ex2(y.y);
                    if constexpr (!PLAIN) {  // even by a query that is NaN
                        if (x.x == -INFINITY) s[u][nt][e] = NOT_SEEN;
                        if (x.y == -INFINITY) s[u][nt][e + 1] = NOT_SEEN;
                    }
                    l[nt][0] += s[u][nt][e];
                    l[nt][NC - 1] += s[u][nt][e + 1];
                }
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            // fp32 results: a run's products sum by themselves, since the tensor core cuts what a
            // long running sum no longer holds
            float fresh[4][NT][4];
#pragma unroll
            for (int u = 0; u < SU; ++u) {
                const float2 v0 = half2_of(vm[u][n][0]), v1 = half2_of(vm[u][n][1]);
                const float s0 = v0.x * cv, s1 = v1.x * cv, b0 = fmaf(8.f, v0.x, v0.y), b1 = fmaf(8.f, v1.x, v1.y);
                const uint4 vw = lds128(st + u * tile_bytes + v_at + 512 * n);
                uint32_t va[8], vb[8];  // dim e of the word: positions 2 t and 2 t + 1; 2 t + 8 and 2 t + 9
                codes_minus_8(__byte_perm(vw.x, vw.y, 0x5410), va);
                codes_minus_8(__byte_perm(vw.x, vw.y, 0x7632), va + 4);
                codes_minus_8(__byte_perm(vw.z, vw.w, 0x5410), vb);
                codes_minus_8(__byte_perm(vw.z, vw.w, 0x7632), vb + 4);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float w[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int e = 0; e < 2 * NC; ++e) {
                        const float p = s[u][nt][e], sv = e < NC ? s0 : s1, bv = e < NC ? b0 : b1;
                        // what a query does not see adds nothing, whatever its page holds; what it sees
                        // does, a NaN even where p underflowed
                        const bool none = !PLAIN && not_seen(p);
                        w[2 * (e / NC) + e % NC] = none ? 0.f : p * sv;
                        ob[n][nt][e % NC] = none ? ob[n][nt][e % NC] : fmaf(p, bv, ob[n][nt][e % NC]);
                    }
#pragma unroll
                    for (int pl = 0; pl < PP; ++pl) {
                        const uint32_t r0 = pack_half2(w[0], w[1]), r8 = pack_half2(w[2], w[3]);
                        if (pl + 1 < PP) {
                            const float2 h0 = half2_of(r0), h8 = half2_of(r8);
                            w[0] -= h0.x;
                            w[1] -= h0.y;
                            w[2] -= h8.x;
                            w[3] -= h8.y;
                        }
                        const uint32_t t0 = transpose8x8(r0), t8 = transpose8x8(r8);
#pragma unroll
                        for (int mt = 0; mt < 4; ++mt) {
                            if (F32 && u == 0 && pl == 0)
                                mma16816_new(fresh[mt][nt], va[2 * mt], va[2 * mt + 1], vb[2 * mt], vb[2 * mt + 1], t0, t8);
                            else
                                mma16816(F32 ? fresh[mt][nt] : o[n][mt][nt], va[2 * mt], va[2 * mt + 1], vb[2 * mt],
                                         vb[2 * mt + 1], t0, t8);
                        }
                    }
                }
            }
            if constexpr (F32)
#pragma unroll
                for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[n][mt][nt][e] += fresh[mt][nt][e];
        }
    };
    const int see = min(all_see, last) / KV4_TILE - tile0;  // whole tiles that every query sees
    int slot = 0, run = wid;
    uint32_t phase = 0;
    for (; run < runs; run += W) {
        if (!__all_sync(FULL, mbar_wait(&s_bar[wid][slot], phase, KV4_WAIT_LIMIT))) break;
        const uint32_t ok = s_ok[wid][slot];
        if (ok == (1u << SU) - 1 && (run + 1) * SU <= see) work(std::true_type{}, run, slot, ok);
        else work(std::false_type{}, run, slot, ok);
        __syncwarp();  // every lane has read the slot
        if (run + ATT_STAGES * W < runs) copy(look(tile0, tiles, run + ATT_STAGES * W), slot);
        if (++slot == ATT_STAGES) {
            slot = 0;
            phase ^= 1;
        }
    }

    if (run < runs) {  // a copy did not come: no result rather than a wrong one, once no other is in flight
        if (lane == 0 && a.status) atomicCAS(a.status, 0u, (unsigned)DEV_WAIT_TIMEOUT);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < NC; ++c) l[nt][c] = NAN;
        for (int i = 0; i < ATT_STAGES && run + i * W < runs; ++i)
            mbar_wait(&s_bar[wid][(slot + i) % ATT_STAGES], phase ^ (uint32_t)((slot + i) / ATT_STAGES));
    }
    for (int i = 0; i < early; ++i)
        if (wid + i * W >= runs) mbar_wait(&s_bar[wid][i], 0);

    // join the warps: unnormalised sums in shared memory (the rings are done with)
    if (W > 1) __syncthreads();
    float* join = reinterpret_cast<float*>(smem);
    const int ld = hd + 4;
    const float up = 1.f / cv;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int r = NC * (nt * 4 + t) + c;
            const float lr = rows_sum(l[nt][c]);
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                const float bias = rows_sum(ob[n][nt][c]);
                float* dst = join + (size_t)(wid * ROWS + r) * ld + 64 * n + 8 * g;
                if (r < rows && 64 * n + 8 * g < hd)
#pragma unroll
                    for (int mt = 0; mt < 4; ++mt)
                        *reinterpret_cast<float2*>(dst + 2 * mt) =
                            make_float2(fmaf(o[n][mt][nt][c], up, bias), fmaf(o[n][mt][nt][2 + c], up, bias));
            }
            if (g == 0) {
                const float mf = m[nt][c] == -INFINITY ? -INFINITY : m[nt][c] * f[nt][c];
                s_m[wid][r] = mf;
                s_l[wid][r] = m[nt][c] > -INFINITY && fabsf(mf) == INFINITY ? NAN : lr;  // a score past fp32's range
            }
        }
    if (W > 1) __syncthreads();
    else __syncwarp();
    const bool whole = n_split == 1;
    for (int r = wid; r < rows; r += W) {
        float mx = -INFINITY, ls = 0.f;
        for (int w = 0; w < W; ++w) mx = fmaxf(mx, s_m[w][r]);
        float v[2 * NG];
#pragma unroll
        for (int k = 0; k < 2 * NG; ++k) v[k] = 0.f;
        for (int w = 0; w < W; ++w) {
            const float fw = s_m[w][r] == -INFINITY ? 0.f : ex2(s_m[w][r] - mx);
            if (s_l[w][r] == 0.f) continue;
            ls = fmaf(s_l[w][r], fw, ls);
#pragma unroll
            for (int k = 0; k < 2 * NG; ++k)
                if (lane + 32 * k < hd) v[k] = fmaf(join[(size_t)(w * ROWS + r) * ld + lane + 32 * k], fw, v[k]);
        }
        const float inv = ls == 0.f ? 0.f : 1.f / ls;  // nothing seen: zeros
        const int qi = over(row0 + r, per), h = kvh * per + (row0 + r - qi * per);
        const long long tok = row.q0 + (long long)qi;
        if (whole) {
            const long long out = tok * a.out_token_stride + h * a.out_head_stride;
#pragma unroll
            for (int k = 0; k < 2 * NG; ++k)
                if (lane + 32 * k < hd) put<T>(a, out + lane + 32 * k, ls != ls ? NAN : v[k] * inv);
        } else {
            const long long each = a.q_tokens * a.heads, at = part_nr * each + tok * a.heads + h;
#pragma unroll
            for (int k = 0; k < 2 * NG; ++k)
                if (lane + 32 * k < hd) sp.part[at * hd + lane + 32 * k] = v[k];
            if (lane == 0) reinterpret_cast<float2*>(sp.part + sp.splits * each * hd)[at] = make_float2(mx, ls);
        }
    }
}

// Joins the CTAs of contexts longer than one chunk, in their order: a (token, head) row has 16
// lanes (32 for more than 64 dims) of four dims each, of one warp, or of all eight of a CTA
// (WIDE) when there are many parts, each warp taking every eighth.  Four parts are loaded at a
// time and added under a running maximum, so that up to four cost one memory latency.
template <class T, bool WIDE>
__global__ void __launch_bounds__(256, 4) kv4_attention_join_kernel(const Kv4Pool pool, const Kv4Attention a,
                                                                    const AttSplit sp) {
    __shared__ float4 s_v[8][32];
    __shared__ float2 s_ml[8][32];
    pdl_wait();
    const int chunk = chunk_of(pool, a, sp);
    const Row row(pool, a, blockIdx.y);
    if (row.len <= chunk) return;  // nothing to join
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, hd = pool.head_dim;
    const int lanes = hd <= 64 ? 16 : 32, sub = lane & (lanes - 1), at_once = (WIDE ? 1 : 8) * (32 / lanes);
    const int per = over(a.heads, pool.kv_heads), tokens = min(row.n, a.max_q);
    const bool dims = 4 * sub < hd;
    const long long each = a.q_tokens * a.heads;
    for (int r0 = blockIdx.x * at_once; r0 < tokens * a.heads; r0 += gridDim.x * at_once) {
        const int r = r0 + (WIDE ? 0 : wid * (32 / lanes)) + lane / lanes, qi = r / a.heads, h = r - qi * a.heads;
        // the CTAs that had this row went by their last row's end
        const int in_head = qi * per + h % per;
        const int last = min(in_head / sp.rows * sp.rows + sp.rows, tokens * per) - 1;
        int n = qi < tokens ? splits_of(row.end(a, over(last, per)), chunk) : 1;
        if (n == 1) n = 0;
        const long long tok = row.q0 + (long long)qi, at = tok * a.heads + h;
        const float2* ml = reinterpret_cast<const float2*>(sp.part + sp.splits * each * hd) + at;
        const float* part = sp.part + at * hd + 4 * sub;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float mx = -INFINITY, ls = 0.f;
        auto add = [&](float2 x, float4 y) {  // a part (maximum, sum) and its values; the sum of one that saw nothing is 0
            if (x.y == 0.f) return;
            const float now = fmaxf(mx, x.x), was = mx == -INFINITY ? 0.f : ex2(mx - now);
            const float f = x.x == -INFINITY ? 0.f : ex2(x.x - now);
            mx = now;
            ls = fmaf(ls, was, x.y * f);
            v = make_float4(fmaf(v.x, was, y.x * f), fmaf(v.y, was, y.y * f), fmaf(v.z, was, y.z * f), fmaf(v.w, was, y.w * f));
        };
        constexpr int STEP = WIDE ? 8 : 1;
        for (int s0 = WIDE ? wid : 0; s0 < n; s0 += 4 * STEP) {
            float2 x[4];
            float4 y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int s = s0 + i * STEP;
                x[i] = s < n ? ml[s * each] : make_float2(-INFINITY, 0.f);
                y[i] = s < n && dims ? *reinterpret_cast<const float4*>(part + s * each * hd) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) add(x[i], y[i]);
        }
        if constexpr (WIDE) {
            s_v[wid][lane] = v;
            s_ml[wid][lane] = make_float2(mx, ls);
            __syncthreads();
            if (wid == 0)
                for (int w = 1; w < 8; ++w) add(s_ml[w][lane], s_v[w][lane]);
            __syncthreads();
        }
        if (n == 0 || !dims || (WIDE && wid != 0)) continue;
        const float inv = ls == 0.f ? 0.f : 1.f / ls, z[4] = {v.x, v.y, v.z, v.w};
        const long long out = tok * a.out_token_stride + h * a.out_head_stride + 4 * sub;
#pragma unroll
        for (int k = 0; k < 4; ++k) put<T>(a, out + k, ls != ls ? NAN : z[k] * inv);
    }
}

template <class T>
cudaError_t launch_join(const Kv4Pool& pool, const Kv4Attention& a, const AttSplit& sp, cudaStream_t s) {
    ++launch_counter();
    const bool pdl = pdl_launches();
    pdl_launches() = true;  // the join waits for the parts in the kernel: its launch overlaps them
    const bool wide = sp.splits > 8;
    const long long at_once = (wide ? 1 : 8) * (pool.head_dim <= 64 ? 2 : 1);
    // few CTAs per row of the batch when there are many: most rows may have nothing to join
    const long long all = ((long long)a.max_q * a.heads + at_once - 1) / at_once, some = std::max(16, 148 * 8 / a.rows);
    const cudaError_t j = launch_kernel(wide ? kv4_attention_join_kernel<T, true> : kv4_attention_join_kernel<T, false>,
                                        dim3((unsigned)std::min(all, some), a.rows), dim3(256), 0, s, pool, a, sp);
    pdl_launches() = pdl;
    return j;
}

template <class T, int NG, int NT, int NC, int HD>
cudaError_t launch_shape(const Kv4Pool& pool, const Kv4Attention& a, const AttSplit& sp, cudaStream_t s) {
    using S = AttShape<T, NG, NT, NC>;
    const size_t smem = S::smem(pool.head_dim, sp.warps);
    const auto fn = kv4_attention_kernel<T, NG, NT, NC, HD>;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(fn),
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    ++launch_counter();
    return launch_kernel(fn, dim3(sp.per_row, a.rows, sp.splits), dim3(32 * sp.warps), smem, s, pool, a, sp,
                         (int)S::ring(pool.head_dim, sp.warps));
}

template <class T, int NG, int HD>
cudaError_t launch_head(const Kv4Pool& pool, const Kv4Attention& a, const AttSplit& sp, cudaStream_t s) {
    if (sp.rows == 4) return launch_shape<T, NG, 1, 1, HD>(pool, a, sp, s);
    if (sp.rows == 8) return launch_shape<T, NG, 1, 2, HD>(pool, a, sp, s);
    if constexpr (!is_step<T>)  // one token per row
        if (sp.rows == 16) return launch_shape<T, NG, 2, 2, HD>(pool, a, sp, s);
    return cudaErrorInvalidValue;
}

template <class T>
cudaError_t launch_type(const Kv4Pool& pool, const Kv4Attention& a, const AttSplit& sp, cudaStream_t s) {
    const int hd = pool.head_dim;
    cudaError_t e = cudaErrorInvalidValue;
    if constexpr (is_step<T>) {  // the decoder's head sizes
        if (hd <= 64) e = hd == 64 ? launch_head<T, 1, 64>(pool, a, sp, s) : launch_head<T, 1, 0>(pool, a, sp, s);
    } else {
        e = hd == 64    ? launch_head<T, 1, 64>(pool, a, sp, s)
            : hd == 128 ? launch_head<T, 2, 128>(pool, a, sp, s)
            : hd < 64   ? launch_head<T, 1, 0>(pool, a, sp, s)
            : launch_head<T, 2, 0>(pool, a, sp, s);
    }
    return e != cudaSuccess || sp.splits == 1 ? e : launch_join<T>(pool, a, sp, s);
}

}  // namespace
#endif  // KV4_ATTENTION_KERNELS

}  // namespace msb
