// 4-bit K/V attention for many query rows per K/V head (prompt chunks, drafted tokens of grouped
// heads): the same products as kv4_attention.cuh on the fifth-generation tensor cores.
//
// One CTA has 128 (token, head) rows of one K/V head and walks its positions 64 at a time:
//   warps 4-7  unpack: the 4-bit tiles of a stage (bulk copies, one tile per warp) into fp16
//              codes d = c - 8, K as rows of positions, V as rows of dims (its byte permute puts
//              two positions side by side, and row 8 (dim % 8) + dim / 8 makes the stores free of
//              bank conflicts), both 128-byte swizzled; scales and biases into shared memory
//   warp 8     one thread issues S_n = Q_n D_n^T for each group n of 64 dims (tcgen05, both
//              operands fp16, q scaled exactly by a power of two per row) and O_n += P_n D_n
//   warps 0-3  softmax, a thread per row: S_n out of tensor memory, scores
//              sum_n s_tn S_n + (b_tn + 8 s_tn) sum(q_n), running reference and sum, and
//              P_n = p_t s_tn back over S_n as the next product's operand, fp16 (two planes for
//              fp16 results); sum p_t (b_tn + 8 s_tn) stays in the thread
// With one group S has two buffers (and unpacked tiles three), so the product of the next stage runs under the softmax of
// this one; two CTAs share an SM and fill each other's gaps.  The reference of a row moves only
// when a probability times a scale could pass fp16's range, 8 bits above where it was set, so
// O is rescaled (tensor memory read and written by the row's thread) a few times per CTA.
// Bound: the softmax, about 9 fp32 operations and one ex2 per (row, position).
#define KV4_ATTENTION_KERNELS
#include "kv4_attention.cuh"

namespace msb {
namespace {

constexpr int WIDE_ROWS = 128;
constexpr int WIDE_STEP = 64;  // positions per stage
constexpr int WIDE_TILES = WIDE_STEP / KV4_TILE;
constexpr int WIDE_RAW = 3;    // stages of packed tiles
constexpr int WIDE_THREADS = 384;  // three warpgroups: softmax, unpacking, products (one warp of it)
constexpr uint32_t WIDE_COLS = 256;  // tensor memory columns: S in 2 buffers of 64 (or 2 groups), O from 128 on
constexpr uint32_t O_COL = 128;

template <int NG>
struct WideSmem {
    static constexpr int NB = NG == 1 ? 3 : 1;  // buffers of unpacked tiles
    static constexpr int NS = NG == 1 ? 2 : 1;  // of S, in tensor memory
    static constexpr int BLOCK = WIDE_STEP * 128;  // 64 rows of 128 bytes
    static constexpr int Q = NG * WIDE_ROWS * 128, K = NB * NG * BLOCK, V = NB * NG * BLOCK;
    static int raw(int hd) { return (WIDE_TILES * kv4_tile_words(hd) * 4 + 127) / 128 * 128; }
    static size_t bytes(int hd) { return (size_t)Q + K + V + WIDE_RAW * raw(hd) + 512 + 1024; }  // + alignment
};

__device__ __forceinline__ uint64_t sw128_desc(uint32_t addr) {  // K-major rows of 128 bytes, 8-row groups
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// fp16 A and B, both K-major, fp32 sums, 128 x n
__device__ __forceinline__ constexpr uint32_t f16_idesc(int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void commit_to(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t at, float* v) {  // the caller waits
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at));
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void sts32(uint32_t a, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ void sts128(uint32_t a, const uint32_t* v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
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

__device__ __forceinline__ float4 four(const float* p) { return *reinterpret_cast<const float4*>(p); }

// Bounded wait that also ends when another role has given up.
__device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity, volatile int* failed) {
    const uint32_t a = smem_u32(bar);
    for (uint32_t i = 0; i < WAIT_LIMIT; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(a), "r"(parity)
            : "memory");
        if (ok) return true;
        if ((i & 255) == 255 && *failed) return false;
    }
    *failed = 1;
    return false;
}

template <class T, int NG>
__global__ void __launch_bounds__(WIDE_THREADS, 2) kv4_attention_wide_kernel(const Kv4Pool pool, const Kv4Attention a,
                                                                             const AttSplit sp) {
    using S = WideSmem<NG>;
    constexpr int NB = S::NB, NS = S::NS, PP = is_bf16<T> ? 1 : 2;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t s_raw_full[WIDE_RAW], s_raw_empty[WIDE_RAW];
    // Stage i: entry i % 2 of s_k, s_s and s_p, i % 4 of s_v and s_pv, so that an entry's next
    // phase always waits, through the other roles, for whoever still has to see this one.
    __shared__ __align__(8) uint64_t s_k[2], s_v[4], s_s[2], s_p[2], s_pv[4];
    __shared__ uint32_t s_okr[WIDE_RAW], s_ok[2], s_tmem;
    __shared__ int s_failed;
    __shared__ __align__(16) float s_meta[2][NG][4][WIDE_STEP];  // K's s and b + 8 s, V's
    __shared__ __align__(16) float s_vmax[2][WIDE_TILES];
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const int hd = pool.head_dim, nw = kv4_words(hd), P = pool.page_size, per = over(a.heads, pool.kv_heads);
    // the last queries first: under a causal mask they see the most
    const int b = blockIdx.z, y = gridDim.y - 1 - blockIdx.y, above = gridDim.y == pool.kv_heads ? 0 : y / pool.kv_heads;
    const int kvh = y - above * pool.kv_heads, row0 = above * WIDE_ROWS;
    pdl_wait();
    const int chunk = chunk_of(pool, a, sp);
    const Row row(pool, a, b);
    const int rows = min(WIDE_ROWS, min(row.n, a.max_q) * per - row0);  // this CTA's (token, head) rows
    if (rows <= 0) return;
    const int end = row.end(a, over(row0 + rows - 1, per)), all_see = row.end(a, over(row0, per));
    const int n_split = splits_of(end, chunk);
    if ((int)blockIdx.x >= n_split) return;
    const int piece = n_split == 1 ? end : ((end + n_split - 1) / n_split + WIDE_STEP - 1) / WIDE_STEP * WIDE_STEP;
    const int first = min(end, (int)blockIdx.x * piece), last = min(end, first + piece);
    const int tile0 = first / KV4_TILE, tiles = (last - first + KV4_TILE - 1) / KV4_TILE;
    const int steps = (tiles + WIDE_TILES - 1) / WIDE_TILES;
    const int active = (rows + 31) / 32;  // softmax warps with rows

    const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
    const uint32_t q_at = base, k_buf = q_at + S::Q, v_buf = k_buf + S::K, raw_at = v_buf + S::V;
    const int tile_words = kv4_tile_words(hd), tpp = P / KV4_TILE;
    const uint32_t tile_bytes = (uint32_t)tile_words * 4, raw_bytes = (WIDE_TILES * tile_bytes + 127) / 128 * 128;
    if (threadIdx.x == 0) {
        for (int i = 0; i < WIDE_RAW; ++i) {
            mbar_init(&s_raw_full[i], 1);
            mbar_init(&s_raw_empty[i], WIDE_TILES);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_k[i], WIDE_TILES);
            mbar_init(&s_s[i], 1);
            mbar_init(&s_p[i], active);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&s_v[i], WIDE_TILES);
            mbar_init(&s_pv[i], 1);
        }
        s_failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (wid == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                     "r"(WIDE_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // K rows end with zeros where the head is shorter than its groups (q is zero there too)
    if (nw < 8 * NG)
        for (uint32_t i = threadIdx.x; i < (uint32_t)S::K / 16; i += WIDE_THREADS) {
            const uint32_t zero[4] = {0, 0, 0, 0};
            sts128(k_buf + 16 * i, zero);
        }
    // q rows, a thread each, in the order that unpacked words have (dims 0 4 1 5 2 6 3 7)
    float f = 1.f, qs[NG];
    int lim = last;
#pragma unroll
    for (int n = 0; n < NG; ++n) qs[n] = 0.f;
    const int r = threadIdx.x;
    const bool mine = wid < 4 && r < rows;
    const int qi = mine ? over(row0 + r, per) : 0, h = mine ? kvh * per + (row0 + r - qi * per) : 0;
    const long long tok = row.q0 + (long long)qi;
    if (wid < 4) {
        const T* qp = reinterpret_cast<const T*>(a.q) + tok * a.q_token_stride + h * a.q_head_stride;
        const bool wide = !((reinterpret_cast<uintptr_t>(qp)) & 15);
        float mx = 0.f;
        bool odd = false;
        auto word = [&](int w, float (&x)[8]) {
            if (!mine || w >= nw) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = 0.f;
            } else if (wide) {
                const uint4 v = *reinterpret_cast<const uint4*>(qp + 8 * w);
                const T* t = reinterpret_cast<const T*>(&v);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = to_f32<T>(t[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = to_f32<T>(qp[8 * w + e]);
            }
        };
#pragma unroll 1
        for (int w = 0; w < nw; ++w) {
            float x[8];
            word(w, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                odd |= !(fabsf(x[e]) < INFINITY);
                mx = fmaxf(mx, fabsf(x[e]));
            }
        }
        const int e2 = mx > 0.f && !odd ? min(100, max(-100, ilogbf(mx))) : 0;
        const float up = a.scale < 0.f ? -pow2(14 - e2) : pow2(14 - e2);
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
                float x[8];
                word(8 * n + c, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = odd ? 0.f : x[e] * up;
                    qs[n] += x[e];
                }
                uint32_t v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = pack_half2(x[e], x[e + 4]);
                sts128(q_at + n * (WIDE_ROWS * 128) + r * 128 + ((c ^ (r & 7)) << 4), v);
            }
        f = odd ? NAN : fmaxf(fabsf(a.scale) * LOG2E * pow2(e2 - 14), 1e-37f);
        if (mine) lim = min(last, row.end(a, qi));
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    fence_before();
    __syncthreads();
    fence_after();
    pdl_trigger();
    const uint32_t tmem = s_tmem;
    volatile int* failed = &s_failed;
    int loaded = 0;  // stages that warp 9 asked for

    // Registers from the 3 x 80 of the launch: 136 for the softmax, 64 to unpack, 40 for the rest.
    if (wid >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        // ---------------------------------------------------------------- products
        if (wid == 8 && lane == 0) {
            constexpr uint32_t idesc = f16_idesc(64);
            const uint64_t q_desc = sw128_desc(q_at), k_desc = sw128_desc(k_buf), v_desc = sw128_desc(v_buf);
            auto scores = [&](int i, int buf) {  // descriptors count in 16 bytes
                if (!wait_on(&s_k[i & 1], (i >> 1) & 1, failed)) return false;
                fence_after();
#pragma unroll
                for (int n = 0; n < NG; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_ss(tmem + (i % NS * NG + n) * 64, q_desc + n * (WIDE_ROWS * 8) + 2 * k,
                               k_desc + (buf * NG + n) * (S::BLOCK / 16) + 2 * k, idesc, k > 0);
                commit_to(&s_s[i & 1]);
                return true;
            };
            auto values = [&](int i, int buf) {
                if (!wait_on(&s_v[i & 3], (i >> 2) & 1, failed) || !wait_on(&s_p[i & 1], (i >> 1) & 1, failed)) return false;
                fence_after();
#pragma unroll
                for (int n = 0; n < NG; ++n)
#pragma unroll
                    for (int pl = 0; pl < PP; ++pl)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_ts(tmem + O_COL + n * 64, tmem + (i % NS * NG + n) * 64 + 32 * pl + 8 * k,
                                   v_desc + (buf * NG + n) * (S::BLOCK / 16) + 2 * k, idesc, i > 0 || pl > 0 || k > 0);
                commit_to(&s_pv[i & 3]);
                return true;
            };
            // with two buffers of S the next stage's scores go first: they run under this softmax
            bool ok = true;
            int next = 0;  // buffer of the next scores
            if (NS == 2 && steps > 0) ok = scores(0, next++);
            for (int i = 0, buf = 0; ok && i < steps; ++i) {
                if (NS == 1 || i + 1 < steps) {
                    ok = scores(i + NS - 1, next);
                    if (++next == NB) next = 0;
                }
                ok = ok && values(i, buf);
                if (++buf == NB) buf = 0;
            }
        } else if (wid == 9) {
            // ------------------------------------------------------------ loads: lane v is tile v of a stage
            const int* table = a.table + (long long)b * a.table_stride;
            const char* head = reinterpret_cast<const char*>(pool.base) + kvh * pool.head_stride;
            auto page_of = [&](int i, int& in_page) {  // -2: copied with the tile before it, or none
                const int u = i * WIDE_TILES + lane, nth = sp.page_shift >= 0 ? (tile0 + u) >> sp.page_shift : (tile0 + u) / tpp;
                in_page = tile0 + u - nth * tpp;
                return lane < WIDE_TILES && u < tiles && (lane == 0 || in_page == 0) ? table[nth] : -2;
            };
            int in_page, page = page_of(0, in_page);
            for (int i = 0; i < steps; ++i) {
                const int slot = i % WIDE_RAW, n = min(WIDE_TILES, tiles - i * WIDE_TILES);
                int in_next, next = page_of(i + 1, in_next);
                if (i >= WIDE_RAW && !wait_on(&s_raw_empty[slot], (i / WIDE_RAW - 1) & 1, failed)) break;
                __syncwarp();
                const bool here = page >= 0 && page < pool.pages;
                const int len = here ? min(n - lane, tpp - in_page) : 0;
                const uint32_t ok = __reduce_or_sync(FULL, here ? ((1u << len) - 1) << lane : 0u);
                if (lane == 0) {
                    s_okr[slot] = ok;
                    mbar_expect_tx(&s_raw_full[slot], __popc(ok) * tile_bytes);
                }
                __syncwarp();
                if (here)
                    bulk_load(smem_raw + (raw_at - smem_u32(smem_raw)) + slot * raw_bytes + lane * tile_bytes,
                              head + page * pool.page_stride + (long long)in_page * tile_bytes, len * tile_bytes,
                              &s_raw_full[slot]);
                loaded = i + 1;
                page = next;
                in_page = in_next;
            }
        }
        __syncwarp();
    } else if (wid >= 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        // ---------------------------------------------------------------- unpacking
        const int u = wid - 4, g = lane >> 2, t = lane & 3;  // this warp's tile of a stage
        uint32_t k_from[2 * NG];
#pragma unroll
        for (int j = 0; j < 2 * NG; ++j) k_from[j] = 4 * (64 * j + 2 * (min(4, max(0, nw - 4 * j)) * g + t));
        for (int i = 0; i < steps; ++i) {
            const int slot = i % WIDE_RAW, nb = i % NB, i2 = i & 1;
            if (!wait_on(&s_raw_full[slot], (i / WIDE_RAW) & 1, failed)) break;
            // Buffers of stage i - NB are free when its second product is done; with one buffer K's
            // when its first is.  The scales' are those of stage i - 2, which its softmax has read.
            if (NB == 1 && i >= 1 && !wait_on(&s_s[1 - i2], ((i - 1) >> 1) & 1, failed)) break;
            if (NB > 1 && i >= NB && !wait_on(&s_pv[(i - NB) & 3], ((i - NB) >> 2) & 1, failed)) break;
            if (NB > 1 && i >= 2 && !wait_on(&s_p[i2], ((i - 2) >> 1) & 1, failed)) break;
            const uint32_t okr = s_okr[slot];
            const bool here = (okr >> u) & 1;
            const uint32_t tile = raw_at + slot * raw_bytes + u * tile_bytes;
            const int pos = first - first % KV4_TILE + (i * WIDE_TILES + u) * KV4_TILE + g;  // and 8 further
            uint2 kw[2 * NG];
            uint4 mw[NG];
#pragma unroll
            for (int j = 0; j < 2 * NG; ++j)  // lanes past the vector's last word read what lies behind
                kw[j] = lds64(tile + k_from[j]);
#pragma unroll
            for (int n = 0; n < NG; ++n) mw[n] = lds128(tile + 4 * (32 * nw + 32 * n + 4 * g));
#pragma unroll
            for (int j = 0; j < 2 * NG; ++j) {
                if (4 * j + t >= nw) continue;
                uint32_t d[4];
                const uint32_t to = k_buf + (nb * NG + j / 2) * S::BLOCK + (16 * u + g) * 128 + ((((j & 1) * 4 + t) ^ g) << 4);
                codes_minus_8(kw[j].x, d);
                sts128(to, d);
                codes_minus_8(kw[j].y, d);
                sts128(to + 8 * 128, d);
            }
            float vmax = 0.f;
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                // lane t: K of position g, K of g + 8, V of g, V of g + 8
                const uint32_t w = t == 0 ? mw[n].x : t == 1 ? mw[n].y : t == 2 ? mw[n].z : mw[n].w;
                float2 sb = half2_of(w);
                sb.y = fmaf(8.f, sb.x, sb.y);
                if (!here || pos + 8 * (t & 1) >= last) sb = make_float2(0.f, 0.f);  // nobody sees it
                float* to = &s_meta[i2][n][t & 2][16 * u + g + 8 * (t & 1)];
                to[0] = sb.x;
                to[WIDE_STEP] = sb.y;
                if (t >= 2) vmax = fmaxf(vmax, sb.x);
            }
            vmax = fminf(warp_max(vmax), 65504.f);
            if (lane == 0) {
                s_vmax[i2][u] = vmax;
                if (u == 0) s_ok[i2] = okr;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_k[i2]);
            if (NB == 1 && i > 0 && !wait_on(&s_pv[(i - 1) & 3], ((i - 1) >> 2) & 1, failed)) break;
#pragma unroll
            for (int n = 0; n < NG; ++n)
                if (8 * n + g < nw) {
                    const uint4 w = lds128(tile + 4 * (16 * nw + 16 * (8 * n + g) + 4 * t));
                    uint32_t d[8];
                    const uint32_t to = v_buf + (nb * NG + n) * S::BLOCK + g * 128 + 4 * t;
                    codes_minus_8(__byte_perm(w.x, w.y, 0x5410), d);
                    codes_minus_8(__byte_perm(w.x, w.y, 0x7632), d + 4);
#pragma unroll
                    for (int e = 0; e < 8; ++e) sts32(to + e * 1024 + (((2 * u) ^ g) << 4), d[e]);
                    codes_minus_8(__byte_perm(w.z, w.w, 0x5410), d);
                    codes_minus_8(__byte_perm(w.z, w.w, 0x7632), d + 4);
#pragma unroll
                    for (int e = 0; e < 8; ++e) sts32(to + e * 1024 + (((2 * u + 1) ^ g) << 4), d[e]);
                }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&s_raw_empty[slot]);
                mbar_arrive(&s_v[i & 3]);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
        if (wid < active) {
        // ---------------------------------------------------------------- softmax
        const uint32_t mine_at = tmem + ((uint32_t)wid << 21);  // 32 lanes per warp
        float ref = -INFINITY;  // log2 reference: p = 2^(score f - ref)
        float2 l2 = make_float2(0.f, 0.f), ob2[NG];
#pragma unroll
        for (int n = 0; n < NG; ++n) ob2[n] = make_float2(0.f, 0.f);
        const float2 f2 = make_float2(f, f);
        bool good = true;
        auto step = [&](auto plain, int i, uint32_t ok) {
            constexpr bool PLAIN = decltype(plain)::value;
            const int sb = i % NS;  // buffer of S
            const float(&meta)[NG][4][WIDE_STEP] = s_meta[i & 1];
            float s[WIDE_STEP];
            float2* s2 = reinterpret_cast<float2*>(s);
            tmem_ld32(mine_at + sb * NG * 64, s);
            tmem_ld32(mine_at + sb * NG * 64 + 32, s + 32);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < WIDE_STEP / 2; j += 2) {
                const float4 ks = four(meta[0][0] + 2 * j), kb = four(meta[0][1] + 2 * j);
                const float2 q2 = make_float2(qs[0], qs[0]);
                s2[j] = fma2(make_float2(kb.x, kb.y), q2, mul2(s2[j], make_float2(ks.x, ks.y)));
                s2[j + 1] = fma2(make_float2(kb.z, kb.w), q2, mul2(s2[j + 1], make_float2(ks.z, ks.w)));
            }
            if constexpr (NG == 2) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float x[16];
                    tmem_ld16(mine_at + 64 + 16 * c, x);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const float4 ks = four(meta[NG - 1][0] + 16 * c + 2 * j);
                        const float4 kb = four(meta[NG - 1][1] + 16 * c + 2 * j);
                        const float2 q2 = make_float2(qs[NG - 1], qs[NG - 1]);
                        float2* d = s2 + 8 * c + j;
                        d[0] = fma2(make_float2(kb.x, kb.y), q2,
                                    fma2(make_float2(x[2 * j], x[2 * j + 1]), make_float2(ks.x, ks.y), d[0]));
                        d[1] = fma2(make_float2(kb.z, kb.w), q2,
                                    fma2(make_float2(x[2 * j + 2], x[2 * j + 3]), make_float2(ks.z, ks.w), d[1]));
                    }
                }
            }
            if constexpr (!PLAIN) {
                const int pos = first - first % KV4_TILE + i * WIDE_STEP;
#pragma unroll
                for (int j = 0; j < WIDE_STEP; ++j)
                    if (!((ok >> (j / KV4_TILE)) & 1) || pos + j >= lim) s[j] = -INFINITY;
            }
            float tops[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) tops[j] = s[j];
#pragma unroll
            for (int j = 8; j < WIDE_STEP; ++j) tops[j & 7] = fmaxf(tops[j & 7], s[j]);
            const float top = fmaxf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])),
                                    fmaxf(fmaxf(tops[4], tops[5]), fmaxf(tops[6], tops[7])));
            // the reference moves when p s could pass 2^15; it is set so that they are below 2^7
            const float4 vm = *reinterpret_cast<const float4*>(s_vmax[i & 1]);
            const float most = top * f + __log2f(fmaxf(fmaxf(fmaxf(vm.x, vm.y), fmaxf(vm.z, vm.w)), 5.9604645e-8f));
            const bool move = most > ref + 15.f;  // also from -inf; never for -inf or NaN scores
            if (__any_sync(FULL, move)) {
                const float to = move ? most - 7.f : ref;
                const float corr = !move || ref == -INFINITY ? (move ? 0.f : 1.f) : ex2(ref - to);
                ref = to;
                l2 = mul2(l2, make_float2(corr, corr));
#pragma unroll
                for (int n = 0; n < NG; ++n) ob2[n] = mul2(ob2[n], make_float2(corr, corr));
                if (i > 0) {
                    good = good && wait_on(&s_pv[(i - 1) & 3], ((i - 1) >> 2) & 1, failed);
                    fence_after();
#pragma unroll 1
                    for (int c = 0; c < 4 * NG; ++c) {
                        float x[16];
                        tmem_ld16(mine_at + O_COL + 16 * c, x);
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 16; ++j) x[j] *= corr;
                        tmem_st16(mine_at + O_COL + 16 * c, reinterpret_cast<const uint32_t*>(x));
                    }
                }
            }
            const float neg = ref == -INFINITY ? 0.f : -ref;
            const float2 neg2 = make_float2(neg, neg);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int j = 16 * c; j < 16 * c + 16; ++j) {
                    const float2 x = fma2(s2[j], f2, neg2);
                    s2[j] = make_float2(ex2(x.x), ex2(x.y));
                    l2 = add2(l2, s2[j]);
                }
#pragma unroll
                for (int n = 0; n < NG; ++n) {
                    uint32_t hi[16];
                    [[maybe_unused]] uint32_t lo[16];
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        const float4 vs = four(meta[n][2] + 32 * c + 2 * k), vb = four(meta[n][3] + 32 * c + 2 * k);
#pragma unroll
                        for (int o = 0; o < 2; ++o) {
                            const float2 p = s2[16 * c + k + o];
                            const float2 bv = o ? make_float2(vb.z, vb.w) : make_float2(vb.x, vb.y);
                            float2 w = mul2(p, o ? make_float2(vs.z, vs.w) : make_float2(vs.x, vs.y));
                            if constexpr (PLAIN) {
                                ob2[n] = fma2(p, bv, ob2[n]);
                            } else {
                                // what a query does not see adds nothing, whatever its page holds
                                if (p.x == 0.f) w.x = 0.f;
                                else ob2[n].x = fmaf(p.x, bv.x, ob2[n].x);
                                if (p.y == 0.f) w.y = 0.f;
                                else ob2[n].y = fmaf(p.y, bv.y, ob2[n].y);
                            }
                            hi[k + o] = pack_half2(w.x, w.y);
                            if constexpr (PP == 2) {
                                const float2 back = half2_of(hi[k + o]);
                                lo[k + o] = pack_half2(w.x - back.x, w.y - back.y);
                            }
                        }
                    }
                    tmem_st16(mine_at + (sb * NG + n) * 64 + 16 * c, hi);
                    if constexpr (PP == 2) tmem_st16(mine_at + (sb * NG + n) * 64 + 32 + 16 * c, lo);
                }
            }
            tmem_st_wait();
        };
        const int whole = (min(all_see, last) - (first - first % KV4_TILE)) / WIDE_STEP;  // stages that all rows see
        for (int i = 0; i < steps && good; ++i) {
            good = wait_on(&s_k[i & 1], (i >> 1) & 1, failed) && wait_on(&s_s[i & 1], (i >> 1) & 1, failed);
            if (!good) break;
            fence_after();
            const uint32_t ok = s_ok[i & 1];
            if (i < whole && ok == (1u << WIDE_TILES) - 1) step(std::true_type{}, i, ok);
            else step(std::false_type{}, i, ok);
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_p[i & 1]);
        }
        if (steps > 0 && good) good = wait_on(&s_pv[(steps - 1) & 3], ((steps - 1) >> 2) & 1, failed);
        fence_after();
        good = __all_sync(FULL, good);
        const float l = good ? l2.x + l2.y : NAN;
        const float inv = l == 0.f ? 0.f : 1.f / l;  // nothing seen: zeros
        const bool done = n_split == 1;
        const long long each = a.q_tokens * a.heads, at = blockIdx.x * each + tok * a.heads + h;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            float x[64];
            if (steps > 0) {
                tmem_ld32(mine_at + O_COL + 64 * n, x);
                tmem_ld32(mine_at + O_COL + 64 * n + 32, x + 32);
                tmem_ld_wait();
            } else {
#pragma unroll
                for (int e = 0; e < 64; ++e) x[e] = 0.f;
            }
            if (!mine) continue;
            const float bias = ob2[n].x + ob2[n].y;
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                if (8 * n + g >= nw) continue;
                if (done) {
                    T* out = reinterpret_cast<T*>(a.out) + tok * a.out_token_stride + h * a.out_head_stride + 64 * n + 8 * g;
                    __align__(16) T v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = from_f32<T>(l != l ? NAN : l == 0.f ? 0.f : (x[8 * e + g] + bias) * inv);
                    if (!(reinterpret_cast<uintptr_t>(out) & 15)) {
                        *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(v);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) out[e] = v[e];
                    }
                } else {
                    float4* out = reinterpret_cast<float4*>(sp.part + at * hd + 64 * n + 8 * g);
                    out[0] = make_float4(x[g] + bias, x[8 + g] + bias, x[16 + g] + bias, x[24 + g] + bias);
                    out[1] = make_float4(x[32 + g] + bias, x[40 + g] + bias, x[48 + g] + bias, x[56 + g] + bias);
                }
            }
        }
        if (mine && !done) reinterpret_cast<float2*>(sp.part + sp.splits * each * hd)[at] = make_float2(ref, l);
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (wid == 9 && *failed)  // a role gave up: its copies in flight end before the CTA does
        for (int i = max(0, loaded - WIDE_RAW); i < loaded; ++i) mbar_wait(&s_raw_full[i % WIDE_RAW], (i / WIDE_RAW) & 1);
    if (wid == 8)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(WIDE_COLS) : "memory");
}

template <class T, int NG>
cudaError_t launch_wide(const Kv4Pool& pool, const Kv4Attention& a, const AttSplit& sp, cudaStream_t s) {
    const size_t smem = WideSmem<NG>::bytes(pool.head_dim);
    const auto fn = kv4_attention_wide_kernel<T, NG>;
    cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return e;
    ++launch_counter();
    e = launch_kernel(fn, dim3(sp.splits, sp.per_row, a.rows), dim3(WIDE_THREADS), smem, s, pool, a, sp);
    return e != cudaSuccess || sp.splits == 1 ? e : launch_join<T>(pool, a, sp, s);
}

}  // namespace

cudaError_t launch_kv4_attention_wide(const Kv4Pool& pool, const Kv4Attention& a, const AttSplit& sp, cudaStream_t s) {
    const bool one = kv4_groups(pool.head_dim) == 1;
    if (a.dtype == KV4_F16) return one ? launch_wide<__half, 1>(pool, a, sp, s) : launch_wide<__half, 2>(pool, a, sp, s);
    if (a.dtype == KV4_BF16)
        return one ? launch_wide<__nv_bfloat16, 1>(pool, a, sp, s) : launch_wide<__nv_bfloat16, 2>(pool, a, sp, s);
    return cudaErrorInvalidValue;
}

}  // namespace msb
