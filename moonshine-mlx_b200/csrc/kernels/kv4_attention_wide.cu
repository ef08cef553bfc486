// 4-bit K/V attention for many query rows per K/V head (prompt chunks, drafted tokens of grouped
// heads): the products of kv4_attention.cuh on the fifth-generation tensor cores.
//
// bf16 results (ROUND): K and V enter the products as fp16(s c + b), three bits more than the
// results keep, one rounding each.  Then S = Q K^T and O += P V are plain products and the softmax
// thread has 4 operations per position, where the exact form has 9.
// fp16 results: the products take the codes d = c - 8 themselves, S_n = Q_n D_n^T for each group n
// of 64 dims, scores sum_n s_tn S_n + (b_tn + 8 s_tn) sum(q_n), and P_n = p_t s_tn (two fp16
// planes); sum p_t (b_tn + 8 s_tn) stays in the thread.
//
// One CTA has 128 (token, head) rows of one K/V head and walks its positions 64 at a time, each
// role on its own (the comment at the barriers says why an entry is never reused too early):
//   loads     one warp, tiles of a stage by bulk copies into a ring
//   unpacking 4 or 8 warps: a tile each into K rows of positions and V rows of dims (a byte permute
//             puts two positions side by side, and row 8 (dim % 8) + dim / 8 makes the stores free
//             of bank conflicts), both 128-byte swizzled
//   S, O      one warp each issues its tcgen05 products; with one warp for both, 8 waits and
//             products per stage took 2000 cycles of its own, the whole stage
//   softmax   4 warps, a thread per row: S out of tensor memory, running reference and sum, P back
//             over S as the next product's operand
// The reference of a row moves only when a probability (times a scale) could pass fp16's range, 8
// bits above where it was set, so O is rescaled (tensor memory read and written by the row's
// thread) a few times per CTA.
//
// Two CTAs share an SM.  Bound: latency inside the roles; of a stage's 1300 cycles (64 dims, bf16)
// the 64 exponentials of a warp are 512, and the tensor pipe is active 16 % of the time.  Measured,
// 592 CTAs of 2048 positions: bf16 116 us (64 dims), 166 us (128); fp16 170 and 292 us.  8 prompts of
// up to 512 tokens over up to 4096 positions, 16 heads on 4: 86 us, of which the longest rows' CTAs,
// which meet on some SMs, take all: cut into pieces of 2048 the parts cost more (7 to 15 us).
#define KV4_ATTENTION_KERNELS
#include "kv4_attention.cuh"

namespace msb {
namespace {

constexpr int WIDE_ROWS = 128;
constexpr int WIDE_STEP = 64;  // positions per stage
constexpr int WIDE_TILES = WIDE_STEP / KV4_TILE;
constexpr uint32_t WIDE_COLS = 256;  // tensor memory columns: O of 64 (or 128) dims behind S in 64s

// ROUND: K and V enter the products as fp16(s c + b), else as codes
template <int NG, bool ROUND>
struct WideSmem {
    static constexpr int GROUPS = ROUND ? 2 : 1;                // warpgroups that unpack
    static constexpr int UNPACK = GROUPS == 1 || NG == 1 ? 4 : 8;  // warps per stage
    static constexpr int LAST = 4 + 4 * GROUPS;                 // first warp of the last warpgroup
    static constexpr int THREADS = 32 * (LAST + 4);
    static constexpr int NK = NG == 1 ? 3 : 1;                  // buffers of unpacked K
    static constexpr int NV = NG == 1 ? 3 : ROUND ? 2 : 1;      // of V
    static constexpr int SG = ROUND ? 1 : NG;                   // sums per score
    static constexpr int NS = NG == 1 ? 3 : SG == 1 ? 2 : 1;    // buffers of S, in tensor memory
    static constexpr int RAW = NG == 1 ? 4 : 3;                 // stages of packed tiles
    static_assert(64 * (NS * SG + NG) <= 256, "columns");
    static constexpr int BLOCK = WIDE_STEP * 128;               // 64 rows of 128 bytes
    static constexpr int Q = NG * WIDE_ROWS * 128, K = NK * NG * BLOCK, V = NV * NG * BLOCK;
    static int raw(int hd) { return (WIDE_TILES * kv4_tile_words(hd) * 4 + 127) / 128 * 128; }
    static size_t bytes(int hd) { return (size_t)Q + K + V + RAW * raw(hd) + 512 + 1024; }  // + alignment
};

__device__ __forceinline__ uint64_t sw128_desc(uint32_t addr) {  // K-major rows of 128 bytes, 8-row groups
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// fp16 A and B, both K-major, fp32 sums, 128 x n
__device__ __forceinline__ constexpr uint32_t f16_idesc(int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// By the lane with `leader` set; the others come along, so that the descriptors stay uniform.
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void commit_to(uint32_t leader, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"(leader)
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
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ void sts32(uint32_t a, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ void sts128(uint32_t a, const uint32_t* v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
// an (s, b) word with an infinity or a NaN
__device__ __forceinline__ bool not_finite(uint32_t w) {
    return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
}
__device__ __forceinline__ uint32_t twice_low(uint32_t w) { return __byte_perm(w, w, 0x1010); }
__device__ __forceinline__ uint32_t twice_high(uint32_t w) { return __byte_perm(w, w, 0x3232); }
// fp16(s c + b) of codes 0 .. 3 of both halves of x, each half with its s and b; `huge`: held
// to fp16's largest values
__device__ __forceinline__ void values_of(uint32_t x, uint32_t s, uint32_t b, bool huge, uint32_t* d) {
    const uint32_t y = x >> 8;
    d[0] = hfma2_of(hfma2_of(on_1024(x, 0x000f000fu), 0x3c003c00u, 0xe400e400u), s, b);  // 1, -1024
    d[1] = hfma2_of(hfma2_of(on_1024(x, 0x00f000f0u), 0x2c002c00u, 0xd400d400u), s, b);  // 1/16, -64
    d[2] = hfma2_of(hfma2_of(on_1024(y, 0x000f000fu), 0x3c003c00u, 0xe400e400u), s, b);
    d[3] = hfma2_of(hfma2_of(on_1024(y, 0x00f000f0u), 0x2c002c00u, 0xd400d400u), s, b);
    if (huge)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            asm("min.NaN.f16x2 %0, %0, %1;" : "+r"(d[e]) : "r"(0x7bff7bffu));
            asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(d[e]) : "r"(0xfbfffbffu));
        }
}

__device__ __forceinline__ float4 four(const float* p) { return *reinterpret_cast<const float4*>(p); }

// Bounded wait of a warp that also ends when another role has given up.  Its lanes agree on how
// it ended: what follows (votes, shuffles, tensor memory) wants all of them or none.
__device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity, volatile int* failed) {
    const uint32_t a = smem_u32(bar);
    uint32_t ok = 0;
    for (uint32_t i = 0; i < WAIT_LIMIT; ++i) {
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(a), "r"(parity)
            : "memory");
        if (ok || ((i & 255) == 255 && *failed)) break;
    }
    if (__all_sync(FULL, ok)) return true;
    *failed = 1;
    return false;
}

// n / d for n below 2^24, `inv` = 1 / d: the product is off by less than one
__device__ __forceinline__ int over_near(int n, int d, float inv) {
    const int q = (int)(n * inv), left = n - q * d;
    return left < 0 ? q - 1 : left >= d ? q + 1 : q;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}

template <class T, int NG>
__global__ void __launch_bounds__(WideSmem<NG, is_bf16<T>>::THREADS, 2) kv4_attention_wide_kernel(const Kv4Pool pool, const Kv4Attention a,
                                                                             const AttSplit sp) {
    constexpr bool ROUND = is_bf16<T>;
    using S = WideSmem<NG, ROUND>;
    constexpr int NK = S::NK, NV = S::NV, SG = S::SG, NS = S::NS, RAW = S::RAW, PP = ROUND ? 1 : 2;
    constexpr uint32_t O_COL = 64 * NS * SG;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t s_raw_full[RAW], s_raw_empty[RAW], s_raw_q, s_q;
    // Stage i has entry i % 4: K and V unpacked, S summed (and K unpacked, with what the softmax
    // reads of it), P written, O summed; what the softmax reads, i % 8.  K of stage i + 4 is
    // unpacked after the softmax of stage i or a later one, V after the second product of stage
    // i + 1, so an entry's next phase waits, through the other roles, for whoever still has to
    // see this one.
    __shared__ __align__(8) uint64_t s_k[4], s_v[4], s_s[4], s_p[4], s_pv[4];
    __shared__ uint32_t s_okr[RAW], s_ok[8], s_tmem;
    __shared__ int s_failed;
    using Meta = float[NG][ROUND ? 1 : 4][WIDE_STEP];  // K's s and b + 8 s, V's
    __shared__ __align__(16) Meta s_meta[ROUND ? 1 : 2];
    __shared__ __align__(16) float s_vmax[2][2 * WIDE_TILES];
    __shared__ __align__(16) uint32_t s_odd[8][2 * WIDE_TILES];  // positions whose V is not finite, 8 bits per group
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const int hd = pool.head_dim, nw = kv4_words(hd), P = pool.page_size, per = over(a.heads, pool.kv_heads);
    // the last queries first: under a causal mask they see the most
    const int b = blockIdx.y, part_nr = blockIdx.z, y = gridDim.x - 1 - blockIdx.x;
    const int above = gridDim.x == pool.kv_heads ? 0 : y / pool.kv_heads;
    const int kvh = y - above * pool.kv_heads, row0 = above * WIDE_ROWS;
    pdl_wait();
    const int chunk = chunk_of(pool, a, sp);
    const Row row(pool, a, b);
    const int rows = min(WIDE_ROWS, min(row.n, a.max_q) * per - row0);  // this CTA's (token, head) rows
    if (rows <= 0) return;
    const int end = row.end(a, over(row0 + rows - 1, per)), all_see = row.end(a, over(row0, per));
    const int n_split = splits_of(end, chunk);
    if (part_nr >= n_split) return;
    const int piece = n_split == 1 ? end : ((end + n_split - 1) / n_split + WIDE_STEP - 1) / WIDE_STEP * WIDE_STEP;
    const int first = min(end, part_nr * piece), last = min(end, first + piece);
    const int tile0 = first / KV4_TILE, tiles = (last - first + KV4_TILE - 1) / KV4_TILE;
    const int steps = (tiles + WIDE_TILES - 1) / WIDE_TILES;
    const int active = (rows + 31) / 32;  // softmax warps with rows

    const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
    const uint32_t q_at = base, k_buf = q_at + S::Q, v_buf = k_buf + S::K, raw_at = v_buf + S::V;
    const int tile_words = kv4_tile_words(hd), tpp = P / KV4_TILE;
    const uint32_t tile_bytes = (uint32_t)tile_words * 4, raw_bytes = (WIDE_TILES * tile_bytes + 127) / 128 * 128;
    int loaded = 0, issued = 0;  // stages that the load warp asked for, and a product warp
    auto load = [&](int i) {  // lane v stands for tile v of stage i
        const int* table = a.table + (long long)b * a.table_stride;
        const char* head = reinterpret_cast<const char*>(pool.base) + kvh * pool.head_stride;
        const int slot = i % RAW, n = min(WIDE_TILES, tiles - i * WIDE_TILES), at = tile0 + i * WIDE_TILES + lane;
        const int nth = sp.page_shift >= 0 ? at >> sp.page_shift : at / tpp, in_page = at - nth * tpp;
        // a page's first tile here copies those that lie behind it
        const int page = lane < n && (lane == 0 || in_page == 0) ? table[nth] : -1;
        const bool here = page >= 0 && page < pool.pages;
        const int len = here ? min(n - lane, tpp - in_page) : 0;
        const uint32_t ok = __reduce_or_sync(FULL, here ? ((1u << len) - 1) << lane : 0u);
        if (i >= RAW && !wait_on(&s_raw_empty[slot], (i / RAW - 1) & 1, &s_failed)) return false;
        __syncwarp();
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
        return true;
    };
    if (wid == S::LAST + 1) {
        if (lane == 0) {
            for (int i = 0; i < RAW; ++i) {
                mbar_init(&s_raw_full[i], 1);
                mbar_init(&s_raw_empty[i], S::UNPACK);
            }
            for (int i = 0; i < 4; ++i) {
                mbar_init(&s_k[i], S::UNPACK);
                mbar_init(&s_s[i], 1 + S::UNPACK);
                mbar_init(&s_p[i], active);
                mbar_init(&s_v[i], S::UNPACK);
                mbar_init(&s_pv[i], 1);
            }
            mbar_init(&s_raw_q, S::LAST);
            mbar_init(&s_q, 4);
            s_failed = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        while (loaded < min(steps, RAW)) load(loaded);
    }
    if (wid == S::LAST) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                     "r"(WIDE_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // q rows as they are, 8 or 16 threads each; nobody waits for them here
    const float each_per = 1.f / per;
    if (wid < S::LAST) {
        constexpr int LANES = 8 * NG;
        const bool wide = !((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)(a.q_token_stride * 2) |
                             (uintptr_t)(a.q_head_stride * 2)) & 15);
#pragma unroll 3
        for (int i = threadIdx.x; i < WIDE_ROWS * LANES; i += 32 * S::LAST) {
            const int r = i / LANES, w = i % LANES;
            const uint32_t to = q_at + w / 8 * (WIDE_ROWS * 128) + r * 128 + (((w & 7) ^ (r & 7)) << 4);
            const int qi = over_near(row0 + min(r, rows - 1), per, each_per), h = kvh * per + (row0 + r - qi * per);
            const T* qp = reinterpret_cast<const T*>(a.q) + (row.q0 + (long long)qi) * a.q_token_stride +
                          h * a.q_head_stride + 8 * w;
            if (r >= rows || w >= nw) {
                const uint32_t zero[4] = {0, 0, 0, 0};
                sts128(to, zero);
            } else if (wide) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to), "l"(qp) : "memory");
            } else {
#pragma unroll 1
                for (int e = 0; e < 4; ++e) {
                    const uint16_t* u = reinterpret_cast<const uint16_t*>(qp + 2 * e);
                    sts32(to + 4 * e, (uint32_t)u[0] | (uint32_t)u[1] << 16);
                }
            }
        }
    }
    // K rows end with zeros where the head is shorter than its groups (q is zero there too)
    if (nw < 8 * NG)
        for (uint32_t i = threadIdx.x; i < (uint32_t)S::K / 16; i += S::THREADS) {
            const uint32_t zero[4] = {0, 0, 0, 0};
            sts128(k_buf + 16 * i, zero);
        }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    fence_before();
    __syncthreads();
    fence_after();
    pdl_trigger();
    const uint32_t tmem = s_tmem;
    volatile int* failed = &s_failed;

    if (wid < S::LAST) {
        asm volatile("cp.async.wait_all;\n" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_raw_q);
    }

    // Registers out of those of the launch: 4 x 64 in 112 for the softmax, 56 to unpack (twice) and
    // 32 for the rest, or 3 x 80 in 136, 64 and 40.
    if (wid >= S::LAST) {
        if constexpr (ROUND) asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        // ---------------------------------------------------------------- products
        const uint32_t leader = lane == 0, tmem = __shfl_sync(FULL, s_tmem, 0);
        if (wid == S::LAST) {
            // S, up to NS stages ahead of the softmax; descriptors count in 16 bytes
            const bool there = wait_on(&s_q, 0, failed);
            const uint64_t q_desc = sw128_desc(q_at), k_desc = sw128_desc(k_buf);
#pragma unroll 1
            for (int i = 0; there && i < steps; issued = ++i) {
                if (!wait_on(&s_k[i & 3], (i >> 2) & 1, failed)) break;
                // P of stage i - NS lies where S goes
                if (i >= NS && !wait_on(&s_pv[(i - NS) & 3], ((i - NS) >> 2) & 1, failed)) break;
                fence_after();
#pragma unroll
                for (int n = 0; n < NG; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_ss(leader, tmem + (i % NS * SG + n % SG) * 64, q_desc + n * (WIDE_ROWS * 8) + 2 * k,
                               k_desc + (i % NK * NG + n) * (S::BLOCK / 16) + 2 * k, f16_idesc(64), n >= SG || k > 0);
                commit_to(leader, &s_s[i & 3]);
            }
        } else if (wid == S::LAST + 2) {
            // O; one P for all groups: one product over the dims of both
            const uint64_t v_desc = sw128_desc(v_buf);
#pragma unroll 1
            for (int i = 0; i < steps; issued = ++i) {
                if (!wait_on(&s_v[i & 3], (i >> 2) & 1, failed) || !wait_on(&s_p[i & 3], (i >> 2) & 1, failed)) break;
                fence_after();
#pragma unroll
                for (int n = 0; n < SG; ++n)
#pragma unroll
                    for (int pl = 0; pl < PP; ++pl)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_ts(leader, tmem + O_COL + n * 64, tmem + (i % NS * SG + n) * 64 + 32 * pl + 8 * k,
                                   v_desc + (i % NV * NG + n) * (S::BLOCK / 16) + 2 * k, f16_idesc(64 * NG / SG),
                                   i > 0 || pl > 0 || k > 0);
                commit_to(leader, &s_pv[i & 3]);
            }
        } else if (wid == S::LAST + 1) {
            // ------------------------------------------------------------ loads
            while (loaded < steps && load(loaded)) {
            }
        }
        __syncwarp();
    } else if (wid >= 4) {
        if constexpr (ROUND) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        // ---------------------------------------------------------------- unpacking
        // This warp's tile of a stage; a half of it (positions g for K and 2 t, 2 t + 1 for V, or 8
        // further), or both; every stage, or every other one.
        constexpr int HALVES = S::UNPACK == 8 ? 1 : 2, EVERY = HALVES == 1 ? 1 : S::GROUPS;
        const int u = wid & 3, group = (wid >> 2) - 1, half0 = HALVES == 1 ? group : 0, g = lane >> 2, t = lane & 3;
        uint32_t k_from[2 * NG];
#pragma unroll
        for (int j = 0; j < 2 * NG; ++j) k_from[j] = 4 * (64 * j + 2 * (min(4, max(0, nw - 4 * j)) * g + t) + half0);
#pragma unroll 1
        for (int i = EVERY == 1 ? 0 : group; i < steps; i += EVERY) {
            const int slot = i % RAW, i4 = i & 3, i8 = i & 7;
            if (!wait_on(&s_raw_full[slot], (i / RAW) & 1, failed)) break;
            // K's buffer is free when the scores of stage i - NK are summed, V's when its second
            // product is; the scales' when the softmax of stage i - 2 has read them.  A group that
            // unpacks every other stage has not seen stage i - 4 through: its entries are free
            // when that softmax is done.
            if (i >= NK && !wait_on(&s_s[(i - NK) & 3], ((i - NK) >> 2) & 1, failed)) break;
            if (!ROUND && i >= 2 && !wait_on(&s_p[(i - 2) & 3], ((i - 2) >> 2) & 1, failed)) break;
            if (EVERY > 1 && i >= 4 && !wait_on(&s_p[i4], ((i - 4) >> 2) & 1, failed)) break;
            const uint32_t k_to = k_buf + i % NK * NG * S::BLOCK, v_to = v_buf + i % NV * NG * S::BLOCK;
            const uint32_t okr = s_okr[slot];
            const bool here = (okr >> u) & 1;
            const uint32_t tile = raw_at + slot * raw_bytes + u * tile_bytes, meta_at = tile + 4 * (32 * nw + half0);
            const int pos = first - first % KV4_TILE + (i * WIDE_TILES + u) * KV4_TILE + 8 * half0;  // of g = 0
            uint32_t kw[HALVES][2 * NG], ks[HALVES][NG], vs[HALVES][NG];  // (s, b) of position g
#pragma unroll
            for (int x = 0; x < HALVES; ++x) {
#pragma unroll
                for (int j = 0; j < 2 * NG; ++j)  // lanes past the vector's last word read what lies behind
                    kw[x][j] = lds32(tile + k_from[j] + 4 * x);
#pragma unroll
                for (int n = 0; n < NG; ++n) {
                    ks[x][n] = lds32(meta_at + 4 * (32 * n + 4 * g + x));
                    vs[x][n] = lds32(meta_at + 4 * (32 * n + 4 * g + 2 + x));
                    if (!here || pos + 8 * x + g >= last) ks[x][n] = vs[x][n] = 0;  // nobody sees it
                }
            }
            [[maybe_unused]] bool huge = false;
            if constexpr (ROUND) {
                uint32_t most = 0;
#pragma unroll
                for (int x = 0; x < HALVES; ++x) {
                    uint32_t odd = 0;
#pragma unroll
                    for (int n = 0; n < NG; ++n) {
                        odd |= not_finite(vs[x][n]) ? 1u << (8 * n + g) : 0u;
                        // what code 15 stands for, in the low half: the group's largest, monotone in c
                        most = max(most, max(hfma2_of(ks[x][n], 0x4b80u, ks[x][n] >> 16) & 0x7fffu,
                                             hfma2_of(vs[x][n], 0x4b80u, vs[x][n] >> 16) & 0x7fffu));
                    }
                    odd = __reduce_or_sync(FULL, odd);
                    if (lane == 0) s_odd[i8][4 * (half0 + x) + u] = odd;
                }
                huge = __any_sync(FULL, most >= 0x7c00u);  // a value of the tile that fp16 does not hold
            } else {
#pragma unroll
                for (int x = 0; x < HALVES; ++x) {
                    float vmax = 0.f;
#pragma unroll
                    for (int n = 0; n < NG; ++n) {
                        // lane t: K's s and b + 8 s, V's
                        const float2 sb = half2_of(t < 2 ? ks[x][n] : vs[x][n]);
                        s_meta[i & 1][n][t][16 * u + 8 * (half0 + x) + g] = t & 1 ? fmaf(8.f, sb.x, sb.y) : sb.x;
                        if (t >= 2) vmax = fmaxf(vmax, sb.x);
                    }
                    vmax = fminf(warp_max(vmax), 65504.f);
                    if (lane == 0) s_vmax[i & 1][4 * (half0 + x) + u] = vmax;
                }
            }
            if (lane == 0 && u == 0 && half0 == 0) s_ok[i8] = okr;
#pragma unroll
            for (int x = 0; x < HALVES; ++x)
#pragma unroll
                for (int j = 0; j < 2 * NG; ++j) {
                    if (4 * j + t >= nw) continue;
                    uint32_t d[4];
                    if constexpr (ROUND) values_of(kw[x][j], twice_low(ks[x][j / 2]), twice_high(ks[x][j / 2]), huge, d);
                    else codes_minus_8(kw[x][j], d);
                    sts128(k_to + j / 2 * S::BLOCK + (16 * u + 8 * (half0 + x) + g) * 128 + ((((j & 1) * 4 + t) ^ g) << 4), d);
                }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&s_k[i4]);
                mbar_arrive(&s_s[i4]);
            }
            if (i >= NV && !wait_on(&s_pv[(i - NV) & 3], ((i - NV) >> 2) & 1, failed)) break;
#pragma unroll
            for (int n = 0; n < NG; ++n)
#pragma unroll
                for (int x = 0; x < HALVES; ++x) {
                    // V of positions 2 t and 2 t + 1: their (s, b) are lane 8 t's and lane 8 t + 4's
                    [[maybe_unused]] uint32_t s2, b2;
                    if constexpr (ROUND) {
                        uint32_t even = __shfl_sync(FULL, vs[x][n], 8 * t), odd = __shfl_sync(FULL, vs[x][n], 8 * t + 4);
                        if (not_finite(even)) even = 0;
                        if (not_finite(odd)) odd = 0;
                        s2 = __byte_perm(even, odd, 0x5410);
                        b2 = __byte_perm(even, odd, 0x7632);
                    }
                    if (8 * n + g >= nw) continue;
                    const uint2 w = lds64(tile + 4 * (16 * nw + 16 * (8 * n + g) + 4 * t + 2 * (half0 + x)));
                    const uint32_t lo = __byte_perm(w.x, w.y, 0x5410), hi = __byte_perm(w.x, w.y, 0x7632);
                    uint32_t d[8];
                    if constexpr (ROUND) {
                        values_of(lo, s2, b2, huge, d);
                        values_of(hi, s2, b2, huge, d + 4);
                    } else {
                        codes_minus_8(lo, d);
                        codes_minus_8(hi, d + 4);
                    }
                    const uint32_t to = v_to + n * S::BLOCK + g * 128 + 4 * t + (((2 * u + half0 + x) ^ g) << 4);
#pragma unroll
                    for (int e = 0; e < 8; ++e) sts32(to + e * 1024, d[e]);
                }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&s_raw_empty[slot]);
                mbar_arrive(&s_v[i4]);
            }
        }
    } else {
        if constexpr (ROUND) asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
        // ---------------------------------------------------------------- softmax
        const int r = threadIdx.x;
        bool good = wait_on(&s_raw_q, 0, failed);
        // This thread's row of q scaled by a power of two, in the order that unpacked words have
        // (dims 0 4 1 5 2 6 3 7).
        float f = 1.f;
        [[maybe_unused]] float qs[NG];
        {
            using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
            const uint32_t at = q_at + r * 128;
            uint4 most = make_uint4(0, 0, 0, 0);
            T2* top = reinterpret_cast<T2*>(&most);
#pragma unroll 4
            for (int w = 0; w < 8 * NG; ++w) {
                const uint4 raw = lds128(at + w / 8 * (WIDE_ROWS * 128) + (((w & 7) ^ (r & 7)) << 4));
#pragma unroll
                for (int e = 0; e < 4; ++e) top[e] = __hmax2_nan(top[e], __habs2(reinterpret_cast<const T2*>(&raw)[e]));
            }
            top[0] = __hmax2_nan(__hmax2_nan(top[0], top[1]), __hmax2_nan(top[2], top[3]));
            const float mx = max_nan(to_f32<T>(top[0].x), to_f32<T>(top[0].y));
            const bool odd = !(mx < INFINITY);
            // its exponent; rows below 2^-100 keep less
            const int e2 = mx > 0.f && !odd ? max(-100, (__float_as_int(mx) >> 23) - 127) : 0;
            const float up = odd ? 0.f : a.scale < 0.f ? -pow2(14 - e2) : pow2(14 - e2);
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                qs[n] = 0.f;
#pragma unroll 4
                for (int c = 0; c < 8; ++c) {
                    const uint32_t to = at + n * (WIDE_ROWS * 128) + ((c ^ (r & 7)) << 4);
                    const uint4 raw = lds128(to);
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[e] = to_f32<T>(reinterpret_cast<const T*>(&raw)[e]);
                        x[e] = odd ? 0.f : x[e] * up;
                        if constexpr (!ROUND) qs[n] += x[e];
                    }
                    uint32_t v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = pack_half2(x[e], x[e + 4]);
                    sts128(to, v);
                }
            }
            f = odd ? NAN : fmaxf(fabsf(a.scale) * LOG2E * pow2(e2 - 14), 1e-37f);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_q);
        if (wid < active) {
        const uint32_t mine_at = tmem + ((uint32_t)wid << 21);  // 32 lanes per warp
        const bool mine = r < rows;
        const int qi = mine ? over_near(row0 + r, per, each_per) : 0, h = mine ? kvh * per + (row0 + r - qi * per) : 0;
        const long long tok = row.q0 + (long long)qi;
        const int lim = mine ? min(last, row.end(a, qi)) : last;
        float ref = -INFINITY, add = 0.f;  // p = 2^((score - ref) f + add)
        float2 l2 = make_float2(0.f, 0.f), ob2[NG];
#pragma unroll
        for (int n = 0; n < NG; ++n) ob2[n] = make_float2(0.f, 0.f);
        const float2 f2 = make_float2(f, f);
        auto step = [&](auto plain, int i, uint32_t ok) {
            constexpr bool PLAIN = decltype(plain)::value;
            const int sb = i % NS;  // buffer of S
            [[maybe_unused]] const Meta& meta = s_meta[ROUND ? 0 : i & 1];
            float s[WIDE_STEP];
            float2* s2 = reinterpret_cast<float2*>(s);
            tmem_ld32(mine_at + sb * SG * 64, s);
            tmem_ld32(mine_at + sb * SG * 64 + 32, s + 32);
            tmem_ld_wait();
            if constexpr (!ROUND) {
#pragma unroll
                for (int j = 0; j < WIDE_STEP / 2; j += 2) {
                    const float4 ks = four(meta[0][0] + 2 * j), kb = four(meta[0][1] + 2 * j);
                    const float2 q2 = make_float2(qs[0], qs[0]);
                    s2[j] = fma2(make_float2(kb.x, kb.y), q2, mul2(s2[j], make_float2(ks.x, ks.y)));
                    s2[j + 1] = fma2(make_float2(kb.z, kb.w), q2, mul2(s2[j + 1], make_float2(ks.z, ks.w)));
                }
            }
            if constexpr (SG == 2) {
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
                const int pos = tile0 * KV4_TILE + i * WIDE_STEP;
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
            // the reference moves when p (s) could pass 2^15; it is set so that they are below 2^7
            float lift = 0.f;
            if constexpr (!ROUND) {
                const float4 a = four(s_vmax[i & 1]), b = four(s_vmax[i & 1] + 4);
                lift = __log2f(fmaxf(fmaxf(fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w)), fmaxf(fmaxf(b.x, b.y), fmaxf(b.z, b.w))),
                                     5.9604645e-8f));
            }
            const bool move = fmaf(top - ref, f, add) + lift > 15.f;  // also from -inf; never for -inf or NaN scores
            if (__any_sync(FULL, move)) {
                const float to = move ? top : ref, gain = move ? 7.f - lift : add;
                const float corr = !move ? 1.f : ref == -INFINITY ? 0.f : ex2(fmaf(ref - to, f, gain - add));
                add = gain;
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
            const float2 neg2 = make_float2(-ref, -ref), add2f = make_float2(add, add);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int j = 16 * c; j < 16 * c + 16; ++j) {
                    const float2 x = fma2(add2(s2[j], neg2), f2, add2f);
                    float2 p = make_float2(ex2(x.x), ex2(x.y));
                    if constexpr (!PLAIN) {  // even by a query that is NaN
                        if (s2[j].x == -INFINITY) p.x = ROUND ? 0.f : NOT_SEEN;
                        if (s2[j].y == -INFINITY) p.y = ROUND ? 0.f : NOT_SEEN;
                    }
                    s2[j] = p;
                    l2 = add2(l2, s2[j]);
                }
                if constexpr (ROUND) {
                    uint32_t hi[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) hi[k] = pack_half2(s2[16 * c + k].x, s2[16 * c + k].y);
                    tmem_st16(mine_at + sb * 64 + 16 * c, hi);
                } else {
#pragma unroll
                    for (int n = 0; n < NG; ++n) {
                        uint32_t hi[16];
                        uint32_t lo[16];
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
                                    if (not_seen(p.x)) w.x = 0.f;
                                    else ob2[n].x = fmaf(p.x, bv.x, ob2[n].x);
                                    if (not_seen(p.y)) w.y = 0.f;
                                    else ob2[n].y = fmaf(p.y, bv.y, ob2[n].y);
                                }
                                hi[k + o] = pack_half2(w.x, w.y);
                                const float2 back = half2_of(hi[k + o]);
                                lo[k + o] = pack_half2(w.x - back.x, w.y - back.y);
                            }
                        }
                        tmem_st16(mine_at + (sb * NG + n) * 64 + 16 * c, hi);
                        tmem_st16(mine_at + (sb * NG + n) * 64 + 32 + 16 * c, lo);
                    }
                }
            }
            tmem_st_wait();
        };
        const int whole = (min(all_see, last) - tile0 * KV4_TILE) / WIDE_STEP;  // stages that all rows see
        for (int i = 0; i < steps && good; ++i) {
            good = wait_on(&s_s[i & 3], (i >> 2) & 1, failed);
            if (!good) break;
            fence_after();
            const uint32_t ok = s_ok[i & 7];
            if constexpr (ROUND) {
                const uint4 x = *reinterpret_cast<const uint4*>(s_odd[i & 7]), y = *reinterpret_cast<const uint4*>(s_odd[i & 7] + 4);
                if (x.x | x.y | x.z | x.w | y.x | y.y | y.z | y.w) {
                    // where V is not finite zeros go into the product; who sees it has a NaN
#pragma unroll 1
                    for (int u = 0; u < 2 * WIDE_TILES; ++u)
#pragma unroll 1
                        for (uint32_t odd = s_odd[i & 7][u]; odd; odd &= odd - 1) {
                            const int bit = __ffs(odd) - 1;
                            if (tile0 * KV4_TILE + i * WIDE_STEP + u % WIDE_TILES * KV4_TILE + u / WIDE_TILES * 8 + (bit & 7) < lim)
                                (bit < 8 ? ob2[0] : ob2[NG - 1]).x = NAN;
                        }
                }
            }
            if (i < whole && ok == (1u << WIDE_TILES) - 1) step(std::true_type{}, i, ok);
            else step(std::false_type{}, i, ok);
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_p[i & 3]);
        }
        if (steps > 0 && good) good = wait_on(&s_pv[(steps - 1) & 3], ((steps - 1) >> 2) & 1, failed);
        fence_after();
        const float log2_ref = ref == -INFINITY ? -INFINITY : fmaf(ref, f, -add);
        const bool past = ref > -INFINITY && fabsf(log2_ref) == INFINITY;  // a score past fp32's range
        const float l = good && !past ? l2.x + l2.y : NAN;
        const float inv = l == 0.f ? 0.f : 1.f / l;  // nothing seen: zeros
        const bool done = n_split == 1;
        const long long each = a.q_tokens * a.heads, at = part_nr * each + tok * a.heads + h;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            float x[64];
            __syncwarp();  // lanes without a row left the group before early
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
        if (mine && !done) reinterpret_cast<float2*>(sp.part + sp.splits * each * hd)[at] = make_float2(log2_ref, l);
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (*failed) {  // a role gave up: what is in flight ends before its memory goes
        for (int i = max(0, loaded - RAW); i < loaded; ++i) mbar_wait(&s_raw_full[i % RAW], (i / RAW) & 1);
        if (issued > 0) mbar_wait(wid == S::LAST ? &s_s[(issued - 1) & 3] : &s_pv[(issued - 1) & 3], ((issued - 1) >> 2) & 1);
        __syncthreads();
    }
    if (wid == S::LAST)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(WIDE_COLS) : "memory");
}

template <class T, int NG>
cudaError_t launch_wide(const Kv4Pool& pool, const Kv4Attention& a, const AttSplit& sp, cudaStream_t s) {
    const size_t smem = WideSmem<NG, is_bf16<T>>::bytes(pool.head_dim);
    const auto fn = kv4_attention_wide_kernel<T, NG>;
    cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem);
    if (e != cudaSuccess) return e;
    ++launch_counter();
    e = launch_kernel(fn, dim3(sp.per_row, a.rows, sp.splits), dim3(WideSmem<NG, is_bf16<T>>::THREADS), smem, s, pool, a, sp);
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
