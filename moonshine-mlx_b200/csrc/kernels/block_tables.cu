// Block tables and slot maps of a paged K/V cache, from request lengths on the device.
//
// Row b holds len_b positions in ceil(len_b / P) pages and appends new_b more: it takes
// take_b = ceil((len_b + new_b) / P) - ceil(len_b / P) pages, numbered start_b + i with
// start_b the sum of the takes before it, and token j's slot is page * P + offset of position
// len_b + j.  One launch and no workspace: every CTA scans the rows itself (both running
// sums packed in one 64-bit word) and writes its own range of the slots and table rows as
// soon as the scan has passed them.
//
// Bound: launch latency for a decode step (64 rows: 8 us from launch to launch), the writes for
// many new tokens: 4096 rows of up to 32K positions append 262144 .. 4.2M slots and the empty ends
// of a table 2112 wide, up to 68 MB, in 25 us, of which two scans of 2048 rows, the same in all
// CTAs, are about 4.  Slots go out four per store (32 bytes), lengths come in four per load (31 us
// without).
#include "common.cuh"

namespace msb {
namespace {

constexpr int BT_THREADS = 512;
constexpr int BT_ITEMS = 4;
constexpr int BT_CHUNK = BT_THREADS * BT_ITEMS;  // rows per scan step

struct BlockTableArgs {
    const int* lengths;
    const int* added;
    const int* free_pages;
    int* table;
    long long* slots;
    int* cu;
    int* counts;
    long long n_slots, table_stride;
    int rows, page, n_free, width;
    int wide, wide_in, wide_table;  // slots 32-byte, lengths and table rows 16-byte aligned
    int shift;  // log2 of the page size, -1 if it is no power of two
    int rows_per_cta;
    long long slots_per_cta;
};

__device__ __forceinline__ unsigned over_page(const BlockTableArgs& a, unsigned n) {
    return a.shift >= 0 ? n >> a.shift : n / (unsigned)a.page;
}
__device__ __forceinline__ unsigned pages_for(const BlockTableArgs& a, unsigned n) {
    const unsigned q = over_page(a, n);
    return q + (q * (unsigned)a.page != n);
}

// page number `i` handed out by this call, -1 past the free ones
__device__ __forceinline__ int fresh_page(const BlockTableArgs& a, unsigned i) {
    if (i >= (unsigned)a.n_free) return -1;
    return a.free_pages ? a.free_pages[i] : (int)i;
}

__global__ void __launch_bounds__(BT_THREADS) block_tables_kernel(const BlockTableArgs a) {
    __shared__ __align__(16) int s_tok[BT_CHUNK + 4];  // tokens before each row of the chunk
    __shared__ __align__(16) int s_pg[BT_CHUNK + 4];   // pages before it
    __shared__ __align__(16) int s_len[BT_CHUNK];
    __shared__ unsigned long long s_warp[BT_THREADS / 32];
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const unsigned P = (unsigned)a.page;
    const long long slot0 = min(a.n_slots, (long long)blockIdx.x * a.slots_per_cta);
    const long long slot1 = min(a.n_slots, slot0 + a.slots_per_cta);
    const int row0 = min(a.rows, (int)blockIdx.x * a.rows_per_cta), row1 = min(a.rows, row0 + a.rows_per_cta);
    const bool last = blockIdx.x == gridDim.x - 1;
    unsigned long long base = 0;  // pages << 32 | tokens before the chunk
    for (int c0 = 0; c0 < a.rows; c0 += BT_CHUNK) {
        const int nr = min(BT_CHUNK, a.rows - c0);
        // this thread's rows, their sums, then the block scan of the sums
        unsigned long long mine[BT_ITEMS], sum = 0;
        int lens[BT_ITEMS] = {0, 0, 0, 0}, adds[BT_ITEMS] = {0, 0, 0, 0};
        static_assert(BT_ITEMS == 4, "a thread's rows are one 16-byte load");
        if (a.wide_in && tid * BT_ITEMS + 3 < nr) {
            *reinterpret_cast<int4*>(lens) = __ldg(reinterpret_cast<const int4*>(a.lengths + c0) + tid);
            *reinterpret_cast<int4*>(adds) = __ldg(reinterpret_cast<const int4*>(a.added + c0) + tid);
        } else {
#pragma unroll
            for (int i = 0; i < BT_ITEMS; ++i)
                if (tid * BT_ITEMS + i < nr) {
                    lens[i] = a.lengths[c0 + tid * BT_ITEMS + i];
                    adds[i] = a.added[c0 + tid * BT_ITEMS + i];
                }
        }
#pragma unroll
        for (int i = 0; i < BT_ITEMS; ++i) {
            const int len = lens[i] = max(0, lens[i]), add = max(0, adds[i]);
            const unsigned have = pages_for(a, (unsigned)len), need = pages_for(a, (unsigned)len + (unsigned)add);
            mine[i] = sum;
            sum += (unsigned long long)(need - have) << 32 | (unsigned)add;
        }
        *reinterpret_cast<int4*>(s_len + tid * BT_ITEMS) = make_int4(lens[0], lens[1], lens[2], lens[3]);
        unsigned long long inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long v = __shfl_up_sync(FULL, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) s_warp[wid] = inc;
        __syncthreads();
        unsigned long long before = base, total = base;
#pragma unroll
        for (int w = 0; w < BT_THREADS / 32; ++w) {
            if (w < wid) before += s_warp[w];
            total += s_warp[w];
        }
        before += inc - sum;
        // rows past the last hold the sums, so entry nr is the end of the last row
        int toks[BT_ITEMS], pgs[BT_ITEMS];
#pragma unroll
        for (int i = 0; i < BT_ITEMS; ++i) {
            toks[i] = (int)(unsigned)(before + mine[i]);
            pgs[i] = (int)((before + mine[i]) >> 32);
        }
        *reinterpret_cast<int4*>(s_tok + tid * BT_ITEMS) = make_int4(toks[0], toks[1], toks[2], toks[3]);
        *reinterpret_cast<int4*>(s_pg + tid * BT_ITEMS) = make_int4(pgs[0], pgs[1], pgs[2], pgs[3]);
        if (tid == 0) {
            s_tok[BT_CHUNK] = (int)(unsigned)total;
            s_pg[BT_CHUNK] = (int)(total >> 32);
        }
        __syncthreads();
        // table rows [row0, row1) of this chunk: new pages, then -1
        for (int b = max(row0, c0) + wid; b < min(row1, c0 + nr); b += BT_THREADS / 32) {
            const int r = b - c0;
            const unsigned have = pages_for(a, (unsigned)s_len[r]), start = (unsigned)s_pg[r];
            const unsigned take = (unsigned)s_pg[r + 1] - start;
            int* t = a.table + b * a.table_stride;
            // new pages, up to a 16-byte boundary of the entries behind them, which take whole stores
            const long long need = (long long)have + take, whole = a.wide_table ? (need + 3) & ~3ll : a.width;
            for (long long k = (long long)have + lane; k < min(whole, (long long)a.width); k += 32)
                t[k] = k < need ? fresh_page(a, start + (unsigned)(k - have)) : -1;
            for (long long k = whole + 4 * lane; k < a.width; k += 128) {
                if (k + 3 < a.width) *reinterpret_cast<int4*>(t + k) = make_int4(-1, -1, -1, -1);
                else
                    for (long long j = k; j < a.width; ++j) t[j] = -1;
            }
            if (lane == 0) a.cu[b + 1] = s_tok[r + 1];
        }
        // slots [slot0, slot1) of this chunk's tokens, four per thread (one 32-byte store)
        const long long t0 = max(slot0, (long long)s_tok[0]), t1 = min(slot1, (long long)s_tok[nr]);
        int lo = 0;  // the last row whose first token is <= t has it
        for (long long t = (t0 & ~3ll) + 4 * tid; t < t1; t += 4 * BT_THREADS) {
            long long slot[4];
            int pg = -1;
            unsigned page = ~0u;  // the table column that pg is of
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const long long ti = t + i;
                if (ti < t0 || ti >= t1) continue;
                if (s_tok[lo + 1] <= ti) {
                    int hi = nr;
                    ++lo;
                    while (hi - lo > 1) {
                        const int mid = (lo + hi) >> 1;
                        if (s_tok[mid] <= ti) lo = mid;
                        else hi = mid;
                    }
                    page = ~0u;
                }
                const unsigned len = (unsigned)s_len[lo], pos = len + (unsigned)(ti - s_tok[lo]);
                const unsigned blk = over_page(a, pos);
                if (blk != page) {
                    const unsigned have = pages_for(a, len);
                    page = blk;
                    pg = -1;
                    if (blk < (unsigned)a.width)
                        pg = blk < have ? a.table[(long long)(c0 + lo) * a.table_stride + blk]
                                        : fresh_page(a, (unsigned)s_pg[lo] + (blk - have));
                }
                slot[i] = pg < 0 ? -1ll : (long long)pg * P + (pos - blk * P);
            }
            if (a.wide && t >= t0 && t + 3 < t1) {
                asm volatile("st.global.v4.b64 [%0], {%1, %2, %3, %4};" ::"l"(a.slots + t), "l"(slot[0]), "l"(slot[1]),
                             "l"(slot[2]), "l"(slot[3])
                             : "memory");
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (t + i >= t0 && t + i < t1) a.slots[t + i] = slot[i];
            }
        }
        base = total;
        // done when the scan has passed this CTA's slots and rows (the last CTA writes the sums)
        if (!last && c0 + nr >= row1 && (long long)(unsigned)base >= slot1) return;
        __syncthreads();
    }
    for (long long t = max(slot0, (long long)(unsigned)base) + tid; t < slot1; t += BT_THREADS) a.slots[t] = -1;
    if (last && tid == 0) {
        a.cu[0] = 0;
        a.counts[0] = (int)(base >> 32);
        a.counts[1] = (int)(unsigned)base;
    }
}

}  // namespace

cudaError_t launch_block_tables(const int* lengths, const int* added, int rows, int page, const int* free_pages,
                                int n_free, int* table, int width, long long table_stride, long long* slots,
                                long long n_slots, int* cu, int* counts, cudaStream_t s) {
    BlockTableArgs a{lengths, added, free_pages, table, slots, cu, counts, n_slots, table_stride,
                     rows, page, n_free, width, 0, 0, 0, -1, 0, 0};
    a.wide = !(reinterpret_cast<uintptr_t>(slots) & 31);
    a.wide_in = !((reinterpret_cast<uintptr_t>(lengths) | reinterpret_cast<uintptr_t>(added)) & 15);
    a.wide_table = !(reinterpret_cast<uintptr_t>(table) & 15) && table_stride % 4 == 0;
    for (int n = 0; n < 31; ++n)
        if (1 << n == page) a.shift = n;
    // one CTA per 16 KB of output, at most three per SM of the 148
    const double out = 8.0 * n_slots + 4.0 * rows * (double)width;
    const int grid = (int)std::min(444.0, std::max(1.0, out / 16384.0));
    a.rows_per_cta = (rows + grid - 1) / grid;
    a.slots_per_cta = ((n_slots + grid - 1) / grid + 3) & ~3ll;
    ++launch_counter();
    return launch_kernel(block_tables_kernel, dim3(grid), dim3(BT_THREADS), 0, s, a);
}

}  // namespace msb
