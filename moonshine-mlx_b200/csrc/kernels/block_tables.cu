// Block tables and slot maps of a paged K/V cache, from request lengths on the device.
//
// Row b holds len_b positions in ceil(len_b / P) pages and appends new_b more: it takes
// take_b = ceil((len_b + new_b) / P) - ceil(len_b / P) pages, numbered start_b + i with
// start_b the sum of the takes before it, and token j's slot is page * P + offset of position
// len_b + j.  One launch and no workspace: every CTA scans the rows itself (both running
// sums packed in one 64-bit word) and writes its own range of the slots and table rows as
// soon as the scan has passed them.
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
    int wide;   // slots are 16-byte aligned
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
    __shared__ int s_tok[BT_CHUNK + 1];  // tokens before each row of the chunk
    __shared__ int s_pg[BT_CHUNK + 1];   // pages before it
    __shared__ int s_len[BT_CHUNK];
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
#pragma unroll
        for (int i = 0; i < BT_ITEMS; ++i) {
            const int r = tid * BT_ITEMS + i;
            int len = 0, add = 0;
            if (r < nr) {
                len = max(0, a.lengths[c0 + r]);
                add = max(0, a.added[c0 + r]);
            }
            const unsigned have = pages_for(a, (unsigned)len), need = pages_for(a, (unsigned)len + (unsigned)add);
            mine[i] = sum;
            sum += (unsigned long long)(need - have) << 32 | (unsigned)add;
            if (r < nr) s_len[r] = len;
        }
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
#pragma unroll
        for (int i = 0; i < BT_ITEMS; ++i) {
            const int r = tid * BT_ITEMS + i;
            const unsigned long long v = before + mine[i];
            if (r < nr) {
                s_tok[r] = (int)(unsigned)v;
                s_pg[r] = (int)(v >> 32);
            }
        }
        if (tid == 0) {
            s_tok[nr] = (int)(unsigned)total;
            s_pg[nr] = (int)(total >> 32);
        }
        __syncthreads();
        // table rows [row0, row1) of this chunk: new pages, then -1
        for (int b = max(row0, c0) + wid; b < min(row1, c0 + nr); b += BT_THREADS / 32) {
            const int r = b - c0;
            const unsigned have = pages_for(a, (unsigned)s_len[r]), start = (unsigned)s_pg[r];
            const unsigned take = (unsigned)s_pg[r + 1] - start;
            int* t = a.table + b * a.table_stride;
            for (long long k = (long long)have + lane; k < a.width; k += 32)
                t[k] = k - have < take ? fresh_page(a, start + (unsigned)(k - have)) : -1;
            if (lane == 0) a.cu[b + 1] = s_tok[r + 1];
        }
        // slots [slot0, slot1) of this chunk's tokens, two per thread (one 16-byte store)
        const long long t0 = max(slot0, (long long)s_tok[0]), t1 = min(slot1, (long long)s_tok[nr]);
        int lo = 0;  // the last row whose first token is <= t has it
        for (long long t = (t0 & ~1ll) + 2 * tid; t < t1; t += 2 * BT_THREADS) {
            long long slot[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
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
                }
                const unsigned len = (unsigned)s_len[lo], pos = len + (unsigned)(ti - s_tok[lo]);
                const unsigned blk = over_page(a, pos), have = pages_for(a, len);
                int pg = -1;
                if (blk < (unsigned)a.width)
                    pg = blk < have ? a.table[(long long)(c0 + lo) * a.table_stride + blk]
                                    : fresh_page(a, (unsigned)s_pg[lo] + (blk - have));
                slot[i] = pg < 0 ? -1ll : (long long)pg * P + (pos - blk * P);
            }
            if (a.wide && t >= t0 && t + 1 < t1) {
                *reinterpret_cast<longlong2*>(a.slots + t) = make_longlong2(slot[0], slot[1]);
            } else {
                if (t >= t0) a.slots[t] = slot[0];
                if (t + 1 >= t0 && t + 1 < t1) a.slots[t + 1] = slot[1];
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
                     rows, page, n_free, width, 0, -1, 0, 0};
    a.wide = !(reinterpret_cast<uintptr_t>(slots) & 15);
    for (int n = 0; n < 31; ++n)
        if (1 << n == page) a.shift = n;
    // one CTA per 16 KB of output, at most three per SM of the 148
    const double out = 8.0 * n_slots + 4.0 * rows * (double)width;
    const int grid = (int)std::min(444.0, std::max(1.0, out / 16384.0));
    a.rows_per_cta = (rows + grid - 1) / grid;
    a.slots_per_cta = ((n_slots + grid - 1) / grid + 1) & ~1ll;
    ++launch_counter();
    return launch_kernel(block_tables_kernel, dim3(grid), dim3(BT_THREADS), 0, s, a);
}

}  // namespace msb
