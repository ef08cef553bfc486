// Attention over 4-bit pages in which every wait for a copy gives up at its first look: the kernel
// then waits for its copies in flight, reports and returns.  Prints the status word and how
// many of the results are not NaN.
#define KV4_WAIT_LIMIT 0
#define KV4_ATTENTION_KERNELS
#include "kv4_attention.cuh"

#include <cstdio>
#include <vector>

namespace msb {
int64_t& launch_counter() {
    static int64_t n = 0;
    return n;
}
bool& pdl_launches() {
    static bool on = false;
    return on;
}
}  // namespace msb
using namespace msb;

int main() {
    constexpr int rows = 3, heads = 4, hd = 64, page = 64, width = 8, n = rows * heads * hd;
    Kv4Pool pool;
    pool.pages = rows * width;
    pool.kv_heads = heads;
    pool.head_dim = hd;
    pool.page_size = page;
    pool.head_stride = (long long)page * 72;
    pool.page_stride = pool.head_stride * heads;
    Kv4Attention a;
    float* q;
    __nv_bfloat16* out;
    int *table, *lens;
    unsigned* status;
    if (cudaMalloc(&pool.base, pool.page_stride * pool.pages) || cudaMalloc(&q, n * 4) || cudaMalloc(&out, n * 2) ||
        cudaMalloc(&table, rows * width * 4) || cudaMalloc(&lens, rows * 4) || cudaMalloc(&status, 4))
        return 1;
    std::vector<int> t(rows * width);
    for (int i = 0; i < rows * width; ++i) t[i] = i;
    const int l[rows] = {1, 300, width * page};
    std::vector<__nv_bfloat16> got(n);
    unsigned word = 0;
    cudaMemset(pool.base, 0, pool.page_stride * pool.pages);
    cudaMemset(q, 0, n * 4);
    cudaMemset(out, 0, n * 2);
    cudaMemset(status, 0, 4);
    cudaMemcpy(table, t.data(), t.size() * 4, cudaMemcpyHostToDevice);
    cudaMemcpy(lens, l, sizeof(l), cudaMemcpyHostToDevice);
    a.q = q;
    a.out = out;
    a.dtype = KV4_STEP;
    a.heads = heads;
    a.q_tokens = a.rows = rows;
    a.q_token_stride = a.out_token_stride = heads * hd;
    a.q_head_stride = a.out_head_stride = hd;
    a.table = table;
    a.table_stride = a.width = width;
    a.lens = lens;
    a.status = status;
    AttSplit sp;
    sp.per_row = heads;
    sp.page_shift = 2;
    if (launch_type<Step>(pool, a, sp, nullptr) || cudaDeviceSynchronize()) return 2;
    cudaMemcpy(&word, status, 4, cudaMemcpyDeviceToHost);
    cudaMemcpy(got.data(), out, n * 2, cudaMemcpyDeviceToHost);
    int numbers = 0;
    for (int i = 0; i < n; ++i) numbers += __bfloat162float(got[i]) == __bfloat162float(got[i]);
    std::printf("%u %d\n", word, numbers);
    return 0;
}
