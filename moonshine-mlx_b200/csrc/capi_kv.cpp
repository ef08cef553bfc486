// extern "C" boundary of the 4-bit paged K/V cache operators: argument checks, the device, and
// the launches (kernels/block_tables.cu, kv4_store.cu, kv4_attention.cu).
#include <algorithm>
#include <cmath>
#include <exception>
#include <string>

#include "../../include/moonshine_b200.h"
#include "runtime/model.hpp"

namespace msb {
void set_last_error(const std::string& m);
namespace {

// `device` current for the scope of one call (-1: the one that is)
struct DeviceScope {
    int before = -1;
    explicit DeviceScope(int device) {
        if (device < 0) return;
        int now = 0;
        MSB_CUDA(cudaGetDevice(&now));
        if (now == device) return;
        MSB_CUDA(cudaSetDevice(device));
        before = now;
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
};

template <class F>
ms_status checked(F&& f) {
    try {
        set_last_error("");
        f();
        return MS_OK;
    } catch (const MsError& e) {
        set_last_error(e.what());
        return e.status;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return MS_ERR_INVALID_ARG;
    }
}

void need(bool ok, const char* what) {
    if (!ok) throw MsError(MS_ERR_INVALID_ARG, what);
}

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int elem_size(int32_t dtype) {
    need(dtype == MS_F32 || dtype == MS_F16 || dtype == MS_BF16, "dtype must be MS_F32, MS_F16 or MS_BF16");
    return dtype == MS_F32 ? 4 : 2;
}

// rows of hd elements at these strides lie apart
bool apart(int64_t tokens, int64_t heads, int64_t token_stride, int64_t head_stride, int hd) {
    return (tokens <= 1 || token_stride >= hd) && (heads <= 1 || head_stride >= hd);
}

int type_of(int32_t dtype) { return dtype == MS_F32 ? KV4_F32 : dtype == MS_F16 ? KV4_F16 : KV4_BF16; }

void check_tokens(const ms_kv4_tokens* t) {
    need(t != nullptr, "null tokens");
    const int es = elem_size(t->dtype);
    need(t->tokens >= 0, "tokens must not be negative");
    if (t->tokens == 0) return;
    need(t->k && t->v && t->slots, "null k, v or slots");
    need(aligned(t->k, es) && aligned(t->v, es), "k and v must be aligned to their type");
}

void check_head_dim(int32_t hd) {
    if (ms_kv4_position_bytes(hd) == 0)
        throw MsError(MS_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 from 8 to 128, not " + std::to_string(hd));
}

Kv4Pool pool_of(const ms_kv4_pool* p) {
    need(p != nullptr, "null pool");
    check_head_dim(p->head_dim);
    need(p->page_size > 0 && p->page_size % 16 == 0 && p->page_size <= 1 << 30,
         "page_size must be a positive multiple of 16, at most 2^30");
    need(p->pages >= 0 && p->kv_heads > 0, "pages must not be negative and kv_heads must be positive");
    need(p->base || p->pages == 0, "null pool base");
    need(aligned(p->base, 16) && p->page_stride % 16 == 0 && p->head_stride % 16 == 0,
         "pool base and strides must be multiples of 16 bytes");
    const int64_t head = (int64_t)p->page_size * ms_kv4_position_bytes(p->head_dim);
    need(p->kv_heads == 1 || p->head_stride >= head, "head_stride is smaller than a head's page");
    need(p->pages <= 1 || p->page_stride >= head, "page_stride is smaller than a page");
    Kv4Pool k;
    k.base = p->base;
    k.pages = p->pages;
    k.kv_heads = p->kv_heads;
    k.head_dim = p->head_dim;
    k.page_size = p->page_size;
    k.page_stride = p->page_stride;
    k.head_stride = p->head_stride;
    return k;
}

Kv4Attention attention_of(const ms_kv4_pool* pool, const ms_kv4_attention_args* a) {
    need(a != nullptr, "null attention arguments");
    const int es = elem_size(a->dtype);
    need(a->rows >= 0 && a->width >= 0 && a->q_tokens >= 0 && a->max_q >= 0, "sizes must not be negative");
    need(a->heads > 0 && a->heads % pool->kv_heads == 0, "heads must be a positive multiple of kv_heads");
    need(a->rows <= 65535, "at most 65535 rows per call");
    need(a->heads <= 65535, "at most 65535 heads");
    const int max_q = a->cu_q ? (int)std::min<int64_t>(a->max_q, a->q_tokens) : 1;
    if (a->rows > 0 && a->q_tokens > 0 && max_q > 0) {
        need(a->q && a->out && a->lens, "null q, out or lens");
        need(a->block_table || a->width == 0, "null block_table");
        need(a->q != a->out, "out may not be q");
        need(aligned(a->q, es) && aligned(a->out, es), "q and out must be aligned to their type");
        need(a->cu_q || a->q_tokens >= a->rows, "without cu_q q holds one token per row");
        need((int64_t)a->width * pool->page_size <= (int64_t)1 << 30, "a row's table spans more than 2^30 positions");
        need(apart(a->q_tokens, a->heads, a->out_token_stride, a->out_head_stride, pool->head_dim),
             "out's strides are smaller than head_dim");
    }
    need(a->scale == a->scale && !std::isinf(a->scale), "scale must be finite");
    Kv4Attention k;
    k.q = a->q;
    k.out = a->out;
    k.dtype = type_of(a->dtype);
    k.heads = a->heads;
    k.q_tokens = a->q_tokens;
    k.q_token_stride = a->q_token_stride;
    k.q_head_stride = a->q_head_stride;
    k.out_token_stride = a->out_token_stride;
    k.out_head_stride = a->out_head_stride;
    k.table = a->block_table;
    k.table_stride = a->table_stride;
    k.rows = a->rows;
    k.width = a->width;
    k.lens = a->lens;
    k.cu_q = a->cu_q;
    k.max_q = max_q;
    k.causal = a->causal != 0;
    const int64_t q_rows = (int64_t)k.max_q * a->heads;
    if (q_rows >= (int64_t)1 << 30 || q_rows / pool->kv_heads >= 1 << 24)
        throw MsError(MS_ERR_UNSUPPORTED, "max_q * heads is too large: give the queries in several calls");
    k.scale = a->scale == 0.f ? (float)(1.0 / std::sqrt((double)pool->head_dim)) : a->scale;
    return k;
}

}  // namespace
}  // namespace msb

using namespace msb;

extern "C" {

int32_t ms_kv4_position_bytes(int32_t head_dim) {
    if (!kv4_head_dim_ok(head_dim)) return 0;
    return head_dim + 8 * ((head_dim + 63) / 64);
}

ms_status ms_kv_block_tables(const ms_kv_tables* t, int32_t device, void* stream) {
    return checked([&] {
        need(t != nullptr, "null arguments");
        need(t->rows >= 0 && t->width >= 0 && t->n_free >= 0, "sizes must not be negative");
        need(t->n_slots >= 0 && t->n_slots < (int64_t)1 << 31, "n_slots must be from 0 to 2^31 - 1");
        need(t->page_size > 0, "page_size must be positive");
        need(t->cu_new && t->counts, "null cu_new or counts");
        need(t->rows == 0 || (t->lengths && t->new_tokens), "null lengths or new_tokens");
        need(t->rows == 0 || t->width == 0 || t->block_table, "null block_table");
        need(t->rows <= 1 || t->table_stride >= t->width, "table_stride is smaller than width");
        need(t->n_slots == 0 || t->slots, "null slots");
        DeviceScope d(device);
        MSB_CUDA(launch_block_tables(t->lengths, t->new_tokens, t->rows, t->page_size, t->free_pages, t->n_free,
                                     t->block_table, t->width, t->table_stride,
                                     reinterpret_cast<long long*>(t->slots), t->n_slots, t->cu_new, t->counts,
                                     reinterpret_cast<cudaStream_t>(stream)));
    });
}

ms_status ms_kv4_append(const ms_kv4_pool* pool, const ms_kv4_tokens* t, int32_t device, void* stream) {
    return checked([&] {
        const Kv4Pool p = pool_of(pool);
        check_tokens(t);
        if (t->tokens == 0 || p.pages == 0) return;
        DeviceScope d(device);
        MSB_CUDA(launch_kv4_append(p, t->k, t->v, type_of(t->dtype), t->tokens, t->k_token_stride, t->k_head_stride,
                                   t->v_token_stride, t->v_head_stride, reinterpret_cast<const long long*>(t->slots),
                                   reinterpret_cast<cudaStream_t>(stream)));
    });
}

ms_status ms_kv4_read(const ms_kv4_pool* pool, const ms_kv4_tokens* t, int32_t device, void* stream) {
    return checked([&] {
        const Kv4Pool p = pool_of(pool);
        check_tokens(t);
        if (t->tokens == 0) return;
        need(apart(t->tokens, p.kv_heads, t->k_token_stride, t->k_head_stride, p.head_dim) &&
                 apart(t->tokens, p.kv_heads, t->v_token_stride, t->v_head_stride, p.head_dim),
             "strides of k or v are smaller than head_dim");
        DeviceScope d(device);
        MSB_CUDA(launch_kv4_read(p, t->k, t->v, type_of(t->dtype), t->tokens, t->k_token_stride, t->k_head_stride,
                                 t->v_token_stride, t->v_head_stride, reinterpret_cast<const long long*>(t->slots),
                                 reinterpret_cast<cudaStream_t>(stream)));
    });
}

int64_t ms_kv4_attention_workspace(const ms_kv4_pool* pool, const ms_kv4_attention_args* args) {
    int64_t n = -1;
    checked([&] {
        const Kv4Pool p = pool_of(pool);
        n = (int64_t)kv4_attention_workspace(p, attention_of(pool, args));
    });
    return n;
}

ms_status ms_kv4_attention(const ms_kv4_pool* pool, const ms_kv4_attention_args* args, void* workspace,
                           int64_t workspace_bytes, int32_t device, void* stream) {
    return checked([&] {
        const Kv4Pool p = pool_of(pool);
        const Kv4Attention a = attention_of(pool, args);
        if (a.rows == 0 || a.q_tokens == 0 || a.max_q == 0) return;
        const int64_t bytes = (int64_t)kv4_attention_workspace(p, a);
        if (bytes > workspace_bytes || (bytes > 0 && (!workspace || !aligned(workspace, 16))))
            throw MsError(MS_ERR_CAPACITY, "attention needs a 16-byte aligned workspace of " + std::to_string(bytes) + " bytes");
        DeviceScope d(device);
        MSB_CUDA(launch_kv4_attention(p, a, workspace, reinterpret_cast<cudaStream_t>(stream)));
    });
}

}  // extern "C"
