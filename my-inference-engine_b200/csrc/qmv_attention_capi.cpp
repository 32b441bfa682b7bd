// C ABI of the attention of many sequences (declared in include/qmv_b200.h):
// argument checks, then one launch helper each.  0 return + per-thread
// message on failure; nothing is launched for a refused call.
#include <cuda_runtime.h>

#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "qmv_attention.h"
#include "qmv_b200.h"
#include "qmv_internal.h"

#define QMV_EXPORT extern "C" __attribute__((visibility("default")))

namespace {

int fail(const char *fmt, ...)
{
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return qmv::set_error(buf);
}

int element_bytes(uint32_t type)
{
    return type == QMV_TYPE_F32 ? 4 : type == QMV_TYPE_F16 || type == QMV_TYPE_BF16 ? 2 : 0;
}

// A device address of the calling thread's device (the kernels follow it).
int check_device(const char *what, const void *p, int dev)
{
    cudaPointerAttributes at{};
    const cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return qmv::set_cuda_error(what, e);
    }
    if (at.type == cudaMemoryTypeManaged) return 1;
    if (at.type != cudaMemoryTypeDevice) return fail("%s is not device memory", what);
    if (at.device != dev) return fail("%s lives on device %d but the calling thread's device is %d", what, at.device, dev);
    return 1;
}

// `count` elements a row, rows `ld` elements apart, each on a 16-byte boundary.
int check_rows(const char *what, const void *p, int64_t ld, int64_t count, int bytes)
{
    if (p == nullptr) return fail("%s is null", what);
    if (ld < count) return fail("%s_ld %lld is less than a row's %lld elements", what, (long long)ld, (long long)count);
    if (ld > (int64_t)1 << 32) return fail("%s_ld %lld is out of range", what, (long long)ld);
    if (((uintptr_t)p & 15u) != 0 || ld * bytes % 16 != 0) return fail("%s must start every row on a 16-byte boundary", what);
    return 1;
}

int check_heads(uint32_t type, int heads, int kv_heads, int head_dim)
{
    if (element_bytes(type) == 0) return fail("unsupported type %u (F32, F16 and BF16 only)", type);
    if (head_dim != 64 && head_dim != 128) return fail("head_dim must be 64 or 128");
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0) return fail("heads must be a positive multiple of kv_heads");
    if (heads / kv_heads > qmv::kMaxGroup) return fail("at most %d query heads per key/value head", qmv::kMaxGroup);
    if (heads > 65535) return fail("too many heads");
    return 1;
}

int check_cache(const QmvPagedCache *c, uint32_t type, qmv::KvView *kv)
{
    if (c == nullptr) return fail("cache is null");
    if (c->type != (type == QMV_TYPE_BF16 ? QMV_TYPE_BF16 : QMV_TYPE_F16))
        return fail("cache type %u does not go with activation type %u (F16 with F32 or F16, BF16 with BF16)", c->type, type);
    int shift = 4;
    while (shift < 9 && c->page_size != 1 << shift) ++shift;
    if (shift == 9) return fail("page_size must be 16, 32, 64, 128 or 256");
    if (c->page_count <= 0) return fail("page_count must be positive");
    if (c->keys == nullptr || c->values == nullptr) return fail("cache keys or values are null");
    if ((((uintptr_t)c->keys | (uintptr_t)c->values) & 15u) != 0) return fail("cache keys and values must be 16-byte aligned");
    const int64_t strides[3] = {c->page_stride, c->position_stride, c->head_stride};
    for (int64_t s : strides)
        if (s < c->head_dim || s % 8 != 0 || s > (int64_t)1 << 38)
            return fail("cache strides must be multiples of 8 elements and at least head_dim");
    *kv = qmv::KvView{c->keys, c->values, c->position_stride, c->position_stride, c->page_stride, c->head_stride,
                      nullptr, 0, shift, c->page_count};
    return 1;
}

int check_batch(const QmvPagedBatch *b, qmv::KvView *kv)
{
    if (b == nullptr) return fail("batch is null");
    if (b->sequences < 0 || b->tokens < 0) return fail("sequences and tokens must not be negative");
    if (b->sequences == 0 || b->tokens == 0) return 1;
    if (b->query_start == nullptr || b->length == nullptr || b->page_table == nullptr)
        return fail("query_start, length or page_table is null");
    // (key counts are rounded up to blocks in 32 bits)
    if (b->max_pages <= 0 || b->max_pages > ((1 << 30) >> kv->page_shift)) return fail("max_pages is out of range (2^30 positions at most)");
    if (b->max_query <= 0) return fail("max_query must be positive");
    kv->table = b->page_table;
    kv->max_pages = b->max_pages;
    return 1;
}

int check_metadata_device(const QmvPagedBatch *b, int dev)
{
    return check_device("query_start", b->query_start, dev) && check_device("length", b->length, dev) &&
           check_device("page_table", b->page_table, dev);
}

int check_scale(float *scale, int head_dim)
{
    if (!(*scale >= 0.f) || !isfinite(*scale)) return fail("scale must be finite and not negative");
    if (*scale == 0.f) *scale = 1.0f / sqrtf((float)head_dim);
    return 1;
}

int current_device(int *dev, unsigned int **status)
{
    cudaError_t e = cudaGetDevice(dev);
    if (e == cudaSuccess) e = qmv::attention_status_word(status);
    return e == cudaSuccess ? 1 : qmv::set_cuda_error("current device", e);
}

}  // namespace

QMV_EXPORT int qmv_paged_append(const QmvPagedCache *cache, const QmvPagedBatch *batch, uint32_t type, int heads,
                                const void *q, int64_t q_ld, const void *k, int64_t k_ld, const void *v, int64_t v_ld,
                                float rope_base, void *q_out, int64_t q_out_ld, void *k_out, int64_t k_out_ld,
                                void *stream)
{
    qmv::KvView kv{};
    if (cache == nullptr) return fail("cache is null");
    if (!check_heads(type, heads, cache->kv_heads, cache->head_dim) || !check_cache(cache, type, &kv) || !check_batch(batch, &kv))
        return 0;
    if (!(rope_base == 0.f || rope_base >= 1.f) || !isfinite(rope_base)) return fail("rope_base must be 0 or at least 1, and finite");
    if (batch->sequences == 0 || batch->tokens == 0) return 1;
    const int bytes = element_bytes(type), d = cache->head_dim;
    if (!check_rows("k", k, k_ld, (int64_t)cache->kv_heads * d, bytes) || !check_rows("v", v, v_ld, (int64_t)cache->kv_heads * d, bytes))
        return 0;
    if (q_out != nullptr &&
        (!check_rows("q", q, q_ld, (int64_t)heads * d, bytes) || !check_rows("q_out", q_out, q_out_ld, (int64_t)heads * d, bytes)))
        return 0;
    if (k_out != nullptr && !check_rows("k_out", k_out, k_out_ld, (int64_t)cache->kv_heads * d, bytes)) return 0;
    if ((q_out == q && q_out != nullptr && q_out_ld != q_ld) || (k_out == k && k_out_ld != k_ld))
        return fail("an output in its input's place needs the same ld");
    int dev = 0;
    unsigned int *status = nullptr;
    if (!current_device(&dev, &status) || !check_device("keys", cache->keys, dev) ||
        !check_device("values", cache->values, dev) || !check_device("k", k, dev) || !check_device("v", v, dev) ||
        (q_out != nullptr && (!check_device("q", q, dev) || !check_device("q_out", q_out, dev))) ||
        (k_out != nullptr && !check_device("k_out", k_out, dev)) || !check_metadata_device(batch, dev))
        return 0;
    const qmv::AppendArgs a{type, cache->type, q, k, v, q_out, k_out, q_ld, k_ld, v_ld, q_out_ld, k_out_ld, kv,
                            batch->query_start, batch->length, batch->sequences, batch->tokens, heads, cache->kv_heads, d,
                            rope_base, status};
    const cudaError_t e = qmv::launch_paged_append(a, (cudaStream_t)stream);
    return e == cudaSuccess ? 1 : qmv::set_cuda_error("append launch", e);
}

QMV_EXPORT int qmv_packed_attention(uint32_t type, int heads, int kv_heads, int head_dim, const int *start,
                                    int sequences, int tokens, const void *q, int64_t q_ld, const void *k, int64_t k_ld,
                                    const void *v, int64_t v_ld, void *out, int64_t out_ld, float scale, void *stream)
{
    if (!check_heads(type, heads, kv_heads, head_dim) || !check_scale(&scale, head_dim)) return 0;
    if (sequences < 0 || tokens < 0) return fail("sequences and tokens must not be negative");
    if (sequences == 0 || tokens == 0) return 1;
    if (start == nullptr) return fail("start is null");
    const int bytes = element_bytes(type);
    const int64_t nq = (int64_t)heads * head_dim, nk = (int64_t)kv_heads * head_dim;
    if (!check_rows("q", q, q_ld, nq, bytes) || !check_rows("k", k, k_ld, nk, bytes) || !check_rows("v", v, v_ld, nk, bytes) ||
        !check_rows("out", out, out_ld, nq, bytes))
        return 0;
    int dev = 0;
    unsigned int *status = nullptr;
    if (!current_device(&dev, &status) || !check_device("q", q, dev) || !check_device("k", k, dev) || !check_device("v", v, dev) ||
        !check_device("out", out, dev) || !check_device("start", start, dev))
        return 0;
    const qmv::KvView kv{k, v, k_ld, v_ld, 0, head_dim, nullptr, 0, 0, 0};
    const qmv::AttnArgs a{type, type, q, out, q_ld, out_ld, kv, start, nullptr, sequences, tokens, heads, kv_heads,
                          heads / kv_heads, head_dim, tokens, scale, status};
    const cudaError_t e = qmv::launch_tc_attention(a, (cudaStream_t)stream);
    return e == cudaSuccess ? 1 : qmv::set_cuda_error("attention launch", e);
}

QMV_EXPORT int qmv_paged_attention(const QmvPagedCache *cache, const QmvPagedBatch *batch, uint32_t type, int heads,
                                   const void *q, int64_t q_ld, void *out, int64_t out_ld, float scale, void *stream)
{
    qmv::KvView kv{};
    if (cache == nullptr) return fail("cache is null");
    if (!check_heads(type, heads, cache->kv_heads, cache->head_dim) || !check_cache(cache, type, &kv) ||
        !check_batch(batch, &kv) || !check_scale(&scale, cache->head_dim))
        return 0;
    if (batch->sequences == 0 || batch->tokens == 0) return 1;
    const int bytes = element_bytes(type), d = cache->head_dim;
    if (!check_rows("q", q, q_ld, (int64_t)heads * d, bytes) || !check_rows("out", out, out_ld, (int64_t)heads * d, bytes)) return 0;
    int dev = 0;
    unsigned int *status = nullptr;
    if (!current_device(&dev, &status) || !check_device("keys", cache->keys, dev) ||
        !check_device("values", cache->values, dev) || !check_device("q", q, dev) || !check_device("out", out, dev) ||
        !check_metadata_device(batch, dev))
        return 0;
    const qmv::AttnArgs a{type, cache->type, q, out, q_ld, out_ld, kv, batch->query_start, batch->length,
                          batch->sequences, batch->tokens, heads, cache->kv_heads, heads / cache->kv_heads, d,
                          batch->max_query, scale, status};
    const bool few = (int64_t)a.max_query * a.group <= 32;
    const cudaError_t e = few ? qmv::launch_decode_attention(a, (cudaStream_t)stream) : qmv::launch_tc_attention(a, (cudaStream_t)stream);
    return e == cudaSuccess ? 1 : qmv::set_cuda_error("attention launch", e);
}
