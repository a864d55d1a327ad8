// Host side of libmcsparse.so, products with matrices that are never stored: argument checks of the embedding and the
// windowed-attention entry points. The status codes used here are explained in api_common.h.
#include <cmath>
#include <new>

#include "api_common.h"

using namespace mcsp_b200;
using namespace mcsp_b200::api;

namespace {

bool operator_type(macaDataType t) { return t == MACA_R_32F || t == MACA_R_16F || t == MACA_R_16BF; }
int64_t type_bytes(macaDataType t) { return t == MACA_R_32F ? 4 : 2; }
bool too_big(int64_t v) { return (v >> 31) != 0; }  // negative, or no int32
bool misaligned(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) != 0; }

ScalarArg<float> scalar(const mcsparseContext* h, const void* p) {
    ScalarArg<float> a;
    a.host = h->ptr_mode == MCSPARSE_POINTER_MODE_HOST ? *static_cast<const float*>(p) : 0.0f;
    a.dev = h->ptr_mode == MCSPARSE_POINTER_MODE_HOST ? nullptr : static_cast<const float*>(p);
    return a;
}

bool gave_up(mcsparseContext* h) {
    return take_device_fault(h->attention_fault_host, "an earlier attention call on this handle gave up a bounded device-side wait; its result is incomplete");
}

// ----------------------------------------------------------------------------- embedding

// table: E or dE (rows x width); tokens: Y or dY (count x width).
St embedding_check(mcsparseHandle_t h, int64_t count, mcsparseIndexType_t indexType, const mcsparseDnMatDescr* table,
                   const mcsparseDnMatDescr* tokens) {
    if (h == nullptr) return BAD_HANDLE;
    if (table == nullptr || tokens == nullptr) return BAD_POINTER;
    if (count < 0) return BAD_SIZE;
    if (indexType != MCSPARSE_INDEX_32I && indexType != MCSPARSE_INDEX_64I) return NOT_IMPL;
    const macaDataType e = table->valueType, y = tokens->valueType;
    if (!operator_type(e) || !operator_type(y) || !(e == y || e == MACA_R_32F || y == MACA_R_32F)) return NOT_IMPL;
    if (table->order != MCSPARSE_ORDER_ROW || tokens->order != MCSPARSE_ORDER_ROW) return NOT_IMPL;
    if (table->batchCount != 1 || tokens->batchCount != 1) return NOT_IMPL;
    if (tokens->row_num != count || tokens->col_num != table->col_num) return BAD_SIZE;
    if (table->ld < table->col_num || tokens->ld < tokens->col_num) return BAD_SIZE;
    // sorted keys, positions and the keys behind the last row are int32; a launch has fewer than 2^31 blocks
    const int64_t width = table->col_num, rows = table->row_num;
    if (too_big(count) || too_big(width) || too_big(rows + 1)) return NOT_IMPL;
    if ((width / 128 + 1) > (int64_t(1) << 33) / (rows + count + 1)) return NOT_IMPL;
    if (misaligned(table->values, type_bytes(e)) || misaligned(tokens->values, type_bytes(y))) return BAD_VALUE;
    return OK;
}

// A descriptor's values may have been taken away (mcsparseDnMatSetValues) after it was made.
bool absent(const mcsparseDnMatDescr* m) { return m->values == nullptr && m->row_num > 0 && m->col_num > 0; }

St embedding_arrays(const void* indices, int64_t count, mcsparseIndexType_t type, mcsparseIndexBase_t base, const mcsparseDnMatDescr* table,
                    const mcsparseDnMatDescr* tokens) {
    if ((indices == nullptr && count > 0) || absent(table) || absent(tokens)) return BAD_POINTER;
    if (base != MCSPARSE_INDEX_BASE_ZERO && base != MCSPARSE_INDEX_BASE_ONE) return BAD_VALUE;
    return misaligned(indices, type == MCSPARSE_INDEX_64I ? 8 : 4) ? BAD_VALUE : OK;
}

EmbeddingArgs embedding_args(int64_t count, const void* indices, mcsparseIndexType_t type, mcsparseIndexBase_t base,
                             const mcsparseDnMatDescr* table, const mcsparseDnMatDescr* tokens) {
    EmbeddingArgs a;
    a.count = count, a.rows = table->row_num, a.width = table->col_num;
    a.ids = indices, a.wide_ids = type == MCSPARSE_INDEX_64I, a.base = base == MCSPARSE_INDEX_BASE_ONE ? 1 : 0;
    a.table = table->values, a.ld_table = table->ld, a.table_type = table->valueType;
    a.tokens = tokens->values, a.ld_tokens = tokens->ld, a.token_type = tokens->valueType;
    return a;
}

// ----------------------------------------------------------------------------- attention

// Whether two elements of the tensor may share an address (outputs must not).
bool folded(int64_t tokens, int64_t token_stride, int heads, int64_t head_stride, int dim) {
    if (tokens <= 1 && heads <= 1) return false;
    if (tokens <= 1) return head_stride < dim;
    if (heads <= 1) return token_stride < dim;
    const bool heads_inside = head_stride >= dim && token_stride >= (heads - 1) * head_stride + dim;
    const bool tokens_inside = token_stride >= dim && head_stride / token_stride >= tokens - 1 &&
                               head_stride >= (tokens - 1) * token_stride + dim;
    return !(heads_inside || tokens_inside);
}

// A stride below 2^32 elements times an index below 2^31 stays inside 63 bits.
bool wild_stride(int64_t s) { return s < 0 || (s >> 32) != 0; }

St heads_check(const mcsparseB200Heads_t* t, int64_t tokens, int heads, const mcsparseB200WindowDescr* d, bool output) {
    if (t == nullptr || (t->values == nullptr && tokens > 0)) return BAD_POINTER;
    if (misaligned(t->values, type_bytes(d->valueType))) return BAD_VALUE;
    if (wild_stride(t->tokenStride) || wild_stride(t->headStride)) return BAD_SIZE;
    if (output && folded(tokens, t->tokenStride, heads, t->headStride, d->head_dim)) return BAD_SIZE;
    return OK;
}

AttentionTensor tensor(const mcsparseB200Heads_t* t) {
    AttentionTensor a;
    a.p = t->values, a.token = t->tokenStride, a.head = t->headStride;
    return a;
}

// Token counts stay below 2^30, so that positions, and positions less a window, are int32; a longer window is all of them.
constexpr int64_t kMostTokens = int64_t(1) << 30;
bool too_many(int64_t v) { return v >= kMostTokens; }
int clip(int64_t v) { return (int)(v > kMostTokens ? kMostTokens : v); }

St attention_sizes(mcsparseHandle_t h, const mcsparseB200WindowDescr* d, int64_t batch, int64_t totalQ, int64_t totalK,
                   AttentionArgs* a) {
    if (h == nullptr) return BAD_HANDLE;
    if (d == nullptr) return BAD_POINTER;
    if (batch < 0 || totalQ < 0 || totalK < 0) return BAD_SIZE;
    // blocks of a launch: one per (row tile or row, head)
    if (too_big(batch) || too_many(totalQ) || too_many(totalK) || (totalQ + totalK) / 8 + batch >= (int64_t(1) << 31) / d->q_heads)
        return NOT_IMPL;
    a->batch = (int)batch, a->total_q = (int)totalQ, a->total_k = (int)totalK;
    a->window = clip(d->window), a->sinks = clip(d->sinks);
    a->q_heads = d->q_heads, a->kv_heads = d->kv_heads, a->dim = d->head_dim;
    a->scale = d->scale, a->type = d->valueType;
    a->sm_count = h->sm_count > 0 ? h->sm_count : 148;
    a->wait.limit_cycles = h->wait_cycles;
    a->wait.fault_word = h->attention_fault_dev;
    return OK;
}

St attention_offsets(int64_t batch, const int32_t* q, const int32_t* k, AttentionArgs* a) {
    if ((q == nullptr) != (k == nullptr)) return BAD_POINTER;
    if (q == nullptr && batch > 1) return BAD_POINTER;
    if (misaligned(q, 4) || misaligned(k, 4)) return BAD_VALUE;
    a->q_offsets = q, a->k_offsets = k;
    return OK;
}

St decode_sizes(mcsparseHandle_t h, const mcsparseB200WindowDescr* d, int64_t batch, int64_t maxPages, int64_t pageSize,
                DecodeArgs* a) {
    if (h == nullptr) return BAD_HANDLE;
    if (d == nullptr) return BAD_POINTER;
    if (batch < 0 || maxPages < 0 || pageSize < 1) return BAD_SIZE;
    if (too_big(batch) || too_big(maxPages) || too_big(pageSize) || (maxPages > 0 && pageSize > (kMostTokens - 1) / maxPages) ||
        batch >= (int64_t(1) << 31) / d->q_heads)
        return NOT_IMPL;
    a->batch = (int)batch, a->max_pages = maxPages, a->page_size = pageSize;
    a->window = clip(d->window), a->sinks = clip(d->sinks);
    a->q_heads = d->q_heads, a->kv_heads = d->kv_heads, a->dim = d->head_dim;
    a->scale = d->scale, a->type = d->valueType;
    a->sm_count = h->sm_count > 0 ? h->sm_count : 148;
    return OK;
}

St cache_check(const mcsparseB200Cache_t* c, const mcsparseB200WindowDescr* d, bool any) {
    if (c == nullptr || (c->values == nullptr && any)) return BAD_POINTER;
    if (misaligned(c->values, type_bytes(d->valueType))) return BAD_VALUE;
    return wild_stride(c->pageStride) || wild_stride(c->tokenStride) || wild_stride(c->headStride) ? BAD_SIZE : OK;
}

}  // namespace

extern "C" {

mcsparseStatus_t mcsparseB200EmbeddingLookup(mcsparseHandle_t handle, const void* alpha, int64_t count,
                                             const void* indices, mcsparseIndexType_t indexType,
                                             mcsparseIndexBase_t idxBase, mcsparseDnMatDescr_t matE,
                                             mcsparseDnMatDescr_t matY) {
    St st = embedding_check(handle, count, indexType, matE, matY);
    if (st != OK) return pub(st);
    if (alpha == nullptr) return pub(BAD_POINTER);
    if ((st = embedding_arrays(indices, count, indexType, idxBase, matE, matY)) != OK) return pub(st);
    DeviceGuard guard(handle->device);
    EmbeddingArgs a = embedding_args(count, indices, indexType, idxBase, matE, matY);
    a.alpha = scalar(handle, alpha);
    return pub(from_cuda(embedding_lookup(handle->stream, a)));
}

mcsparseStatus_t mcsparseB200EmbeddingGradient_bufferSize(mcsparseHandle_t handle, int64_t count,
                                                          mcsparseIndexType_t indexType, mcsparseDnMatDescr_t matDY,
                                                          mcsparseDnMatDescr_t matDE, size_t* bufferSize) {
    const St st = embedding_check(handle, count, indexType, matDE, matDY);
    if (st != OK) return pub(st);
    if (bufferSize == nullptr) return pub(BAD_POINTER);
    *bufferSize = embedding_gradient_bytes(count, matDE->row_num, matDE->col_num);
    return MCSPARSE_STATUS_SUCCESS;
}

mcsparseStatus_t mcsparseB200EmbeddingGradient(mcsparseHandle_t handle, const void* alpha, int64_t count,
                                               const void* indices, mcsparseIndexType_t indexType,
                                               mcsparseIndexBase_t idxBase, mcsparseDnMatDescr_t matDY, const void* beta,
                                               mcsparseDnMatDescr_t matDE, void* externalBuffer) {
    St st = embedding_check(handle, count, indexType, matDE, matDY);
    if (st != OK) return pub(st);
    if (alpha == nullptr || beta == nullptr || externalBuffer == nullptr) return pub(BAD_POINTER);
    if ((st = embedding_arrays(indices, count, indexType, idxBase, matDE, matDY)) != OK) return pub(st);
    DeviceGuard guard(handle->device);
    EmbeddingArgs a = embedding_args(count, indices, indexType, idxBase, matDE, matDY);
    a.alpha = scalar(handle, alpha);
    a.beta = scalar(handle, beta);
    if (handle->sm_count > 0) a.sm_count = handle->sm_count;
    return pub(from_cuda(embedding_gradient(handle->stream, a, externalBuffer)));
}

mcsparseStatus_t mcsparseB200CreateWindow(mcsparseB200WindowDescr_t* descr, int64_t window, int64_t sinks, int qHeads,
                                          int kvHeads, int headDim, float scale, macaDataType valueType) {
    if (descr == nullptr) return pub(BAD_POINTER);
    if (window < 1 || sinks < 0 || qHeads < 1 || kvHeads < 1 || qHeads % kvHeads != 0 || headDim < 1) return pub(BAD_SIZE);
    if (!std::isfinite(scale)) return pub(BAD_VALUE);
    if (headDim > 128 || !operator_type(valueType)) return pub(NOT_IMPL);
    mcsparseB200WindowDescr* d = new (std::nothrow) mcsparseB200WindowDescr();
    if (d == nullptr) return MCSPARSE_STATUS_ALLOC_FAILED;
    d->window = window, d->sinks = sinks;
    d->q_heads = qHeads, d->kv_heads = kvHeads, d->head_dim = headDim;
    d->scale = scale, d->valueType = valueType;
    *descr = d;
    return MCSPARSE_STATUS_SUCCESS;
}

mcsparseStatus_t mcsparseB200DestroyWindow(mcsparseB200WindowDescr_t descr) {
    delete descr;
    return MCSPARSE_STATUS_SUCCESS;
}

mcsparseStatus_t mcsparseB200WindowAttention(mcsparseHandle_t handle, mcsparseB200WindowDescr_t descr, int64_t batch,
                                             const int32_t* qOffsets, const int32_t* kOffsets, int64_t totalQ,
                                             int64_t totalK, const mcsparseB200Heads_t* q, const mcsparseB200Heads_t* k,
                                             const mcsparseB200Heads_t* v, const mcsparseB200Heads_t* o, float* lse) {
    AttentionArgs a;
    St st = attention_sizes(handle, descr, batch, totalQ, totalK, &a);
    if (st == OK) st = attention_offsets(batch, qOffsets, kOffsets, &a);
    if (st == OK) st = heads_check(q, totalQ, descr->q_heads, descr, false);
    if (st == OK) st = heads_check(k, totalK, descr->kv_heads, descr, false);
    if (st == OK) st = heads_check(v, totalK, descr->kv_heads, descr, false);
    if (st == OK) st = heads_check(o, totalQ, descr->q_heads, descr, true);
    if (st != OK) return pub(st);
    if (misaligned(lse, 4)) return pub(BAD_VALUE);
    a.q = tensor(q), a.k = tensor(k), a.v = tensor(v), a.o = tensor(o), a.lse = lse;
    if (gave_up(handle)) return pub(EXEC_FAILED);
    DeviceGuard guard(handle->device);
    return pub(from_cuda(window_attention(handle->stream, a)));
}

mcsparseStatus_t mcsparseB200WindowAttentionBackward_bufferSize(mcsparseHandle_t handle, mcsparseB200WindowDescr_t descr,
                                                                int64_t batch, int64_t totalQ, int64_t totalK,
                                                                size_t* bufferSize) {
    AttentionArgs a;
    const St st = attention_sizes(handle, descr, batch, totalQ, totalK, &a);
    if (st != OK) return pub(st);
    if (bufferSize == nullptr) return pub(BAD_POINTER);
    *bufferSize = window_attention_backward_bytes(a);
    return MCSPARSE_STATUS_SUCCESS;
}

mcsparseStatus_t mcsparseB200WindowAttentionBackward(
    mcsparseHandle_t handle, mcsparseB200WindowDescr_t descr, int64_t batch, const int32_t* qOffsets,
    const int32_t* kOffsets, int64_t totalQ, int64_t totalK, const mcsparseB200Heads_t* q, const mcsparseB200Heads_t* k,
    const mcsparseB200Heads_t* v, const mcsparseB200Heads_t* o, const float* lse, const mcsparseB200Heads_t* dO,
    const mcsparseB200Heads_t* dQ, const mcsparseB200Heads_t* dK, const mcsparseB200Heads_t* dV, void* externalBuffer) {
    AttentionArgs a;
    St st = attention_sizes(handle, descr, batch, totalQ, totalK, &a);
    if (st == OK) st = attention_offsets(batch, qOffsets, kOffsets, &a);
    const mcsparseB200Heads_t* const queries[] = {q, o, dO, dQ};
    const mcsparseB200Heads_t* const keys[] = {k, v, dK, dV};
    for (int i = 0; i < 4 && st == OK; ++i) st = heads_check(queries[i], totalQ, descr->q_heads, descr, i == 3);
    for (int i = 0; i < 4 && st == OK; ++i) st = heads_check(keys[i], totalK, descr->kv_heads, descr, i >= 2);
    if (st != OK) return pub(st);
    if ((lse == nullptr && totalQ > 0) || externalBuffer == nullptr) return pub(BAD_POINTER);
    if (misaligned(lse, 4)) return pub(BAD_VALUE);
    a.q = tensor(q), a.k = tensor(k), a.v = tensor(v), a.o = tensor(o), a.lse = const_cast<float*>(lse);
    a.d_o = tensor(dO), a.dq = tensor(dQ), a.dk = tensor(dK), a.dv = tensor(dV);
    if (gave_up(handle)) return pub(EXEC_FAILED);
    DeviceGuard guard(handle->device);
    return pub(from_cuda(window_attention_backward(handle->stream, a, externalBuffer)));
}

mcsparseStatus_t mcsparseB200WindowAttentionDecode_bufferSize(mcsparseHandle_t handle, mcsparseB200WindowDescr_t descr,
                                                              int64_t batch, int64_t maxPages, int64_t pageSize,
                                                              size_t* bufferSize) {
    DecodeArgs a;
    const St st = decode_sizes(handle, descr, batch, maxPages, pageSize, &a);
    if (st != OK) return pub(st);
    if (bufferSize == nullptr) return pub(BAD_POINTER);
    *bufferSize = window_attention_decode_bytes(a);
    return MCSPARSE_STATUS_SUCCESS;
}

mcsparseStatus_t mcsparseB200WindowAttentionDecode(mcsparseHandle_t handle, mcsparseB200WindowDescr_t descr, int64_t batch,
                                                   const int32_t* lengths, const mcsparseB200Heads_t* q,
                                                   const mcsparseB200Cache_t* kCache, const mcsparseB200Cache_t* vCache,
                                                   int64_t numPages, int64_t pageSize, const int32_t* pageTable,
                                                   int64_t maxPages, const mcsparseB200Heads_t* o, float* lse,
                                                   void* externalBuffer) {
    DecodeArgs a;
    St st = decode_sizes(handle, descr, batch, maxPages, pageSize, &a);
    if (st == OK) st = heads_check(q, batch, descr->q_heads, descr, false);
    if (st == OK) st = heads_check(o, batch, descr->q_heads, descr, true);
    if (st == OK) st = cache_check(kCache, descr, numPages > 0);
    if (st == OK) st = cache_check(vCache, descr, numPages > 0);
    if (st != OK) return pub(st);
    if (numPages < 0 || (pageTable == nullptr && maxPages != 1)) return pub(BAD_SIZE);
    if (too_big(numPages)) return pub(NOT_IMPL);
    if ((lengths == nullptr && batch > 0) || externalBuffer == nullptr) return pub(BAD_POINTER);
    if (misaligned(lengths, 4) || misaligned(pageTable, 4) || misaligned(lse, 4)) return pub(BAD_VALUE);
    a.lengths = lengths, a.page_table = pageTable, a.num_pages = numPages;
    a.q = tensor(q), a.o = tensor(o), a.lse = lse;
    a.k.p = kCache->values, a.k.token = kCache->tokenStride, a.k.head = kCache->headStride, a.k_page = kCache->pageStride;
    a.v.p = vCache->values, a.v.token = vCache->tokenStride, a.v.head = vCache->headStride, a.v_page = vCache->pageStride;
    DeviceGuard guard(handle->device);
    return pub(from_cuda(window_attention_decode(handle->stream, a, externalBuffer)));
}

}  // extern "C"
