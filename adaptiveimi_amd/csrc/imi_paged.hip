// Attention over a paged KV cache: checks, entry points, and the kernels for
// rows in bf16 and fp16 (imi_paged.hpp).
#include "imi_paged.hpp"

namespace imi {

int validate_batch(const imi_paged_batch* b) {
    IMI_REQUIRE(b->n_seqs >= 0 && b->n_tokens >= 0, IMI_ERR_INVALID, "negative batch (n_seqs=%d, n_tokens=%d)",
                b->n_seqs, b->n_tokens);
    IMI_REQUIRE(b->n_seqs <= 1 << 30 && b->n_tokens <= 1 << 30, IMI_ERR_UNSUPPORTED,
                "more than 2^30 sequences or tokens (n_seqs=%d, n_tokens=%d)", b->n_seqs, b->n_tokens);
    if (b->n_seqs == 0 || b->n_tokens == 0) return IMI_OK;
    IMI_REQUIRE(b->lens && b->query_start, IMI_ERR_INVALID, "null lens or query_start");
    IMI_REQUIRE(b->max_query >= 1, IMI_ERR_INVALID, "max_query=%d must be >= 1", b->max_query);
    IMI_REQUIRE(b->n_pages >= 1, IMI_ERR_INVALID, "n_pages=%d must be >= 1", b->n_pages);
    IMI_REQUIRE(b->page_size >= 1, IMI_ERR_INVALID, "page_size=%d must be >= 1", b->page_size);
    if (b->page_table) {
        IMI_REQUIRE((b->page_size & (b->page_size - 1)) == 0, IMI_ERR_UNSUPPORTED,
                    "page_size=%d must be a power of two", b->page_size);
        IMI_REQUIRE(b->max_pages >= 0 && b->table_stride >= b->max_pages, IMI_ERR_INVALID,
                    "table_stride=%lld < max_pages=%d", static_cast<long long>(b->table_stride), b->max_pages);
    } else {
        IMI_REQUIRE(b->n_pages >= b->n_seqs, IMI_ERR_INVALID, "n_pages=%d < n_seqs=%d with no page table", b->n_pages,
                    b->n_seqs);
    }
    IMI_REQUIRE(batch_capacity(b) <= int64_t(1) << 30, IMI_ERR_UNSUPPORTED, "more than 2^30 rows in a sequence");
    return IMI_OK;
}

// Rows a sequence can have: what the page table (or the page) holds.
int64_t batch_capacity(const imi_paged_batch* b) {
    return b->page_table ? static_cast<int64_t>(b->max_pages) * b->page_size : b->page_size;
}

// Checks of a pool's format: codes (strides in bytes) and their exponents.
int validate_format(int format, int dim, const void* key_exps, const void* value_exps, int64_t page_s, int64_t head_s,
                    int64_t row_s, int64_t e_page, int64_t e_head, int64_t e_row, int64_t page_size) {
    IMI_REQUIRE(format >= IMI_ROWS && format <= IMI_FP4, IMI_ERR_UNSUPPORTED, "format=%d is not one of the formats",
                format);
    if (format == IMI_ROWS) return IMI_OK;
    const int64_t blocks = dim / kBlock;
    IMI_REQUIRE(key_exps && value_exps, IMI_ERR_INVALID, "null exponents");
    for (const int64_t s : {page_s, head_s, row_s})
        IMI_REQUIRE(s >= 0 && s % 16 == 0, IMI_ERR_INVALID, "strides of codes must be multiples of 16 bytes (got %lld)",
                    static_cast<long long>(s));
    for (const int64_t s : {e_page, e_head, e_row})
        IMI_REQUIRE(s >= 0 && s % blocks == 0, IMI_ERR_INVALID,
                    "strides of exponents must be multiples of %lld bytes (got %lld)", static_cast<long long>(blocks),
                    static_cast<long long>(s));
    for (const void* p : {key_exps, value_exps})
        IMI_REQUIRE(reinterpret_cast<uintptr_t>(p) % blocks == 0, IMI_ERR_INVALID,
                    "exponents must be aligned to %lld bytes", static_cast<long long>(blocks));
    IMI_REQUIRE(e_page <= UINT_MAX && e_row <= UINT_MAX / page_size, IMI_ERR_UNSUPPORTED,
                "a page's exponents span more than 2^32 bytes");
    return IMI_OK;
}

int paged_attention_raw(const imi_paged_attention_args* a, hipStream_t stream) { return run<Raw16>(a, stream); }

namespace {

int validate(const imi_paged_attention_args* a) {
    const imi_paged_batch* const b = &a->batch;
    if (const int rc = validate_batch(b)) return rc;
    IMI_REQUIRE(!b->shared == !b->members && !b->shared == !b->leaders && !b->shared == !b->saved, IMI_ERR_INVALID,
                "shared, members, leaders and saved go together");
    IMI_REQUIRE(b->share_bytes >= 0, IMI_ERR_INVALID, "share_bytes=%lld must be >= 0",
                static_cast<long long>(b->share_bytes));
    IMI_REQUIRE(a->dtype == IMI_BF16 || a->dtype == IMI_FP16, IMI_ERR_UNSUPPORTED, "dtype=%d is not bf16 or fp16",
                a->dtype);
    IMI_REQUIRE(a->dim == 64 || a->dim == 128, IMI_ERR_UNSUPPORTED, "dim=%d is not 64 or 128", a->dim);
    IMI_REQUIRE(a->kv_heads >= 1 && a->groups >= 1 && static_cast<int64_t>(a->kv_heads) * a->groups <= 65535,
                IMI_ERR_INVALID, "bad heads (kv_heads=%d, groups=%d)", a->kv_heads, a->groups);
    IMI_REQUIRE(a->window >= 0 && a->sinks >= 0, IMI_ERR_INVALID, "window=%d and sinks=%d must be >= 0", a->window,
                a->sinks);
    IMI_REQUIRE(a->scale > 0.0f && a->scale <= 1e30f, IMI_ERR_INVALID, "scale=%g must be positive and finite",
                static_cast<double>(a->scale));
    if (a->batch.n_seqs == 0 || a->batch.n_tokens == 0) return IMI_OK;
    IMI_REQUIRE(a->query && a->keys && a->values && a->out, IMI_ERR_INVALID, "null query, keys, values or out");
    const int64_t strides[] = {a->query_token_stride, a->query_head_stride, a->out_token_stride, a->out_head_stride,
                               a->page_stride,        a->head_stride,       a->row_stride};
    for (const int64_t s : strides)
        IMI_REQUIRE(s >= 0 && s % 8 == 0, IMI_ERR_INVALID, "strides must be multiples of 8 elements (got %lld)",
                    static_cast<long long>(s));
    if (const int rc = validate_format(a->format, a->dim, a->key_exponents, a->value_exponents, a->page_stride,
                                       a->head_stride, a->row_stride, a->exponent_page_stride,
                                       a->exponent_head_stride, a->exponent_row_stride, b->page_size))
        return rc;
    const void* ptrs[] = {a->query, a->keys, a->values, a->out};
    for (const void* p : ptrs)
        IMI_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, IMI_ERR_INVALID,
                    "query, keys, values and out must be 16-byte aligned");
    IMI_REQUIRE(a->page_stride <= UINT_MAX && (a->batch.page_size - 1) * a->row_stride <= UINT_MAX, IMI_ERR_UNSUPPORTED,
                "a page spans more than 2^32 elements");
    IMI_REQUIRE(static_cast<int64_t>(a->batch.n_tokens) * a->groups <= (int64_t(1) << 30), IMI_ERR_UNSUPPORTED,
                "more than 2^30 query rows per KV head");
    // the units that are shared out (each at least 128 rows of a sequence), times workgroups, in 64 bits
    const double units = (static_cast<double>(a->batch.n_tokens) * a->groups / kTileRows + a->batch.n_seqs) *
                         (batch_capacity(&a->batch) / 128 + 1) * a->kv_heads;
    IMI_REQUIRE(units <= 1e15, IMI_ERR_UNSUPPORTED, "too much work for one call");
    return IMI_OK;
}

}  // namespace
}  // namespace imi

extern "C" int imi_paged_attention_workspace_size(const imi_paged_attention_args* a, size_t* bytes) {
    using namespace imi;
    clear_error();
    IMI_REQUIRE(a && bytes, IMI_ERR_INVALID, "null argument");
    if (const int rc = validate(a)) return rc;
    *bytes = work_of(a, nullptr).bytes;
    return IMI_OK;
}

extern "C" int imi_paged_attention(const imi_paged_attention_args* a, imi_stream_t stream) {
    using namespace imi;
    clear_error();
    IMI_REQUIRE(a, IMI_ERR_INVALID, "null argument");
    if (const int rc = validate(a)) return rc;
    if (a->batch.n_seqs == 0 || a->batch.n_tokens == 0) return IMI_OK;
    const size_t need = work_of(a, nullptr).bytes;
    IMI_REQUIRE(need == 0 || (a->workspace && a->workspace_bytes >= need), IMI_ERR_WORKSPACE,
                "workspace of %zu bytes, need %zu", a->workspace_bytes, need);
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (a->format) {
        case IMI_FP8: return paged_attention_fp8(a, st);
        case IMI_INT8: return paged_attention_int8(a, st);
        case IMI_FP4: return paged_attention_fp4(a, st);
        default: return paged_attention_raw(a, st);
    }
}
