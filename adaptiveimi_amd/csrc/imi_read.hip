// Cached rows read back from their pages into contiguous rows in bf16 or fp16.
//
// A copy that is bound by memory: D / 8 lanes hold a row, 16 bytes of the
// output each, and a thread has the keys and values of kRows rows under way.
#include <algorithm>

#include "imi_blocks.hpp"

namespace imi {
namespace {

// Rows of a thread.  32768 rows of 8 heads of 128 dims, fp8: 45.2 us with 2 (4.5 TB/s,
// a large copy runs at 4.98), 48 with 4, 51 with 8.
constexpr int kRows = 2;
constexpr int kThreads = 256;

struct ReadParams {
    const uint8_t *k, *v, *ke, *ve;
    uint16_t *ko, *vo;
    const int32_t *table, *lens, *first;
    int64_t table_s, page_s, head_s, row_s;       // in bytes
    int64_t e_page_s, e_head_s, e_row_s;
    int64_t o_ss, o_hs, o_rs;                     // in elements
    int H, n_pages, page_shift, capacity, rows, chunks;
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }

template <bool HALF, int D, typename C>
__global__ __launch_bounds__(kThreads) void read_kernel(ReadParams a) {
    constexpr int L = D / 8, NG = kThreads / L;   // lanes of a row, rows at a time
    const int c = threadIdx.x % L, g = threadIdx.x / L;
    const int chunk = blockIdx.x % a.chunks, h = blockIdx.x / a.chunks % a.H, s = blockIdx.x / a.chunks / a.H;
    const int len = clampi(a.lens[s], 0, a.capacity);
    const int64_t first = a.first ? a.first[s] : 0;
    uint32_t kw[kRows][C::kWords], vw[kRows][C::kWords], kx[kRows], vx[kRows];
    bool live[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const int r = (chunk * kRows + i) * NG + g;
        const int64_t j64 = first + r;
        live[i] = r < a.rows && j64 >= 0 && j64 < len;
        if (!live[i]) continue;
        const int j = static_cast<int>(j64);
        const int page = clampi(a.table ? a.table[s * a.table_s + (j >> a.page_shift)] : s, 0, a.n_pages - 1);
        const uint32_t slot = static_cast<uint32_t>(j) & ((1u << a.page_shift) - 1u);
        const int64_t o = page * a.page_s + slot * a.row_s + h * a.head_s + c * (4 * C::kWords);
        auto load = [](const uint8_t* p, uint32_t (&w)[C::kWords]) {
            if constexpr (C::kWords == 4) {
                const uint4 x = *reinterpret_cast<const uint4*>(p);
                w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
            } else if constexpr (C::kWords == 2) {
                const uint2 x = *reinterpret_cast<const uint2*>(p);
                w[0] = x.x, w[1] = x.y;
            } else {
                w[0] = *reinterpret_cast<const uint32_t*>(p);
            }
        };
        load(a.k + o, kw[i]);
        load(a.v + o, vw[i]);
        if constexpr (C::kBits != 16) {
            const int64_t e = page * a.e_page_s + slot * a.e_row_s + h * a.e_head_s + c / 4;
            kx[i] = a.ke[e];
            vx[i] = a.ve[e];
        }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        if (!live[i]) continue;
        const int r = (chunk * kRows + i) * NG + g;
        const int64_t o = s * a.o_ss + h * a.o_hs + r * a.o_rs + 8 * c;
        blk_u32x4 k, v;
        if constexpr (C::kBits == 16) {
            k = blk_u32x4{kw[i][0], kw[i][1], kw[i][2], kw[i][3]};
            v = blk_u32x4{vw[i][0], vw[i][1], vw[i][2], vw[i][3]};
        } else {
            k = C::template decode<HALF>(kw[i], kx[i]);
            v = C::template decode<HALF>(vw[i], vx[i]);
        }
        *reinterpret_cast<blk_u32x4*>(a.ko + o) = k;
        *reinterpret_cast<blk_u32x4*>(a.vo + o) = v;
    }
}

template <bool HALF, int D>
void launch(const ReadParams& P, int format, unsigned grid, hipStream_t st) {
    switch (format) {
        case IMI_FP8: read_kernel<HALF, D, Fp8><<<grid, kThreads, 0, st>>>(P); break;
        case IMI_INT8: read_kernel<HALF, D, Int8><<<grid, kThreads, 0, st>>>(P); break;
        case IMI_FP4: read_kernel<HALF, D, Fp4><<<grid, kThreads, 0, st>>>(P); break;
        default: read_kernel<false, D, Raw16><<<grid, kThreads, 0, st>>>(P);
    }
}

}  // namespace
}  // namespace imi

extern "C" int imi_read_pages(const imi_read_pages_args* a, imi_stream_t stream) {
    using namespace imi;
    clear_error();
    IMI_REQUIRE(a, IMI_ERR_INVALID, "null argument");
    const imi_paged_batch& b = a->batch;
    IMI_REQUIRE(a->dtype == IMI_BF16 || a->dtype == IMI_FP16, IMI_ERR_UNSUPPORTED, "dtype=%d is not bf16 or fp16",
                a->dtype);
    IMI_REQUIRE(a->dim == 64 || a->dim == 128, IMI_ERR_UNSUPPORTED, "dim=%d is not 64 or 128", a->dim);
    IMI_REQUIRE(a->kv_heads >= 1 && a->kv_heads <= 65535, IMI_ERR_INVALID, "bad heads (kv_heads=%d)", a->kv_heads);
    IMI_REQUIRE(a->rows >= 0 && a->rows <= 1 << 30, IMI_ERR_INVALID, "rows=%d", a->rows);
    imi_paged_batch all = b;   // (the batch's new tokens are not read)
    all.n_tokens = all.max_query = 1;
    if (!all.query_start) all.query_start = all.lens;
    if (const int rc = validate_batch(&all)) return rc;
    if (b.n_seqs == 0 || a->rows == 0) return IMI_OK;
    if (const int rc = validate_format(a->format, a->dim, a->key_exponents, a->value_exponents, a->page_stride,
                                       a->head_stride, a->row_stride, a->exponent_page_stride, a->exponent_head_stride,
                                       a->exponent_row_stride, b.page_size))
        return rc;
    IMI_REQUIRE(a->key_pages && a->value_pages && a->keys && a->values, IMI_ERR_INVALID, "null tensor");
    for (const void* p : {a->key_pages, a->value_pages, static_cast<const void*>(a->keys),
                          static_cast<const void*>(a->values)})
        IMI_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, IMI_ERR_INVALID, "tensors must be 16-byte aligned");
    for (const int64_t s : {a->page_stride, a->head_stride, a->row_stride, a->out_seq_stride, a->out_head_stride,
                            a->out_row_stride})
        IMI_REQUIRE(s >= 0 && s % 8 == 0, IMI_ERR_INVALID, "strides must be multiples of 8 elements (got %lld)",
                    static_cast<long long>(s));
    const int per = kRows * (kThreads / (a->dim / 8));
    const int64_t chunks = (static_cast<int64_t>(a->rows) + per - 1) / per;
    IMI_REQUIRE(chunks * a->kv_heads * b.n_seqs <= (1 << 24) - 1, IMI_ERR_UNSUPPORTED,
                "too many rows for one call (%d sequences of %d rows, %d heads)", b.n_seqs, a->rows, a->kv_heads);
    const int64_t width = a->format == IMI_ROWS ? 2 : 1;
    const ReadParams P{static_cast<const uint8_t*>(a->key_pages), static_cast<const uint8_t*>(a->value_pages),
                       a->key_exponents, a->value_exponents, a->keys, a->values, b.page_table, b.lens, a->first,
                       b.table_stride, a->page_stride * width, a->head_stride * width, a->row_stride * width,
                       a->exponent_page_stride, a->exponent_head_stride, a->exponent_row_stride, a->out_seq_stride,
                       a->out_head_stride, a->out_row_stride, a->kv_heads, b.n_pages,
                       b.page_table ? __builtin_ctz(static_cast<unsigned>(b.page_size)) : 31,
                       static_cast<int>(batch_capacity(&b)), a->rows, static_cast<int>(chunks)};
    const unsigned grid = static_cast<unsigned>(chunks * a->kv_heads * b.n_seqs);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (a->dtype == IMI_BF16) {
        if (a->dim == 128) launch<false, 128>(P, a->format, grid, st);
        else launch<false, 64>(P, a->format, grid, st);
    } else {
        if (a->dim == 128) launch<true, 128>(P, a->format, grid, st);
        else launch<true, 64>(P, a->format, grid, st);
    }
    IMI_LAUNCH_CHECK("read_kernel");
    return IMI_OK;
}
