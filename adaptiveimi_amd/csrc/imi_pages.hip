// Page tables of a paged KV cache: forking and freeing sequences, taking
// pages for new tokens, moving live pages to the lowest ids.
//
// State: pages [S][max_pages] (sequence s holds its first ceil(len / page)
// entries), lens [S], refs [n_pages] = sequences that hold each page; a page
// with refs 0 is free.  Nothing else is kept, so every result is a function of
// these three arrays and no order of threads can change it: free pages are
// taken lowest first, in sequence order, and the only atomics are integer
// additions.
//
// The counting (free pages, pages needed) is one workgroup's pass over refs
// and lens (4 bytes per page, 16 pages per thread at a time: 7 us to extend 32
// sequences, 15 us to compact a pool of 10401 pages, mostly the chain of
// loads and scans).  It stays so at any size, 16384 pages to a turn of about 7 us:
// extend looks no further than the free pages it needs, but in a full pool of
// 100000 pages (one sequence of 128k rows takes 8192 of 16) a call takes 58 us, of
// 10^6 pages 500, and compact, which always looks at all and twice, 105 and 975.
// The table entries and the page copies, which are what moves bytes, are
// spread over the chip (0.67 GB of pages moved in 256 us, 5.3 TB/s both ways).
#include <algorithm>

#include "imi_common.hpp"

namespace imi {
namespace {

typedef __attribute__((ext_vector_type(4))) unsigned int u32x4_t;

constexpr int kThreads = 1024;
constexpr int kMaxPools = 64;    // pools of one launch

struct Pools {
    u32x4_t* base[kMaxPools];
    int64_t stride[kMaxPools];   // 16-byte units from page to page
    int32_t words[kMaxPools];    // 16-byte units of a page
};

struct TableParams {
    int32_t* pages;
    int32_t* lens;
    int32_t* refs;
    int64_t stride;
    int S, cols, P, page;
};

__device__ __forceinline__ int held_of(const TableParams& t, int s) {
    return (min(max(t.lens[s], 0), t.cols * t.page) + t.page - 1) / t.page;
}
__device__ __forceinline__ int entry(const TableParams& t, int s, int c) { return t.pages[s * t.stride + c]; }
__device__ __forceinline__ bool in_pool(const TableParams& t, int p) { return p >= 0 && p < t.P; }

// Inclusive scan of one value per thread of the workgroup, and the total.
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t* s_wave, int64_t& total) {
    const int lane = lane_id(), wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) s_wave[wave] = x;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int w = 0; w < kThreads / 64; ++w) {
        if (w < wave) before += s_wave[w];
        total += s_wave[w];
    }
    return x + before;
}

// ---------------------------------------------------------------- fork ----
__global__ __launch_bounds__(256) void fork_copy_kernel(TableParams in, TableParams out, const int32_t* parents,
                                                        int row_blocks) {
    if (blockIdx.x >= static_cast<unsigned>(row_blocks)) {   // refs
        const int n = gridDim.x - row_blocks;
        for (int p = (blockIdx.x - row_blocks) * 256 + threadIdx.x; p < in.P; p += n * 256) out.refs[p] = in.refs[p];
        return;
    }
    for (int s = blockIdx.x; s < in.S; s += row_blocks) {
        const int from = parents[s];
        const bool alive = from >= 0 && from < in.S;
        const int held = alive ? held_of(in, from) : 0;
        for (int c = threadIdx.x; c < in.cols; c += 256)
            out.pages[s * out.stride + c] = c < held ? entry(in, from, c) : -1;
        if (threadIdx.x == 0) out.lens[s] = alive ? max(in.lens[from], 0) : 0;
    }
}

__global__ __launch_bounds__(256) void fork_refs_kernel(TableParams in, TableParams out, const int32_t* parents) {
    __shared__ int s_n[4];
    for (int s = blockIdx.x; s < in.S; s += gridDim.x) {
        int n = 0;
        for (int x = threadIdx.x; x < in.S; x += 256) n += parents[x] == s;
        n = wave_sum_i(n);
        __syncthreads();
        if (lane_id() == 0) s_n[threadIdx.x >> 6] = n;
        __syncthreads();
        const int more = s_n[0] + s_n[1] + s_n[2] + s_n[3] - 1;   // children instead of the sequence itself
        if (more == 0) continue;
        const int held = held_of(in, s);
        for (int c = threadIdx.x; c < held; c += 256) {
            const int p = entry(in, s, c);
            if (in_pool(in, p)) atomicAdd(&out.refs[p], more);
        }
    }
}

// Both steps in one workgroup, for tables of up to kForkSmall words: a launch
// less (7.4 us on the GPU for 32 sequences of 258 pages, 2.8 + 2.8 and the gap
// in two; fork and extend called in a loop take 27 us together instead of 31).
constexpr int kForkSmall = 32768;

__global__ __launch_bounds__(kThreads) void fork_small_kernel(TableParams in, TableParams out, const int32_t* parents) {
    const int tid = threadIdx.x;
    for (int p = tid; p < in.P; p += kThreads) out.refs[p] = in.refs[p];
    const int waves = kThreads / 64, wave = tid >> 6;
    for (int s = wave; s < in.S; s += waves) {
        const int from = parents[s];
        const bool alive = from >= 0 && from < in.S;
        const int held = alive ? held_of(in, from) : 0;
        for (int c = lane_id(); c < in.cols; c += 64) out.pages[s * out.stride + c] = c < held ? entry(in, from, c) : -1;
        if (lane_id() == 0) out.lens[s] = alive ? max(in.lens[from], 0) : 0;
    }
    __threadfence_block();
    __syncthreads();
    for (int s = wave; s < in.S; s += waves) {
        int n = 0;
        for (int x0 = 0; x0 < in.S; x0 += 64) {
            const int x = x0 + lane_id();
            n += __builtin_popcountll(__ballot(x < in.S && parents[x] == s));
        }
        if (n == 1) continue;
        const int held = held_of(in, s);
        for (int c = lane_id(); c < held; c += 64) {
            const int p = entry(in, s, c);
            if (in_pool(in, p)) atomicAdd(&out.refs[p], n - 1);
        }
    }
}

// -------------------------------------------------------------- extend ----
// What extend_count_kernel leaves for each sequence.
struct Grant {
    int first, n;       // new table entries [first, first + n)
    int at;             // their pages: free list from here on
    int copy;           // page that is copied to the first of them, or -1
};

__global__ __launch_bounds__(kThreads) void extend_count_kernel(TableParams t, const int32_t* counts, Grant* grants,
                                                                int32_t* free_list, uint8_t* granted) {
    __shared__ int64_t s_wave[kThreads / 64];
    const int tid = threadIdx.x;
    // pages that every sequence needs
    int64_t need_all = 0;
    for (int s0 = 0; s0 < t.S; s0 += kThreads) {
        const int s = s0 + tid;
        int need = 0;
        Grant g{0, 0, 0, -1};
        bool fits = true;
        if (s < t.S) {
            const int len = max(t.lens[s], 0), count = max(counts[s], 0);
            const int held = (len + t.page - 1) / t.page;
            const int64_t after = (static_cast<int64_t>(len) + count + t.page - 1) / t.page;
            fits = after <= t.cols;
            if (fits) {
                if (count > 0 && len % t.page != 0) {
                    const int last = entry(t, s, held - 1);
                    if (in_pool(t, last) && t.refs[last] > 1) g.copy = last;
                }
                g.first = held - (g.copy >= 0 ? 1 : 0);
                g.n = need = static_cast<int>(after) - g.first;
            }
        }
        int64_t total;
        const int64_t upto = need_all + block_scan(need, s_wave, total);
        if (s < t.S) {
            // offsets past the pool cannot be granted: kept in 32 bits
            g.at = static_cast<int>(min(upto - need, static_cast<int64_t>(t.P) + 1));
            if (!fits) g.n = -1;
            grants[s] = g;
        }
        need_all += total;
    }
    // that many of the lowest free pages
    int64_t found = 0;
    for (int p0 = 0; p0 < t.P && found < need_all; p0 += kThreads * 16) {
        int32_t r[16];
        const int p = p0 + tid * 16;
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = p + i < t.P ? t.refs[p + i] : 1;
        int n = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) n += r[i] == 0;
        int64_t total;
        int64_t at = found + block_scan(n, s_wave, total) - n;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (r[i] == 0) {
                if (at < need_all) free_list[at] = p + i;
                ++at;
            }
        found += total;
    }
    found = min(found, need_all);
    for (int s = tid; s < t.S; s += kThreads) {   // each thread its own entries of the first loop
        Grant g = grants[s];
        const bool ok = g.n == 0 || (g.n > 0 && static_cast<int64_t>(g.at) + g.n <= found);
        granted[s] = ok;
        if (ok) {
            t.lens[s] = max(t.lens[s], 0) + max(counts[s], 0);
        } else {
            g.n = 0;
            g.copy = -1;
            grants[s] = g;
        }
    }
}

__device__ __forceinline__ void copy_page(const Pools& pools, int i, int from, int to) {
    constexpr int kAhead = 8;   // loads under way per thread: 32 KB per workgroup
    const u32x4_t* src = pools.base[i] + from * pools.stride[i];
    u32x4_t* dst = pools.base[i] + to * pools.stride[i];
    const int n = pools.words[i];
    for (int w = threadIdx.x; w < n; w += 256 * kAhead) {
        u32x4_t x[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (w + 256 * k < n) x[k] = src[w + 256 * k];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (w + 256 * k < n) dst[w + 256 * k] = x[k];
    }
}

// y = 0: table entries and refs; y > 0: the copies of pool y - 1.
__global__ __launch_bounds__(256) void extend_write_kernel(TableParams t, const Grant* grants,
                                                           const int32_t* free_list, Pools pools, bool tables) {
    for (int s = blockIdx.x; s < t.S; s += gridDim.x) {
        const Grant g = grants[s];
        if (blockIdx.y > 0) {
            if (g.copy >= 0) copy_page(pools, blockIdx.y - 1, g.copy, free_list[g.at]);
            continue;
        }
        if (!tables) continue;
        for (int i = threadIdx.x; i < g.n; i += 256) {
            const int p = free_list[g.at + i];
            t.pages[s * t.stride + g.first + i] = p;
            t.refs[p] = 1;
        }
        if (threadIdx.x == 0 && g.copy >= 0) atomicSub(&t.refs[g.copy], 1);
    }
}

// ------------------------------------------------------------- compact ----
__global__ __launch_bounds__(kThreads) void compact_count_kernel(TableParams t, int32_t* from, int32_t* to,
                                                                 int32_t* where, int32_t* info, int32_t* n_live) {
    __shared__ int64_t s_wave[kThreads / 64];
    const int tid = threadIdx.x;
    constexpr int kChunk = kThreads * 16;   // 16 pages per thread
    auto live_of = [&](int p0) {            // bit i: page p0 + 16 tid + i is live
        const int p = p0 + tid * 16;
        int32_t r[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = p + i < t.P ? t.refs[p + i] : 0;
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) m |= (r[i] > 0 ? 1u : 0u) << i;
        return m;
    };
    int64_t live = 0, total;
    int n = 0;
    uint32_t bits = 0;
    for (int p0 = 0; p0 < t.P; p0 += kChunk) {
        bits = live_of(p0);
        n += __builtin_popcount(bits);
    }
    block_scan(n, s_wave, live);
    int64_t holes = 0, movers = 0;
    for (int p0 = 0; p0 < t.P; p0 += kChunk) {
        if (t.P > kChunk) bits = live_of(p0);   // else it is at hand
        const int p = p0 + tid * 16;
        const int below = static_cast<int>(min(max(live - p, static_cast<int64_t>(0)), static_cast<int64_t>(16)));
        const uint32_t low = (1u << below) - 1u;
        const uint32_t mask = (~bits & low) | (bits & ~low);   // holes below the new end, live pages from it on
        const int nh = __builtin_popcount(mask & low), nm = __builtin_popcount(mask) - nh;
        const int64_t both = block_scan((static_cast<int64_t>(nh) << 32) + nm, s_wave, total);
        int64_t h = holes + (both >> 32) - nh, m = movers + (both & 0xFFFFFFFF) - nm;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (p + i < t.P && p + i >= live) where[p + i] = p + i;
            if (mask >> i & 1) {
                if (i < below) to[h++] = p + i;
                else from[m++] = p + i;
            }
        }
        holes += total >> 32;
        movers += total & 0xFFFFFFFF;
    }
    __syncthreads();
    for (int i = tid; i < movers; i += kThreads) {
        const int f = from[i], d = to[i];
        where[f] = d;
        t.refs[d] = t.refs[f];
        t.refs[f] = 0;
    }
    if (tid == 0) {
        info[0] = static_cast<int>(movers);
        info[1] = static_cast<int>(live);
        *n_live = static_cast<int>(live);
    }
}

__global__ __launch_bounds__(256) void compact_move_kernel(TableParams t, const int32_t* from, const int32_t* to,
                                                           const int32_t* where, const int32_t* info, Pools pools,
                                                           bool tables) {
    const int moves = info[0], live = info[1];
    if (blockIdx.y > 0) {
        for (int i = blockIdx.x; i < moves; i += gridDim.x) copy_page(pools, blockIdx.y - 1, from[i], to[i]);
        return;
    }
    if (!tables || moves == 0) return;
    for (int s = blockIdx.x; s < t.S; s += gridDim.x) {
        const int held = held_of(t, s);
        for (int c = threadIdx.x; c < held; c += 256) {
            const int p = entry(t, s, c);
            if (p >= live && p < t.P) t.pages[s * t.stride + c] = where[p];
        }
    }
}

// ---------------------------------------------------------------- host ----
int check_table(const imi_page_table* t, const char* what) {
    IMI_REQUIRE(t->n_seqs >= 0 && t->max_pages >= 0 && t->n_pages >= 0, IMI_ERR_INVALID, "%s: negative size", what);
    IMI_REQUIRE(t->n_pages <= 1 << 30 && t->n_seqs <= 1 << 30, IMI_ERR_UNSUPPORTED,
                "%s: more than 2^30 pages or sequences", what);
    IMI_REQUIRE(t->page_size >= 1, IMI_ERR_INVALID, "%s: page_size=%d must be >= 1", what, t->page_size);
    IMI_REQUIRE(t->stride >= t->max_pages, IMI_ERR_INVALID, "%s: stride=%lld < max_pages=%d", what,
                static_cast<long long>(t->stride), t->max_pages);
    IMI_REQUIRE(t->n_seqs == 0 || (t->lens && (t->pages || t->max_pages == 0)), IMI_ERR_INVALID, "%s: null pointer",
                what);
    IMI_REQUIRE(t->n_pages == 0 || t->refs, IMI_ERR_INVALID, "%s: null refs", what);
    // (a page more than the table holds, for the rounding up to whole pages)
    IMI_REQUIRE((static_cast<int64_t>(t->max_pages) + 1) * t->page_size <= INT_MAX, IMI_ERR_UNSUPPORTED,
                "%s: 2^31 rows or more in a sequence and a page (max_pages=%d, page_size=%d)", what, t->max_pages, t->page_size);
    return IMI_OK;
}

TableParams params(const imi_page_table* t) {
    return TableParams{t->pages, t->lens, t->refs, t->stride, t->n_seqs, t->max_pages, t->n_pages, t->page_size};
}

int check_pools(const imi_page_pool* pools, int32_t n) {
    IMI_REQUIRE(n >= 0 && (n == 0 || pools), IMI_ERR_INVALID, "bad pools (n_pools=%d)", n);
    for (int i = 0; i < n; ++i) {
        IMI_REQUIRE(pools[i].base && reinterpret_cast<uintptr_t>(pools[i].base) % 16 == 0, IMI_ERR_INVALID,
                    "pool %d is null or not 16-byte aligned", i);
        IMI_REQUIRE(pools[i].page_bytes > 0 && pools[i].page_bytes % 16 == 0 && pools[i].page_stride % 16 == 0 &&
                        pools[i].page_stride >= pools[i].page_bytes && pools[i].page_bytes / 16 <= INT_MAX,
                    IMI_ERR_INVALID, "pool %d: page_bytes=%lld and page_stride=%lld must be multiples of 16", i,
                    static_cast<long long>(pools[i].page_bytes), static_cast<long long>(pools[i].page_stride));
    }
    return IMI_OK;
}

Pools take_pools(const imi_page_pool* pools, int n) {
    Pools p{};
    for (int i = 0; i < n; ++i) {
        p.base[i] = static_cast<u32x4_t*>(pools[i].base);
        p.stride[i] = pools[i].page_stride / 16;
        p.words[i] = static_cast<int32_t>(pools[i].page_bytes / 16);
    }
    return p;
}

struct ExtendWork {
    Grant* grants;
    int32_t* free_list;
    size_t bytes;
    ExtendWork(const imi_page_table* t, void* ws) {
        Carver c(ws);
        grants = c.take<Grant>(t->n_seqs);
        free_list = c.take<int32_t>(t->n_pages);
        bytes = c.used();
    }
};

struct CompactWork {
    int32_t *from, *to, *where, *info;
    size_t bytes;
    CompactWork(const imi_page_table* t, void* ws) {
        Carver c(ws);
        from = c.take<int32_t>(t->n_pages);
        to = c.take<int32_t>(t->n_pages);
        where = c.take<int32_t>(t->n_pages);
        info = c.take<int32_t>(2);
        bytes = c.used();
    }
};

}  // namespace
}  // namespace imi

extern "C" int imi_fork_pages(const imi_page_table* in, const int32_t* parents, const imi_page_table* out,
                              imi_stream_t stream) {
    using namespace imi;
    clear_error();
    IMI_REQUIRE(in && out, IMI_ERR_INVALID, "null argument");
    if (const int rc = check_table(in, "in")) return rc;
    if (const int rc = check_table(out, "out")) return rc;
    IMI_REQUIRE(in->n_seqs == out->n_seqs && in->max_pages == out->max_pages && in->n_pages == out->n_pages &&
                    in->page_size == out->page_size,
                IMI_ERR_INVALID, "in and out differ in size");
    IMI_REQUIRE(in->n_seqs == 0 || parents, IMI_ERR_INVALID, "null parents");
    IMI_REQUIRE((in->n_seqs == 0 || (in->lens != out->lens && (in->pages != out->pages || in->max_pages == 0))) &&
                    (in->n_pages == 0 || in->refs != out->refs),
                IMI_ERR_INVALID, "out must not be in");
    if (in->n_seqs == 0 && in->n_pages == 0) return IMI_OK;
    const TableParams I = params(in), O = params(out);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (static_cast<int64_t>(in->n_seqs) * in->max_pages + in->n_pages <= kForkSmall && in->n_seqs <= kThreads) {
        fork_small_kernel<<<1, kThreads, 0, st>>>(I, O, parents);
        IMI_LAUNCH_CHECK("fork_small_kernel");
        return IMI_OK;
    }
    const int rows = std::min(in->n_seqs, 4096), refs = std::min(in->n_pages / 2048 + 1, 1024);
    fork_copy_kernel<<<rows + refs, 256, 0, st>>>(I, O, parents, rows);
    IMI_LAUNCH_CHECK("fork_copy_kernel");
    if (rows) {
        fork_refs_kernel<<<rows, 256, 0, st>>>(I, O, parents);
        IMI_LAUNCH_CHECK("fork_refs_kernel");
    }
    return IMI_OK;
}

extern "C" int imi_extend_pages_workspace_size(const imi_page_table* t, size_t* bytes) {
    using namespace imi;
    clear_error();
    IMI_REQUIRE(t && bytes, IMI_ERR_INVALID, "null argument");
    if (const int rc = check_table(t, "table")) return rc;
    *bytes = ExtendWork(t, nullptr).bytes;
    return IMI_OK;
}

extern "C" int imi_extend_pages(const imi_page_table* t, const int32_t* counts, uint8_t* granted,
                                const imi_page_pool* pools, int32_t n_pools, void* workspace, size_t workspace_bytes,
                                imi_stream_t stream) {
    using namespace imi;
    clear_error();
    IMI_REQUIRE(t, IMI_ERR_INVALID, "null argument");
    if (const int rc = check_table(t, "table")) return rc;
    if (const int rc = check_pools(pools, n_pools)) return rc;
    if (t->n_seqs == 0) return IMI_OK;
    IMI_REQUIRE(counts && granted, IMI_ERR_INVALID, "null counts or granted");
    const ExtendWork w(t, workspace);
    IMI_REQUIRE(workspace && workspace_bytes >= w.bytes, IMI_ERR_WORKSPACE, "workspace of %zu bytes, need %zu",
                workspace_bytes, w.bytes);
    const TableParams T = params(t);
    hipStream_t st = static_cast<hipStream_t>(stream);
    extend_count_kernel<<<1, kThreads, 0, st>>>(T, counts, w.grants, w.free_list, granted);
    IMI_LAUNCH_CHECK("extend_count_kernel");
    for (int at = 0; at == 0 || at < n_pools; at += kMaxPools) {
        const int n = std::min(n_pools - at, kMaxPools);
        extend_write_kernel<<<dim3(std::min(t->n_seqs, 4096), 1 + n), 256, 0, st>>>(
            T, w.grants, w.free_list, take_pools(pools + at, n), at == 0);
        IMI_LAUNCH_CHECK("extend_write_kernel");
    }
    return IMI_OK;
}

extern "C" int imi_compact_pages_workspace_size(const imi_page_table* t, size_t* bytes) {
    using namespace imi;
    clear_error();
    IMI_REQUIRE(t && bytes, IMI_ERR_INVALID, "null argument");
    if (const int rc = check_table(t, "table")) return rc;
    *bytes = CompactWork(t, nullptr).bytes;
    return IMI_OK;
}

extern "C" int imi_compact_pages(const imi_page_table* t, int32_t* n_live, const imi_page_pool* pools,
                                 int32_t n_pools, void* workspace, size_t workspace_bytes, imi_stream_t stream) {
    using namespace imi;
    clear_error();
    IMI_REQUIRE(t, IMI_ERR_INVALID, "null argument");
    if (const int rc = check_table(t, "table")) return rc;
    if (const int rc = check_pools(pools, n_pools)) return rc;
    IMI_REQUIRE(n_live, IMI_ERR_INVALID, "null n_live");
    const CompactWork w(t, workspace);
    IMI_REQUIRE(workspace && workspace_bytes >= w.bytes, IMI_ERR_WORKSPACE, "workspace of %zu bytes, need %zu",
                workspace_bytes, w.bytes);
    const TableParams T = params(t);
    hipStream_t st = static_cast<hipStream_t>(stream);
    compact_count_kernel<<<1, kThreads, 0, st>>>(T, w.from, w.to, w.where, w.info, n_live);
    IMI_LAUNCH_CHECK("compact_count_kernel");
    for (int at = 0; at == 0 || at < n_pools; at += kMaxPools) {
        const int n = std::min(n_pools - at, kMaxPools);
        compact_move_kernel<<<dim3(1024, 1 + n), 256, 0, st>>>(T, w.from, w.to, w.where, w.info,
                                                               take_pools(pools + at, n), at == 0);
        IMI_LAUNCH_CHECK("compact_move_kernel");
    }
    return IMI_OK;
}
