// Which sequences of a batch begin with the same pages.
//
// Pairs first: a workgroup per sequence compares its table with its neighbour's
// (a(s) = equal leading pages of s - 1 and s, at most those before the new
// tokens of either; none where another page follows before kMinShared rows).
// Pages are equal for all of a run where they are for each pair, so a run is a
// stretch of a(s) >= 1 behind its first sequence and shares the smallest of them:
// a wave per run.  Reads each table twice at most; one
// call serves every layer of a step.  64 sequences of 512 common pages: 4.8 us and
// 4.8 us, most of it the chain of loads; the host's call takes 8.6.
#include "imi_common.hpp"

namespace imi {
namespace {

constexpr int kPairThreads = 256;
constexpr int kMinShared = 64;   // fewer common rows are left to each sequence

struct ShareParams {
    const int32_t *table, *lens, *start, *labels;
    int64_t table_s;
    int S, page_size, capacity;
    int32_t *shared, *members, *leaders, *pairs;
    int64_t* saved;
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }

// Full pages before the new tokens of sequence s.
__device__ __forceinline__ int old_pages(const ShareParams& a, int s) {
    const int64_t n = static_cast<int64_t>(a.start[s + 1]) - a.start[s];
    const int64_t old = clampi(a.lens[s], 0, a.capacity) - max(n, static_cast<int64_t>(0));
    return static_cast<int>(max(old, static_cast<int64_t>(0))) / a.page_size;
}

__global__ __launch_bounds__(kPairThreads) void pairs_kernel(ShareParams a) {
    __shared__ int s_first;
    const int s = blockIdx.x;
    if (s == 0 && threadIdx.x == 0) *a.saved = 0;   // for runs_kernel
    int most = s > 0 ? min(old_pages(a, s), old_pages(a, s - 1)) : 0;
    if (s > 0 && a.labels && a.labels[s] != a.labels[s - 1]) most = 0;
    if (threadIdx.x == 0) s_first = most;
    __syncthreads();
    const int32_t* const x = a.table + static_cast<int64_t>(s) * a.table_s;
    const int32_t* const y = x - a.table_s;
    constexpr int kAtOnce = 4;
    for (int c0 = 0; c0 < most; c0 += kAtOnce * kPairThreads) {
        int first = most;
#pragma unroll
        for (int i = kAtOnce - 1; i >= 0; --i) {
            const int c = c0 + i * kPairThreads + static_cast<int>(threadIdx.x);
            if (c < most && x[c] != y[c]) first = c;
        }
        if (first < most) atomicMin(&s_first, first);
        __syncthreads();
        const bool found = s_first < most;
        __syncthreads();
        if (found) break;
    }
    // tables that part within kMinShared rows part the runs: chained, the pair would
    // leave those on either side of it nothing to share
    if (threadIdx.x == 0) a.pairs[s] = s_first < most && s_first * a.page_size < kMinShared ? 0 : s_first;
}

__global__ __launch_bounds__(64) void runs_kernel(ShareParams a) {
    const int s = blockIdx.x;
    if (a.pairs[s] > 0) return;   // its run's first sequence writes for it
    const int lane = threadIdx.x;
    int end = s + 1, least = INT_MAX;
    for (; end < a.S; end += 64) {
        const int t = end + lane;
        const int p = t < a.S ? a.pairs[t] : 0;
        const uint64_t out = __ballot(p <= 0);
        const int n = out ? __builtin_ctzll(out) : 64;
        int m = lane < n ? p : INT_MAX;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = min(m, __shfl_xor(m, o));
        least = min(least, m);
        if (n < 64) {
            end += n;
            break;
        }
    }
    end = min(end, a.S);
    int rows = end - s > 1 ? (least * a.page_size) & ~7 : 0;   // (least pages lie within the table)
    if (rows < kMinShared) rows = 0;
    if (lane == 0 && rows > 0)   // (whole numbers: in any order)
        atomicAdd(reinterpret_cast<unsigned long long*>(a.saved),
                  static_cast<unsigned long long>(end - s - 1) * static_cast<unsigned long long>(rows));
    for (int t = s + lane; t < end; t += 64) {
        a.shared[t] = rows;
        a.members[t] = t == s && rows > 0 ? end - s : 0;
        a.leaders[t] = rows > 0 ? s : t;
    }
}

int validate(const imi_paged_batch* b) {
    imi_paged_batch all = *b;   // pools and query rows are not read
    all.n_tokens = all.max_query = all.n_pages = 1;
    if (const int rc = validate_batch(&all)) return rc;
    IMI_REQUIRE(b->n_seqs == 0 || b->page_table, IMI_ERR_INVALID, "sequences without a page table share no pages");
    return IMI_OK;
}

}  // namespace
}  // namespace imi

extern "C" int imi_share_prefixes_workspace_size(const imi_paged_batch* b, size_t* bytes) {
    using namespace imi;
    clear_error();
    IMI_REQUIRE(b && bytes, IMI_ERR_INVALID, "null argument");
    if (const int rc = validate(b)) return rc;
    *bytes = static_cast<size_t>(b->n_seqs) * sizeof(int32_t);
    return IMI_OK;
}

extern "C" int imi_share_prefixes(const imi_paged_batch* b, const int32_t* labels, int32_t* shared, int32_t* members,
                                  int32_t* leaders, int64_t* saved, void* workspace, size_t workspace_bytes,
                                  imi_stream_t stream) {
    using namespace imi;
    clear_error();
    IMI_REQUIRE(b, IMI_ERR_INVALID, "null argument");
    if (const int rc = validate(b)) return rc;
    if (b->n_seqs == 0) return IMI_OK;
    IMI_REQUIRE(shared && members && leaders && saved, IMI_ERR_INVALID, "null shared, members, leaders or saved");
    const size_t need = static_cast<size_t>(b->n_seqs) * sizeof(int32_t);
    IMI_REQUIRE(workspace && workspace_bytes >= need, IMI_ERR_WORKSPACE, "workspace of %zu bytes, need %zu",
                workspace_bytes, need);
    const ShareParams P{b->page_table, b->lens, b->query_start, labels, b->table_stride, b->n_seqs,
                        b->page_size, static_cast<int>(batch_capacity(b)), shared, members, leaders,
                        static_cast<int32_t*>(workspace), saved};
    hipStream_t st = static_cast<hipStream_t>(stream);
    pairs_kernel<<<P.S, kPairThreads, 0, st>>>(P);
    IMI_LAUNCH_CHECK("pairs_kernel");
    runs_kernel<<<P.S, 64, 0, st>>>(P);
    IMI_LAUNCH_CHECK("runs_kernel");
    return IMI_OK;
}
