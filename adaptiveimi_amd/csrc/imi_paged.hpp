// Attention of a batch of new tokens over a paged KV cache on gfx950.
//
// Sequence s has len rows, of which the last n = start[s + 1] - start[s] are
// new; its new token i stands at position p = len - n + i and sees the rows
//   V(p) = { j : 0 <= j <= p, and j > p - window or j < sinks }
// (window 0: no limit).  For query head x of KV head h = x / G:
//   out = sum_{j in V} w_j v_j,  w = softmax over V of scale * q . k_j,
//   lse = ln sum_{j in V} exp(scale * q . k_j);  V empty: out 0, lse -inf.
//
// The G query heads of a KV head and the new tokens of a sequence form the
// rows r = i * G + g of one problem.  Both kernels compute the transposed
// scores S^T = K Q^T, so that a lane holds one query row (a column of S^T):
// the running maximum, the sum and the rescaling of that row need no lane
// exchange but the last steps of the maximum, and P^T in the registers of S^T
// is the second operand of O^T += V^T P^T as it stands: the keys of a matrix
// instruction are summed over, so their order is free, and V^T is read from
// LDS in the order that the registers of S^T have (by ds_read_b64_tr_b16 in
// the few-row kernel, transposed on its way there in the tile kernel).
//
// The rows that a tile of new tokens sees are numbered without gaps: the
// first min(sinks, lo) rows, then lo .. hi - 1, lo being the first row inside
// the window of the tile's first token.
//
// Softmax statistics and sums are fp32 in base 2; P is rounded to the cache's
// type for the matrix instruction, unnormalised (half a step of that type
// relative to each weight, the rounding that the output itself takes: bf16
// outputs are 2.0e-3 off where an fp32 P leaves 1.7e-3, and P in two halves
// would take the matrix instructions of the second product twice).  The running
// maximum moves only when it grows by more than kSlack in base 2, which leaves
// the sums exact to fp32 and saves most rescalings; a row's largest weight lies
// in 2^kShift .. 2^(kShift + kSlack).  bf16 has fp32's range (shift 0, slack 8).
// fp16 has steps of 2^-24 under 2^-14, so its weights use the range up to 2^15
// (shift 11, slack 4): one under 2^-25 of the largest is off by at most 2^-36 of
// it, and 131072 rows of such weights, which one row outweighs, by 2^-19 in all
// (unshifted they would be lost: 2^-25 of it each, 2^-8 in all).  Either way 8192
// fp16 tokens over 32768 rows take 3.91-4.0 ms.
//
// Rows may be held as codes of 8 or 4 bits (C, imi_blocks.hpp).  They become bf16
// or fp16 in registers, which rounds nothing in bf16, on the way to the matrix
// instruction (K of the few-row kernel) or to LDS (all others), and from there on
// both kernels are the same: the masks, the statistics and the look for infinities
// and NaN see values, and no scale enters a score or a weight.
#pragma once

#include <algorithm>

#include "imi_blocks.hpp"

namespace imi {

// The formats of the pools, a source each (every one holds many kernels).
int paged_attention_raw(const imi_paged_attention_args* a, hipStream_t stream);
int paged_attention_fp8(const imi_paged_attention_args* a, hipStream_t stream);
int paged_attention_int8(const imi_paged_attention_args* a, hipStream_t stream);
int paged_attention_fp4(const imi_paged_attention_args* a, hipStream_t stream);

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;
typedef __attribute__((ext_vector_type(8))) short s16x8_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;
typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(4))) unsigned int u32x4_t;
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// A weight is 2^(s c - m c) in one fma, whose m c is rounded: a common factor of
// the weights of one maximum, of up to half a step of m c in base 2.  Past 2^12
// (a factor of 1 + 2^-13) the maximum is subtracted from the scores instead, which
// is exact next to it: from 2^24 on the factor could leave fp16's range, from 2^31
// on fp32's (keys padded with the type's lowest value have such scores), and
// before that it differs between the maxima that are joined.
constexpr float kFar = 4096.0f;

// The two element types: pairs rounded to nearest even, matrix instructions;
// kShift: base 2 exponent of the weight of a row at the running maximum, kSlack:
// growth of a running maximum (base 2) that is left unapplied.
struct BF16 {
    typedef bf16x8_t v8;
    static constexpr bool kHalf = false;
    static constexpr uint32_t kExp = 0x7F80;
    static constexpr float kShift = 0.0f, kSlack = 8.0f;
    static __device__ __forceinline__ float wide(uint32_t h) { return __uint_as_float(h << 16); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        typedef __attribute__((ext_vector_type(2))) float f2;
        typedef __attribute__((ext_vector_type(2))) __bf16 b2;
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), b2));
    }
    static __device__ __forceinline__ f32x4_t mma16(u32x4_t a, u32x4_t b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16_t mma32(u32x4_t a, u32x4_t b, f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
};
struct FP16 {
    typedef f16x8_t v8;
    static constexpr bool kHalf = true;
    static constexpr uint32_t kExp = 0x7C00;
    static constexpr float kShift = 11.0f, kSlack = 4.0f;
    static __device__ __forceinline__ float wide(uint32_t h) {
        return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        typedef __attribute__((ext_vector_type(2))) _Float16 h2;
        return __builtin_bit_cast(uint32_t, (h2{static_cast<_Float16>(a), static_cast<_Float16>(b)}));
    }
    static __device__ __forceinline__ f32x4_t mma16(u32x4_t a, u32x4_t b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16_t mma32(u32x4_t a, u32x4_t b, f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
};

// LDS row of D elements plus a pad: eight rows' 16-byte pieces (the K reads)
// and four rows' 32-byte pieces (the transposed V reads) fall on different
// banks.
template <int D>
constexpr int kRow = D == 128 ? 144 : 72;

struct Join;

// Threads of the kernels that attend (a constant, as all sizes of launches: a kernel
// that asks for them has 256 bytes of arguments more).
constexpr int kThreads = 512;

struct BaseParams {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* out;
    float* lse;                // or null
    const int32_t* table;      // or null: sequence s's rows are "page" s
    const int32_t* lens;
    const int32_t* start;
    int64_t q_ts, q_hs;        // strides in elements: token, head
    int64_t o_ts, o_hs;
    int64_t l_ts;              // lse token stride (heads are adjacent)
    int64_t head_s;
    uint32_t page_s, tok_s;    // from page to page, from row to row
    int64_t table_s;
    int S, N, H, G;
    int n_pages;               // pages in the pool
    int page_shift;            // 31 with no table
    int capacity;              // rows a sequence can have
    int window, sinks;
    float c;                   // scale * log2(e)
    int min_rows, max_rows;    // rows (n * G) of the sequences this launch takes
    int w_log;                 // 2^w_log workgroups share the work
    Join* joins;        // [W]
    float* part;               // [2 W][cap][D]
    float* part_ml;            // [2 W][cap][2]
    int cap;                   // rows of a partial
    int32_t* plan;             // tile kernel: see plan_kernel
    int slots;                 // tile kernel: tiles that the plan can hold
};
struct ExpParams {   // codes (strides above in bytes then): exponents of their blocks
    const uint8_t *ke, *ve;
    int64_t e_head_s;
    uint32_t e_page_s, e_tok_s;
};
struct SharedParams {   // shared first rows (see Seq)
    const int32_t* shared;     // [S] rows
    const int32_t* members;    // [S] sequences of the run that s leads, or 0
    const int64_t* saved;      // rows that sharing saves, and how many it has to
    int64_t least_saved;
    bool common;               // the shared rows are attended, not the others
    float* keep;               // [N][H G][D] rows that one range attended whole, before the division,
    float* keep_ml;            // [N][H G][2] their maxima and sums
    int32_t* place;            // [keys][H] where a tile's rows are: see place_key
};
// A kernel's arguments are those that it reads.
template <int>
struct NoParams {};
template <typename C, bool SH>
struct PagedParams : BaseParams,
                     std::conditional_t<C::kBits != 16, ExpParams, NoParams<0>>,
                     std::conditional_t<SH, SharedParams, NoParams<1>> {};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }

// New tokens [t0, t0 + n), length, position of the first new token and first
// row to attend of sequence s, forced into the tensors.
//
// With shared first rows (SH) a call attends two kinds of problem: of each run
// of sequences that begin with the same pages, the rows that all of them share,
// by the tokens of all (common: led by the run's first sequence, and all tokens
// see all rows, p0 being their end); and of each sequence its rows from `lo` on.
// What either gives a query row is joined afterwards (join_kernel).
struct Seq {
    int t0, n, len, p0, lo;
};
template <bool SH, typename P>
__device__ __forceinline__ Seq seq_of(const P& a, int s) {
    const int b = clampi(a.start[s], 0, a.N);
    if constexpr (SH) {
        const int rows = *a.saved >= a.least_saved ? clampi(a.shared[s], 0, a.capacity) : 0;
        if (a.common) {
            const int m = clampi(a.members[s], 0, a.S - s);
            const int e = m > 1 && rows > 0 ? clampi(a.start[s + m], 0, a.N) : b;
            return Seq{b, max(e - b, 0), rows, rows, 0};
        }
        const int e = clampi(a.start[s + 1], 0, a.N), n = max(e - b, 0), len = clampi(a.lens[s], 0, a.capacity);
        return Seq{b, n, len, len - n, clampi(rows, 0, max(len - n, 0)) & ~7};
    } else {
        const int e = clampi(a.start[s + 1], 0, a.N), n = max(e - b, 0), len = clampi(a.lens[s], 0, a.capacity);
        return Seq{b, n, len, len - n, 0};
    }
}

// Rows visible to the new tokens at positions p0 .. p1: [0, sink) and [lo, hi).
struct Span {
    int lo, hi, sink;
    __device__ __forceinline__ int count() const { return sink + hi - lo; }
    __device__ __forceinline__ int row(int v) const { return v < sink ? v : v - sink + lo; }
};
__device__ __forceinline__ Span span_of(const BaseParams& a, const Seq& q, int p0, int p1) {
    Span r;
    r.hi = clampi(p1 + 1, 0, q.len);
    r.lo = a.window > 0 ? clampi(p0 - a.window + 1, 0, r.hi) : q.lo;   // (not both)
    r.sink = min(a.sinks, r.lo);
    return r;
}

// The rows of a span (row v is cached row v up to the sinks, v + shift from
// there on) that a token at position pos (-1: none) sees: v <= last, and from
// `from` on or under `sinks`.
struct Sees {
    int last, from, sinks;
    __device__ __forceinline__ Sees(const BaseParams& a, int pos, int shift, int sink, int vis)
        : last(min(pos - shift, vis - 1)),
          from(a.window > 0 ? pos - a.window + 1 - shift : 0),
          sinks(shift ? sink : a.sinks) {}
    __device__ __forceinline__ bool row(int k, int base) const {   // v = base + k
        return (k <= last - base) & ((k >= from - base) | (k < sinks - base));
    }
};

// Whether the rows of a problem are kept for the join, where a range holds them whole.
template <bool SH, typename P>
__device__ __forceinline__ bool keeps(const P& a, const Seq& q) {
    if constexpr (SH) return a.common || q.lo > 0;
    else return false;
}

// Element offset of cached row j of sequence s (head offset not included).
// A page id outside the pool is forced into it.
__device__ __forceinline__ int page_of(const BaseParams& a, int s, int j) {
    return a.table ? a.table[static_cast<int64_t>(s) * a.table_s + (j >> a.page_shift)] : s;
}
__device__ __forceinline__ int64_t row_offset(const BaseParams& a, int page, int j) {
    const uint32_t slot = static_cast<uint32_t>(j) & ((1u << a.page_shift) - 1u);
    return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(clampi(page, 0, a.n_pages - 1))) * a.page_s +
                                slot * a.tok_s);
}
// Of the exponents of cached row j.
template <typename P>
__device__ __forceinline__ int64_t exp_offset(const P& a, int page, int j) {
    const uint32_t slot = static_cast<uint32_t>(j) & ((1u << a.page_shift) - 1u);
    const uint64_t id = static_cast<uint32_t>(clampi(page, 0, a.n_pages - 1));
    return static_cast<int64_t>(id * a.e_page_s + slot * a.e_tok_s);
}

__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The loads into LDS that this wave has under way are done.  The compiler
// counts only those whose result it sees in a register.
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ u32x4_t load16(const uint16_t* p) { return *reinterpret_cast<const u32x4_t*>(p); }

// N words at p (aligned to 16 bytes, or to all of them where they are fewer)
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
    if constexpr (N >= 4) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const u32x4_t x = reinterpret_cast<const u32x4_t*>(p)[i];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[4 * i + k] = x[k];
        }
    } else if constexpr (N == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        w[0] = x.x;
        w[1] = x.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}
// codes 8 i .. of some words as 8 bf16 or fp16
template <typename T, typename C, int N>
__device__ __forceinline__ u32x4_t decode8(const uint32_t (&w)[N], int i, uint32_t e) {
    uint32_t x[C::kWords];
#pragma unroll
    for (int k = 0; k < C::kWords; ++k) x[k] = w[C::kWords * i + k];
    return C::template decode<T::kHalf>(x, e);
}

__device__ __forceinline__ s16x4_t read_tr(const uint16_t* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(p));
}
__device__ __forceinline__ u32x4_t join(s16x4_t a, s16x4_t b) {
    return __builtin_bit_cast(u32x4_t, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// A row of V that only some of a workgroup's tokens see meets the others with
// weight 0 in the matrix instruction, and 0 times an infinity or a NaN would
// reach them.  Where rows are masked in part such values are looked for and
// replaced by 0; a workgroup that found one adds it, after its rows are
// written, to those that see it (patch_rows: slow, for data that is broken).
template <typename T>
__device__ __forceinline__ uint32_t finite_halves(uint32_t x) {   // 0xFFFF per finite half
    return ((x & T::kExp) == T::kExp ? 0u : 0xFFFFu) | (((x >> 16) & T::kExp) == T::kExp ? 0u : 0xFFFF0000u);
}
template <typename T, int N>
__device__ __forceinline__ bool all_finite(const u32x4_t (&x)[N]) {
    uint32_t m = ~0u;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) m &= finite_halves<T>(x[i][k]);
    return m == ~0u;
}
template <typename T, int N>
__device__ __forceinline__ void keep_finite(u32x4_t (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) x[i][k] &= finite_halves<T>(x[i][k]);
}

// Rows [first, end) of one (sequence s, KV head h): adds the infinities and NaN
// of the span's rows [v0, v1) that each sees, to the output (slot < 0) or to
// the partial.  The workgroup's own writes of these rows are done.
template <typename T, int D, typename C, bool SH, typename SpanT>
__device__ __forceinline__ void patch_rows(const PagedParams<C, SH>& a, const Seq& sq, int s, int h, const SpanT& sp,
                                           int first, int end, int v0, int v1, int64_t slot) {
    for (int x = threadIdx.x; x < (end - first) * (D / 2); x += kThreads) {
        const int r = first + x / (D / 2), d = 2 * (x % (D / 2));
        const int p = sq.p0 + r / a.G;
        float add[2] = {0.0f, 0.0f};
        for (int v = v0; v < v1; ++v) {
            const int j = sp.row(v);
            if (j > p || (a.window > 0 && j <= p - a.window && j >= a.sinks)) continue;
            const int page = page_of(a, s, j);
            uint32_t w;
            if constexpr (C::kBits == 16) {
                w = *reinterpret_cast<const uint32_t*>(a.v + row_offset(a, page, j) +
                                                       static_cast<int64_t>(h) * a.head_s + d);
            } else {
                const uint8_t* const row =
                    reinterpret_cast<const uint8_t*>(a.v) + row_offset(a, page, j) + static_cast<int64_t>(h) * a.head_s;
                uint32_t codes[C::kWords] = {};   // the two that count, first
                codes[0] = C::kBits == 8 ? *reinterpret_cast<const uint16_t*>(row + d) : row[d / 2];
                w = C::template decode<T::kHalf>(
                    codes, a.ve[exp_offset(a, page, j) + static_cast<int64_t>(h) * a.e_head_s + d / kBlock])[0];
            }
            const uint32_t m = finite_halves<T>(w);
            if (!(m & 0xFFFFu)) add[0] += T::wide(w & 0xFFFFu);
            if (!(m >> 16)) add[1] += T::wide(w >> 16);
        }
        if (add[0] == 0.0f && add[1] == 0.0f) continue;
        if (slot >= 0 || keeps<SH>(a, sq)) {
            float* o = a.part + (slot * a.cap + r - first) * D + d;
            if constexpr (SH)
                if (slot < 0)
                    o = a.keep + (static_cast<int64_t>(sq.t0 + r / a.G) * (a.H * a.G) + h * a.G + r % a.G) * D + d;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                o[i] = __hip_atomic_load(o + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + add[i];
        } else {
            uint32_t* const o = reinterpret_cast<uint32_t*>(a.out + static_cast<int64_t>(sq.t0 + r / a.G) * a.o_ts +
                                                            static_cast<int64_t>(h * a.G + r % a.G) * a.o_hs + d);
            const uint32_t w = __hip_atomic_load(o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            *o = T::pack(T::wide(w & 0xFFFFu) + add[0], T::wide(w >> 16) + add[1]);
        }
    }
}

__device__ __forceinline__ float exp2_weight(float m, float M, float c) {
    return m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - M) * c);
}

constexpr int kTileRows = 256;   // rows of a tile of the tile kernel

// Where the rows of a problem (r0 ..: its first row, or of a tile) are with
// shared rows, for each head: -1, in `keep`, or the range that holds its first
// unit, in that range's partials and those after it.  Problems begin at query
// rows t0 G in the order of s, so no two tiles have the same key.
__device__ __forceinline__ int place_key(const BaseParams& a, int t0, int s, int r0) {
    return static_cast<int>((static_cast<int64_t>(t0) * a.G + r0) / kTileRows) + s;
}

// What a row's sum L of weights divides by: nothing for a row that sees nothing
// (blind: 0), and 1 / 0 where all that it sees has a score of -infinity, which
// makes NaN of its zeros, as 0 / 0 is and as for a NaN among the scores.
__device__ __forceinline__ float inverse(float L, bool blind) { return blind ? 0.0f : 1.0f / L; }

// ln sum exp of a row: maximum M, sum L of its weights.
template <typename T>
__device__ __forceinline__ float log_sum(float M, float L, float c) {
    return L == 0.0f ? -INFINITY : M * (c * kLn2) + (__log2f(L) - T::kShift) * kLn2;   // (M c may be past fp32)
}

// ---------------------------------------------------------- few rows ------
// Sequences of at most 16 NB rows (decode, verification of a few tokens):
// the rows fit one matrix tile, so K and V are streamed once and the kernel
// is bound by that stream.  Work is counted in units of UNIT cached rows of
// one (sequence, KV head); the units of all, in order, are cut into W equal
// ranges, one per workgroup, whatever the lengths (each workgroup adds the
// lengths up itself: no host knows them).  A workgroup whose range covers a
// whole (sequence, head) writes its output; the others (its first and its
// last at most) write a partial that merge_kernel joins.
//
// A wave's 32 rows of the next unit are loaded while it computes on this one's:
// 128 KB per CU under way (64 for 64 dims; twice the rows there, two
// workgroups per CU, or loads two units ahead were no faster).  K is loaded as
// the matrix instruction wants it, 64 bytes of 16 rows at a time; V goes through
// LDS and is loaded in whole rows, which the cache serves faster (768 rows in a
// workgroup 16.0 -> 14.1 us; K in the same way 12.0, but then the long streams
// lose 3 percent to LDS).  One token over 131072 rows of 8 heads of 128: 94 us,
// 5.7 TB/s (a large copy runs at 4.84); 64 dims, 4 x 30000 rows: 44 us with its
// join.
//
// Of codes there are half or a quarter of the bytes under way, and the same number
// of rows, so the work on a row tells: over 131072 rows of 8 heads of 128 fp8 takes
// 56 us (5.0 TB/s), int8, whose codes take five instructions a pair where the others
// take one, 59-67, fp4 36 (4.0 TB/s).  In a ragged int8 batch vector instructions hold
// half of the issue slots.  Two workgroups per CU (128 registers, spilled) took 88
// us for the 61 with its join in fp8; with 64 dims, where they fit, 41 for 37.
constexpr int kFewWaves = kThreads / 64;
// Rows of K / V per wave and step: 32, or 64 of 64 dims in 4 bits, which then
// have as many bytes under way as others (3 tokens each of 12 sequences over 4000 ..
// 60000 rows, 8 heads: 46 us instead of 54, one over 131072 28.6 instead of 29.9).
// At 64 bytes a row the larger step is no better (one token each of 40 sequences
// over 300 .. 40000, 4 heads: 75 us instead of 71 in 4 bits, 71 instead of 67 in 8
// of 64 dims), at 128 worse.
template <int BITS, int D>
constexpr int kFewTile = D * BITS <= 8 * 32 ? 64 : 32;

// How both kernels cut their work: range w of 2^log is the units
// [cut(w), cut(w + 1)), with a range per workgroup, or for little work about
// as many ranges as units (at most half of them empty: merge_kernel visits
// every range of a tile).  What one range holds of a (sequence, head) or tile
// with units [lo, hi) that it does not hold whole goes to a partial: 2 w for
// the first that the range meets, 2 w + 1 for the last.  The range that holds
// unit lo leaves a Join where hi lies past its end, and merge_kernel joins the
// partials of the ranges from there on, in order.
//
// To begin and to end a (sequence, head) costs about as much time as two units
// of codes (6 us: lookups, queries, first loads, the join of the waves), so
// FewLoads::kLead units that hold no rows come before each in the count, and a
// range that holds none but these has no part in it.  One token each of 40
// sequences over 300 .. 40000 rows, 4 heads of 128 dims: int8 107 -> 82 us, fp8 98
// -> 85, fp4 88 -> 72 (1: 91, 87, 78; 4: 85, 87, 73).
struct Join {
    int64_t total;      // units in all
    int64_t lo, hi;     // lo = hi: nothing to join
    int t0;             // the sequence's first query row
    int first, end;     // rows (token, head of the group) [first, end)
    int h;
    int blind;          // the sequence's rows before this one see nothing (more new tokens than rows)
};
__device__ __forceinline__ int ranges_log(int w_log, int64_t total) {
    return total <= 1 ? 0 : min(w_log, 64 - __builtin_clzll(static_cast<uint64_t>(total - 1)));
}
__device__ __forceinline__ int64_t cut(int64_t total, int64_t w, int log) { return (total * w) >> log; }

template <int UNIT, int LEAD>
__device__ __forceinline__ int few_units(const BaseParams& a, const Seq& q) {
    const int rows = q.n * a.G;
    if (q.n <= 0 || rows < a.min_rows || rows > a.max_rows) return 0;
    const Span sp = span_of(a, q, max(q.p0, 0), q.len - 1);
    return max((sp.count() + UNIT - 1) / UNIT, 1) + LEAD;
}

// a / b, fast where it fits 32 bits
__device__ __forceinline__ int quotient(int64_t a, int b) {
    return a <= UINT_MAX ? static_cast<int>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b))
                         : static_cast<int>(a / b);
}

// This workgroup's range of the units of all sequences, the sequence in which
// it begins and the units (of one KV head) before that sequence.
struct FewRange {
    int64_t total, g0, g1, before;
    int s;
};
template <bool SH, int UNIT, int LEAD, typename P>
__device__ __forceinline__ FewRange few_range(const P& a, int block) {
    FewRange r{0, 0, 0, 0, 0};
    int u = 0, incl = 0;
    for (int s0 = 0; s0 < a.S; s0 += 64) {
        const int s = s0 + lane_id();
        u = s < a.S ? few_units<UNIT, LEAD>(a, seq_of<SH>(a, s)) : 0;
        incl = wave_incl_scan(u);
        r.total += __builtin_amdgcn_readlane(incl, 63);
    }
    r.total *= a.H;
    const int log = ranges_log(a.w_log, r.total);
    if (block >> log) return r;
    r.g0 = cut(r.total, block, log);
    r.g1 = cut(r.total, block + 1, log);
    if (r.g0 >= r.g1) return r;
    for (int s0 = 0; s0 < a.S; s0 += 64) {
        if (a.S > 64) {   // else the only 64 are still at hand
            const int s = s0 + lane_id();
            u = s < a.S ? few_units<UNIT, LEAD>(a, seq_of<SH>(a, s)) : 0;
            incl = wave_incl_scan(u);
        }
        const uint64_t past = __ballot((r.before + incl) * a.H > r.g0);
        if (past) {
            const int l = __builtin_ctzll(past);
            r.s = s0 + l;
            r.before += __builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(u, l);
            return r;
        }
        r.before += __builtin_amdgcn_readlane(incl, 63);
    }
    return r;
}

// Codes (C): a lane loads D / 4 of a K row's dims for the matrix instruction,
// in pieces of up to 16 bytes; which of them an instruction takes is free, as
// long as the queries come in the same order (frag_dim).  They become bf16 or
// fp16 in registers, those of V on the way to LDS.  A row's place and exponents
// are looked up by one lane and go to the others by lane exchange: a load for each
// piece (a byte) and 64-bit addresses in every lane cost 45 registers more.
template <typename C, int D>
struct FewLoads {
    static constexpr int kWords = C::kBits == 16 ? 4 : D * C::kBits / 128;       // a lane's words of a K row
    static constexpr int kPiece = (kWords < 4 ? kWords : 4) * 32 / C::kBits;     // dims of a piece
    static constexpr int kFrags = kPiece / 8;                                    // matrix instructions of a piece
    static constexpr int CH = D * C::kBits / 128;                                // 16-byte pieces of a V row
    static constexpr int kTile = kFewTile<C::kBits, D>;
    static constexpr int kLead = C::kBits == 16 ? 0 : 2;
    static constexpr int NV = kTile * CH / 64;                                   // loads of a tile of V
    static constexpr int kDims = 128 / C::kBits;                                 // dims of such a piece
    // first of the 8 dims that instruction c takes from lane group lg
    static __device__ __forceinline__ int frag_dim(int c, int lg) {
        return (c / kFrags) * 4 * kPiece + lg * kPiece + 8 * (c % kFrags);
    }
};

// The kernel's LDS: tiles of V (partials afterwards), maxima and sums, and the
// queries where they are not in registers, as two blocks of 128 dims (32 registers
// more than there are).
template <typename C, int D, int NB>
struct FewLds {
    static constexpr bool kQuery = NB * D > 128;
    static constexpr int kRows = FewLoads<C, D>::kTile * kRow<D>;
    static constexpr int kWave = kRows > 16 * D * 2 ? kRows : 16 * D * 2;   // u16
    static constexpr int kBuf = kFewWaves * kWave, kQ = kQuery ? 16 * NB * kRow<D> : 8;
    static constexpr int kBytes = 2 * (kBuf + kQ) + kFewWaves * 16 * NB * 8 + 4;
    typedef float Ml[16 * NB][2];
    uint16_t* buf;
    uint16_t* q;
    Ml* ml;     // [kFewWaves]
    int* odd;   // a masked tile held infinities or NaN
};

template <typename T, int D, int NB, typename C, bool SH>
__device__ __forceinline__ void few_body(const PagedParams<C, SH>& a, int direct, int block,
                                         const FewLds<C, D, NB>& lds) {
    constexpr int KK = D / 32;     // matrix instructions over the head dim
    constexpr int DB = D / 16;     // output blocks of 16 dims
    constexpr int LR = kRow<D>;
    typedef FewLoads<C, D> Lo;
    constexpr int LEAD = Lo::kLead;
    constexpr bool kCodes = C::kBits != 16;
    constexpr int CH = Lo::CH, NV = Lo::NV;          // 16-byte pieces of a row, loads of a tile of V
    constexpr int TILE = Lo::kTile, UNIT = TILE * kFewWaves, KB = TILE / 16;   // KB: blocks of 16 rows
    constexpr int kWaveLds = FewLds<C, D, NB>::kWave;
    constexpr bool kQueryLds = FewLds<C, D, NB>::kQuery;
    static_assert(kWaveLds * 2 % 16 == 0 && LR * 2 % 16 == 0,
                  "rows and partials are read and written 16 bytes at a time");
    uint16_t* const s_buf = lds.buf;
    uint16_t* const s_q = lds.q;
    auto* const s_ml = lds.ml;
    int& s_odd = *lds.odd;
    const int tid = threadIdx.x, lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ln = lane & 15, lg = lane >> 4;
    uint16_t* const sv = s_buf + wave * kWaveLds;
    if (tid == 0) s_odd = 0;
    __syncthreads();

    FewRange range;
    if (direct) {     // a workgroup per (sequence, head): nothing to join
        range.s = block / a.H;
        range.before = 0;
        const int u = few_units<UNIT, LEAD>(a, seq_of<SH>(a, range.s));
        if (u == 0) return;
        range.g0 = static_cast<int64_t>(block % a.H) * u;
        range.g1 = range.g0 + u;
    } else {
        range = few_range<SH, UNIT, LEAD>(a, block);
    }
    int64_t g0 = range.g0;
    const int64_t g1 = range.g1;
    int s = range.s;
    int64_t base = range.before * a.H;   // units before sequence s, all heads
    bool first = true;
    Join rest{};
    while (g0 < g1) {
        const Seq sq = seq_of<SH>(a, s);
        const int units = few_units<UNIT, LEAD>(a, sq);
        if (g0 >= base + static_cast<int64_t>(units) * a.H) {   // next sequence
            base += static_cast<int64_t>(units) * a.H;
            ++s;
            continue;
        }
        const int h = direct ? block % a.H : quotient(g0 - base, units);
        const int at = static_cast<int>(g0 - base - static_cast<int64_t>(h) * units);
        const int end = static_cast<int>(min(static_cast<int64_t>(units), at + g1 - g0));
        const int u0 = max(at - LEAD, 0), u1 = end - LEAD;   // of the units that hold rows
        if (LEAD > 0 && u1 <= u0) {
            g0 += end - at;
            continue;
        }
        const int rows = sq.n * a.G;
        const int p0 = sq.p0;
        const Span sp = span_of(a, sq, max(p0, 0), sq.len - 1);
        const int vis = sp.count();

        // queries: row r = 16 b + ln of lane, dims 32 c + 8 lg ..
        u32x4_t qf[kQueryLds ? 1 : NB][KK];
        int pos[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int r = 16 * b + ln;
            const int i = r / a.G;
            pos[b] = r < rows ? p0 + i : -1;
            const int rr = min(r, rows - 1);
            const uint16_t* qp = a.q + static_cast<int64_t>(sq.t0 + rr / a.G) * a.q_ts +
                                 static_cast<int64_t>(h * a.G + rr % a.G) * a.q_hs;
            if constexpr (!kQueryLds)
#pragma unroll
                for (int c = 0; c < KK; ++c) qf[b][c] = load16(qp + Lo::frag_dim(c, lg));
            else if (wave == b)   // (a segment's end has a barrier)
#pragma unroll
                for (int c = 0; c < KK; ++c)
                    *reinterpret_cast<u32x4_t*>(s_q + r * LR + 32 * c + 8 * lg) = load16(qp + Lo::frag_dim(c, lg));
        }
        if constexpr (kQueryLds) __syncthreads();
        auto query = [&](int b, int c) {
            if constexpr (kQueryLds) return *reinterpret_cast<const u32x4_t*>(s_q + (16 * b + ln) * LR + 32 * c + 8 * lg);
            else return qf[b][c];
        };
        f32x4_t acc[NB][DB];
        float m[NB], l[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            m[b] = -INFINITY;
            l[b] = 0.0f;
#pragma unroll
            for (int d = 0; d < DB; ++d) acc[b][d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
        const uint16_t* const kh = a.k + static_cast<int64_t>(h) * a.head_s + 8 * lg;
        const uint16_t* const vh = a.v + static_cast<int64_t>(h) * a.head_s + 8 * (lane % CH);
        // (codes)
        const uint8_t* const kc = reinterpret_cast<const uint8_t*>(a.k) + static_cast<int64_t>(h) * a.head_s +
                                  lg * (Lo::kPiece * C::kBits / 8);
        const uint8_t* const vc = reinterpret_cast<const uint8_t*>(a.v) + static_cast<int64_t>(h) * a.head_s +
                                  16 * (lane % CH);
        const uint8_t *kx = nullptr, *vx = nullptr;
        if constexpr (kCodes) {
            kx = (TILE == 64 || lane < 32 ? a.ke : a.ve) + static_cast<int64_t>(h) * a.e_head_s;
            vx = a.ve + static_cast<int64_t>(h) * a.e_head_s;
        }
        // lane's rows of a step's tile: of K ln and 16 + ln (the matrix
        // instruction's), of V, which goes through LDS, whole rows of CH lanes
        auto row_of = [&](int u, int r) { return sp.row(min(u * UNIT + wave * TILE + r, vis - 1)); };
        auto k_row = [&](int u, int e) { return row_of(u, 16 * e + ln); };
        auto v_row = [&](int u, int i) { return row_of(u, (64 / CH) * i + lane / CH); };
        // (codes: lane r looks row r up and holds its exponents, of K and of V, in
        // a tile of 32 rows lane 32 + r those of V; lanes get them from there)
        int idk[2] = {s, s}, idv[NV], id = s;
#pragma unroll
        for (int i = 0; i < NV; ++i) idv[i] = s;
        auto fetch_ids = [&](int u) {
            if (!a.table) return;
            if constexpr (kCodes) {
                id = page_of(a, s, row_of(u, lane % TILE));
                return;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) idk[e] = page_of(a, s, k_row(u, e));
#pragma unroll
            for (int i = 0; i < NV; ++i) idv[i] = page_of(a, s, v_row(u, i));
        };
        u32x4_t kb[kCodes ? 1 : 2][KK], vb[kCodes ? 1 : NV];
        uint32_t kw[KB][Lo::kWords], vw[NV][4], ke = 0, ve = 0;   // codes and exponents
        auto from = [](int lane, uint32_t x) {
            return static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(4 * lane, x));
        };
        auto fetch = [&](int u) {
            if constexpr (!kCodes) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int64_t o = row_offset(a, idk[e], k_row(u, e));
#pragma unroll
                    for (int c = 0; c < KK; ++c) kb[e][c] = load16(kh + o + 32 * c);
                }
#pragma unroll
                for (int i = 0; i < NV; ++i) vb[i] = load16(vh + row_offset(a, idv[i], v_row(u, i)));
            } else {
                const int j = row_of(u, lane % TILE);
                const uint64_t mine = row_offset(a, id, j);
                auto offset = [&](int lane) {
                    return static_cast<uint64_t>(from(lane, mine >> 32)) << 32 | from(lane, mine);
                };
#pragma unroll
                for (int e = 0; e < KB; ++e) {
                    const uint8_t* const row = kc + offset(16 * e + ln);
                    if constexpr (Lo::kWords > 4) {   // two pieces
#pragma unroll
                        for (int p = 0; p < 2; ++p) {
                            uint32_t w[4];
                            load_words<4>(row + 64 * p, w);
#pragma unroll
                            for (int i = 0; i < 4; ++i) kw[e][4 * p + i] = w[i];
                        }
                    } else {
                        load_words<Lo::kWords>(row, kw[e]);
                    }
                }
#pragma unroll
                for (int i = 0; i < NV; ++i) load_words<4>(vc + offset((64 / CH) * i + lane / CH), vw[i]);
                auto load_exps = [&](const uint8_t* p) -> uint32_t {
                    if constexpr (D == 128) return *reinterpret_cast<const uint32_t*>(p);
                    else return *reinterpret_cast<const uint16_t*>(p);
                };
                const int64_t x = exp_offset(a, id, j);
                ke = load_exps(kx + x);
                if constexpr (TILE == 64) ve = load_exps(vx + x);
            }
        };
        // a wave with no row in its share of a unit still runs the step (all
        // of its keys masked): only a unit's tail has such waves
        const bool any = vis > 0;
        if (any) {
            fetch_ids(u0);
            fetch(u0);
            fetch_ids(min(u0 + 1, u1 - 1));
        }
        for (int u = u0; any && u < u1; ++u) {
            const int v0 = u * UNIT + wave * TILE;   // first row of the tile
            if (!kCodes && v0 + TILE > vis) {   // rows past the end weigh nothing: no NaN may enter through V
#pragma unroll
                for (int i = 0; i < (kCodes ? 0 : NV); ++i)
                    if (v0 + (64 / CH) * i + lane / CH >= vis) vb[i] = u32x4_t{0, 0, 0, 0};
            }
            const int j_lo = sp.row(v0), j_hi = sp.row(v0 + TILE - 1);
            const bool full = v0 + TILE <= vis && j_hi <= p0 &&
                              (a.window == 0 || j_lo >= sq.len - a.window || j_hi < a.sinks);
            uint16_t* const sv_row = sv + lane / CH * LR + Lo::kDims * (lane % CH);
            if constexpr (!kCodes) {
                if (!full && sq.n > 1) {   // (one token sees every row of its span)
                    if (__builtin_amdgcn_ballot_w64(!all_finite<T>(vb))) {
                        keep_finite<T>(vb);
                        s_odd = 1;
                    }
                }
#pragma unroll
                for (int i = 0; i < NV; ++i) *reinterpret_cast<u32x4_t*>(sv_row + (64 / CH) * i * LR) = vb[i];
            } else {   // the same, piece by piece
                const bool look = !full && sq.n > 1;
                bool odd = false;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int r = (64 / CH) * i + lane / CH;
                    const uint32_t x4 = TILE == 64 ? from(r, ve) : from(32 + r, ke);
                    const uint32_t e = (x4 >> (8 * (Lo::kDims * (lane % CH) / kBlock))) & 255u;
#pragma unroll
                    for (int k = 0; k < Lo::kDims / 8; ++k) {
                        u32x4_t x[1] = {decode8<T, C>(vw[i], k, e)};
                        if (!full) {
                            if (v0 + (64 / CH) * i + lane / CH >= vis) x[0] = u32x4_t{0, 0, 0, 0};
                            if (look) {
                                odd |= !all_finite<T>(x);
                                keep_finite<T>(x);
                            }
                        }
                        *reinterpret_cast<u32x4_t*>(sv_row + (64 / CH) * i * LR + 8 * k) = x[0];
                    }
                }
                if (look && __builtin_amdgcn_ballot_w64(odd)) s_odd = 1;
            }
            f32x4_t sc[NB][KB];
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < KB; ++e) {
                    sc[b][e] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
                    if constexpr (!kCodes)
#pragma unroll
                        for (int c = 0; c < KK; ++c) sc[b][e] = T::mma16(kb[e][c], query(b, c), sc[b][e]);
                }
            if constexpr (kCodes)
#pragma unroll
                for (int e = 0; e < KB; ++e) {
                    const uint32_t x4 = from(16 * e + ln, ke);
#pragma unroll
                    for (int c = 0; c < KK; ++c) {
                        const u32x4_t k8 = decode8<T, C>(kw[e], c, (x4 >> (8 * (Lo::frag_dim(c, lg) / kBlock))) & 255u);
#pragma unroll
                        for (int b = 0; b < NB; ++b) sc[b][e] = T::mma16(k8, query(b, c), sc[b][e]);
                    }
                }
            if (u + 1 < u1) {
                // a wave that gets here issues its loads ahead of the other's work
                // (131072 bf16 rows: 99.8 us, 102 without; codes as fast either way)
                __builtin_amdgcn_s_setprio(3);
                fetch(u + 1);
                __builtin_amdgcn_s_setprio(0);
                fetch_ids(min(u + 2, u1 - 1));
            }
            wave_lds_sync();
            // lane: keys v0 + 16 e + 4 lg + i of row ln
            u32x4_t pf[NB][KB / 2];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (!full) {
                    const Sees sees(a, pos[b], sp.lo - sp.sink, sp.sink, vis);
#pragma unroll
                    for (int e = 0; e < KB; ++e)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            sc[b][e][i] = sees.row(16 * e + i, v0 + 4 * lg) ? sc[b][e][i] : -INFINITY;
                }
                float mx = -INFINITY;
#pragma unroll
                for (int e = 0; e < KB; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[b][e][i]);
                mx = fmaxf(mx, xor16(mx));
                mx = fmaxf(mx, xor32(mx));
                const bool grow = (mx - m[b]) * a.c > T::kSlack;
                if (__builtin_amdgcn_ballot_w64(grow)) {
                    const float f = grow ? __builtin_amdgcn_exp2f((m[b] - mx) * a.c) : 1.0f;
                    m[b] = grow ? mx : m[b];
                    l[b] *= f;
#pragma unroll
                    for (int d = 0; d < DB; ++d) acc[b][d] *= f;
                }
                float mc = m[b] == -INFINITY ? 0.0f : m[b] * a.c;
                if (__builtin_amdgcn_ballot_w64(fabsf(mc) > kFar)) {
                    const float off = fabsf(mc) > kFar ? m[b] : 0.0f;
                    mc = fabsf(mc) > kFar ? 0.0f : mc;
#pragma unroll
                    for (int i = 0; i < 4 * KB; ++i) sc[b][i >> 2][i & 3] -= off;
                }
                mc -= T::kShift;
#pragma unroll
                for (int x = 0; x < KB / 2; ++x) {
                    float p[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[b][2 * x + (i >> 2)][i & 3], a.c, -mc));
                    l[b] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                    pf[b][x] = u32x4_t{T::pack(p[0], p[1]), T::pack(p[2], p[3]), T::pack(p[4], p[5]), T::pack(p[6], p[7])};
                }
            }
#pragma unroll
            for (int x = 0; x < KB / 2; ++x) {
                const uint16_t* const vp = sv + (32 * x + 4 * lg + (ln >> 2)) * LR + 4 * (ln & 3);
                u32x4_t vt[DB];   // all reads under way before the first is waited for
#pragma unroll
                for (int d = 0; d < DB; ++d) vt[d] = join(read_tr(vp + 16 * d), read_tr(vp + 16 * d + 16 * LR));
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int b = 0; b < NB; ++b) acc[b][d] = T::mma16(vt[d], pf[b][x], acc[b][d]);
            }
            wave_lds_sync();
        }
        // join the waves: sums over the lane groups, then LDS, block by block
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            l[b] += xor16(l[b]);
            l[b] += xor32(l[b]);
            if (lg == 0) {
                s_ml[wave][16 * b + ln][0] = m[b];
                s_ml[wave][16 * b + ln][1] = l[b];
            }
        }
        const bool whole = u0 == 0 && u1 == units - LEAD;
        bool odd = false;
        const int64_t slot = 2 * static_cast<int64_t>(block) + (first ? 0 : 1);
        float* const so = reinterpret_cast<float*>(sv);   // [16 rows][D]
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (16 * b >= rows) break;
            if (b) __syncthreads();
            // O^T: lane has dims 16 d + 4 lg + i of row ln
#pragma unroll
            for (int d = 0; d < DB; ++d)
                *reinterpret_cast<f32x4_t*>(so + ln * D + 16 * d + 4 * lg) = acc[b][d];
            __syncthreads();
            odd = s_odd != 0;   // set before, and not again until all are past the loop
            for (int x = tid; x < 16 * D / 4; x += 64 * kFewWaves) {
                const int rr = x / (D / 4), d4 = x % (D / 4), r = 16 * b + rr;
                if (r >= rows) break;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < kFewWaves; ++w) M = fmaxf(M, s_ml[w][r][0]);
                float L = 0.0f;
                f32x4_t A = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < kFewWaves; ++w) {
                    const float wt = exp2_weight(s_ml[w][r][0], M, a.c);
                    L += s_ml[w][r][1] * wt;
                    A += *reinterpret_cast<const f32x4_t*>(reinterpret_cast<float*>(s_buf + w * kWaveLds) + rr * D +
                                                           4 * d4) *
                         wt;
                }
                if (whole) {
                    const int64_t t = sq.t0 + r / a.G;
                    const int x_head = h * a.G + r % a.G;
                    if constexpr (SH) {
                        if (keeps<SH>(a, sq)) {
                            const int64_t e = t * (a.H * a.G) + x_head;
                            *reinterpret_cast<f32x4_t*>(a.keep + e * D + 4 * d4) = A;
                            if (d4 == 0) {
                                a.keep_ml[2 * e] = M;
                                a.keep_ml[2 * e + 1] = L;
                            }
                            continue;
                        }
                    }
                    const float inv = inverse(L, p0 + r / a.G < 0);
                    uint2 o;
                    o.x = T::pack(A[0] * inv, A[1] * inv);
                    o.y = T::pack(A[2] * inv, A[3] * inv);
                    *reinterpret_cast<uint2*>(a.out + t * a.o_ts + x_head * a.o_hs + 4 * d4) = o;
                    if (a.lse && d4 == 0)
                        a.lse[t * a.l_ts + x_head] = log_sum<T>(M, L, a.c);
                } else {
                    *reinterpret_cast<f32x4_t*>(a.part + (slot * a.cap + r) * D + 4 * d4) = A;
                    if (d4 == 0) {
                        a.part_ml[(slot * a.cap + r) * 2] = M;
                        a.part_ml[(slot * a.cap + r) * 2 + 1] = L;
                    }
                }
            }
        }
        __syncthreads();
        if (odd) {
            __threadfence();
            __syncthreads();
            patch_rows<T, D, C, SH>(a, sq, s, h, sp, 0, rows, u0 * UNIT, min(u1 * UNIT, vis), whole ? -1 : slot);
            __syncthreads();
            if (tid == 0) s_odd = 0;
            __syncthreads();
        }
        if constexpr (SH)
            if (u0 == 0 && tid == 0)
                a.place[static_cast<int64_t>(place_key(a, sq.t0, s, 0)) * a.H + h] = whole ? -1 : block;
        if (u0 == 0 && u1 < units - LEAD)
            rest = Join{range.total, g0 - at, g0 - at + units, sq.t0, 0, rows, h, max(-p0, 0) * a.G};
        g0 += end - at;
        first = false;
    }
    if (!direct && tid == 0) a.joins[block] = rest;
}

template <typename T, int D, int NB, typename C, bool SH>
__global__ __launch_bounds__(kThreads, 2) void few_kernel(PagedParams<C, SH> a, int direct) {
    typedef FewLds<C, D, NB> Lds;   // arrays of their own: in one, the writes of V hold up the reads of others
    __shared__ __align__(16) uint16_t s_buf[Lds::kBuf];
    __shared__ typename Lds::Ml s_ml[kFewWaves];
    __shared__ int s_odd;
    __shared__ __align__(16) uint16_t s_q[Lds::kQ];
    few_body<T, D, NB, C, SH>(a, direct, blockIdx.x, Lds{s_buf, s_q, s_ml, &s_odd});
}

// What merge_kernel needs: the partials of the few-row launch and of the tiles.
struct Parts {
    const Join* joins;
    const float* rows;   // [2 W][cap][D]
    const float* ml;     // [2 W][cap][2]
    int cap;
};
struct MergeParams {
    Parts few, tiles;
    uint16_t* out;
    float* lse;
    int64_t o_ts, o_hs, l_ts;
    int few_blocks;      // workgroups for the few-row launch: W cap, or none
    int tile_blocks;     // and for the tiles
    int G, w_log;
    float c;
};

template <int D>
struct Partial {
    float M = -INFINITY, L = 0.0f;
    f32x4_t A = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    __device__ __forceinline__ void add(float m, float l, f32x4_t x, float c) {
        const float Mn = fmaxf(M, m);
        const float f0 = exp2_weight(M, Mn, c), f1 = exp2_weight(m, Mn, c);
        L = L * f0 + l * f1;
        A = A * f0 + x * f1;
        M = Mn;
    }
    // row r's partials of ranges w0 + first, w0 + first + step .. w1, four
    // loads under way at a time (behind a branch each they would be one); an
    // empty range, whose slot holds anything, and one past w1 are left out
    __device__ __forceinline__ void gather(const Parts& p, const Join& j, int log, int w0, int w1, int r, int d4,
                                           int first, int step, float c, int lead) {
        constexpr int N = 4;
        for (int w = w0 + first; w <= w1; w += N * step) {
            float m[N], l[N];
            f32x4_t x[N];
            bool use[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int wi = min(w + i * step, w1);
                const int64_t b = cut(j.total, wi, log);
                use[i] = w + i * step <= w1 && (lead > 0 ? max(b, j.lo + lead) : b) < cut(j.total, wi + 1, log);
                const int64_t e = (2 * static_cast<int64_t>(wi) + (b < j.lo ? 1 : 0)) * p.cap + r;
                m[i] = p.ml[2 * e];
                l[i] = p.ml[2 * e + 1];
                x[i] = *reinterpret_cast<const f32x4_t*>(p.rows + e * D + 4 * d4);
            }
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (use[i]) add(m[i], l[i], x[i], c);
        }
    }
    template <typename T>
    __device__ __forceinline__ void write(const MergeParams& a, const Join& j, int row, int d4) const {
        const int64_t tok = j.t0 + row / a.G;
        const int head = j.h * a.G + row % a.G;
        const float inv = inverse(L, row < j.blind);
        uint2 o;
        o.x = T::pack(A[0] * inv, A[1] * inv);
        o.y = T::pack(A[2] * inv, A[3] * inv);
        *reinterpret_cast<uint2*>(a.out + tok * a.o_ts + head * a.o_hs + 4 * d4) = o;
        if (a.lse && d4 == 0) a.lse[tok * a.l_ts + head] = log_sum<T>(M, L, a.c);
    }
};

// the last range that holds some of a join: about hi W / total, then exactly
__device__ __forceinline__ int last_of(const Join& j, int w0, int log) {
    int w1 = max(w0, static_cast<int>(static_cast<float>(j.hi - 1) / static_cast<float>(j.total) * (1 << log)) - 1);
    while (cut(j.total, w1 + 1, log) < j.hi) ++w1;
    return w1;
}

// groups of D / 4 threads to a row of so many partials, of P
__device__ __forceinline__ int groups_of(int parts, int P) {
    int K = 1;
    while (K < P && 4 * K < parts) K *= 2;
    return K;
}

// Joins what the ranges left.  D / 4 threads hold a row's partial, so a
// workgroup holds P of them: P / K rows with K groups each, K about a quarter
// of a join's partials, so that a long sequence of few rows and a large chunk
// both wait for one or two loads.
//
// The few-row launch has a workgroup per (range, P / K rows) and most find
// nothing to do.  Tiles have up to 256 rows, far more such workgroups, so
// theirs first list the joins and share out (join, rows) pairs: a tile of 120
// rows in 38 ranges takes 6 us so, 73 with a fixed share of the rows per
// workgroup.  Decoding takes 5 us the first way and 7 the second.
constexpr int kMergeThreads = 256;
constexpr int kMaxRanges = kMergeThreads;   // (a thread looks at one)

template <typename T, int D, int LEAD>
__global__ __launch_bounds__(kMergeThreads) void merge_kernel(MergeParams a) {
    constexpr int Q = D / 4, P = kMergeThreads / Q;
    __shared__ float s_ml[P][2];
    __shared__ __align__(16) float s_acc[P][D];
    static_assert(__alignof__(s_acc) >= 16 && D * 4 % 16 == 0, "rows are read and written 16 bytes at a time");
    __shared__ int s_range[kMaxRanges];
    __shared__ int s_n[kMergeThreads / 64];
    const int tid = threadIdx.x, W = 1 << a.w_log;
    const int d4 = tid % Q, g = tid / Q;
    // rows r0 .. of a join that range w0 left, K groups to a row
    auto merge = [&](const Parts& from, const Join& j, int w0, int w1, int log, int r0, int K, int lead) {
        const int r = r0 + g / K, k = g % K;
        const bool live = r < j.end - j.first;
        Partial<D> p;
        if (live) p.gather(from, j, log, w0, w1, r, d4, k, K, a.c, lead);
        if (K > 1) {
            __syncthreads();
            if (d4 == 0) {
                s_ml[g][0] = p.M;
                s_ml[g][1] = p.L;
            }
            *reinterpret_cast<f32x4_t*>(&s_acc[g][4 * d4]) = p.A;
            __syncthreads();
            if (k == 0)
                for (int x = g + 1; x < g + K; ++x)
                    p.add(s_ml[x][0], s_ml[x][1], *reinterpret_cast<const f32x4_t*>(&s_acc[x][4 * d4]), a.c);
        }
        if (live && k == 0) p.template write<T>(a, j, j.first + r, d4);
    };
    if (static_cast<int>(blockIdx.x) < a.few_blocks) {
        const int w0 = blockIdx.x % W, y = blockIdx.x / W;
        const Join j = a.few.joins[w0];
        if (j.lo == j.hi) return;
        const int log = ranges_log(a.w_log, j.total), w1 = last_of(j, w0, log);
        const int K = groups_of(w1 - w0 + 1, P), r0 = y * (P / K);
        if (r0 < j.end - j.first) merge(a.few, j, w0, w1, log, r0, K, LEAD);
        return;
    }
    // the ranges that hold a join
    const bool has = tid < W && a.tiles.joins[tid].lo != a.tiles.joins[tid].hi;
    const uint64_t mask = __ballot(has);
    if (lane_id() == 0) s_n[tid >> 6] = __builtin_popcountll(mask);
    __syncthreads();
    int before = 0, n = 0;
#pragma unroll
    for (int w = 0; w < kMergeThreads / 64; ++w) {
        if (w < tid >> 6) before += s_n[w];
        n += s_n[w];
    }
    if (n == 0) return;
    if (has) s_range[before + __builtin_popcountll(mask & ((1ull << lane_id()) - 1))] = tid;
    __syncthreads();
    const int log = ranges_log(a.w_log, a.tiles.joins[s_range[0]].total);
    const int K = groups_of(((1 << log) + n - 1) / n, P);
    const int blocks = (a.tiles.cap * K + P - 1) / P;
    for (int item = blockIdx.x - a.few_blocks; item < n * blocks; item += a.tile_blocks) {
        const int w0 = __builtin_amdgcn_readfirstlane(s_range[item / blocks]);
        const Join j = a.tiles.joins[w0];
        const int r0 = item % blocks * (P / K);
        if (r0 < j.end - j.first) merge(a.tiles, j, w0, last_of(j, w0, log), log, r0, K, 0);
    }
}

// --------------------------------------------------------- many rows ------
// Sequences of more rows (prefill chunks): tiles of 256 rows of one (sequence,
// KV head), 32 per wave; the waves share each step's 128 rows of K and V in
// LDS.  The steps of all tiles, KV head by KV head, are again cut
// into W equal ranges, so a causal triangle, a short prompt and a chunk over
// a long prefix load the chip evenly; partials as above.
//
// A CU's eight waves have its registers (acc, scores, queries: 248 of 256) and
// LDS to themselves.  Bound by matrix and vector instructions together (50 and
// 60 percent of a SIMD's time): 8192 tokens of 32 heads over 32768 rows take
// 3.8-4.0 ms, 960-1010 TFLOP/s (a large matrix product runs at 1381).  Without
// the staging the same loop runs at 1190, without the softmax at 1100.  Tiles
// of 128 rows read K and V twice as often and were slower, 64 rows per wave
// (half as many reads of LDS) no faster.
//
// Codes are loaded a step ahead into registers (as many as V's rows take in 16
// bits) and become bf16 or fp16 on their way to LDS, once for all waves; the
// exponents of a wave's 16 rows are one load of a lane each.  A byte for each piece
// spilled 74 registers, in every step: 2.21 ms for 4096 fp8 tokens over 16384 rows
// (32 heads), now 0.96-1.02, 950-1000 TFLOP/s (of one card: fp8 1.016, int8 1.105,
// fp4 0.974, in 16 bits 1.035).
constexpr int kStage = 64;            // cached rows of a stage in LDS
constexpr int kStep = 2 * kStage;     // and of a step

// A step's cached rows in LDS, two stages of 64, shared by the eight waves;
// waves 0-3 fill the first stage, waves 4-7 the second.
//
// Thread (g, ch) of a wave holds piece ch (16 bytes, 8 dims) of NR rows in a
// row, 16 wave + NR g + i, so one page lookup and one address serve K and V.
// K goes from memory to LDS without registers (global_load_lds writes 64 x 16
// bytes in lane order): load i of a wave is a block of consecutive LDS rows,
// and a row's pieces lie at piece ^ k_swz(row).  A 16-byte read takes the lanes
// 0-3, 12-15, 20-27 of a half wave together, then 4-11, 16-19, 28-31: sixteen
// rows whose pieces then cover the 64 banks once.  V is transposed in registers on its way to LDS
// ([dim][64 rows], 128 bytes a dim): the matrix instruction wants eight rows
// of one dim per lane, and stored in the order that the registers of S^T have
// (rows 4 hi .. and 8 + 4 hi .. of 16) they are one 16-byte read.  Dim d's
// pieces lie at piece ^ ((d ^ d / 8) & 7): so do a read's dims, and the dims 8
// apart of a write fall on different banks.
template <int D>
struct Stage {
    static constexpr int CH = D / 8;          // 16-byte pieces of a row
    static constexpr int NR = kStage * CH / 256;   // (four waves fill a stage)
    static constexpr int G = 64 / CH;         // lane groups of a wave
    static constexpr int kBytes = kStage * D * 2;   // of K, and of V
    // what a lane adds to a stage's base, for the pieces that differ in the
    // low bits xored in
    static constexpr int KX = CH / 2;
    int k_read[KX], v_read[4], v_write, v_swz, k_piece, l_ch, l_row;

    // what row r's pieces of K are xored with
    static __device__ __forceinline__ int k_swz(int r) { return D == 128 ? r & 15 : (r & 1) | ((r >> 1) & 6); }

    __device__ __forceinline__ void init() {
        const int lane = lane_id(), wave = threadIdx.x >> 6;
        const int g = lane / CH;
        l_ch = lane % CH;
        l_row = 16 * wave + NR * g;   // in the step; the waves of a stage: 16 (wave & 3)
        k_piece = l_ch ^ k_swz(NR * g);
        const int q = lane & 31, hi = lane >> 5;
        // LDS row of cached row q (of 16): load i = q % NR, lane group q / NR
        const int slot = (q & 16) + (q % NR) * G + (q / NR) % G;
        const int f = (q & 7) ^ (q >> 3);
#pragma unroll
        for (int x = 0; x < KX; ++x) k_read[x] = slot * (2 * D) + 16 * ((2 * x + hi) ^ k_swz(q));
#pragma unroll
        for (int x = 0; x < 4; ++x) v_read[x] = q * 128 + 16 * ((f ^ hi) ^ (2 * x));
        // this thread's rows in the transposed order
        const int y = l_row & 15;
        const int piece = 2 * (wave & 3) + ((y >> 2) & 1);
        v_write = l_ch * 8 * 128 + 8 * ((y >> 3) & 1) + 2 * (y & 3);
        v_swz = 16 * ((piece ^ l_ch) & 7);
    }
    // K: row i of the thread, from the row's first element to its LDS place
    __device__ __forceinline__ void load_k(const uint16_t* row, int i, char* stage) const {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        typedef __attribute__((address_space(1))) const void gvoid;
        typedef __attribute__((address_space(3))) void lvoid;
        __builtin_amdgcn_global_load_lds((gvoid*)(row + 8 * (k_piece ^ i)), (lvoid*)(stage + (wave >> 2) * kBytes + ((wave & 3) * NR + i) * 1024), 16,
                                         0, 0);
    }
    // the same from registers, 8 dims from piece k_piece ^ i of the row
    __device__ __forceinline__ void store_k(u32x4_t x, int i, char* stage) const {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        *reinterpret_cast<u32x4_t*>(stage + (wave >> 2) * kBytes + ((wave & 3) * NR + i) * 1024 + 16 * lane_id()) = x;
    }
    __device__ __forceinline__ void store_v(const u32x4_t (&r)[NR], char* stage) const {
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            char* const at = stage + (threadIdx.x >> 8) * kBytes + v_write + (v_swz ^ (16 * d)) + 128 * d;
            const uint32_t sel = d & 1 ? 0x07060302u : 0x05040100u;
            const uint32_t lo = __builtin_amdgcn_perm(r[1][d >> 1], r[0][d >> 1], sel);
            if constexpr (NR == 4) {
                const uint32_t up = __builtin_amdgcn_perm(r[3][d >> 1], r[2][d >> 1], sel);
                *reinterpret_cast<uint2*>(at) = make_uint2(lo, up);
            } else {
                *reinterpret_cast<uint32_t*>(at) = lo;
            }
        }
    }
    // S^T operand: rows 32 e .. of the step, dims 16 c ..
    __device__ __forceinline__ u32x4_t k_frag(const char* stage, int e, int c) const {
        return *reinterpret_cast<const u32x4_t*>(stage + k_read[c] + 32 * e * 2 * D);
    }
    // O^T operand: dims 32 d .., rows 32 e + 16 c ..
    __device__ __forceinline__ u32x4_t v_frag(const char* stage, int e, int c, int d) const {
        return *reinterpret_cast<const u32x4_t*>(stage + v_read[((2 * e + c) ^ (2 * (d & 1))) & 3] + 32 * d * 128);
    }
};

__device__ __forceinline__ int seq_tiles(const BaseParams& a, const Seq& q) {
    const int64_t rows = static_cast<int64_t>(q.n) * a.G;
    if (q.n <= 0 || rows < a.min_rows || rows > a.max_rows) return 0;
    return static_cast<int>((rows + kTileRows - 1) / kTileRows);
}

// Rows of a tile of new tokens, bounds moved out to multiples of 8 so that
// four rows from a multiple of 4 on are neighbours in memory (pages of four
// rows or more): row v of the span is cached row v, v < pad, or v + shift.
// The rows in between that no token sees (dead) weigh nothing.
struct TileSpan {
    int sink, lo, hi;     // visible: [0, sink) and [lo, hi)
    int pad, shift, vis;  // rows of the span: vis
    int edge;             // dead rows but for those past vis come before
    __device__ __forceinline__ int row(int v) const { return v < pad ? v : v + shift; }
    __device__ __forceinline__ bool dead(int v) const {
        const int j = row(v);
        return v >= vis || (j >= sink && j < lo);
    }
};
__device__ __forceinline__ TileSpan tile_span(const BaseParams& a, const Seq& q, int first) {
    const int p0 = q.p0;
    const int i0 = first / a.G;
    const int i1 = min((first + kTileRows - 1) / a.G, q.n - 1);
    const Span x = span_of(a, q, max(p0 + i0, 0), p0 + i1);
    TileSpan r;
    r.sink = x.sink;
    r.lo = x.lo;
    r.hi = x.hi;
    r.pad = (x.sink + 7) & ~7;
    r.shift = max((x.lo & ~7) - r.pad, 0);
    r.vis = x.hi - r.shift;
    if (r.shift == 0) r.pad = 0;
    r.edge = x.lo > x.sink ? x.lo - r.shift : 0;
    return r;
}

// Up to so many tiles every workgroup of tile_kernel makes the plan for itself,
// a tile per thread: one new sequence of 100 tokens takes 18.5 us so, 21.2 with
// a launch of plan_kernel before (and 8192 over 32768 rows 4.00 ms, 4.06).
constexpr int kOwnPlan = 512;

// The plan: tiles in use; per tile its sequence and first row, and the
// inclusive prefix of the steps; per sequence the inclusive prefix of the
// tiles (scratch of plan_kernel).
struct Plan {
    int32_t* n;
    int2* tiles;       // [slots]
    int64_t* steps;    // [slots]
    int32_t* seqs;     // [S]
};
__host__ __device__ inline size_t plan_bytes(int slots, int S) { return 16 + size_t(slots) * 16 + size_t(S) * 4; }
__device__ __forceinline__ Plan plan_of(const BaseParams& a) {
    Plan p;
    p.n = a.plan;
    p.tiles = reinterpret_cast<int2*>(a.plan + 4);
    p.steps = reinterpret_cast<int64_t*>(p.tiles + a.slots);
    p.seqs = reinterpret_cast<int32_t*>(p.steps + a.slots);
    return p;
}

template <int THREADS, typename V>
__device__ __forceinline__ V block_incl_scan(V x, V* s_wave, V& total) {
    const int lane = lane_id(), wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const V y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) s_wave[wave] = x;
    __syncthreads();
    V before = 0;
    total = 0;
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w < wave) before += s_wave[w];
        total += s_wave[w];
    }
    return x + before;
}

// Fills the plan (all of the workgroup's threads; what it wrote is there after
// the next barrier) and returns the number of tiles.
template <bool SH, int THREADS, typename P>
__device__ __forceinline__ int make_plan(const P& a, const Plan& p, int64_t* s_wave) {
    int64_t n = 0;
    for (int s0 = 0; s0 < a.S; s0 += THREADS) {
        const int s = s0 + threadIdx.x;
        int64_t total;
        const int64_t tiles = s < a.S ? seq_tiles(a, seq_of<SH>(a, s)) : 0;
        const int64_t incl = block_incl_scan<THREADS>(tiles, s_wave, total);
        if (s < a.S) p.seqs[s] = static_cast<int32_t>(min(n + incl, static_cast<int64_t>(a.slots)));
        n += total;
    }
    const int n_tiles = static_cast<int>(min(n, static_cast<int64_t>(a.slots)));
    __syncthreads();   // the prefix is read by other threads of this workgroup
    int64_t before = 0;
    for (int t0 = 0; t0 < n_tiles; t0 += THREADS) {
        const int t = t0 + threadIdx.x;
        int64_t u = 0;
        if (t < n_tiles) {
            int lo = 0, hi = a.S - 1;   // first sequence whose prefix is past t
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (p.seqs[mid] > t) hi = mid;
                else lo = mid + 1;
            }
            const int row = (t - (lo ? p.seqs[lo - 1] : 0)) * kTileRows;
            p.tiles[t] = make_int2(lo, row);
            u = max((tile_span(a, seq_of<SH>(a, lo), row).vis + kStep - 1) / kStep, 1);
        }
        int64_t total;
        const int64_t incl = block_incl_scan<THREADS>(u, s_wave, total);
        if (t < n_tiles) p.steps[t] = before + incl;
        before += total;
    }
    return n_tiles;
}

template <bool SH, typename P>
__global__ __launch_bounds__(1024) void plan_kernel(P a) {
    __shared__ int64_t s_wave[16];
    const Plan p = plan_of(a);
    const int n_tiles = make_plan<SH, 1024>(a, p, s_wave);
    if (threadIdx.x == 0) *p.n = n_tiles;
}

// First tile whose steps reach past x.
__device__ __forceinline__ int find_tile(const int64_t* steps, int n, int64_t x) {
    int lo = 0, hi = n;   // steps[lo - 1] <= x < steps[hi - 1]
    while (hi - lo > 1) {
        const int stride = (hi - lo + 63) / 64;
        const int i = lo + (lane_id() + 1) * stride - 1;
        const uint64_t past = __ballot(i >= hi - 1 || steps[i] > x);
        const int l = __builtin_ctzll(past);
        const int nlo = lo + l * stride;
        hi = min(hi, nlo + stride);
        lo = nlo;
    }
    return lo;
}

// LDS of the tile kernel, one array: with two, the compiler makes every read of
// K wait for the loads into LDS that are under way for the next step
template <int D, bool OWN>
constexpr int kTileLds = 8 * Stage<D>::kBytes + 16 + (OWN ? kOwnPlan * 20 + 128 : 0);

template <typename T, int D, bool OWN, typename C, bool SH>
__device__ __forceinline__ void tile_body(const PagedParams<C, SH>& a, int block, char* const s_stage) {
    constexpr int KK = D / 16;
    constexpr int DB = D / 32;
    constexpr int NF = 4;                   // operand blocks read ahead of their use (2, 6, 8 cost 2, 0, 4 percent)
    constexpr int NR = Stage<D>::NR;
    constexpr int SB = Stage<D>::kBytes;
    constexpr bool kCodes = C::kBits != 16;
    char* const s_k = s_stage;
    char* const s_v = s_stage + 4 * SB;
    // a masked step held infinities or NaN: this tile's word and the next one's
    int* const s_odd = reinterpret_cast<int*>(s_stage + 8 * SB);
    static_assert(SB % 16 == 0, "read and written 16 bytes at a time");
    int turn = 0;
    if (threadIdx.x == 0) s_odd[0] = 0;
    Stage<D> st;
    st.init();
    const int tid = threadIdx.x, lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q32 = lane & 31, hi = lane >> 5;

    Plan plan;
    int n_tiles;
    if constexpr (OWN) {
        plan.steps = reinterpret_cast<int64_t*>(s_stage + 8 * SB + 16);
        plan.tiles = reinterpret_cast<int2*>(plan.steps + kOwnPlan);
        plan.seqs = reinterpret_cast<int32_t*>(plan.tiles + kOwnPlan);
        n_tiles = make_plan<SH, kThreads>(a, plan, reinterpret_cast<int64_t*>(plan.seqs + kOwnPlan));
        __syncthreads();
    } else {
        plan = plan_of(a);
        n_tiles = *plan.n;
    }
    const int64_t* const steps = plan.steps;
    const int64_t per_head = n_tiles ? steps[n_tiles - 1] : 1;
    const int64_t total = n_tiles ? per_head * a.H : 0;
    // workgroups go round robin over the 8 dies: die x takes the x-th eighth
    // of the steps, so that its workgroups read the same head's K and V
    const int log = ranges_log(a.w_log, total), W = 1 << log;
    const bool used = block < W;
    const int wg = W >= 8 && used ? (block % 8) * (W / 8) + block / 8 : block;
    int64_t g0 = used ? cut(total, wg, log) : 0;
    const int64_t g1 = used ? cut(total, wg + 1, log) : 0;
    bool first = true;
    Join rest{};
    int h = static_cast<int>(g0 / per_head);
    int t = g0 < g1 ? find_tile(steps, n_tiles, g0 - h * per_head) : 0;
    while (g0 < g1) {
        const int2 tile = plan.tiles[t];
        const int64_t t_lo = h * per_head + (t ? steps[t - 1] : 0);
        const int units = static_cast<int>(h * per_head + steps[t] - t_lo);
        const int u0 = static_cast<int>(g0 - t_lo);
        const int u1 = static_cast<int>(min(static_cast<int64_t>(units), u0 + g1 - g0));
        const int s = tile.x;
        const Seq sq = seq_of<SH>(a, s);
        const int64_t rows = static_cast<int64_t>(sq.n) * a.G;
        const int p0 = sq.p0;
        const TileSpan sp = tile_span(a, sq, tile.y);
        const int vis = sp.vis;

        // this lane's query row (both halves of the wave), dims 16 c + 8 hi ..
        const int r = tile.y + wave * 32 + q32;
        const bool live = r < rows;
        const int rr = live ? r : static_cast<int>(rows) - 1;
        const int tok = rr / a.G;
        const int pos = live ? p0 + tok : -1;
        const int64_t q_tok = sq.t0 + tok;
        const int x_head = h * a.G + rr % a.G;
        const uint16_t* qp = a.q + q_tok * a.q_ts + x_head * a.q_hs + 8 * hi;
        u32x4_t qf[KK];
#pragma unroll
        for (int c = 0; c < KK; ++c) qf[c] = load16(qp + 16 * c);
        const int w_first = tile.y + wave * 32;
        const bool idle = w_first >= rows;
        const int t_end = static_cast<int>(min(static_cast<int64_t>(tile.y) + kTileRows, rows));
        // Which steps need what, once per tile.  Row v of the span is cached row
        // v + shift (from pad on), so a bound on rows is one on steps.
        // A step whose rows are all there, and neighbours four by four:
        const int easy_lo = (sp.pad + kStep - 1) / kStep, easy_hi = a.page_shift >= 2 ? vis / kStep : 0;
        // a step with nothing to look for in V: no dead row, no row that only
        // some of the tile's tokens see
        const int t_min = p0 + tile.y / a.G, t_max = p0 + (t_end - 1) / a.G;
        const int gone = a.window > 0 ? max(t_max - a.window - sp.shift + 1, sp.pad) : 0;
        const int plain_lo = (max(gone, sp.edge) + kStep - 1) / kStep;
        const int plain_hi = min(vis, max(t_min + 1 - sp.shift, 0)) / kStep;
        // stages (64 rows) that all of the wave's tokens see, and that some do
        const int p_min = p0 + min(w_first, static_cast<int>(rows) - 1) / a.G;
        const int p_max = p0 + static_cast<int>(min(static_cast<int64_t>(w_first) + 31, rows - 1)) / a.G;
        const int full_lo = a.window > 0 ? (max(p_max - a.window + 1 - sp.shift, sp.pad) + kStage - 1) / kStage : 0;
        const int full_hi = w_first + 32 <= rows ? min(vis, max(p_min + 1 - sp.shift, 0)) / kStage : 0;
        const int seen_hi = idle ? 0 : (p_max - sp.shift) / kStage + 1;
        // of the rows before, first tokens that stay visible: full up to here
        const int sink_hi = w_first + 32 <= rows ? min(a.sinks, sp.shift ? sp.sink : p_min + 1) / kStage : 0;
        __syncthreads();   // all have read the last tile's word: it is the next one's
        if (tid == 0) s_odd[turn ^ 1] = 0;

        f32x16_t acc[DB];
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
        float m = -INFINITY, l = 0.0f;
        float mc = -T::kShift;   // what a score's exponent loses, and whether a row of the wave is far (kFar)
        bool far = false;

        const uint16_t* const kh = a.k + static_cast<int64_t>(h) * a.head_s;
        const uint16_t* const vh = a.v + static_cast<int64_t>(h) * a.head_s + 8 * st.l_ch;
        // (codes: pieces of 8 dims are kWords words)
        const uint8_t* const kc = reinterpret_cast<const uint8_t*>(a.k) + static_cast<int64_t>(h) * a.head_s;
        const uint8_t* const vc = reinterpret_cast<const uint8_t*>(a.v) + static_cast<int64_t>(h) * a.head_s +
                                  4 * C::kWords * st.l_ch;
        // and the exponents of a wave's 16 rows of K are in lanes 0 .. 15 (and
        // 32 ..), of V in 16 .. 31
        const uint8_t* ex = nullptr;
        if constexpr (kCodes) ex = (lane & 16 ? a.ve : a.ke) + static_cast<int64_t>(h) * a.e_head_s;
        const int ex_row = 16 * wave + (lane & 15);
        // an easy step: one page lookup, one step ahead of its use, and one
        // address per thread
        int id = s, ex_id = s;
        auto fetch_id = [&](int u) {
            if (a.table) id = page_of(a, s, sp.row(min(u * kStep + st.l_row, vis - 1)));
            if constexpr (kCodes)
                if (a.table) ex_id = page_of(a, s, sp.row(min(u * kStep + ex_row, vis - 1)));
        };
        u32x4_t vb[NR];
        uint32_t kw[NR][C::kWords], vw[NR][C::kWords], exps = 0;   // codes and exponents
        auto fetch_row = [&](int i, int64_t o) {
            load_words<C::kWords>(kc + o + 4 * C::kWords * (st.k_piece ^ i), kw[i]);
            load_words<C::kWords>(vc + o, vw[i]);
        };
        auto fetch_exps = [&](int u) {
            if constexpr (kCodes) {
                const uint8_t* const p = ex + exp_offset(a, ex_id, sp.row(min(u * kStep + ex_row, vis - 1)));
                if constexpr (D == 128) exps = *reinterpret_cast<const uint32_t*>(p);
                else exps = *reinterpret_cast<const uint16_t*>(p);
            }
        };
        auto fetch = [&](int u) {
            char* const sk = s_k + (u & 1) * 2 * SB;
            fetch_exps(u);
            if (u >= easy_lo && u < easy_hi) {
                const int j = u * kStep + st.l_row + sp.shift;
                const int64_t o = row_offset(a, id, j);
                if constexpr (kCodes) {
#pragma unroll
                    for (int i = 0; i < NR; ++i) fetch_row(i, o + i * a.tok_s);
                } else {
#pragma unroll
                    for (int i = 0; i < NR; ++i) {
                        st.load_k(kh + o + i * a.tok_s, i, sk);
                        vb[i] = load16(vh + o + i * a.tok_s);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    const int j = sp.row(min(u * kStep + st.l_row + i, vis - 1));
                    const int page = page_of(a, s, j);
                    const int64_t o = row_offset(a, page, j);
                    if constexpr (kCodes) {
                        fetch_row(i, o);
                    } else {
                        st.load_k(kh + o, i, sk);
                        vb[i] = load16(vh + o);
                    }
                }
            }
        };
        auto store = [&](int u) {
            if constexpr (kCodes) {
                char* const sk = s_k + (u & 1) * 2 * SB;
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    const int from = 4 * (NR * (lane / Stage<D>::CH) + i);
                    const uint32_t e = __builtin_amdgcn_ds_bpermute(from, exps);
                    st.store_k(decode8<T, C>(kw[i], 0, (e >> (8 * ((st.k_piece ^ i) / 4))) & 255u), i, sk);
                }
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    const int from = 4 * (16 + NR * (lane / Stage<D>::CH) + i);
                    const uint32_t e = __builtin_amdgcn_ds_bpermute(from, exps);
                    vb[i] = decode8<T, C>(vw[i], 0, (e >> (8 * (st.l_ch / 4))) & 255u);
                }
            }
            if (u < plain_lo || u >= plain_hi) {   // no NaN may enter through a row that is not seen
#pragma unroll
                for (int i = 0; i < NR; ++i)
                    if (sp.dead(u * kStep + st.l_row + i)) vb[i] = u32x4_t{0, 0, 0, 0};
                if (__builtin_amdgcn_ballot_w64(!all_finite<T>(vb))) {
                    keep_finite<T>(vb);
                    s_odd[turn] = 1;
                }
            }
            st.store_v(vb, s_v + (u & 1) * 2 * SB);
            if constexpr (!kCodes) wait_loads();   // K is in LDS
        };
        // block n of a step's V: rows 16 (n / DB), dims 32 (n % DB)
        auto v_at = [&](const char* sv, int n) { return st.v_frag(sv, n / DB >> 1, n / DB & 1, n % DB); };
        auto order = [] { __builtin_amdgcn_sched_barrier(0); };   // reads stay ahead of their use
#pragma unroll
        for (int c = 0; c < KK; ++c) asm volatile("" : "+v"(qf[c]));   // loaded here, not waited for in every step
        if (vis > 0) {
            fetch_id(u0);
            fetch(u0);
            fetch_id(min(u0 + 1, u1 - 1));
            store(u0);
        }
        for (int u = u0; vis > 0 && u < u1; ++u) {
            const bool more = u + 1 < u1;
            __syncthreads();
            if (more) {
                fetch(u + 1);
                fetch_id(min(u + 2, u1 - 1));
            }
#pragma unroll 1
            for (int sub = 0; sub < 2; ++sub) {
                const char* const sk = s_k + ((u & 1) * 2 + sub) * SB;
                const char* const sv = s_v + ((u & 1) * 2 + sub) * SB;
                const int v0 = u * kStep + sub * kStage;
                if (sub > 0 && more) store(u + 1);   // between two stages, not where the waves meet
                if (v0 >= vis) break;
                const int stage = 2 * u + sub;
                // rows that none of the wave's tokens sees are skipped
                const bool skip = stage >= seen_hi;
                if (!skip) {
                    f32x16_t sc[2];
                    // K's blocks (32 rows, 16 dims), then V's, NF reads ahead
                    u32x4_t fr[NF];
                    auto frag = [&](int n) {
                        return n < 2 * KK ? st.k_frag(sk, n & 1, n >> 1) : v_at(sv, n - 2 * KK);
                    };
#pragma unroll
                    for (int n = 0; n < NF; ++n) fr[n] = frag(n);
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int i = 0; i < 16; ++i) sc[e][i] = 0.0f;
                    order();
#pragma unroll
                    for (int n = 0; n < 2 * KK; ++n) {
                        sc[n & 1] = T::mma32(fr[n % NF], qf[n >> 1], sc[n & 1]);
                        fr[n % NF] = frag(n + NF);
                        order();
                    }
                    // lane: keys v0 + 32 e + 8 (i / 4) + 4 hi + i % 4 of row q32
                    const bool full = (stage >= full_lo && stage < full_hi) || stage < sink_hi;
                    u32x4_t pf[4];   // weights of 16 rows each
                    {
                        if (!full) {
                            const Sees sees(a, pos, sp.shift, sp.sink, vis);
#pragma unroll
                            for (int e = 0; e < 2; ++e)
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    const int k = 32 * e + 8 * (i >> 2) + (i & 3);
                                    sc[e][i] = sees.row(k, v0 + 4 * hi) ? sc[e][i] : -INFINITY;
                                }
                        }
                        float mx = sc[0][0];
#pragma unroll
                        for (int i = 1; i < 32; ++i) mx = fmaxf(mx, sc[i >> 4][i & 15]);
                        mx = fmaxf(mx, xor32(mx));
                        const bool grow = (mx - m) * a.c > T::kSlack;
                        if (far || __builtin_amdgcn_ballot_w64(grow)) {
                            const float f = grow ? __builtin_amdgcn_exp2f((m - mx) * a.c) : 1.0f;
                            m = grow ? mx : m;
                            l *= f;
#pragma unroll
                            for (int d = 0; d < DB; ++d) acc[d] *= f;
                            mc = m == -INFINITY ? 0.0f : m * a.c;
                            far = __builtin_amdgcn_ballot_w64(fabsf(mc) > kFar) != 0;
                            if (far) {
                                const float off = fabsf(mc) > kFar ? m : 0.0f;
                                mc = fabsf(mc) > kFar ? 0.0f : mc;
#pragma unroll
                                for (int i = 0; i < 32; ++i) sc[i >> 4][i & 15] -= off;
                            }
                            mc -= T::kShift;
                        }
                        float ls[2] = {0.0f, 0.0f};
                        // weights 2 i, 2 i + 1 of the lane's 32; those of the next
                        // 16 rows come between the matrix instructions of these, in
                        // the compiler's order (1 percent of a chunk's time, 2 more
                        // of a mixed batch than in this one's)
                        auto weigh = [&](int i) {
                            const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i >> 3][2 * (i & 7)], a.c, -mc));
                            const float w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i >> 3][2 * (i & 7) + 1], a.c, -mc));
                            pf[i >> 2][i & 3] = T::pack(w0, w1);
                            ls[0] += w0;
                            ls[1] += w1;
                        };
#pragma unroll
                        for (int i = 0; i < 4; ++i) weigh(i);
                        order();
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
#pragma unroll
                            for (int d = 0; d < DB; ++d) {
                                const int n = 2 * KK + DB * x + d;
                                acc[d] = T::mma32(fr[n % NF], pf[x], acc[d]);
                                if (n + NF < 2 * KK + 4 * DB) fr[n % NF] = frag(n + NF);
                                if (x < 3) {
#pragma unroll
                                    for (int k = 0; k < 4 / DB; ++k) weigh(4 * (x + 1) + (4 / DB) * d + k);
                                }
                            }
                        }
                        l += ls[0] + ls[1];
                    }
                }
            }
        }
        l += xor32(l);
        if (live) {
            const bool keep = u0 == 0 && u1 == units && keeps<SH>(a, sq);
            if (u0 == 0 && u1 == units && !keep) {
                const float inv = inverse(l, pos < 0);
                uint16_t* const op = a.out + q_tok * a.o_ts + x_head * a.o_hs + 4 * hi;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint2 o;
                        o.x = T::pack(acc[d][4 * i] * inv, acc[d][4 * i + 1] * inv);
                        o.y = T::pack(acc[d][4 * i + 2] * inv, acc[d][4 * i + 3] * inv);
                        *reinterpret_cast<uint2*>(op + 32 * d + 8 * i) = o;
                    }
                if (a.lse && hi == 0)
                    a.lse[q_tok * a.l_ts + x_head] = log_sum<T>(m, l, a.c);
            } else {
                int64_t e = (2 * static_cast<int64_t>(wg) + (first ? 0 : 1)) * a.cap + wave * 32 + q32;
                float *rows_at = a.part, *ml = a.part_ml;
                if constexpr (SH)
                    if (keep) e = q_tok * (a.H * a.G) + x_head, rows_at = a.keep, ml = a.keep_ml;
                float* const op = rows_at + e * D + 4 * hi;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<f32x4_t*>(op + 32 * d + 8 * i) =
                            f32x4_t{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
                if (hi == 0) {
                    ml[2 * e] = m;
                    ml[2 * e + 1] = l;
                }
            }
        }
        __syncthreads();   // the next tile's first store reuses the stages
        if (s_odd[turn]) {
            __threadfence();
            __syncthreads();
            for (int u = u0; u < u1; ++u)
                if (u < plain_lo || u >= plain_hi)
                    patch_rows<T, D, C, SH>(a, sq, s, h, sp, tile.y, t_end, u * kStep, min((u + 1) * kStep, vis),
                                     u0 == 0 && u1 == units ? -1 : 2 * static_cast<int64_t>(wg) + (first ? 0 : 1));
        }
        turn ^= 1;
        if constexpr (SH)
            if (u0 == 0 && tid == 0)
                a.place[static_cast<int64_t>(place_key(a, sq.t0, s, tile.y)) * a.H + h] = u1 == units ? -1 : wg;
        if (u0 == 0 && u1 < units)
            rest = Join{total, t_lo, t_lo + units, sq.t0, tile.y, t_end, h, max(-p0, 0) * a.G};
        g0 += u1 - u0;
        first = false;
        if (++t == n_tiles) {
            t = 0;
            ++h;
        }
    }
    if (tid == 0) a.joins[wg] = rest;
}

template <typename T, int D, bool OWN, typename C, bool SH>
__global__ __launch_bounds__(kThreads, 2) void tile_kernel(PagedParams<C, SH> a) {
    __shared__ __align__(1024) char s_stage[kTileLds<D, OWN>];
    tile_body<T, D, OWN, C, SH>(a, blockIdx.x, s_stage);
}

// ------------------------------------------------------------ shared rows --
// A launch for the shared rows (the first 2^w_log workgroups, tiles: a run of 64
// sequences of 4 heads has 256 rows, and reads K and V once for all) and for the
// rows of the sequences' own (few rows each).  A CU holds one workgroup (its LDS), so
// these begin where a CU is done with the former, and not when all are.
// (Twice the whole arguments, 912 bytes instead of 392, cost 1.5 us a launch.)
struct Common {   // what differs in the launch's arguments for the shared rows
    Join* joins;
    float *part, *part_ml, *keep, *keep_ml;
    int32_t* place;
    int min_rows, max_rows, cap, slots;
};
template <typename T, int D, int NB, typename C>
__global__ __launch_bounds__(kThreads, 2) void both_kernel(PagedParams<C, true> own, Common c) {
    typedef FewLds<C, D, NB> Lds;
    constexpr int kLds = std::max(kTileLds<D, true>, Lds::kBytes);
    __shared__ __align__(1024) char s_lds[kLds];
    const int W = 1 << own.w_log;
    if (static_cast<int>(blockIdx.x) < W) {
        own.common = true;
        own.joins = c.joins;
        own.part = c.part;
        own.part_ml = c.part_ml;
        own.keep = c.keep;
        own.keep_ml = c.keep_ml;
        own.place = c.place;
        own.min_rows = c.min_rows;
        own.max_rows = c.max_rows;
        own.cap = c.cap;
        own.slots = c.slots;
        tile_body<T, D, true, C, true>(own, blockIdx.x, s_lds);
    } else {
        char* const q = s_lds + 2 * Lds::kBuf;
        char* const ml = q + 2 * Lds::kQ;
        few_body<T, D, NB, C, true>(own, 0, blockIdx.x - W,
                                    Lds{reinterpret_cast<uint16_t*>(s_lds), reinterpret_cast<uint16_t*>(q),
                                        reinterpret_cast<typename Lds::Ml*>(ml),
                                        reinterpret_cast<int*>(ml + kFewWaves * sizeof(typename Lds::Ml))});
    }
}

struct JoinParams {
    PagedParams<Raw16, true> own;        // sequences, and where their own rows' results are
    int few_rows;                // up to so many rows they are in few, above in tiles
    int blocks;                  // to a (sequence, head)
    Parts few, tiles, common;
    const float *keep, *keep_ml;         // of the shared rows
    const int32_t *place, *leaders;
};

// Joins what the shared rows and its own rows gave each query row: a workgroup
// per (sequence, head) and some rows, D / 4 threads to a partial as in
// merge_kernel.  All of a workgroup's for a row after the other, or, where there
// are more than kJoinRows rows (CHUNKS: many rows, of few partials each), a row for
// each group of D / 4: a chunk of 4096 tokens of 32 heads beside 8 single tokens
// that share nothing takes 490 us so, 774 with all of the workgroup's for each row
// (and 470 without looking for shared rows).  Batches that cannot have so many rows
// have a kernel without that branch, which costs them 1 us (144 -> 146).
constexpr int kJoinRows = 64;
template <typename T, int D, int LEAD, bool CHUNKS>
__global__ __launch_bounds__(kMergeThreads) void join_kernel(JoinParams p) {
    constexpr int Q = D / 4, K = kMergeThreads / Q;
    __shared__ float s_ml[K][2];
    __shared__ __align__(16) float s_acc[K][D];
    const auto& a = p.own;
    const int s = blockIdx.x / a.H, h = blockIdx.x % a.H;
    const int d4 = threadIdx.x % Q, k = threadIdx.x / Q;
    const Seq sq = seq_of<true>(a, s);
    const int64_t rows = static_cast<int64_t>(sq.n) * a.G;
    if (rows == 0 || rows > a.max_rows) return;
    const int heads = a.H * a.G;
    const int lead = sq.lo > 0 ? clampi(p.leaders[s], 0, s) : s;
    const int lead_t0 = clampi(a.start[lead], 0, sq.t0);
    // row r's, as far as this one of `groups` groups takes them: returns how many hold
    // something, none where the row's range has written it
    auto gather = [&](int64_t r, int k, int groups, Partial<D>& x) {
        const int i = static_cast<int>(r / a.G), g = static_cast<int>(r % a.G);
        const int64_t t = sq.t0 + i, e = t * heads + h * a.G + g;
        int used = groups;
        auto add = [&](int place, const Parts& from, const float* keep, const float* keep_ml, int row, int lead) {
            if (place < 0) {
                if (k == 0)
                    x.add(keep_ml[2 * e], keep_ml[2 * e + 1], *reinterpret_cast<const f32x4_t*>(keep + e * D + 4 * d4),
                          a.c);
                return;
            }
            const int w0 = place & ((1 << a.w_log) - 1);
            const Join j = from.joins[w0];
            if (j.lo >= j.hi) return;
            const int log = ranges_log(a.w_log, j.total), w1 = last_of(j, w0, log);
            if (sq.lo == 0) used = groups_of(w1 - w0 + 1, groups);   // the order of merge_kernel
            if (k < used) x.gather(from, j, log, w0, w1, row, d4, k, used, a.c, lead);
        };
        const int tile = static_cast<int>(r) & ~(kTileRows - 1);
        const int mine = a.place[static_cast<int64_t>(place_key(a, sq.t0, s, tile)) * a.H + h];
        if (sq.lo == 0 && mine < 0) return 0;
        const bool in_few = rows <= p.few_rows;
        add(mine, in_few ? p.few : p.tiles, a.keep, a.keep_ml, static_cast<int>(r) - tile, in_few ? LEAD : 0);
        if (sq.lo > 0) {
            const int64_t rc = (t - lead_t0) * a.G + g;
            const int first = static_cast<int>(rc) & ~(kTileRows - 1);
            add(p.place[static_cast<int64_t>(place_key(a, lead_t0, lead, first)) * a.H + h], p.common, p.keep,
                p.keep_ml, static_cast<int>(rc) - first, 0);
        }
        return used;
    };
    auto write = [&](int64_t r, const Partial<D>& x) {
        const int i = static_cast<int>(r / a.G);
        const int64_t t = sq.t0 + i;
        const int head = h * a.G + static_cast<int>(r % a.G);
        const float inv = inverse(x.L, sq.p0 + i < 0);
        uint2 o;
        o.x = T::pack(x.A[0] * inv, x.A[1] * inv);
        o.y = T::pack(x.A[2] * inv, x.A[3] * inv);
        *reinterpret_cast<uint2*>(a.out + t * a.o_ts + head * a.o_hs + 4 * d4) = o;
        if (a.lse && d4 == 0) a.lse[t * a.l_ts + head] = log_sum<T>(x.M, x.L, a.c);
    };
    if (CHUNKS && rows > kJoinRows) {
        for (int64_t r = static_cast<int64_t>(blockIdx.y) * K + k; r < rows; r += static_cast<int64_t>(p.blocks) * K) {
            Partial<D> x;
            if (gather(r, 0, 1, x)) write(r, x);
        }
        return;
    }
    for (int64_t r = blockIdx.y; r < rows; r += p.blocks) {
        Partial<D> x;
        const int used = gather(r, k, K, x);
        if (used == 0) continue;
        __syncthreads();
        if (d4 == 0) {
            s_ml[k][0] = x.M;
            s_ml[k][1] = x.L;
        }
        *reinterpret_cast<f32x4_t*>(&s_acc[k][4 * d4]) = x.A;
        __syncthreads();
        if (k == 0) {
            for (int y = 1; y < used; ++y)
                x.add(s_ml[y][0], s_ml[y][1], *reinterpret_cast<const f32x4_t*>(&s_acc[y][4 * d4]), a.c);
            write(r, x);
        }
    }
}

// ------------------------------------------------------------- host -------

// The launches of one call.  Sequences of at most few_rows rows go to the
// few-row kernel (blocks of 16 rows), the others to the tile kernel.
struct Shape {
    int few_rows = 0;       // 0: no few-row launch
    int w_log = 0;          // 2^w_log workgroups
    int max_rows = 0;       // rows a sequence can have: one with more has no room in the partials and is left out
    int most = 0;           // rows a few-row sequence can have
    bool direct = false;    // a workgroup per (sequence, head), no join
    bool tiles = false;
    int tile_most = 0;      // rows of a tile that can be in use
    int slots = 0;
    size_t few_part = 0, tile_part = 0, plan = 0;   // workspace bytes
};

// A workgroup per (sequence, head) up to this many rows.  One sequence of 519
// rows of 128 dims called in a loop takes 13.3 us so, 15.4-15.9 with a join, whose
// workspace and second launch cost the host more than the GPU gains (replayed
// in a graph: 512, 768, 1024 rows 11.3, 14.1, 16.8 us without, 11.4 each with).
constexpr int kDirectRows = 768;
constexpr int kDirectGrid = 1 << 22;   // workgroups of 512 threads in a launch of at most 2^32 - 1

inline Shape shape_of(const imi_paged_attention_args* a) {
    Shape p;
    const imi_paged_batch& b = a->batch;
    if (b.n_seqs == 0 || b.n_tokens == 0) return p;
    const int64_t most = static_cast<int64_t>(std::min(b.max_query, b.n_tokens)) * a->groups;
    p.max_rows = static_cast<int>(most);
    // a workgroup of eight waves per CU: its registers and LDS fill one
    while ((2 << p.w_log) <= std::min(device_cus(), kMaxRanges)) ++p.w_log;
    if (most <= 32) {
        p.few_rows = most <= 16 ? 16 : 32;
    } else {
        // Beside tiles the few-row kernel takes one block where it holds a token,
        // so sequences of 17 to 32 rows become tiles: the batch says how long its
        // chunks may be, not whether there are any, and what such steps mostly
        // hold is single tokens.  With two blocks 40 of these over 300..40000 rows
        // (4 heads of 128, 8 queries each) take 166 us instead of 146, 24 over
        // 600..20000 (8 heads, 4 queries) 134 instead of 124, of 64 dims 71 instead
        // of 65; with one block 24 sequences of 5 tokens (20 rows each) take 173
        // instead of 148 (100 instead of 81 in a window of 4096; beside a chunk of
        // 500 tokens 229 either way, of 64 dims 170 instead of 131).
        p.tiles = true;
        if (b.n_seqs > 1 && a->groups <= 32) p.few_rows = a->groups <= 16 ? 16 : 32;
    }
    if (p.few_rows) {
        p.most = static_cast<int>(std::min<int64_t>(most, p.few_rows));
        const int64_t cap = std::min<int64_t>(batch_capacity(&b), b.max_len > 0 ? b.max_len : INT_MAX);
        int64_t longest = cap;   // visible rows of the longest sequence
        if (a->window > 0)
            longest = std::min<int64_t>(cap, static_cast<int64_t>(a->window) + a->sinks + p.few_rows / a->groups);
        p.direct = longest <= kDirectRows &&
                   static_cast<int64_t>(b.n_seqs) * a->kv_heads <= kDirectGrid;
        if (!p.direct) p.few_part = (size_t(2) << p.w_log) * p.most * (a->dim + 2) * sizeof(float);
    }
    if (p.tiles) {
        p.slots = static_cast<int>(static_cast<int64_t>(b.n_tokens) * a->groups / kTileRows + b.n_seqs);
        p.tile_most = static_cast<int>(std::min<int64_t>(most, kTileRows));
        p.tile_part = (size_t(2) << p.w_log) * p.tile_most * (a->dim + 2) * sizeof(float);
        if (p.slots > kOwnPlan) p.plan = plan_bytes(p.slots, b.n_seqs);
    }
    return p;
}

// The launches that attend shared rows: tiles alone, whose sequences are the
// runs (as many rows as the batch has, all of one KV head).
inline Shape common_shape_of(const imi_paged_attention_args* a) {
    Shape p;
    const imi_paged_batch& b = a->batch;
    const int64_t most = static_cast<int64_t>(b.n_tokens) * a->groups;
    p.max_rows = static_cast<int>(most);
    while ((2 << p.w_log) <= std::min(device_cus(), kMaxRanges)) ++p.w_log;
    p.tiles = true;
    p.slots = static_cast<int>(most / kTileRows + b.n_seqs);
    p.tile_most = static_cast<int>(std::min<int64_t>(most, kTileRows));
    p.tile_part = (size_t(2) << p.w_log) * p.tile_most * (a->dim + 2) * sizeof(float);
    if (p.slots > kOwnPlan) p.plan = plan_bytes(p.slots, b.n_seqs);
    return p;
}

struct Rooms {
    float *few, *tile;
    int32_t* plan;
    Join* joins;
};
inline size_t carve(const Shape& p, void* base, Rooms& r) {
    Carver c(base);
    r.joins = c.take<Join>(size_t(2) << p.w_log);   // of the few-row launch, of the tile launch
    r.few = c.take<float>(p.few_part / sizeof(float));
    r.tile = c.take<float>(p.tile_part / sizeof(float));
    r.plan = c.take<int32_t>(p.plan / sizeof(int32_t));
    return p.few_part || p.tile_part ? c.used() : 0;
}

// Shared rows are attended together where no window hides some of them and that
// saves kShareBytes of keys and values.  A cache behind the dies' L2 holds as much,
// so that rows which many sequences read are soon read from there, and sharing
// costs a longer chain (the tiles and the join).  One token each, 20 .. 200 own
// rows, 4 query heads per KV head of 128 dims, us without and with sharing:
//   8 heads, bf16:  32 sequences behind 1024 rows (130 MB saved) 24.7, 32.9
//                   32 behind 2048 (260 MB)                      35.9, 34.5
//                   32 behind 16384 (2.1 GB)                    172.7, 47.1
//                   4 behind 16384 (201 MB)                      36.1, 42.5
//                   8 behind 16384 (470 MB)                      57.0, 39.0
//   8 heads, fp8:   32 behind 2048 (134 MB)                      27.4, 33.4
//                   8 behind 16384 (242 MB)                      41.6, 38.7
//   1 head, bf16:   32 behind 16384 (260 MB)                     36.0, 27.7
// What is saved is known on the device alone; the host knows a bound.
constexpr int64_t kShareBytes = int64_t(230) << 20;
inline int64_t least_saved(const imi_paged_attention_args* a) {
    static constexpr int kBits[] = {16, 8, 8, 4};
    const int row_bytes = a->dim * kBits[a->format] / 8 + (a->format == IMI_ROWS ? 0 : a->dim / kBlock);
    const int64_t row = int64_t(2) * a->kv_heads * row_bytes;
    return std::max<int64_t>((a->batch.share_bytes ? a->batch.share_bytes : kShareBytes) / row, 1);
}
constexpr int kJoinPairs = 1 << 22;    // (sequence, head) pairs, at most: 2^30 threads along x
inline bool shares(const imi_paged_attention_args* a) {
    const imi_paged_batch& b = a->batch;
    if (!b.shared || !b.page_table || b.n_seqs < 2 || b.n_tokens == 0) return false;
    if (static_cast<int64_t>(b.n_seqs) * a->kv_heads > kJoinPairs) return false;
    const int64_t capacity = batch_capacity(&b);
    if (a->window > 0 && a->window < capacity) return false;
    const int64_t longest = b.max_len > 0 ? std::min<int64_t>(capacity, b.max_len) : capacity;
    return (b.n_seqs - 1) * longest >= least_saved(a);
}

// The workspace: what whole ranges gave the rows, and where the rows are, of the
// shared rows and of the sequences' own (if any are looked for), then the
// partials of the launches.
struct Work {
    Shape own, common;
    bool shared;
    float *keep[2], *keep_ml[2];
    int32_t* place[2];
    Rooms of_own, of_common;
    size_t bytes;
};
inline Work work_of(const imi_paged_attention_args* a, void* base) {
    Work w{};
    w.own = shape_of(a);
    w.shared = shares(a);
    if (!w.shared) {
        w.bytes = carve(w.own, base, w.of_own);
        return w;
    }
    w.common = common_shape_of(a);
    if (w.own.direct) {
        w.own.direct = false;
        w.own.few_part = (size_t(2) << w.own.w_log) * w.own.most * (a->dim + 2) * sizeof(float);
    }
    const size_t rows = static_cast<size_t>(a->batch.n_tokens) * a->kv_heads * a->groups;
    Carver c(base);
    for (int i = 0; i < 2; ++i) {
        w.keep[i] = c.take<float>(rows * a->dim);
        w.keep_ml[i] = c.take<float>(rows * 2);
        w.place[i] = c.take<int32_t>(static_cast<size_t>(w.common.slots + 1) * a->kv_heads);
    }
    const size_t before = c.used();
    auto at = [&](size_t off) { return base ? static_cast<char*>(base) + off : nullptr; };
    const size_t common = carve(w.common, at(before), w.of_common);
    w.bytes = before + common + carve(w.own, at(before + common), w.of_own);
    return w;
}

template <typename P>
P few_params(const Shape& p, P a, const Rooms& room, int D) {
    a.w_log = p.w_log;
    a.min_rows = 1;
    a.max_rows = p.most;
    a.cap = p.most;
    a.joins = room.joins;
    a.part = room.few;
    a.part_ml = room.few + (size_t(2) << p.w_log) * p.most * D;
    return a;
}
template <typename P>
P tile_params(const Shape& p, P a, const Rooms& room, int D) {
    a.w_log = p.w_log;
    a.min_rows = p.few_rows + 1;
    a.max_rows = p.max_rows;
    a.cap = p.tile_most;
    a.joins = room.joins + (1 << p.w_log);
    a.part = room.tile;
    a.part_ml = room.tile + (size_t(2) << p.w_log) * p.tile_most * D;
    a.plan = room.plan;
    a.slots = p.slots;
    return a;
}

template <typename T, int D, typename C, bool SH>
int launch_tiles(const Shape& p, const PagedParams<C, SH>& Q, hipStream_t stream) {
    const int W = 1 << p.w_log;
    if (p.slots <= kOwnPlan) {
        tile_kernel<T, D, true, C, SH><<<W, kThreads, 0, stream>>>(Q);
    } else {
        plan_kernel<SH, PagedParams<C, SH>><<<1, 1024, 0, stream>>>(Q);
        IMI_LAUNCH_CHECK("plan_kernel");
        tile_kernel<T, D, false, C, SH><<<W, kThreads, 0, stream>>>(Q);
    }
    IMI_LAUNCH_CHECK("tile_kernel");
    return IMI_OK;
}
template <typename T, int D, typename C, bool SH>
int launch_few(const Shape& p, const PagedParams<C, SH>& F, hipStream_t stream) {
    const int grid = p.direct ? F.S * F.H : 1 << p.w_log;
    if (p.few_rows == 16)
        few_kernel<T, D, 1, C, SH><<<grid, kThreads, 0, stream>>>(F, p.direct ? 1 : 0);
    else
        few_kernel<T, D, 2, C, SH><<<grid, kThreads, 0, stream>>>(F, p.direct ? 1 : 0);
    IMI_LAUNCH_CHECK("few_kernel");
    return IMI_OK;
}

inline Parts parts_of(const BaseParams& P) { return Parts{P.joins, P.part, P.part_ml, P.cap}; }

template <typename T, int D, typename C>
int launch(const Shape& p, const PagedParams<C, false>& P, const Rooms& room, hipStream_t stream) {
    const int W = 1 << p.w_log;
    PagedParams<C, false> F = P, Q = P;
    if (p.tiles) {
        Q = tile_params(p, P, room, D);
        if (const int rc = launch_tiles<T, D, C, false>(p, Q, stream)) return rc;
    }
    if (p.few_rows) {
        F = few_params(p, P, room, D);
        if (const int rc = launch_few<T, D, C, false>(p, F, stream)) return rc;
    }
    const int few_blocks = p.few_rows && !p.direct ? W * p.most : 0;
    if (few_blocks || p.tiles) {
        // for the tiles: the pairs there can be, as far as workgroups are worth it
        const int64_t pairs = std::min<int64_t>(W, int64_t(p.slots) * P.H) * p.tile_most;
        const int more = p.tiles ? static_cast<int>(std::min<int64_t>(8 * W, pairs)) : 0;
        const MergeParams M{parts_of(F), parts_of(Q), P.out, P.lse, P.o_ts, P.o_hs, P.l_ts,
                            few_blocks, more, P.G, p.w_log, P.c};
        merge_kernel<T, D, FewLoads<C, D>::kLead><<<few_blocks + more, kMergeThreads, 0, stream>>>(M);
        IMI_LAUNCH_CHECK("merge_kernel");
    }
    return IMI_OK;
}

// Shared and own rows: a launch, where the workgroups can plan for themselves,
// one for sequences of many new tokens, and the join.
//
// Workgroups of a join of long chunks, but at least kJoinRows to a (sequence, head):
// most find no row.  2^13, 2^15, 2^17: the chunk of 4096 tokens above 491, 490, 545
// us, one of 8192 beside 32 single tokens 1093, 1084, 1121.
constexpr int kJoinGrid = 1 << 15;
template <typename T, int D, typename C>
int launch_shared(const Work& w, const imi_paged_batch& b, PagedParams<C, true> P, int64_t least, hipStream_t stream) {
    P.shared = b.shared;
    P.members = b.members;
    P.saved = b.saved;
    P.least_saved = least;
    P.keep = w.keep[0];
    P.keep_ml = w.keep_ml[0];
    P.place = w.place[0];
    PagedParams<C, true> common = tile_params(w.common, P, w.of_common, D);
    common.common = true;
    P.keep = w.keep[1];
    P.keep_ml = w.keep_ml[1];
    P.place = w.place[1];
    PagedParams<C, true> few = P, tiles = P;
    if (w.own.few_rows) few = few_params(w.own, P, w.of_own, D);
    if (w.own.few_rows && w.common.slots <= kOwnPlan) {
        const int grid = 2 << w.own.w_log;
        const Common c{common.joins, common.part,     common.part_ml,  common.keep, common.keep_ml,
                       common.place, common.min_rows, common.max_rows, common.cap,  common.slots};
        if (w.own.few_rows == 16) both_kernel<T, D, 1, C><<<grid, kThreads, 0, stream>>>(few, c);
        else both_kernel<T, D, 2, C><<<grid, kThreads, 0, stream>>>(few, c);
        IMI_LAUNCH_CHECK("both_kernel");
    } else {
        if (const int rc = launch_tiles<T, D, C, true>(w.common, common, stream)) return rc;
        if (w.own.few_rows)
            if (const int rc = launch_few<T, D, C, true>(w.own, few, stream)) return rc;
    }
    if (w.own.tiles) {
        tiles = tile_params(w.own, P, w.of_own, D);
        if (const int rc = launch_tiles<T, D, C, true>(w.own, tiles, stream)) return rc;
    }
    // workgroups to a (sequence, head): one for a row, or, where chunks may be long,
    // as many as kJoinGrid leaves for their groups of rows
    const int64_t pairs = static_cast<int64_t>(P.S) * P.H;
    const int64_t most = (w.own.max_rows + kMergeThreads / (D / 4) - 1) / (kMergeThreads / (D / 4));
    const int blocks = static_cast<int>(std::max<int64_t>(std::min(w.own.max_rows, kJoinRows),
                                                          std::min<int64_t>(most, kJoinGrid / pairs)));
    JoinParams J{{},           w.own.few_rows, blocks,     parts_of(few), parts_of(tiles), parts_of(common),
                 w.keep[0],    w.keep_ml[0],   w.place[0], b.leaders};
    static_cast<BaseParams&>(J.own) = P;
    static_cast<SharedParams&>(J.own) = P;
    J.own.w_log = w.own.w_log;
    J.own.max_rows = w.own.max_rows;
    const dim3 grid(static_cast<unsigned>(pairs), static_cast<unsigned>(blocks));
    if (w.own.max_rows > kJoinRows) join_kernel<T, D, FewLoads<C, D>::kLead, true><<<grid, kMergeThreads, 0, stream>>>(J);
    else join_kernel<T, D, FewLoads<C, D>::kLead, false><<<grid, kMergeThreads, 0, stream>>>(J);
    IMI_LAUNCH_CHECK("join_kernel");
    return IMI_OK;
}

template <typename C, bool SH>
PagedParams<C, SH> params_of(const imi_paged_attention_args* a) {
    const imi_paged_batch& b = a->batch;
    PagedParams<C, SH> P{};
    P.q = a->query;
    P.k = static_cast<const uint16_t*>(a->keys);
    P.v = static_cast<const uint16_t*>(a->values);
    P.out = a->out;
    P.lse = a->out_lse;
    P.table = b.page_table;
    P.lens = b.lens;
    P.start = b.query_start;
    P.q_ts = a->query_token_stride;
    P.q_hs = a->query_head_stride;
    P.o_ts = a->out_token_stride;
    P.o_hs = a->out_head_stride;
    P.l_ts = a->lse_token_stride;
    P.page_s = static_cast<uint32_t>(a->page_stride);
    P.head_s = a->head_stride;
    P.tok_s = static_cast<uint32_t>(a->row_stride);
    P.table_s = b.table_stride;
    P.S = b.n_seqs;
    P.N = b.n_tokens;
    P.H = a->kv_heads;
    P.G = a->groups;
    P.n_pages = b.n_pages;
    P.page_shift = b.page_table ? __builtin_ctz(static_cast<unsigned>(b.page_size)) : 31;
    P.capacity = static_cast<int>(batch_capacity(&b));
    P.window = a->window < P.capacity ? a->window : 0;   // (a window of all rows is none)
    P.sinks = P.window > 0 ? a->sinks : 0;
    P.c = a->scale * kLog2e;
    if constexpr (C::kBits != 16) {
        P.ke = a->key_exponents;
        P.ve = a->value_exponents;
        P.e_head_s = a->exponent_head_stride;
        P.e_page_s = static_cast<uint32_t>(a->exponent_page_stride);
        P.e_tok_s = static_cast<uint32_t>(a->exponent_row_stride);
    }
    return P;
}

template <typename T, int D, typename C>
int run_on(const imi_paged_attention_args* a, hipStream_t stream) {
    const Work w = work_of(a, a->workspace);
    return w.shared ? launch_shared<T, D, C>(w, a->batch, params_of<C, true>(a), least_saved(a), stream)
                    : launch<T, D, C>(w.own, params_of<C, false>(a), w.of_own, stream);
}

template <typename C>
int run(const imi_paged_attention_args* a, hipStream_t stream) {
    if (a->dtype == IMI_BF16)
        return a->dim == 128 ? run_on<BF16, 128, C>(a, stream) : run_on<BF16, 64, C>(a, stream);
    return a->dim == 128 ? run_on<FP16, 128, C>(a, stream) : run_on<FP16, 64, C>(a, stream);
}

}  // namespace
}  // namespace imi
