// RMS norm of every query and key head and the rotation by position, in one
// pass over a projection's output; keys and values go straight to their pages.
//
//   y = x / sqrt(mean(x^2) + eps) * w            (no w: y = x)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * f_i
// over pairs (y_i, y_{i + r/2}), or (y_2i, y_2i+1) interleaved, i < r / 2;
// dims from r on stay.  fp32, rounded once at the end.
//
// The angle: position * f_i in fp64, reduced to a fraction of a turn there
// (exact to 2^-53 of the turns: an fp32 product at position 2^17 would be off
// by 2^-8), then sine and cosine of the fraction in fp32.  The fraction's own
// rounding, up to 2^-26 of a turn, is far under half a step of a 16-bit result
// next to the largest of its head; a block of small numbers in codes is scaled up
// (next to a quarter turn it put 1 code in 400 on the other side of a border), so
// with codes its rest is applied to both.
//
// Bound by memory (a 128-wide head is 256 bytes in and out): D / 8 lanes hold
// a head, 16 bytes each, so the sum of squares is a short lane reduction and
// the partner of a pair is a lane exchange.  A workgroup takes a few tokens;
// its sines and cosines are computed once into LDS while the loads of the
// heads are in flight.
//
// Pages in 8 or 4 bits (C): a block of 32 dims is four lanes, whose largest
// magnitude two lane exchanges find; the codes are made of the fp32 results, so
// a key is rounded once there too.  10529 tokens of 48 heads into fp8, int8 or fp4: 63
// us, bound by vector instructions (0.77 of the issue slots; in fp8 237 MB, 3.8 TB/s).  A row's four
// exponents gathered for one store were no faster than a byte by each block's first
// lane.  Keys and values take one path: with one each, 4 bits spill two registers,
// which costs 6 us (8 bits gain 1).
#include <algorithm>

#include "imi_blocks.hpp"

namespace imi {
namespace {

typedef __attribute__((ext_vector_type(4))) unsigned int u32x4_t;

constexpr int kMaxTokens = 8;   // tokens of a workgroup
// Heads a lane group loads before it computes, and twice as many in a
// workgroup's share, where there are tokens enough to fill the chip: 58 us for
// 10529 tokens of 48 heads (4.45 TB/s, a large copy runs at 4.84).  With 4 at a
// time 60, 6 at a time 76, one batch per workgroup 71; a batch loaded ahead of
// its use costs the registers that six waves per SIMD need (104).
constexpr int kInFlight = 3;

struct QkParams {
    const uint16_t *q, *k, *v;
    uint16_t *qo, *ko, *vo;
    int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
    int64_t qo_ts, qo_hs, ko_ts, ko_hs;    // ko: token and head strides, or head and row strides in pages
    int64_t page_s;
    const float* inv_freq;
    const void *qw, *kw;
    const void* positions;                 // or null: from the batch
    const int32_t *table, *lens, *start;
    int64_t table_s;
    int S, N, Hq, Hk, n_pages, page_shift, capacity;
    int half;                              // r / 2, 0: no rotation
    int tokens;                            // per workgroup
    uint32_t div;                          // floor(2^32 / heads) + 1: x / heads = (x div) >> 32
    float eps;
    bool w32, pos64, interleaved, paged;
    uint8_t *ke, *ve;                      // codes (page, head and row strides in bytes then): exponents
    int64_t e_page_s, e_hs, e_ts;
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }

struct BF16 {
    static constexpr bool kHalf = false;
    static __device__ __forceinline__ float lo(uint32_t x) { return bf16_lo(x); }
    static __device__ __forceinline__ float hi(uint32_t x) { return bf16_hi(x); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        typedef __attribute__((ext_vector_type(2))) float f2;
        typedef __attribute__((ext_vector_type(2))) __bf16 b2;
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), b2));
    }
};
struct FP16 {
    static constexpr bool kHalf = true;
    typedef __attribute__((ext_vector_type(2))) _Float16 h2;
    static __device__ __forceinline__ float lo(uint32_t x) { return __builtin_bit_cast(h2, x)[0]; }
    static __device__ __forceinline__ float hi(uint32_t x) { return __builtin_bit_cast(h2, x)[1]; }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, (h2{static_cast<_Float16>(a), static_cast<_Float16>(b)}));
    }
};

template <typename T>
__device__ __forceinline__ void unpack8(u32x4_t x, float (&y)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[2 * i] = T::lo(x[i]);
        y[2 * i + 1] = T::hi(x[i]);
    }
}

template <typename T>
__device__ __forceinline__ float weight_at(const void* w, bool w32, int d) {
    if (!w) return 1.0f;
    return w32 ? static_cast<const float*>(w)[d] : T::lo(static_cast<const uint16_t*>(w)[d]);
}

// Sequence that owns token t (the last one that starts at or before it), or -1.
__device__ __forceinline__ int owner_of(const QkParams& a, int t) {
    int lo = 0, n = a.S;
    while (true) {
        const int stride = (n + 63) / 64;
        const int i = lane_id() * stride;
        const uint64_t m = __ballot(i < n && a.start[lo + i] <= t);
        if (m == 0) return -1;
        const int k = 63 - __builtin_clzll(m);
        lo += k * stride;
        n = min(stride, n - k * stride);
        if (stride == 1) return t < a.start[lo + 1] ? lo : -1;
    }
}

// 8 dims of a lane to a row of codes and, by the first lane of a block, its
// exponent.
template <typename T, typename C>
__device__ __forceinline__ void store_codes(const float (&y)[8], uint8_t* row, uint8_t* exps, int c) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(y[j]) & 0x7FFFFFFFu);
    top = max(top, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(top), 0xB1, 0xF, 0xF, true)));
    top = max(top, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(top), 0x4E, 0xF, 0xF, true)));
    const uint32_t e = block_exponent<C, T::kHalf>(top);
    uint32_t w[C::kWords];
    block_encode<C, T::kHalf>(y, e, w);
    if constexpr (C::kWords == 2)
        *reinterpret_cast<uint2*>(row + 8 * c) = make_uint2(w[0], w[1]);
    else
        *reinterpret_cast<uint32_t*>(row + 4 * c) = w[0];
    if (c % 4 == 0) exps[c / 4] = static_cast<uint8_t>(e);
}

template <typename T, int D, typename C>
__global__ __launch_bounds__(256, 6) void qk_norm_rope_kernel(QkParams a) {
    constexpr int L = D / 8;        // lanes of a head
    constexpr int NG = 256 / L;     // heads at a time
    __shared__ float2 s_cs[kMaxTokens][D / 2];
    constexpr bool kCodes = C::kBits != 16;
    __shared__ int64_t s_slot[kMaxTokens];   // element offset of the token's row in the pages, -1: not stored
    __shared__ int64_t s_exp[kCodes ? kMaxTokens : 1];   // and of its exponents
    __shared__ __align__(16) float s_w[2][D];
    __shared__ int s_pos[kMaxTokens];
    __shared__ int s_own[kMaxTokens];
    const int tid = threadIdx.x, c = tid % L, g = tid / L;
    const int t0 = blockIdx.x * a.tokens;
    const int nt = min(a.tokens, a.N - t0);
    const int HT = a.Hq + a.Hk + (a.paged ? a.Hk : 0);
    const int pairs = nt * HT;

    // heads of this lane group: loads first
    u32x4_t x[kInFlight];
    auto token_of = [&](int p) { return HT > 1 ? static_cast<int>(__umulhi(static_cast<uint32_t>(p), a.div)) : p; };
    auto source = [&](int p) -> const uint16_t* {
        const int ti = token_of(p);
        const int64_t t = t0 + ti;
        const int h = p - ti * HT;
        if (h < a.Hq) return a.q + t * a.q_ts + h * a.q_hs + 8 * c;
        if (h < a.Hq + a.Hk) return a.k + t * a.k_ts + (h - a.Hq) * a.k_hs + 8 * c;
        return a.v + t * a.v_ts + (h - a.Hq - a.Hk) * a.v_hs + 8 * c;
    };
    auto fetch = [&](int p0) {
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            const int p = p0 + i * NG;
            if (p < pairs) x[i] = *reinterpret_cast<const u32x4_t*>(source(p));
        }
    };
    fetch(g);
    if (tid < 2 * D) s_w[tid / D][tid % D] = weight_at<T>(tid < D ? a.qw : a.kw, a.w32, tid % D);

    // positions and slots: a wave per token
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    for (int i = wave; i < nt; i += 4) {
        const int t = t0 + i;
        int pos = 0, own = 1;
        int64_t slot = -1, exp = 0;
        if (a.positions) {
            pos = a.pos64 ? static_cast<int>(static_cast<const int64_t*>(a.positions)[t])
                          : static_cast<const int32_t*>(a.positions)[t];
        } else {
            const int s = owner_of(a, t);
            own = s >= 0;
            if (own) {
                const int b = max(a.start[s], 0), e = min(a.start[s + 1], a.N);
                pos = clampi(a.lens[s], 0, a.capacity) - (e - b) + (t - b);
                if (pos >= 0) {
                    const int page = a.table ? a.table[s * a.table_s + (pos >> a.page_shift)] : s;
                    if (page >= 0 && page < a.n_pages) {
                        slot = page * a.page_s + (pos & ((1u << a.page_shift) - 1u)) * a.ko_ts;
                        if constexpr (kCodes) exp = page * a.e_page_s + (pos & ((1u << a.page_shift) - 1u)) * a.e_ts;
                    }
                }
            }
        }
        if (lane_id() == 0) {
            s_pos[i] = pos;
            s_own[i] = own;
            s_slot[i] = slot;
            if constexpr (kCodes) s_exp[i] = exp;
        }
    }
    __syncthreads();
    for (int i = tid; i < nt * a.half; i += 256) {
        const int t = i / a.half, f = i % a.half;
        const double turns = static_cast<double>(s_pos[t]) * static_cast<double>(a.inv_freq[f]) *
                             0.15915494309189533577;
        float sn, cs;
        const double d = turns - rint(turns);
        const float near = static_cast<float>(d);
        sincospif(2.0f * near, &sn, &cs);
        if constexpr (kCodes) {   // sine and cosine of the rest, r and 1
            const float r = 6.2831855f * static_cast<float>(d - near);
            const float sn0 = sn;
            sn = fmaf(cs, r, sn);
            cs = fmaf(-sn0, r, cs);
        }
        s_cs[t][f] = make_float2(cs, sn);
    }
    __syncthreads();

    const int hc = a.half / 8;      // lanes of half a rotation
    const int lane = lane_id();
    const int partner = (lane & ~(L - 1)) | (c < hc ? c + hc : (c < 2 * hc ? c - hc : c));
    const float sign = c < hc ? -1.0f : 1.0f;
    for (int p0 = g; p0 < pairs; p0 += kInFlight * NG) {
        if (p0 != g) fetch(p0);
#pragma unroll
        for (int i = 0; i < kInFlight; ++i) {
            const int p = p0 + i * NG;
            if (p >= pairs) break;
            const int ti = token_of(p), h = p - ti * HT;
            const int64_t t = t0 + ti;
            if (!s_own[ti]) continue;
            const bool is_v = h >= a.Hq + a.Hk, is_q = h < a.Hq;
            if (!kCodes && is_v) {   // copied
                if (s_slot[ti] >= 0)
                    *reinterpret_cast<u32x4_t*>(a.vo + s_slot[ti] + (h - a.Hq - a.Hk) * a.ko_hs + 8 * c) = x[i];
                continue;
            }
            float y[8];
            unpack8<T>(x[i], y);
            if (!(kCodes && is_v) && (is_q ? a.qw != nullptr : a.kw != nullptr)) {
                float ss = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) ss += y[j] * y[j];
                ss += dpp_f32<0xB1>(ss);
                ss += dpp_f32<0x4E>(ss);
                ss += dpp_f32<0x141>(ss);
                if (L == 16) ss += dpp_f32<0x140>(ss);
                const float inv = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = y[j] * inv * s_w[is_q ? 0 : 1][8 * c + j];
            }
            if (!(kCodes && is_v) && a.half) {
                if (a.interleaved) {
                    if (8 * c < 2 * a.half) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 cs = s_cs[ti][4 * c + j];
                            const float u = y[2 * j], w = y[2 * j + 1];
                            y[2 * j] = u * cs.x - w * cs.y;
                            y[2 * j + 1] = w * cs.x + u * cs.y;
                        }
                    }
                } else {
                    float z[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[j] = __shfl(y[j], partner);
                    if (c < 2 * hc) {
                        const int f0 = 8 * (c < hc ? c : c - hc);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float2 cs = s_cs[ti][f0 + j];
                            y[j] = y[j] * cs.x + sign * z[j] * cs.y;
                        }
                    }
                }
            }
            if constexpr (kCodes) {
                if (!is_q) {
                    const int kv = h - a.Hq - (is_v ? a.Hk : 0);
                    if (s_slot[ti] >= 0)
                        store_codes<T, C>(y, reinterpret_cast<uint8_t*>(is_v ? a.vo : a.ko) + s_slot[ti] + kv * a.ko_hs,
                                          (is_v ? a.ve : a.ke) + s_exp[ti] + kv * a.e_hs, c);
                    continue;
                }
            }
            const u32x4_t o = u32x4_t{T::pack(y[0], y[1]), T::pack(y[2], y[3]), T::pack(y[4], y[5]), T::pack(y[6], y[7])};
            if (is_q)
                *reinterpret_cast<u32x4_t*>(a.qo + t * a.qo_ts + h * a.qo_hs + 8 * c) = o;
            else if (!a.paged)
                *reinterpret_cast<u32x4_t*>(a.ko + t * a.ko_ts + (h - a.Hq) * a.ko_hs + 8 * c) = o;
            else if (s_slot[ti] >= 0)
                *reinterpret_cast<u32x4_t*>(a.ko + s_slot[ti] + (h - a.Hq) * a.ko_hs + 8 * c) = o;
        }
    }
}

template <typename T, int D>
void launch(const QkParams& P, int format, int grid, hipStream_t st) {
    switch (format) {
        case IMI_FP8: qk_norm_rope_kernel<T, D, Fp8><<<grid, 256, 0, st>>>(P); break;
        case IMI_INT8: qk_norm_rope_kernel<T, D, Int8><<<grid, 256, 0, st>>>(P); break;
        case IMI_FP4: qk_norm_rope_kernel<T, D, Fp4><<<grid, 256, 0, st>>>(P); break;
        default: qk_norm_rope_kernel<T, D, Raw16><<<grid, 256, 0, st>>>(P);
    }
}

}  // namespace
}  // namespace imi

extern "C" int imi_qk_norm_rope(const imi_qk_norm_rope_args* a, imi_stream_t stream) {
    using namespace imi;
    clear_error();
    IMI_REQUIRE(a, IMI_ERR_INVALID, "null argument");
    const imi_paged_batch& b = a->batch;
    const bool paged = a->key_pages != nullptr;
    IMI_REQUIRE(a->dtype == IMI_BF16 || a->dtype == IMI_FP16, IMI_ERR_UNSUPPORTED, "dtype=%d is not bf16 or fp16",
                a->dtype);
    IMI_REQUIRE(a->dim == 64 || a->dim == 128, IMI_ERR_UNSUPPORTED, "dim=%d is not 64 or 128", a->dim);
    IMI_REQUIRE(a->query_heads >= 0 && a->kv_heads >= 0 &&
                    static_cast<int64_t>(a->query_heads) + 2 * static_cast<int64_t>(a->kv_heads) <= 65535,
                IMI_ERR_INVALID, "bad heads (query_heads=%d, kv_heads=%d)", a->query_heads, a->kv_heads);
    IMI_REQUIRE(a->rotary >= 0 && a->rotary <= a->dim && a->rotary % 16 == 0, IMI_ERR_UNSUPPORTED,
                "rotary=%d must be a multiple of 16 up to dim=%d", a->rotary, a->dim);
    IMI_REQUIRE(a->rotary == 0 || a->inv_freq, IMI_ERR_INVALID, "rotary=%d without inv_freq", a->rotary);
    IMI_REQUIRE(a->eps >= 0.0f && a->eps <= 1e30f, IMI_ERR_INVALID, "eps=%g must be finite and >= 0",
                static_cast<double>(a->eps));
    IMI_REQUIRE(b.n_tokens >= 0, IMI_ERR_INVALID, "n_tokens=%d", b.n_tokens);
    if (b.n_tokens == 0 || a->query_heads + a->kv_heads == 0) return IMI_OK;
    IMI_REQUIRE(paged || a->positions, IMI_ERR_INVALID, "neither positions nor pages");
    IMI_REQUIRE((a->query_heads == 0 || (a->query && a->query_out)) &&
                    (a->kv_heads == 0 || (a->key && (paged ? a->value && a->value_pages : a->key_out != nullptr))),
                IMI_ERR_INVALID, "null tensor");
    const void* ptrs[] = {a->query, a->key, a->value, a->query_out, a->key_out, a->key_pages, a->value_pages};
    for (const void* p : ptrs)
        IMI_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, IMI_ERR_INVALID, "tensors must be 16-byte aligned");
    const int64_t strides[] = {a->query_token_stride, a->query_head_stride, a->key_token_stride,
                               a->key_head_stride,    a->value_token_stride, a->value_head_stride,
                               a->query_out_token_stride, a->query_out_head_stride, a->key_out_token_stride,
                               a->key_out_head_stride, a->page_stride, a->head_stride, a->row_stride};
    for (const int64_t s : strides)
        IMI_REQUIRE(s >= 0 && s % 8 == 0, IMI_ERR_INVALID, "strides must be multiples of 8 elements (got %lld)",
                    static_cast<long long>(s));
    QkParams P{};
    if (paged) {
        if (b.n_seqs == 0) return IMI_OK;
        if (const int rc = validate_batch(&b)) return rc;
        P.table = b.page_table;
        P.lens = b.lens;
        P.start = b.query_start;
        P.table_s = b.table_stride;
        P.S = b.n_seqs;
        P.n_pages = b.n_pages;
        P.page_shift = b.page_table ? __builtin_ctz(static_cast<unsigned>(b.page_size)) : 31;
        P.capacity = static_cast<int>(batch_capacity(&b));
        if (const int rc = validate_format(a->format, a->dim, a->key_exponents, a->value_exponents, a->page_stride,
                                           a->head_stride, a->row_stride, a->exponent_page_stride,
                                           a->exponent_head_stride, a->exponent_row_stride, b.page_size))
            return rc;
        P.ko = static_cast<uint16_t*>(a->key_pages);
        P.vo = static_cast<uint16_t*>(a->value_pages);
        P.ke = a->key_exponents;
        P.ve = a->value_exponents;
        P.e_page_s = a->exponent_page_stride;
        P.e_hs = a->exponent_head_stride;
        P.e_ts = a->exponent_row_stride;
        P.ko_ts = a->row_stride;
        P.ko_hs = a->head_stride;
        P.page_s = a->page_stride;
    } else {
        P.ko = a->key_out;
        P.ko_ts = a->key_out_token_stride;
        P.ko_hs = a->key_out_head_stride;
        P.positions = a->positions;
        P.pos64 = a->positions_64 != 0;
    }
    P.paged = paged;
    P.q = a->query;
    P.k = a->key;
    P.v = a->value;
    P.qo = a->query_out;
    P.q_ts = a->query_token_stride;
    P.q_hs = a->query_head_stride;
    P.k_ts = a->key_token_stride;
    P.k_hs = a->key_head_stride;
    P.v_ts = a->value_token_stride;
    P.v_hs = a->value_head_stride;
    P.qo_ts = a->query_out_token_stride;
    P.qo_hs = a->query_out_head_stride;
    P.inv_freq = a->inv_freq;
    P.qw = a->query_weight;
    P.kw = a->key_weight;
    P.w32 = a->weight_fp32 != 0;
    P.N = b.n_tokens;
    P.Hq = a->query_heads;
    P.Hk = a->kv_heads;
    P.half = a->rotary / 2;
    P.interleaved = a->interleaved != 0;
    P.eps = a->eps;
    const int heads = P.Hq + P.Hk * (paged ? 2 : 1);
    const int at_once = 256 / (a->dim / 8);
    P.tokens = std::min(kMaxTokens, std::max(1, 2 * kInFlight * at_once / heads));
    P.tokens = std::max(1, std::min(P.tokens, P.N / (2 * device_cus())));
    P.div = static_cast<uint32_t>((uint64_t(1) << 32) / heads + 1);
    const int grid = (P.N + P.tokens - 1) / P.tokens;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int format = paged ? a->format : IMI_ROWS;
    if (a->dtype == IMI_BF16) {
        if (a->dim == 128) launch<BF16, 128>(P, format, grid, st);
        else launch<BF16, 64>(P, format, grid, st);
    } else {
        if (a->dim == 128) launch<FP16, 128>(P, format, grid, st);
        else launch<FP16, 64>(P, format, grid, st);
    }
    IMI_LAUNCH_CHECK("qk_norm_rope_kernel");
    return IMI_OK;
}
