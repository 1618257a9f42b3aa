// Paged 8-bit KV cache (vrt_kv8_*): what its kernels and host entry points
// share.  The layout and the rule of quantisation stand in vortexrt_b200.h.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "vrt_device.cuh"
#include "vrt_internal.hpp"

namespace vrt {

constexpr uint32_t kKv8Page = VRT_KV8_PAGE;
constexpr uint32_t kKv8MaxGroup = 8;  // query heads per KV head

// Device status bit: a length, an offset or a page id outside its array.
constexpr uint32_t kStatusKv8Range = 1u << 5;

struct Kv8View {
    int8_t* k;
    int8_t* v;
    float* k_scale;
    float* v_scale;
    void* k_tail;
    void* v_tail;
    const int32_t* table;
    uint32_t kv, pages, max_seqs, pps;
};

// A row of `rows` tokens: which sequences, where.
struct Kv8Append {
    Kv8View c;
    const void* k;
    const void* v;
    uint64_t stride;  // elements between rows
    const int32_t* start;
    const int32_t* cu;  // NULL: one row for each sequence
    uint32_t max_new;
    uint32_t* status;
};

struct Kv8Read {
    Kv8View c;
    const int32_t* start;
    const int32_t* cu;
    uint32_t max_rows;
    float* k_out;
    float* v_out;
    uint32_t* status;
};

struct Kv8Attn {
    Kv8View c;
    const void* q;
    void* out;
    float* lse;
    uint64_t q_stride, out_stride;
    const int32_t* len;
    const int32_t* cu;  // NULL: one query for each sequence
    const int32_t* prefix;
    uint32_t H, count, max_new, max_len, window;
    float scale, softcap;
    int dtype;
    uint32_t* status;
};

// The visible pages of a row split over `splits` CTAs, whose outputs a second
// kernel joins (kv8_join).
struct Kv8Split {
    Kv8Attn a;
    uint32_t tile;    // query tokens that see their pages together
    uint32_t chunk;   // pages of one split at most
    uint32_t splits;  // of the longest sequence
    float* part;      // [count][max_new][H][splits][head_dim] outputs of a split alone
    float* part_ml;   // [count][max_new][H][splits][2] its maximum (base 2) and sum of weights
};

// Pool index of page `page` of sequence `seq`, -1 (and the status bit) when
// the table names none.
__device__ __forceinline__ int kv8_page(const Kv8View& c, uint32_t seq, uint32_t page, uint32_t* status) {
    const int id = page < c.pps ? c.table[static_cast<uint64_t>(seq) * c.pps + page] : -1;
    if (static_cast<uint32_t>(id) < c.pages) return id;
    atomicOr(status, kStatusKv8Range);
    return -1;
}

// Rows [r0, r0 + n) of sequence `seq` among the call's rows.
__device__ __forceinline__ uint32_t kv8_rows(const int32_t* cu, uint32_t seq, uint32_t most, uint32_t* status,
                                             int64_t& r0) {
    if (!cu) {
        r0 = seq;
        return 1;
    }
    r0 = cu[seq];
    const int64_t n = static_cast<int64_t>(cu[seq + 1]) - r0;
    if (r0 >= 0 && n >= 0 && n <= static_cast<int64_t>(most)) return static_cast<uint32_t>(n);
    atomicOr(status, kStatusKv8Range);
    return r0 < 0 || n < 0 ? 0u : most;
}

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N consecutive elements (a multiple of 16 bytes, 16-byte aligned) as fp32.
template <typename T, int N>
__device__ __forceinline__ void load_row(const T* p, float (&x)[N]) {
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < N / E; ++i) {
        const uint4 u = reinterpret_cast<const uint4*>(p)[i];
        const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int j = 0; j < E; ++j) x[i * E + j] = to_f32(e[j]);
    }
}

// The largest magnitude of a row piece, NaN ignored.
template <int N>
__device__ __forceinline__ float max_abs(const float (&x)[N]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, fabsf(x[i]));
    return m;
}

// The smallest key a query of position `pos` may see through the window.
__host__ __device__ inline int64_t kv8_window_lo(int64_t pos, uint32_t window) {
    return window && pos + 1 > static_cast<int64_t>(window) ? pos + 1 - window : 0;
}

// Pages that the queries i0 .. i1 (of the call's n rows of a sequence) see:
// [0, a) and [b0, b1).  lo: first key in the window of query i0.
struct Kv8Span {
    int64_t len, lo, prefix;
    uint32_t a, b0, b1;
    __device__ __forceinline__ uint32_t count() const { return a + b1 - b0; }
    __device__ __forceinline__ uint32_t page(uint32_t i) const { return i < a ? i : b0 + i - a; }
};

__device__ __forceinline__ Kv8Span kv8_span(const Kv8Attn& p, uint32_t seq, uint32_t n, uint32_t i0, uint32_t i1) {
    Kv8Span s;
    const int64_t limit = min(static_cast<int64_t>(p.max_len), static_cast<int64_t>(p.c.pps) * kKv8Page);
    const int64_t len = p.len[seq];
    if (len < 0 || len > limit) atomicOr(p.status, kStatusKv8Range);
    s.len = max(static_cast<int64_t>(0), min(len, limit));
    s.lo = kv8_window_lo(s.len - n + i0, p.window);
    s.prefix = p.prefix ? max(static_cast<int64_t>(0), min(static_cast<int64_t>(p.prefix[seq]), s.len)) : 0;
    const int64_t end = max(static_cast<int64_t>(0), s.len - n + i1 + 1);
    s.a = static_cast<uint32_t>((s.prefix + kKv8Page - 1) / kKv8Page);
    s.b1 = max(s.a, static_cast<uint32_t>((end + kKv8Page - 1) / kKv8Page));
    s.b0 = min(s.b1, max(s.a, static_cast<uint32_t>(s.lo / kKv8Page)));
    return s;
}

// The splits that n visible pages use (none longer than `chunk`) and the
// pages of each: even shares.
__device__ __forceinline__ uint32_t kv8_used(uint32_t n, uint32_t chunk) { return n ? (n + chunk - 1) / chunk : 1u; }
__device__ __forceinline__ uint32_t kv8_share(uint32_t n, uint32_t used) { return (n + used - 1) / used; }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kKv8Lift = 14.0f;  // weights are held times 2^14

// What a row of maximum mx weighs its scores from (base 2): the lift below it.
// From 2^24 up a step of fp32 is 2 and more, and the lift could round up to 16,
// past fp16: then from the maximum itself.
__device__ __forceinline__ float kv8_base(float mx) {
    const float m = mx - kKv8Lift;
    return mx - m > 15.0f ? mx : m;
}

// ln of a sum l of weights 2^(z - m): nothing seen -> -inf, NaN stays.
__device__ __forceinline__ float kv8_lse(float m, float l) {
    return l == 0.0f ? -INFINITY : (m == -INFINITY ? l : m / kLog2e + logf(l));
}

// What a query row is multiplied by, so that its largest magnitude m comes to
// [2^14, 2^15): a power of two among the normal numbers, 1 for 0, infinity and NaN.
__device__ __forceinline__ float kv8_row_unit(float m) {
    const int ex = static_cast<int>(__float_as_uint(m) >> 23);
    const int up = m > 0.0f && ex < 255 ? max(-126, min(126, 14 - (ex - 127))) : 0;
    return __uint_as_float(static_cast<uint32_t>(up + 127) << 23);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Codes 0, 1 (lo) or 2, 3 (hi) of a word whose bytes were offset by 128, as
// two fp16: the byte under the exponent of 1024, less 1024 + 128.
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) {
    const uint32_t b = __byte_perm(w, 0x64646464u, 0x4140u);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&b), __float2half2_rn(1152.0f));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) {
    const uint32_t b = __byte_perm(w, 0x64646464u, 0x4342u);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&b), __float2half2_rn(1152.0f));
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The same times 2^-kKv8Lift (exact), for values: they meet weights that are held
// times 2^kKv8Lift, and the products are sums of at most the values' own size,
// which fp32 holds as far as it holds the values.
__device__ __forceinline__ uint32_t value_codes(uint32_t b) {
    const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&b), __float2half2_rn(0x1p-14f), __float2half2_rn(-1152.0f * 0x1p-14f));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t value_codes_lo(uint32_t w) { return value_codes(__byte_perm(w, 0x64646464u, 0x4140u)); }
__device__ __forceinline__ uint32_t value_codes_hi(uint32_t w) { return value_codes(__byte_perm(w, 0x64646464u, 0x4342u)); }
constexpr float kKv8Unlift = 16384.0f;  // what such a sum is multiplied by before it is divided by the weights'

__device__ __forceinline__ uint32_t pack_half(__half a, __half b) {
    return static_cast<uint32_t>(__half_as_ushort(a)) | static_cast<uint32_t>(__half_as_ushort(b)) << 16;
}

// softcap * tanh(x / softcap), in base-2 units.  f32 rows take tanhf, off by a
// few steps of the score.  16-bit rows take cap - 2 cap / (1 + e^2y), two special
// functions, whose difference is off by some 2^-23 of the cap whatever the
// score: up to a cap of 128 that is 2^-16 at most, far below a weight's rounding
// (2^-11).  Larger caps take tanhf for all rows.
constexpr float kKv8FastCap = 128.0f;
// 1 / cap, finite for the smallest caps too, and times 2 log2(e): a score of 0 stays 0
__device__ __forceinline__ float kv8_inv_cap(float cap) { return fminf(1.0f / cap, 1.0e38f); }
__device__ __forceinline__ float capped_fast(float x, float cap, float inv_cap) {
    const float e = ex2(x * inv_cap * (2.0f * kLog2e));
    return cap * kLog2e * (1.0f - __fdividef(2.0f, e + 1.0f));
}
__device__ __forceinline__ float capped_exact(float x, float cap, float inv_cap) { return cap * tanhf(x * inv_cap) * kLog2e; }
template <bool EXACT>
__device__ __forceinline__ float capped(float x, float cap, float inv_cap) {
    return EXACT || cap > kKv8FastCap ? capped_exact(x, cap, inv_cap) : capped_fast(x, cap, inv_cap);
}

// Splits of one (sequence, head) at most: the joining kernel's weights.
constexpr uint32_t kKv8MaxSplits = 128;

cudaError_t kv8_append(const Kv8Append& p, uint32_t hd, int dtype, uint32_t count, cudaStream_t s);
cudaError_t kv8_join(const Kv8Split& p, uint32_t hd, int dtype, cudaStream_t s);
cudaError_t kv8_decode(const Kv8Attn& p, uint32_t hd, int sms, void* workspace, cudaStream_t s);
cudaError_t kv8_prefill(const Kv8Attn& p, uint32_t hd, int sms, void* workspace, cudaStream_t s);
uint64_t kv8_prefill_workspace(int sms, uint32_t hd, int dtype, uint32_t kv, uint32_t heads, uint32_t count,
                               uint32_t max_new, uint32_t max_len);
cudaError_t kv8_prefill_tc(const Kv8Split& p, uint32_t hd, cudaStream_t s);
uint32_t kv8_prefill_tc_rows(uint32_t hd);  // rows of one of its CTAs
uint64_t kv8_decode_workspace(int sms, uint32_t hd, uint32_t kv, uint32_t heads, uint32_t count, uint32_t max_len);

}  // namespace vrt
