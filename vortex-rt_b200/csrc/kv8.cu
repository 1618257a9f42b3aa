// Paged 8-bit KV cache: the kernels that write and read its pages, and the C
// entry points (vrt_kv8_*).  Its attention kernels are in kv8_decode.cu and kv8_prefill.cu.

#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "kv8.cuh"

namespace vrt {


// x / s rounded half to even, to a code.  The exact form: two 24-bit numbers'
// quotient is no nearer to a half than 2^-33 unless it is one, which a
// division in 64 bits tells apart.
__device__ __noinline__ int kv8_code_exact(float x, float s) {
    if (!(s > 0.0f)) return 0;  // a page of zeros, or with a NaN
    return static_cast<int>(fmin(fmax(rint(static_cast<double>(x) / static_cast<double>(s)), -127.0), 127.0));
}

__device__ __forceinline__ uint32_t pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040u), __byte_perm(c, d, 0x0040u), 0x5410u);
}

// Codes of N values, four to a word.  x * inv is within 127 * 2^-24 = 7.6e-6
// of x / s, so its nearest whole number, the low byte of x * inv + 1.5 * 2^23,
// is right unless it falls next to a half (then the exact form decides, as it
// does for a scale so small that 1 / s is not finite).
template <int N>
__device__ __forceinline__ void kv8_codes(const float (&x)[N], float s, float inv, uint32_t (&w)[N / 4]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        float far = 0.0f, sum = 0.0f;  // the largest distance from the whole number; NaN, if one is
        uint32_t b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float m = fmaf(x[i + j], inv, 12582912.0f), d = fmaf(x[i + j], inv, 12582912.0f - m);
            far = fmaxf(far, fabsf(d));
            sum += d;
            b[j] = __float_as_uint(m);
        }
        w[i / 4] = pack_bytes(b[0], b[1], b[2], b[3]);
        if (!(far < 0.49999f && sum == sum)) {
            w[i / 4] = pack_bytes(kv8_code_exact(x[i], s), kv8_code_exact(x[i + 1], s), kv8_code_exact(x[i + 2], s),
                                  kv8_code_exact(x[i + 3], s));
        }
    }
}

// Four rows of four bytes -> four columns.
__device__ __forceinline__ void transpose4(uint32_t (&a)[4]) {
    const uint32_t lo0 = __byte_perm(a[0], a[1], 0x5140u), lo1 = __byte_perm(a[2], a[3], 0x5140u);
    const uint32_t hi0 = __byte_perm(a[0], a[1], 0x7362u), hi1 = __byte_perm(a[2], a[3], 0x7362u);
    a[0] = __byte_perm(lo0, lo1, 0x5410u);
    a[1] = __byte_perm(lo0, lo1, 0x7632u);
    a[2] = __byte_perm(hi0, hi1, 0x5410u);
    a[3] = __byte_perm(hi0, hi1, 0x7632u);
}

// Pages that n rows touch at most, wherever they start.
static uint32_t kv8_touched(uint32_t n) { return (n + kKv8Page - 2) / kKv8Page + 1; }

// CTA (b, g + kv * {K, V}, i): the b-th page of sequence i that the new rows
// touch, KV head g.  The page's rows (from the tail below `start`, else from
// the call) are held in registers, 4 threads a row with every fourth 16-byte
// piece each: maximum, scale, codes.  The CTA of a sequence's first page also
// brings the tail up to date, after it has read it: no other CTA touches that
// tail.  A page whose scale did not change keeps its old codes, so that a step
// of one token writes one row.  8192 tokens of 16 heads of 128, bf16: 35 us for
// 16 us of bytes.  18 instructions a value (conversion, maximum, the two FMAs of
// the rounding, their check, transposes) are 18 us at full issue, which is 62%
// filled: 7 rounds of 8 CTAs an SM, each one chain of loads, a reduction, a
// barrier, a division and stores, with nothing else under way.  Single rows are
// bound by a round of dependent loads.
constexpr int kKaThreads = 128;

template <typename T, int HD>
__global__ void __launch_bounds__(kKaThreads) kv8_append_kernel(const Kv8Append p) {
    constexpr int P = 16 / sizeof(T), N = HD / 4, C = N / P;  // values of a piece, of a thread; its pieces
    __shared__ uint32_t top[kKaThreads / 32];
    __shared__ uint32_t tile[kKv8Page * (HD / 4 + 1)];
    const uint32_t g = blockIdx.y % p.c.kv, seq = blockIdx.z;
    const bool is_v = blockIdx.y >= p.c.kv;
    int64_t r0;
    const uint32_t n = kv8_rows(p.cu, seq, p.max_new, p.status, r0);
    const int64_t start = p.start[seq], limit = static_cast<int64_t>(p.c.pps) * kKv8Page;
    if (n == 0) return;
    if (start < 0 || start + n > limit) {
        if (threadIdx.x == 0) atomicOr(p.status, kStatusKv8Range);
        if (start < 0 || start >= limit) return;
    }
    // positions are below 2^31 from here on, and row 0 of the page is at `at`
    const int from = static_cast<int>(start), end = static_cast<int>(min(start + n, limit));
    const int page = from / static_cast<int>(kKv8Page) + static_cast<int>(blockIdx.x);
    if (page > (end - 1) / static_cast<int>(kKv8Page)) return;
    const int id = kv8_page(p.c, seq, static_cast<uint32_t>(page), p.status);

    const T* rows = static_cast<const T*>(is_v ? p.v : p.k) + static_cast<uint64_t>(g) * HD;
    T* tail = static_cast<T*>(is_v ? p.c.v_tail : p.c.k_tail) + (static_cast<uint64_t>(seq) * p.c.kv + g) * kKv8Page * HD;
    const int row = threadIdx.x / 4, first = threadIdx.x % 4 * P;
    const int pos = page * static_cast<int>(kKv8Page) + row;
    float x[N];
    if (pos >= end) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = 0.0f;
    } else {
        const T* src = (pos < from ? tail + row * HD : rows + static_cast<uint64_t>(r0 + (pos - from)) * p.stride) + first;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float y[P];
            load_row<T, P>(src + c * 4 * P, y);
#pragma unroll
            for (int j = 0; j < P; ++j) x[c * P + j] = y[j];
        }
    }
    // |x| as bits: ordered like the values, infinities and NaN on top
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    if (threadIdx.x % 32 == 0) top[threadIdx.x / 32] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kKaThreads / 32; ++w) m = max(m, top[w]);
    const float s = m < 0x7f800000u ? __uint_as_float(m) / 127.0f : NAN;
    const float inv = s > 0.0f ? 1.0f / s : 0.0f;

    // the tail: new rows of the last page, when that is not full
    if (blockIdx.x == 0 && end % static_cast<int>(kKv8Page)) {
        const int at = end / static_cast<int>(kKv8Page) * static_cast<int>(kKv8Page) + row;
        if (at >= from && at < end) {
            const T* src = rows + static_cast<uint64_t>(r0 + (at - from)) * p.stride + first;
            T* dst = tail + row * HD + first;
#pragma unroll
            for (int c = 0; c < C; ++c) *reinterpret_cast<uint4*>(dst + c * 4 * P) = *reinterpret_cast<const uint4*>(src + c * 4 * P);
        }
    }

    if (id < 0) return;
    const uint64_t head = static_cast<uint64_t>(id) * p.c.kv + g;
    float* scale = (is_v ? p.c.v_scale : p.c.k_scale) + head;
    const int kept = max(0, from - page * static_cast<int>(kKv8Page));  // rows that the page already held
    bool same = false;
    if (kept > 0) {
        same = *scale == s;
        __syncthreads();  // every thread has read the old scale
    }
    if (threadIdx.x == 0) *scale = s;
    uint32_t w[N / 4];
    kv8_codes<N>(x, s, inv, w);
    const bool fresh = !same || (row >= kept && pos < end);  // codes of this row are to be written
    if (!is_v) {
        if (!fresh) return;
        int8_t* dst = p.c.k + (head * kKv8Page + row) * HD + first;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if constexpr (P == 8) {
                *reinterpret_cast<uint2*>(dst + c * 4 * P) = make_uint2(w[2 * c], w[2 * c + 1]);
            } else {
                *reinterpret_cast<uint32_t*>(dst + c * 4 * P) = w[c];
            }
        }
        return;
    }
    int8_t* vp = p.c.v + head * HD * kKv8Page;
    if (same) {
        if (!fresh) return;
#pragma unroll
        for (int i = 0; i < N; ++i) vp[(i / P * 4 * P + first + i % P) * kKv8Page + row] = static_cast<int8_t>(w[i / 4] >> 8 * (i % 4));
        return;
    }
    // values lie [dim][token]: transposed through shared memory
#pragma unroll
    for (int i = 0; i < N / 4; ++i) tile[row * (HD / 4 + 1) + (i * 4 / P * 4 * P + first + i * 4 % P) / 4] = w[i];
    __syncthreads();
    // four tokens by four dims a thread; the eight lanes of a token group write whole 32-byte sectors
#pragma unroll
    for (int c = threadIdx.x; c < HD * 2; c += kKaThreads) {
        const int r = c % 8 * 4, d = c / 8;  // dims 4 d .. 4 d + 3
        uint32_t a[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = tile[(r + j) * (HD / 4 + 1) + d];
        transpose4(a);
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t*>(vp + (4 * d + j) * kKv8Page + r) = a[j];
    }
}

constexpr int kKv8Threads = 256;

// CTA (b, g + kv * {K, V}, i): code * scale of the b-th page that the rows of
// sequence i touch -> fp32 rows.  Values are transposed in shared memory.
// Bound by the writes: 4 bytes out for each byte in.
template <int HD>
__global__ void __launch_bounds__(kKv8Threads) kv8_read_kernel(const Kv8Read p) {
    constexpr int W = HD / 4 + 1;  // words of a tile row
    __shared__ uint32_t tile[kKv8Page * W];
    const uint32_t g = blockIdx.y % p.c.kv, seq = blockIdx.z;
    const bool is_v = blockIdx.y >= p.c.kv;
    int64_t r0;
    const uint32_t n = kv8_rows(p.cu, seq, p.max_rows, p.status, r0);
    const int64_t start = p.start[seq], limit = static_cast<int64_t>(p.c.pps) * kKv8Page;
    if (n == 0) return;
    if (start < 0 || start + n > limit) {
        if (threadIdx.x == 0) atomicOr(p.status, kStatusKv8Range);
        if (start < 0 || start >= limit) return;
    }
    const int64_t end = min(start + n, limit), page = start / kKv8Page + blockIdx.x;
    if (page * kKv8Page >= end) return;
    const int id = kv8_page(p.c, seq, static_cast<uint32_t>(page), p.status);
    if (id < 0) return;
    const uint64_t head = static_cast<uint64_t>(id) * p.c.kv + g;
    const float s = (is_v ? p.c.v_scale : p.c.k_scale)[head];
    const int8_t* src = (is_v ? p.c.v : p.c.k) + head * kKv8Page * HD;
    for (int c = threadIdx.x; c < HD * 2; c += kKv8Threads) {
        uint32_t w[4];
        if (!is_v) {
            const uint4 u = reinterpret_cast<const uint4*>(src)[c];
            w[0] = u.x;
            w[1] = u.y;
            w[2] = u.z;
            w[3] = u.w;
#pragma unroll
            for (int j = 0; j < 4; ++j) tile[c / (HD / 16) * W + c % (HD / 16) * 4 + j] = w[j];
        } else {
            const int r = c % 8 * 4, d = c / 8;  // four tokens by four dims
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint32_t*>(src + (4 * d + j) * kKv8Page + r);
            transpose4(w);
#pragma unroll
            for (int j = 0; j < 4; ++j) tile[(r + j) * W + d] = w[j];
        }
    }
    __syncthreads();
    float* out = (is_v ? p.v_out : p.k_out) + static_cast<uint64_t>(g) * HD;
    const uint64_t stride = static_cast<uint64_t>(p.c.kv) * HD;
    for (int c = threadIdx.x; c < static_cast<int>(kKv8Page) * HD / 4; c += kKv8Threads) {
        const int r = c / (HD / 4), d = c % (HD / 4);
        const int64_t pos = page * kKv8Page + r;
        if (pos < start || pos >= end) continue;
        // a byte offset by 128 under the exponent of 2^23, less 2^23 + 128: the code, without a conversion
        const uint32_t w = tile[r * W + d] ^ 0x80808080u;
        float4 f;
        f.x = (__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7550u)) - 8388736.0f) * s;
        f.y = (__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7551u)) - 8388736.0f) * s;
        f.z = (__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7552u)) - 8388736.0f) * s;
        f.w = (__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7553u)) - 8388736.0f) * s;
        reinterpret_cast<float4*>(out + static_cast<uint64_t>(r0 + (pos - start)) * stride)[d] = f;
    }
}

cudaError_t kv8_append(const Kv8Append& p, uint32_t hd, int dtype, uint32_t count, cudaStream_t s) {
    const dim3 grid(kv8_touched(p.max_new), 2 * p.c.kv, count);
#define VRT_KA(TY, T, HD) \
    if (dtype == TY && hd == HD) return launch(kv8_append_kernel<T, HD>, grid, dim3(kKaThreads), 0, s, false, p);
#define VRT_KA3(HD) VRT_KA(VRT_F32, float, HD) VRT_KA(VRT_F16, __half, HD) VRT_KA(VRT_BF16, __nv_bfloat16, HD)
    VRT_KA3(64) VRT_KA3(128) VRT_KA3(256)
#undef VRT_KA3
#undef VRT_KA
    return cudaErrorInvalidValue;
}

static cudaError_t kv8_read(const Kv8Read& p, uint32_t hd, uint32_t count, cudaStream_t s) {
    const dim3 grid(kv8_touched(p.max_rows), 2 * p.c.kv, count), block(kKv8Threads);
    switch (hd) {
        case 64: return launch(kv8_read_kernel<64>, grid, block, 0, s, false, p);
        case 128: return launch(kv8_read_kernel<128>, grid, block, 0, s, false, p);
        case 256: return launch(kv8_read_kernel<256>, grid, block, 0, s, false, p);
        default: return cudaErrorInvalidValue;
    }
}

// ------------------------------------------------------------- host checks

namespace {

// The context's device for the length of a call, then the caller's again.
struct DeviceScope {
    int before = -1;
    cudaError_t e;
    explicit DeviceScope(int device) {
        e = cudaGetDevice(&before);
        if (e == cudaSuccess && before != device) {
            e = cudaSetDevice(device);
        } else {
            before = -1;
        }
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
};

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

uint32_t type_size(int dtype) { return dtype == VRT_F32 ? 4u : 2u; }

uint32_t* status_word(vrt_ctx* ctx) { return reinterpret_cast<uint32_t*>(ctx->d_key) + 2; }

int check_shape(const vrt_kv8_cache* c) {
    if (!c) return fail(VRT_E_INVALID, "kv8: null argument");
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
        return fail(VRT_E_UNSUPPORTED, "kv8: head_dim %u is not 64, 128 or 256", c->head_dim);
    }
    if (c->dtype != VRT_F32 && c->dtype != VRT_F16 && c->dtype != VRT_BF16) return fail(VRT_E_INVALID, "kv8: unknown dtype %d", c->dtype);
    if (!c->kv_heads || c->kv_heads > 1024) return fail(VRT_E_INVALID, "kv8: kv_heads must be 1..1024");
    if (!c->pages || c->pages > 0x7fffffffu) return fail(VRT_E_INVALID, "kv8: pages must be 1..2^31-1");
    if (!c->max_seqs || c->max_seqs > 65535u) return fail(VRT_E_INVALID, "kv8: max_seqs must be 1..65535");
    if (!c->pages_per_seq || c->pages_per_seq > 0x7fffffffu / kKv8Page) {
        return fail(VRT_E_INVALID, "kv8: pages_per_seq must be 1..%u", 0x7fffffffu / kKv8Page);
    }
    return VRT_OK;
}

int check_cache(const vrt_kv8_cache* c) {
    VRT_TRY(check_shape(c));
    const void* ptrs[] = {c->d_k, c->d_v, c->d_k_scale, c->d_v_scale, c->d_k_tail, c->d_v_tail, c->d_table};
    for (const void* p : ptrs) {
        if (!p) return fail(VRT_E_INVALID, "kv8: the cache lacks an array");
    }
    if (!aligned16(c->d_k) || !aligned16(c->d_v) || !aligned16(c->d_k_tail) || !aligned16(c->d_v_tail)) {
        return fail(VRT_E_INVALID, "kv8: pages and tails must be 16-byte aligned");
    }
    return VRT_OK;
}

int check_batch(const vrt_kv8_cache* c, uint32_t count, uint32_t most, const char* what) {
    if (count > c->max_seqs) return fail(VRT_E_INVALID, "kv8: count %u exceeds the cache's %u sequences", count, c->max_seqs);
    if (!most || most > c->pages_per_seq * kKv8Page) {
        return fail(VRT_E_INVALID, "kv8: %s must be 1..%u, the tokens of a table row", what, c->pages_per_seq * kKv8Page);
    }
    return VRT_OK;
}

int check_rows(const void* p, uint64_t& stride, uint64_t width, int dtype, const char* what) {
    if (!p) return fail(VRT_E_INVALID, "kv8: %s is null", what);
    if (!stride) stride = width;
    if (stride < width) return fail(VRT_E_INVALID, "kv8: rows of %s overlap", what);
    if (!aligned16(p) || stride * type_size(dtype) % 16) {
        return fail(VRT_E_INVALID, "kv8: rows of %s must start on 16-byte boundaries", what);
    }
    return VRT_OK;
}

Kv8View view_of(const vrt_kv8_cache* c) {
    Kv8View v{};
    v.k = c->d_k;
    v.v = c->d_v;
    v.k_scale = c->d_k_scale;
    v.v_scale = c->d_v_scale;
    v.k_tail = c->d_k_tail;
    v.v_tail = c->d_v_tail;
    v.table = c->d_table;
    v.kv = c->kv_heads;
    v.pages = c->pages;
    v.max_seqs = c->max_seqs;
    v.pps = c->pages_per_seq;
    return v;
}

int check_heads(const vrt_kv8_cache* c, uint32_t heads) {
    if (!heads || heads % c->kv_heads || heads / c->kv_heads > kKv8MaxGroup) {
        return fail(VRT_E_INVALID, "kv8: %u query heads are not 1..%u for each of %u KV heads", heads, kKv8MaxGroup, c->kv_heads);
    }
    return VRT_OK;
}

int attention(vrt_ctx* ctx, const vrt_kv8_cache* cache, const vrt_kv8_attn* attn, const void* d_q, uint64_t q_stride,
              const int32_t* d_len, const int32_t* d_cu, uint32_t count, uint32_t max_new, uint32_t max_len,
              void* d_out, uint64_t out_stride, float* d_lse, void* d_workspace, uint64_t workspace_bytes,
              void* stream) {
    VRT_TRY(check_cache(cache));
    if (!attn || !d_len) return fail(VRT_E_INVALID, "kv8 attention: null argument");
    VRT_TRY(check_batch(cache, count, max_len, "max_len"));
    VRT_TRY(check_heads(cache, attn->heads));
    if (!std::isfinite(attn->scale)) return fail(VRT_E_INVALID, "kv8 attention: scale is not finite");
    if (!(attn->softcap >= 0.0f) || !std::isfinite(attn->softcap)) return fail(VRT_E_INVALID, "kv8 attention: softcap must be finite and >= 0");
    const uint64_t width = static_cast<uint64_t>(attn->heads) * cache->head_dim;
    VRT_TRY(check_rows(d_q, q_stride, width, cache->dtype, "q"));
    VRT_TRY(check_rows(d_out, out_stride, width, cache->dtype, "out"));
    VRT_TRY(check_batch(cache, count, max_new, "max_new"));
    uint64_t need = 0;
    VRT_TRY(vrt_kv8_workspace(ctx, cache, attn->heads, count, max_new, max_len, &need));
    if (need && (!d_workspace || workspace_bytes < need || !aligned16(d_workspace))) {
        return fail(VRT_E_INVALID, "kv8 attention: workspace of %llu bytes needed, 16-byte aligned (%llu given)",
                    static_cast<unsigned long long>(need), static_cast<unsigned long long>(d_workspace ? workspace_bytes : 0));
    }
    if (!ctx) return fail(VRT_E_INVALID, "kv8: null context");
    if (count == 0) return VRT_OK;
    if (static_cast<uint64_t>(max_new) / 16 * cache->kv_heads > 0x7fffffffull) {
        return fail(VRT_E_UNSUPPORTED, "kv8 attention: max_new %u on %u KV heads exceeds a grid", max_new, cache->kv_heads);
    }
    Kv8Attn p{};
    p.c = view_of(cache);
    p.q = d_q;
    p.out = d_out;
    p.lse = d_lse;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.len = d_len;
    p.cu = d_cu;
    p.prefix = attn->d_prefix;
    p.H = attn->heads;
    p.count = count;
    p.max_new = max_new;
    p.max_len = max_len;
    p.window = attn->window;
    p.scale = attn->scale;
    p.softcap = attn->softcap;
    p.dtype = cache->dtype;
    p.status = status_word(ctx);
    DeviceScope dev(ctx->device);
    VRT_CUDA(dev.e);
    const int sms = ctx->prop.multiProcessorCount;
    const auto run = d_cu ? kv8_prefill : kv8_decode;
    VRT_CUDA(run(p, cache->head_dim, sms, d_workspace, as_stream(ctx, stream)));
    return VRT_OK;
}

}  // namespace
}  // namespace vrt

using namespace vrt;

extern "C" {

int vrt_kv8_append(vrt_ctx* ctx, const vrt_kv8_cache* cache, const void* d_k, const void* d_v, uint64_t row_stride,
                   const int32_t* d_start, const int32_t* d_cu, uint32_t count, uint32_t max_new, void* stream) {
    clear_error();
    VRT_TRY(check_cache(cache));
    if (!d_start) return fail(VRT_E_INVALID, "kv8 append: null argument");
    if (!d_cu) max_new = 1;
    VRT_TRY(check_batch(cache, count, max_new, "max_new"));
    const uint64_t width = static_cast<uint64_t>(cache->kv_heads) * cache->head_dim;
    VRT_TRY(check_rows(d_k, row_stride, width, cache->dtype, "k"));
    VRT_TRY(check_rows(d_v, row_stride, width, cache->dtype, "v"));
    if (!ctx) return fail(VRT_E_INVALID, "kv8: null context");
    if (count == 0) return VRT_OK;
    Kv8Append p{};
    p.c = view_of(cache);
    p.k = d_k;
    p.v = d_v;
    p.stride = row_stride;
    p.start = d_start;
    p.cu = d_cu;
    p.max_new = max_new;
    p.status = status_word(ctx);
    DeviceScope dev(ctx->device);
    VRT_CUDA(dev.e);
    VRT_CUDA(kv8_append(p, cache->head_dim, cache->dtype, count, as_stream(ctx, stream)));
    return VRT_OK;
}

int vrt_kv8_read(vrt_ctx* ctx, const vrt_kv8_cache* cache, const int32_t* d_start, const int32_t* d_cu,
                 uint32_t count, uint32_t max_rows, float* d_k_out, float* d_v_out, void* stream) {
    clear_error();
    VRT_TRY(check_cache(cache));
    if (!d_start || !d_k_out || !d_v_out) return fail(VRT_E_INVALID, "kv8 read: null argument");
    if (!aligned16(d_k_out) || !aligned16(d_v_out)) return fail(VRT_E_INVALID, "kv8 read: outputs must be 16-byte aligned");
    if (!d_cu) max_rows = 1;
    VRT_TRY(check_batch(cache, count, max_rows, "max_rows"));
    if (!ctx) return fail(VRT_E_INVALID, "kv8: null context");
    if (count == 0) return VRT_OK;
    Kv8Read p{};
    p.c = view_of(cache);
    p.start = d_start;
    p.cu = d_cu;
    p.max_rows = max_rows;
    p.k_out = d_k_out;
    p.v_out = d_v_out;
    p.status = status_word(ctx);
    DeviceScope dev(ctx->device);
    VRT_CUDA(dev.e);
    VRT_CUDA(kv8_read(p, cache->head_dim, count, as_stream(ctx, stream)));
    return VRT_OK;
}

int vrt_kv8_workspace(vrt_ctx* ctx, const vrt_kv8_cache* cache, uint32_t heads, uint32_t count, uint32_t max_new,
                      uint32_t max_len, uint64_t* bytes) {
    clear_error();
    VRT_TRY(check_shape(cache));  // the arrays may come later
    if (!bytes) return fail(VRT_E_INVALID, "kv8 workspace: null argument");
    VRT_TRY(check_batch(cache, count, max_len, "max_len"));
    VRT_TRY(check_batch(cache, count, max_new, "max_new"));
    VRT_TRY(check_heads(cache, heads));
    if (!ctx) return fail(VRT_E_INVALID, "kv8: null context");
    const int sms = ctx->prop.multiProcessorCount;
    // of a single row each, either kernel may be meant
    *bytes = kv8_prefill_workspace(sms, cache->head_dim, cache->dtype, cache->kv_heads, heads, count, max_new, max_len);
    if (max_new == 1) {
        *bytes = std::max(*bytes, kv8_decode_workspace(sms, cache->head_dim, cache->kv_heads, heads, count, max_len));
    }
    return VRT_OK;
}

int vrt_kv8_decode(vrt_ctx* ctx, const vrt_kv8_cache* cache, const vrt_kv8_attn* attn, const void* d_q,
                   uint64_t q_stride, const int32_t* d_len, uint32_t count, uint32_t max_len, void* d_out,
                   uint64_t out_stride, float* d_lse, void* d_workspace, uint64_t workspace_bytes, void* stream) {
    clear_error();
    return attention(ctx, cache, attn, d_q, q_stride, d_len, nullptr, count, 1, max_len, d_out, out_stride, d_lse,
                     d_workspace, workspace_bytes, stream);
}

int vrt_kv8_prefill(vrt_ctx* ctx, const vrt_kv8_cache* cache, const vrt_kv8_attn* attn, const void* d_q,
                    uint64_t q_stride, const int32_t* d_len, const int32_t* d_cu, uint32_t count, uint32_t max_new,
                    uint32_t max_len, void* d_out, uint64_t out_stride, float* d_lse, void* d_workspace,
                    uint64_t workspace_bytes, void* stream) {
    clear_error();
    if (!d_cu) return fail(VRT_E_INVALID, "kv8 prefill: null argument");
    return attention(ctx, cache, attn, d_q, q_stride, d_len, d_cu, count, max_new, max_len, d_out, out_stride, d_lse,
                     d_workspace, workspace_bytes, stream);
}

}  // extern "C"
