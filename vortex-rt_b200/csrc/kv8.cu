// Paged 8-bit KV cache: the kernels that write and read its pages, and the C
// entry points (vrt_kv8_*).  Its attention kernels are in kv8_decode.cu and kv8_prefill.cu.

#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "kv8.cuh"

namespace vrt {

constexpr int kKv8Threads = 256;

// x / s rounded half to even.  x * inv is within 127 * 2^-23 of x / s, so its
// rounding is right unless it falls next to a half; there, and for a scale so
// small that 1 / s is not finite, a division in 64 bits decides (two 24-bit
// numbers' quotient is no nearer to a half than 2^-33 unless it is one).
__device__ __forceinline__ int kv8_code(float x, float s, float inv) {
    const float t = x * inv;
    float r = rintf(t);
    if (!(fabsf(t - r) < 0.4999f)) {
        r = s > 0.0f ? static_cast<float>(rint(static_cast<double>(x) / static_cast<double>(s))) : 0.0f;
    }
    return static_cast<int>(fminf(fmaxf(r, -127.0f), 127.0f));
}

__device__ __forceinline__ uint32_t pack4(const int (&q)[4]) {
    return (q[0] & 0xff) | (q[1] & 0xff) << 8 | (q[2] & 0xff) << 16 | static_cast<uint32_t>(q[3]) << 24;
}

// Pages that n rows touch at most, wherever they start.
static uint32_t kv8_touched(uint32_t n) { return (n + kKv8Page - 2) / kKv8Page + 1; }

// CTA (b, g + kv * {K, V}, i): the b-th page of sequence i that the new rows
// touch, KV head g.  The page's rows (from the tail below `start`, else from
// the call) are held in registers, 8 threads a row: maximum, scale, codes.
// The CTA of a sequence's first page also brings the tail up to date, after
// it has read it: no other CTA touches that tail.  A page whose scale did not
// change keeps its old codes, so that a step of one token writes one row.
// Bound by HBM for prompts, by one round of dependent loads for single rows.
template <typename T, int HD>
__global__ void __launch_bounds__(kKv8Threads) kv8_append_kernel(const Kv8Append p) {
    constexpr int N = HD / 8;  // elements of a thread
    __shared__ uint32_t top[kKv8Threads / 32];
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
    const int64_t end = min(start + n, limit);
    const int64_t first = start / kKv8Page, page = first + blockIdx.x;
    if (page * kKv8Page >= end) return;

    const T* rows = static_cast<const T*>(is_v ? p.v : p.k) + static_cast<uint64_t>(g) * HD;
    T* tail = static_cast<T*>(is_v ? p.c.v_tail : p.c.k_tail) + (static_cast<uint64_t>(seq) * p.c.kv + g) * kKv8Page * HD;
    const int row = threadIdx.x / 8, col = threadIdx.x % 8 * N;
    const int64_t pos = page * kKv8Page + row;
    float x[N];
    if (pos >= end) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = 0.0f;
    } else {
        load_row<T, N>((pos < start ? tail + row * HD : rows + static_cast<uint64_t>(r0 + (pos - start)) * p.stride) + col, x);
    }
    // |x| as bits: ordered like the values, infinities and NaN on top
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    m = __reduce_max_sync(0xffffffffu, m);
    if (threadIdx.x % 32 == 0) top[threadIdx.x / 32] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kKv8Threads / 32; ++w) m = max(m, top[w]);
    const float s = m < 0x7f800000u ? __uint_as_float(m) / 127.0f : NAN;
    const float inv = s > 0.0f ? 1.0f / s : 0.0f;

    // the tail: new rows of the last page, when that is not full
    if (blockIdx.x == 0 && end % kKv8Page) {
        const int64_t lp = end / kKv8Page, at = lp * kKv8Page + row;
        if (at >= start && at < end) {
            const uint4* src = reinterpret_cast<const uint4*>(rows + static_cast<uint64_t>(r0 + (at - start)) * p.stride + col);
            uint4* dst = reinterpret_cast<uint4*>(tail + row * HD + col);
#pragma unroll
            for (int i = 0; i < static_cast<int>(N * sizeof(T) / 16); ++i) dst[i] = src[i];
        }
    }

    const int id = kv8_page(p.c, seq, static_cast<uint32_t>(page), p.status);
    if (id < 0) return;
    const uint64_t head = static_cast<uint64_t>(id) * p.c.kv + g;
    float* scale = (is_v ? p.c.v_scale : p.c.k_scale) + head;
    const int64_t kept = page * kKv8Page < start ? start - page * kKv8Page : 0;  // rows that the page already held
    const bool same = kept > 0 && *scale == s;
    __syncthreads();  // every thread has read the old scale
    if (threadIdx.x == 0) *scale = s;
    uint32_t w[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        int q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = s >= 0.0f ? kv8_code(x[4 * i + j], s, inv) : 0;
        w[i] = pack4(q);
    }
    if (!is_v) {
        if (same && (row < kept || pos >= end)) return;
        uint32_t* dst = reinterpret_cast<uint32_t*>(p.c.k + (head * kKv8Page + row) * HD + col);
        if constexpr (N == 8) {
            *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int i = 0; i < N / 16; ++i)
                reinterpret_cast<uint4*>(dst)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        }
        return;
    }
    int8_t* vp = p.c.v + head * HD * kKv8Page;
    if (same) {
        if (row >= kept && pos < end) {
#pragma unroll
            for (int i = 0; i < N; ++i) vp[(col + i) * kKv8Page + row] = static_cast<int8_t>(w[i / 4] >> 8 * (i % 4));
        }
        return;
    }
    // values lie [dim][token]: transposed through shared memory
#pragma unroll
    for (int i = 0; i < N / 4; ++i) tile[row * (HD / 4 + 1) + col / 4 + i] = w[i];
    __syncthreads();
    const uint8_t* t8 = reinterpret_cast<const uint8_t*>(tile);
    for (int c = threadIdx.x; c < HD * 2; c += kKv8Threads) {
        const int d = c % HD, r = c / HD * 16;
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            o[e] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) o[e] |= static_cast<uint32_t>(t8[(r + 4 * e + j) * (HD + 4) + d]) << 8 * j;
        }
        *reinterpret_cast<uint4*>(vp + d * kKv8Page + r) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

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
    const uint4* src = reinterpret_cast<const uint4*>((is_v ? p.c.v : p.c.k) + head * kKv8Page * HD);
    for (int c = threadIdx.x; c < HD * 2; c += kKv8Threads) {
        const uint4 u = src[c];
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        if (!is_v) {
            const int r = c / (HD / 16), d = c % (HD / 16) * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) tile[r * W + d + e] = w[e];
        } else {
            const int d = c / 2, r = c % 2 * 16;
            uint8_t* t8 = reinterpret_cast<uint8_t*>(tile);
#pragma unroll
            for (int e = 0; e < 16; ++e) t8[(r + e) * (W * 4) + d] = static_cast<uint8_t>(w[e / 4] >> 8 * (e % 4));
        }
    }
    __syncthreads();
    float* out = (is_v ? p.v_out : p.k_out) + static_cast<uint64_t>(g) * HD;
    const uint64_t stride = static_cast<uint64_t>(p.c.kv) * HD;
    for (int c = threadIdx.x; c < static_cast<int>(kKv8Page) * HD / 4; c += kKv8Threads) {
        const int r = c / (HD / 4), d = c % (HD / 4);
        const int64_t pos = page * kKv8Page + r;
        if (pos < start || pos >= end) continue;
        const uint32_t w = tile[r * W + d];
        float4 f;
        f.x = static_cast<float>(static_cast<int8_t>(w)) * s;
        f.y = static_cast<float>(static_cast<int8_t>(w >> 8)) * s;
        f.z = static_cast<float>(static_cast<int8_t>(w >> 16)) * s;
        f.w = static_cast<float>(static_cast<int8_t>(w >> 24)) * s;
        reinterpret_cast<float4*>(out + static_cast<uint64_t>(r0 + (pos - start)) * stride)[d] = f;
    }
}

cudaError_t kv8_append(const Kv8Append& p, uint32_t hd, int dtype, uint32_t count, cudaStream_t s) {
    const dim3 grid(kv8_touched(p.max_new), 2 * p.c.kv, count);
#define VRT_KA(TY, T, HD) \
    if (dtype == TY && hd == HD) return launch(kv8_append_kernel<T, HD>, grid, dim3(kKv8Threads), 0, s, false, p);
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

int check_cache(const vrt_kv8_cache* c) {
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
    VRT_TRY(check_cache(cache));
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
