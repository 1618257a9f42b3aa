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
    uint32_t* status;
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

// The smallest key a query of position `pos` may see through the window.
__host__ __device__ inline int64_t kv8_window_lo(int64_t pos, uint32_t window) {
    return window && pos + 1 > static_cast<int64_t>(window) ? pos + 1 - window : 0;
}

cudaError_t kv8_append(const Kv8Append& p, uint32_t hd, int dtype, uint32_t count, cudaStream_t s);
cudaError_t kv8_attention(const Kv8Attn& p, uint32_t hd, int dtype, cudaStream_t s);
cudaError_t kv8_decode(const Kv8Attn& p, uint32_t hd, int dtype, int sms, void* workspace, cudaStream_t s);
uint64_t kv8_decode_workspace(int sms, uint32_t hd, uint32_t kv, uint32_t heads, uint32_t count, uint32_t max_len);

}  // namespace vrt
