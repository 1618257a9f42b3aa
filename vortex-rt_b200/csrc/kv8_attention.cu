// Attention over the paged 8-bit KV cache (kv8.cuh), one warp for each query
// token and head: a page's 32 tokens are the warp's 32 lanes.

#include "kv8.cuh"

namespace vrt {

// Lane t computes the score of token t of the page (its code row against the
// query row in shared memory), the warp keeps the running maximum and sum of
// the softmax, and lane l accumulates dims l + 32 j of the output from the
// transposed value page.
template <typename T, int HD>
__global__ void __launch_bounds__(32) kv8_attention_kernel(const Kv8Attn p) {
    __shared__ float qs[HD];
    __shared__ float ps[32];
    const int lane = threadIdx.x;
    const uint32_t j = blockIdx.x, h = blockIdx.y, seq = blockIdx.z, g = h / (p.H / p.c.kv);
    int64_t r0;
    const uint32_t n = kv8_rows(p.cu, seq, p.max_new, p.status, r0);
    if (j >= n) return;
    int64_t len = p.len[seq];
    const int64_t limit = min(static_cast<int64_t>(p.max_len), static_cast<int64_t>(p.c.pps) * kKv8Page);
    if (len < 0 || len > limit) {
        if (lane == 0) atomicOr(p.status, kStatusKv8Range);
        len = len < 0 ? 0 : limit;
    }
    const int64_t pos = len - n + j;
    const int64_t prefix = p.prefix ? min(max(static_cast<int64_t>(p.prefix[seq]), static_cast<int64_t>(0)), len) : 0;
    const T* q = static_cast<const T*>(p.q) + static_cast<uint64_t>(r0 + j) * p.q_stride + static_cast<uint64_t>(h) * HD;
    for (int d = lane; d < HD; d += 32) qs[d] = to_f32(q[d]);
    __syncwarp();
    const int64_t lo = kv8_window_lo(pos, p.window);
    float mx = -INFINITY, sum = 0.0f, acc[HD / 32];
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) acc[i] = 0.0f;
    const int64_t hi = max(min(pos + 1, len), prefix);
    for (int64_t pg = 0; pg * kKv8Page < hi; ++pg) {
        const int64_t t = pg * kKv8Page + lane;
        if (pg * kKv8Page >= prefix && (pg + 1) * kKv8Page <= lo) continue;  // before the window
        const int id = kv8_page(p.c, seq, static_cast<uint32_t>(pg), p.status);
        if (id < 0) continue;
        const uint64_t head = static_cast<uint64_t>(id) * p.c.kv + g;
        const bool ok = t < len && (t < prefix || (t <= pos && t >= lo));
        const int8_t* kr = p.c.k + (head * kKv8Page + lane) * HD;
        float s = 0.0f;
        for (int d = 0; d < HD; ++d) s = fmaf(qs[d], static_cast<float>(kr[d]), s);
        s = s * p.c.k_scale[head] * p.scale;
        if (p.softcap > 0.0f) s = p.softcap * tanhf(s / p.softcap);
        if (!ok) s = -INFINITY;
        float m = s;  // NaN is kept: fmaxf drops it, the exponential below does not
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        m = fmaxf(m, mx);
        const float c = mx == -INFINITY ? 0.0f : expf(mx - m);
        const float e = ok ? expf(s - (m == -INFINITY ? 0.0f : m)) : 0.0f;
        mx = m;
        sum = sum * c + warp_sum(e);
        ps[lane] = e;
        __syncwarp();
        const float vs = p.c.v_scale[head];
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
            const int8_t* vr = p.c.v + (head * HD + lane + 32 * i) * kKv8Page;
            float a = 0.0f;
            for (int u = 0; u < 32; ++u) a = fmaf(ps[u], static_cast<float>(vr[u]), a);
            acc[i] = fmaf(a, vs, acc[i] * c);
        }
        __syncwarp();
    }
    const bool none = sum == 0.0f;
    T* out = static_cast<T*>(p.out) + static_cast<uint64_t>(r0 + j) * p.out_stride + static_cast<uint64_t>(h) * HD;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) out[lane + 32 * i] = from_f32<T>(none ? 0.0f : acc[i] / sum);
    if (p.lse && lane == 0) p.lse[static_cast<uint64_t>(r0 + j) * p.H + h] = none ? -INFINITY : mx + logf(sum);
}

cudaError_t kv8_attention(const Kv8Attn& p, uint32_t hd, int dtype, cudaStream_t s) {
    const dim3 grid(p.max_new, p.H, p.count);
#define VRT_KT(TY, T, HD) \
    if (dtype == TY && hd == HD) return launch(kv8_attention_kernel<T, HD>, grid, dim3(32), 0, s, false, p);
#define VRT_KT3(HD) VRT_KT(VRT_F32, float, HD) VRT_KT(VRT_F16, __half, HD) VRT_KT(VRT_BF16, __nv_bfloat16, HD)
    VRT_KT3(64) VRT_KT3(128) VRT_KT3(256)
#undef VRT_KT3
#undef VRT_KT
    return cudaErrorInvalidValue;
}

}  // namespace vrt
