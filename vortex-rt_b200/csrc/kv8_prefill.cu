// Prompt attention over the paged 8-bit KV cache (kv8.cuh): many query tokens
// of each sequence at once.  The form for f32 rows (and few rows of 64 dims),
// the choice between it and the tcgen05 form (kv8_prefill_tc.cu), and the
// kernels that join a split history.

#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>

#include "kv8.cuh"

namespace vrt {

// ------------------------------------------------------------ warp products
//
// CTA (tile, KV head, sequence x split): 64 rows = 64 / R query tokens of the
// R heads that share a KV head, 16 rows a warp, against one page of 32 tokens
// at a time.  The page's codes are turned into fp16 once for the CTA (shared
// memory, rows padded so that ldmatrix meets no bank conflict) while the next
// page's codes are on their way in registers; scores and outputs are
// mma.sync m16n8k16 with fp32 sums.  As in the single-token kernel
// (kv8_decode.cu) codes are exact, query rows and weights are fp16 or, for
// f32 rows, fp16 + fp16 remainder, and a page's products start from zero and
// join the fp32 sums by one FMA with the page's value scale.  tcgen05 sums in
// TMEM and cuts them at every step, which f32 outputs of long histories would
// show; its fp32 sums would have to leave TMEM for every key tile.
// Bound by latency: f32 rows of 128 dims take 255 registers, so 8 warps an SM,
// whose tensor pipe is active 37% of the time.  3x512 tokens behind histories
// to 4096, window 1024 (32/16 heads of 128): 186 us, with spills of 32 bytes (196
// at 256 dims).  Query fragments from
// shared memory and 12 warps an SM took 201-221 us.
constexpr int kKpRows = 64;
constexpr int kKpThreads = 128;

template <int HD, int TERMS>
struct KpShape {
    static constexpr int kQ = HD + 8, kK = HD + 8, kV = kKv8Page + 8;  // fp16 a row, padded
    static constexpr bool kQRegs = HD * TERMS <= 256;                  // query fragments stay in registers
    static constexpr uint32_t kBytes = (TERMS * kKpRows * kQ + kKv8Page * kK + HD * kV) * 2 + kKpRows * 4;
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const __half* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_addr(p))
                 : "memory");
}

// 16 codes -> 16 fp16
template <bool VALUES>
__device__ __forceinline__ void store_codes(__half* dst, uint4 u) {
    const uint32_t w[4] = {u.x ^ 0x80808080u, u.y ^ 0x80808080u, u.z ^ 0x80808080u, u.w ^ 0x80808080u};
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[2 * i] = VALUES ? value_codes_lo(w[i]) : codes_lo(w[i]);
        h[2 * i + 1] = VALUES ? value_codes_hi(w[i]) : codes_hi(w[i]);
    }
    reinterpret_cast<uint4*>(dst)[0] = make_uint4(h[0], h[1], h[2], h[3]);
    reinterpret_cast<uint4*>(dst)[1] = make_uint4(h[4], h[5], h[6], h[7]);
}

template <typename T, int HD, int TERMS>
__global__ void __launch_bounds__(kKpThreads) kv8_prefill_kernel(const Kv8Split p) {
    using Shape = KpShape<HD, TERMS>;
    constexpr int KS = HD / 16, NT = HD / 8;
    constexpr int C = 2 * HD / kKpThreads;  // 16-byte pieces of a page that a thread brings: 1, 2 or 4
    extern __shared__ __align__(16) uint8_t sm[];
    __half* qs = reinterpret_cast<__half*>(sm);           // [TERMS][rows][kQ]
    __half* ks = qs + TERMS * kKpRows * Shape::kQ;        // [page][kK]
    __half* vs = ks + kKv8Page * Shape::kK;               // [HD][kV]
    float* unit = reinterpret_cast<float*>(vs + HD * Shape::kV);  // [rows]

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
    const uint32_t R = p.a.H / p.a.c.kv, g = blockIdx.y, seq = blockIdx.z / p.splits, split = blockIdx.z % p.splits;
    pdl_trigger();
    int64_t r0;
    const uint32_t n = kv8_rows(p.a.cu, seq, p.a.max_new, p.a.status, r0);
    // the latest tokens, which see the most, start first
    const uint32_t tiles = (p.a.max_new + p.tile - 1) / p.tile, i0 = (tiles - 1 - blockIdx.x) * p.tile;
    if (i0 >= n) return;
    const uint32_t tokens = min(p.tile, n - i0);
    const Kv8Span span = kv8_span(p.a, seq, n, i0, i0 + tokens - 1);
    const uint32_t all = span.count(), used = kv8_used(all, p.chunk), share = kv8_share(all, used);
    if (split >= used) return;
    const uint32_t j0 = min(all, split * share), j1 = min(all, j0 + share);
    const int64_t pos0 = span.len - n + i0, pos1 = pos0 + tokens - 1, lo1 = kv8_window_lo(pos1, p.a.window);

    // pages travel: codes of the next one in registers
    uint4 kr[C], vr[C];
    float k_scale = 0.0f, v_scale = 0.0f;
    bool there = false;
    auto fetch = [&](uint32_t j) {
        const int id = kv8_page(p.a.c, seq, span.page(j), p.a.status);
        there = id >= 0;
        const uint64_t head = static_cast<uint64_t>(there ? id : 0) * p.a.c.kv + g;
        const uint4* kp = reinterpret_cast<const uint4*>(p.a.c.k + head * kKv8Page * HD);
        const uint4* vp = reinterpret_cast<const uint4*>(p.a.c.v + head * kKv8Page * HD);
#pragma unroll
        for (int i = 0; i < C; ++i) {
            kr[i] = __ldg(kp + tid + i * kKpThreads);
            vr[i] = __ldg(vp + tid + i * kKpThreads);
        }
        k_scale = there ? __ldg(p.a.c.k_scale + head) : 0.0f;
        v_scale = there ? __ldg(p.a.c.v_scale + head) : 0.0f;
    };
    if (j0 < j1) fetch(j0);

    // query rows: two threads a row
    {
        const uint32_t r = tid / 2, token = r / R, h = r % R;
        const int half = tid % 2 * (HD / 2);
        const bool live = token < tokens;
        const T* q = static_cast<const T*>(p.a.q) + static_cast<uint64_t>(r0 + i0 + (live ? token : 0)) * p.a.q_stride +
                     static_cast<uint64_t>(g * R + h) * HD + half;
        float m = 0.0f;
        for (int d = 0; d < HD / 2; d += 8) {
            float x[8];
            load_row<T, 8>(q + d, x);
            m = fmaxf(m, max_abs(x));
        }
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        const float mul = kv8_row_unit(m);
        if (half == 0) unit[r] = m < INFINITY ? 1.0f / mul : NAN;  // an infinity makes the row NaN, capped or not
        for (int d = 0; d < HD / 2; d += 8) {
            float x[8];
            load_row<T, 8>(q + d, x);
            __align__(16) __half hi[8];
            __align__(16) __half lo[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) split_f16(live ? x[e] * mul : 0.0f, hi[e], lo[e]);
            *reinterpret_cast<uint4*>(qs + r * Shape::kQ + half + d) = *reinterpret_cast<const uint4*>(hi);
            if (TERMS == 2) *reinterpret_cast<uint4*>(qs + (kKpRows + r) * Shape::kQ + half + d) = *reinterpret_cast<const uint4*>(lo);
        }
    }
    __syncthreads();
    const bool cap = p.a.softcap > 0.0f;
    const float factor = cap ? p.a.scale : p.a.scale * kLog2e, inv_cap = cap ? kv8_inv_cap(p.a.softcap) : 0.0f;
    float sc[2];
    int64_t pos[2], lo[2];  // this lane's rows 16 warp + g8 (+ 8)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t r = 16 * warp + g8 + 8 * i;
        sc[i] = unit[r] * factor;
        pos[i] = pos0 + r / R;
        lo[i] = kv8_window_lo(pos[i], p.a.window);
    }
    const __half* qrow = qs + (16 * warp + lane % 16) * Shape::kQ + lane / 16 * 8;
    uint32_t qf[Shape::kQRegs ? TERMS * KS : 1][4];
    if (Shape::kQRegs) {
#pragma unroll
        for (int t = 0; t < TERMS; ++t)
#pragma unroll
            for (int s = 0; s < KS; ++s) ldmatrix4(qf[t * KS + s], qrow + t * kKpRows * Shape::kQ + 16 * s);
    }

    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] = 0.0f;
    float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};

    for (uint32_t j = j0; j < j1; ++j) {
        __syncthreads();  // the page before has been read
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int c = tid + i * kKpThreads;
            store_codes<false>(ks + c / (HD / 16) * Shape::kK + c % (HD / 16) * 16, kr[i]);
            store_codes<true>(vs + c / 2 * Shape::kV + c % 2 * 16, vr[i]);
        }
        const float k_now = k_scale, v_now = v_scale;
        const bool here = there;
        const int64_t t0 = static_cast<int64_t>(span.page(j)) * kKv8Page;
        __syncthreads();
        if (j + 1 < j1) fetch(j + 1);

        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][e] = 0.0f;
        const __half* krow = ks + (lane % 8 + lane / 16 * 8) * Shape::kK + lane / 8 % 2 * 8;
        float part[4][4];  // f32 rows: each 64 dims on their own, joined by rounding additions
        float (&acc_s)[4][4] = TERMS == 2 ? part : s;
#pragma unroll
        for (int st = 0; st < KS; ++st) {
            if (TERMS == 2 && st % 4 == 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) part[i][e] = 0.0f;
            }
            uint32_t b0[4], b1[4];  // keys 0-7 and 8-15, 16-23 and 24-31, both k halves
            ldmatrix4(b0, krow + 16 * st);
            ldmatrix4(b1, krow + 16 * Shape::kK + 16 * st);
#pragma unroll
            for (int t = TERMS - 1; t >= 0; --t) {
                uint32_t a[4];
                if (Shape::kQRegs) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[e] = qf[t * KS + st][e];
                } else {
                    ldmatrix4(a, qrow + t * kKpRows * Shape::kQ + 16 * st);
                }
                mma_f16(acc_s[0], a[0], a[1], a[2], a[3], make_uint2(b0[0], b0[1]));
                mma_f16(acc_s[1], a[0], a[1], a[2], a[3], make_uint2(b0[2], b0[3]));
                mma_f16(acc_s[2], a[0], a[1], a[2], a[3], make_uint2(b1[0], b1[1]));
                mma_f16(acc_s[3], a[0], a[1], a[2], a[3], make_uint2(b1[2], b1[3]));
            }
            if (TERMS == 2 && st % 4 == 3) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[i][e] += part[i][e];
            }
        }
        // softmax: s[i][e] is row e / 2, key 8 i + 2 t4 + e % 2
        const bool full = here && (t0 + 32 <= span.prefix || (t0 + 31 <= pos0 && t0 >= lo1 && t0 + 32 <= span.len));
        float top[2] = {mx[0], mx[1]};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float& z = s[i][e];
                z = z * (k_now * sc[e >> 1]);
                if (cap) z = capped<TERMS == 2>(z, p.a.softcap, inv_cap);
                if (!full) {
                    const int64_t t = t0 + 8 * i + 2 * t4 + (e & 1);
                    const bool see = here && t < span.len && (t < span.prefix || (t <= pos[e >> 1] && t >= lo[e >> 1]));
                    if (!see) z = -INFINITY;
                }
                top[e >> 1] = fmaxf(top[e >> 1], z);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
        }
        if (__any_sync(0xffffffffu, top[0] != mx[0] || top[1] != mx[1])) {
            float f[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                f[i] = mx[i] == -INFINITY ? 0.0f : ex2(mx[i] - top[i]);
                sum[i] *= f[i];
                mx[i] = top[i];
            }
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][e] *= f[e >> 1];
        }
        const float m0[2] = {mx[0] == -INFINITY ? 0.0f : kv8_base(mx[0]), mx[1] == -INFINITY ? 0.0f : kv8_base(mx[1])};
        uint32_t ph[2][4], pl[2][4];  // weights as the A operand of two k-steps of 16 keys
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {  // this lane's two keys of row r
                const float w0 = ex2(s[i][2 * r] - m0[r]), w1 = ex2(s[i][2 * r + 1] - m0[r]);
                sum[r] += w0 + w1;
                const __half2 hi = __floats2half2_rn(w0, w1);
                ph[i >> 1][2 * (i & 1) + r] = *reinterpret_cast<const uint32_t*>(&hi);
                if (TERMS == 2) {
                    const float2 f = __half22float2(hi);
                    const __half2 lw = __floats2half2_rn(w0 - f.x, w1 - f.y);
                    pl[i >> 1][2 * (i & 1) + r] = *reinterpret_cast<const uint32_t*>(&lw);
                }
            }
        }
        // a page that a row does not see adds nothing to it, even if its scale is NaN
        float vz[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t a = max(t0, lo[i]), b = min(min(pos[i], span.len - 1), t0 + 31);
            vz[i] = full || (here && (t0 < span.prefix || a <= b)) ? v_now : 0.0f;
        }
        const __half* vrow = vs + (lane % 8) * Shape::kV + lane / 8 * 8;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            uint32_t b[4];  // 8 dims x 32 keys
            ldmatrix4(b, vrow + i * 8 * Shape::kV);
            float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (TERMS == 2) {
                mma_f16(o, pl[0][0], pl[0][1], pl[0][2], pl[0][3], make_uint2(b[0], b[1]));
                mma_f16(o, pl[1][0], pl[1][1], pl[1][2], pl[1][3], make_uint2(b[2], b[3]));
            }
            mma_f16(o, ph[0][0], ph[0][1], ph[0][2], ph[0][3], make_uint2(b[0], b[1]));
            mma_f16(o, ph[1][0], ph[1][1], ph[1][2], ph[1][3], make_uint2(b[2], b[3]));
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][e] = fmaf(o[e], vz[e >> 1], acc[i][e]);
        }
    }

#pragma unroll
    for (int i = 0; i < 2; ++i) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
        const uint32_t r = 16 * warp + g8 + 8 * i, token = r / R, h = g * R + r % R;
        if (token >= tokens) continue;
        const float l = sum[i], inv = l == 0.0f ? 0.0f : kKv8Unlift / l;
        if (used == 1) {
            const uint64_t row = static_cast<uint64_t>(r0 + i0 + token);
            T* out = static_cast<T*>(p.a.out) + row * p.a.out_stride + static_cast<uint64_t>(h) * HD;
#pragma unroll
            for (int d = 0; d < NT; ++d) {
                out[8 * d + 2 * t4] = from_f32<T>(acc[d][2 * i] * inv);
                out[8 * d + 2 * t4 + 1] = from_f32<T>(acc[d][2 * i + 1] * inv);
            }
            if (p.a.lse && t4 == 0) p.a.lse[row * p.a.H + h] = kv8_lse(kv8_base(mx[i]), l);
        } else {
            const uint64_t row = ((static_cast<uint64_t>(seq) * p.a.max_new + i0 + token) * p.a.H + h) * p.splits + split;
            float* part = p.part + row * HD;
#pragma unroll
            for (int d = 0; d < NT; ++d) {
                part[8 * d + 2 * t4] = acc[d][2 * i] * inv;
                part[8 * d + 2 * t4 + 1] = acc[d][2 * i + 1] * inv;
            }
            if (t4 == 0) {
                p.part_ml[row * 2] = kv8_base(mx[i]);
                p.part_ml[row * 2 + 1] = l;
            }
        }
    }
}

// -------------------------------------------------------------------- join

constexpr int kKjThreads = 256, kKjWarps = kKjThreads / 32;
constexpr uint32_t kKjFew = 8;  // splits that one warp joins

// Splits of query token i of sequence `seq` (0: the row does not exist), and
// its row among the call's.
__device__ __forceinline__ uint32_t kv8_row_splits(const Kv8Split& p, uint32_t seq, uint32_t i, uint64_t& row) {
    int64_t r0;
    const uint32_t rows = kv8_rows(p.a.cu, seq, p.a.max_new, p.a.status, r0);
    if (i >= rows) return 0;
    row = static_cast<uint64_t>(r0 + i);
    const uint32_t i0 = i / p.tile * p.tile, i1 = min(rows, i0 + p.tile) - 1;
    return kv8_used(kv8_span(p.a, seq, rows, i0, i1).count(), p.chunk);
}

// Up to kKjFew splits: a warp for each (query token, head), the splits' loads
// in flight together; CTA (token group, sequence) of 8 warps.  One CTA a row
// took 60 us for 8x128 tokens of 32 heads in two splits.
template <typename T, int HD>
__global__ void __launch_bounds__(kKjThreads) kv8_join_few_kernel(const Kv8Split p) {
    const uint32_t at = blockIdx.x * kKjWarps + threadIdx.x / 32, i = at / p.a.H, h = at % p.a.H, seq = blockIdx.y;
    const int lane = threadIdx.x % 32;
    pdl_wait();
    if (i >= p.a.max_new) return;
    uint64_t row = 0;
    const uint32_t used = kv8_row_splits(p, seq, i, row);
    if (used <= 1) return;  // the only split wrote the output itself
    const uint64_t first = ((static_cast<uint64_t>(seq) * p.a.max_new + i) * p.a.H + h) * p.splits;
    const float* ml = p.part_ml + first * 2;
    const float* part = p.part + first * HD;
    float m = -INFINITY, l = 0.0f, f[kKjFew], v[HD / 32];
#pragma unroll
    for (uint32_t s = 0; s < kKjFew; ++s) m = s < used ? fmaxf(m, ml[2 * s]) : m;
#pragma unroll
    for (uint32_t s = 0; s < kKjFew; ++s) {
        const bool there = s < used;
        const float ms = there ? ml[2 * s] : -INFINITY;
        f[s] = there ? ml[2 * s + 1] * (ms == -INFINITY ? 1.0f : ex2(ms - m)) : 0.0f;
        l += f[s];
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) v[e] = 0.0f;
#pragma unroll
    for (uint32_t s = 0; s < kKjFew; ++s) {
        if (s < used) {
#pragma unroll
            for (int e = 0; e < HD / 32; ++e) v[e] = fmaf(part[s * HD + lane + 32 * e], f[s] * inv, v[e]);
        }
    }
    T* out = static_cast<T*>(p.a.out) + row * p.a.out_stride + static_cast<uint64_t>(h) * HD;
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) out[lane + 32 * e] = from_f32<T>(v[e]);
    if (p.a.lse && lane == 0) p.a.lse[row * p.a.H + h] = kv8_lse(m, l);
}

// More splits: CTA (head, query token, sequence), 8 warps over the splits, in
// split order, then over each other.
template <typename T, int HD>
__global__ void __launch_bounds__(kKjThreads) kv8_join_kernel(const Kv8Split p) {
    __shared__ float f[kKv8MaxSplits];
    __shared__ float o[kKjWarps][HD];
    __shared__ float total;
    const uint32_t h = blockIdx.x, i = blockIdx.y, seq = blockIdx.z;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    pdl_wait();
    uint64_t row = 0;
    const uint32_t used = kv8_row_splits(p, seq, i, row);
    if (used <= 1) return;
    const uint64_t first = ((static_cast<uint64_t>(seq) * p.a.max_new + i) * p.a.H + h) * p.splits;
    const float* ml = p.part_ml + first * 2;
    if (warp == 0) {
        float m = -INFINITY, l = 0.0f;
        for (uint32_t s = lane; s < used; s += 32) m = fmaxf(m, ml[2 * s]);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
        for (uint32_t s = lane; s < used; s += 32) {
            f[s] = ml[2 * s + 1] * (ml[2 * s] == -INFINITY ? 1.0f : ex2(ml[2 * s] - m));
            l += f[s];
        }
        l = warp_sum(l);
        if (lane == 0) {
            total = l;
            if (p.a.lse) p.a.lse[row * p.a.H + h] = kv8_lse(m, l);
        }
    }
    __syncthreads();
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const float* part = p.part + first * HD;
    float v[HD / 32];
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) v[e] = 0.0f;
#pragma unroll 4
    for (uint32_t s = warp; s < used; s += kKjWarps) {
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) v[e] = fmaf(part[static_cast<uint64_t>(s) * HD + lane + 32 * e], f[s] * inv, v[e]);
    }
#pragma unroll
    for (int e = 0; e < HD / 32; ++e) o[warp][lane + 32 * e] = v[e];
    __syncthreads();
    T* out = static_cast<T*>(p.a.out) + row * p.a.out_stride + static_cast<uint64_t>(h) * HD;
    for (int d = threadIdx.x; d < HD; d += kKjThreads) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < kKjWarps; ++w) x += o[w][d];
        out[d] = from_f32<T>(x);
    }
}

// -------------------------------------------------------------------- host

cudaError_t kv8_join(const Kv8Split& p, uint32_t hd, int dtype, cudaStream_t s) {
    const bool few = p.splits <= kKjFew;
    const uint64_t rows = static_cast<uint64_t>(p.a.max_new) * p.a.H;
    const dim3 grid = few ? dim3(static_cast<uint32_t>((rows + kKjWarps - 1) / kKjWarps), p.a.count) : dim3(p.a.H, p.a.max_new, p.a.count);
#define VRT_KJ(TY, T, HD)                                                                                             \
    if (dtype == TY && hd == HD)                                                                                      \
        return launch(few ? kv8_join_few_kernel<T, HD> : kv8_join_kernel<T, HD>, grid, dim3(kKjThreads), 0, s, true, p);
#define VRT_KJ3(HD) VRT_KJ(VRT_F32, float, HD) VRT_KJ(VRT_F16, __half, HD) VRT_KJ(VRT_BF16, __nv_bfloat16, HD)
    VRT_KJ3(64) VRT_KJ3(128) VRT_KJ3(256)
#undef VRT_KJ3
#undef VRT_KJ
    return cudaErrorInvalidValue;
}

// Query tokens of a CTA, and whether the tcgen05 form runs: for 16-bit rows,
// always from head_dim 128 up, at head_dim 64 from 512 rows a sequence.
// Measured, tcgen05 and warp form (bf16, us): 32/16 heads of 128, 2 tokens
// behind 8192 31.9 and 34.7, 64 tokens 43.6 and 67.2, 1024 tokens 190 and 848;
// 4/1 heads of 256, 2 tokens behind 1024 23.5 and 34.3; 8/2 heads of 64, 32
// tokens behind 1024 16.1 and 14.1, 64 behind 8192 20.9 and 18.4, 128 behind
// 8192 21.5 and 28.2.
static bool kp_tile(uint32_t hd, int dtype, uint32_t group, uint32_t max_new, uint32_t& tile) {
    const bool tc = dtype != VRT_F32 && (hd >= 128 || static_cast<uint64_t>(max_new) * group >= 512);
    tile = tc ? kv8_prefill_tc_rows(hd) / 128 * (128 / group) : kKpRows / group;
    return tc;
}

// Splits of a history when there are too few query tiles for the GPU: up to
// two CTAs an SM of the warp form, one of the tcgen05 form, kKpMinPages pages
// each at least.
constexpr uint32_t kKpMinPages = 8;

static uint64_t kp_cap(int sms, bool tc, uint32_t tile, uint32_t kv, uint32_t count, uint32_t max_new) {
    const uint64_t ctas = (static_cast<uint64_t>(max_new) + tile - 1) / tile * kv * std::max(1u, count);
    const uint64_t want = std::min<uint64_t>((tc ? 1ull : 2ull) * sms / std::max<uint64_t>(1, ctas), kKv8MaxSplits);
    return max_new > 65535u ? 1 : std::max<uint64_t>(1, std::min<uint64_t>(want, 65535u / std::max(1u, count)));  // grid limits
}

static bool kp_plan(int sms, uint32_t hd, const Kv8Attn& a, uint32_t& tile, uint32_t& chunk, uint32_t& splits) {
    const bool tc = kp_tile(hd, a.dtype, a.H / a.c.kv, a.max_new, tile);
    const uint64_t pages = (static_cast<uint64_t>(a.max_len) + kKv8Page - 1) / kKv8Page;
    const uint64_t cap = kp_cap(sms, tc, tile, a.c.kv, a.count, a.max_new);
    const uint64_t c = std::max<uint64_t>((pages + cap - 1) / cap, kKpMinPages);
    chunk = static_cast<uint32_t>(c);
    splits = static_cast<uint32_t>((pages + c - 1) / c);
    return tc;
}

// For any max_len up to this one, as in kv8_decode_workspace.
uint64_t kv8_prefill_workspace(int sms, uint32_t hd, int dtype, uint32_t kv, uint32_t heads, uint32_t count,
                               uint32_t max_new, uint32_t max_len) {
    uint32_t tile;
    const bool tc = kp_tile(hd, dtype, heads / kv, max_new, tile);
    const uint64_t pages = (static_cast<uint64_t>(max_len) + kKv8Page - 1) / kKv8Page;
    const uint64_t splits = std::min<uint64_t>(kp_cap(sms, tc, tile, kv, count, max_new),
                                               (pages + kKpMinPages - 1) / kKpMinPages);
    return splits > 1 ? static_cast<uint64_t>(count) * max_new * heads * splits * (hd + 2) * 4 : 0;
}

template <typename T, int HD, int TERMS>
static cudaError_t kp_launch(const Kv8Split& p, cudaStream_t s) {
    constexpr uint32_t smem = KpShape<HD, TERMS>::kBytes;
    static std::mutex mu;
    static uint64_t done = 0;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    {
        std::lock_guard<std::mutex> lock(mu);
        const uint64_t bit = dev < 64 ? 1ull << dev : 0ull;
        if (!(done & bit)) {
            e = cudaFuncSetAttribute(kv8_prefill_kernel<T, HD, TERMS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
            if (e != cudaSuccess) return e;
            done |= bit;
        }
    }
    const dim3 grid((p.a.max_new + p.tile - 1) / p.tile, p.a.c.kv, p.a.count * p.splits);
    e = launch(kv8_prefill_kernel<T, HD, TERMS>, grid, dim3(kKpThreads), smem, s, false, p);
    if (e != cudaSuccess || p.splits == 1) return e;
    return kv8_join(p, HD, p.a.dtype, s);
}

cudaError_t kv8_prefill(const Kv8Attn& a, uint32_t hd, int sms, void* workspace, cudaStream_t s) {
    Kv8Split p{};
    p.a = a;
    const bool tc = kp_plan(sms, hd, a, p.tile, p.chunk, p.splits);
    p.part = static_cast<float*>(workspace);
    p.part_ml = p.part + static_cast<uint64_t>(a.count) * a.max_new * a.H * p.splits * hd;
    if (tc) return kv8_prefill_tc(p, hd, s);
    if (a.dtype == VRT_F32) {
        if (hd == 64) return kp_launch<float, 64, 2>(p, s);
        if (hd == 128) return kp_launch<float, 128, 2>(p, s);
        if (hd == 256) return kp_launch<float, 256, 2>(p, s);
    } else if (hd == 64) {
        return a.dtype == VRT_F16 ? kp_launch<__half, 64, 1>(p, s) : kp_launch<__nv_bfloat16, 64, 1>(p, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace vrt
