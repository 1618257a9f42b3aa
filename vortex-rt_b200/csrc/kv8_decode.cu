// Single-token attention over the paged 8-bit KV cache (kv8.cuh): one pass
// over the visible pages, split over the GPU, joined by a second kernel.
//
// Bound by HBM: 2 * head_dim bytes a token and KV head, read once whatever
// the number of query heads.  An int8 code is exact in fp16, so the products
// run on mma.sync m16n8k16 (fp16 in, fp32 sums) with the page as the 16-row
// operand and the query heads of one KV head as the 8 columns: no row of the
// instruction is padding, where tcgen05 would take the 1..8 heads as 128
// rows.  The tensor work is far below its peak (11 SM cycles of HBM time for
// one mma at 6.4 TB/s), so what counts is bytes in flight.
//
// CTA (split, KV head, sequence): 4 warps, each with its own ring of bulk
// copies (192 KB an SM); page j of the split belongs to warp j % 4, its keys
// and its values are two ring items.
//   scores  S^T[token][head] = K[token][dim] Q^T[dim][head]: the 16-byte piece
//           of a key row that a lane holds is 4 k-steps of its A fragment,
//           the dims are permuted alike in Q's fragments;
//   softmax running maximum and sum a head in registers, base 2;
//   output  O^T[dim][head] += V^T[dim][token] P^T[token][head]: the value page
//           lies [dim][token], so 8 bytes of a lane are again A fragments; P
//           goes from the accumulator layout to the operand layout by
//           movmatrix, with the page's tokens dealt to rows so that it fits.
// A page's products start from zero and join the fp32 sums by one FMA with
// the page's value scale: the tensor core cuts its sums at every step, which
// would add up over a long history.
//
// Operands: a query row is brought to [2^14, 2^15) by a power of two, then
// fp16 (exact for f16 and bf16 rows) or, for f32 rows, fp16 + fp16 remainder
// (22 bits).  Weights are 2^14 exp(s - maximum) in fp16, value codes are stored
// times 2^-14 against that: half a step is 2^-11
// of a weight (averaged over the keys below half a step of a 16-bit output),
// and what falls under fp16's smallest step is 2^-39 of the largest weight;
// for f32 rows fp16 + fp16 remainder.  The remainders take columns 4..7 when
// there are at most 4 heads, a second mma otherwise.

#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>

#include "kv8.cuh"

namespace vrt {

constexpr int kKdWarps = 4;
constexpr int kKdThreads = kKdWarps * 32;

template <int HD>
struct KdShape {
    static constexpr uint32_t kItem = kKv8Page * HD;   // bytes of one page of one head: a ring item
    // Warps resident on an SM are what the dependent steps of a page need most
    // (8x32768 f16: 8 warps an SM 224 us, 16 warps 175-181 us), then CTAs
    // small enough that one starts while others stream (32x2304 bf16, 16
    // warps: 2 CTAs 66 us, 4 CTAs 62 us).  At head_dim 256 the output
    // accumulators allow 8 warps.
    static constexpr int kCtas = HD == 256 ? 2 : 4;
    static constexpr uint32_t kRing = 192 * 1024 / kCtas;
    static constexpr int kItems = kRing / kItem / kKdWarps;  // 6, 3 or 3 items of ring a warp
    static_assert(kRing % (kKdWarps * kItem) == 0, "a warp's ring holds whole items");
    static constexpr int kSteps = HD / 16;             // k-steps of the scores, row tiles of the output
};

// TERMS: fp16 terms of an operand (2 for f32 rows).  SETS: mma of each step
// (2: more than 4 heads with remainders).
template <typename T, int HD, int TERMS, int SETS>
__global__ void __launch_bounds__(kKdThreads, KdShape<HD>::kCtas) kv8_decode_kernel(const Kv8Split p) {
    using Shape = KdShape<HD>;
    constexpr bool kPacked = TERMS == 2 && SETS == 1;  // columns 4..7 are the remainders of heads 0..3
    constexpr int D = Shape::kItems, KS = Shape::kSteps, W = kKdWarps;
    constexpr uint32_t kWarpRing = D * Shape::kItem;
    extern __shared__ __align__(128) uint8_t sm[];
    uint2* qf = reinterpret_cast<uint2*>(sm + Shape::kRing);        // [SETS][KS][32] query fragments
    uint64_t* bars = reinterpret_cast<uint64_t*>(qf + SETS * KS * 32);    // [warps][D]
    float* q_unit = reinterpret_cast<float*>(bars + W * D);        // [8] what a query row was divided by

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, t4 = lane & 3;
    const uint32_t split = blockIdx.x, g = blockIdx.y, seq = blockIdx.z, R = p.a.H / p.a.c.kv;
    pdl_trigger();
    const Kv8Span span = kv8_span(p.a, seq, 1, 0, 0);
    const uint32_t n = span.count(), used_splits = kv8_used(n, p.chunk), share = kv8_share(n, used_splits);
    if (split >= used_splits) return;
    const uint32_t j0 = min(n, split * share), j1 = min(n, j0 + share);

    uint64_t* bar = bars + warp * D;
    uint8_t* ring = sm + warp * kWarpRing;
    if (lane < D) mbar_init(bar + lane, 1);
    fence_mbar_init();
    __syncwarp();

    // This warp's pages: j0 + warp + 4 i for i < mine.  Lane l knows page l of
    // the current group of 32: pool index and scales.
    const uint32_t mine = j0 + warp < j1 ? (j1 - j0 - warp + W - 1) / W : 0;
    const int64_t kv = p.a.c.kv;
    auto look_up = [&](uint32_t i, int& id, float& ks, float& vs) {
        id = 0;
        ks = vs = 0.0f;
        if (i >= mine) return;
        id = kv8_page(p.a.c, seq, span.page(j0 + warp + W * i), p.a.status);
        if (id < 0) return;
        ks = __ldg(p.a.c.k_scale + id * kv + g);
        vs = __ldg(p.a.c.v_scale + id * kv + g);
    };
    int id_now, id_next = 0;
    float ks_now, vs_now, ks_next = 0.0f, vs_next = 0.0f;
    look_up(lane, id_now, ks_now, vs_now);
    if (mine > 32) look_up(32 + lane, id_next, ks_next, vs_next);
    uint32_t issued = 0;  // ring items asked for: keys of page i are item 2 i, values 2 i + 1
    auto issue = [&](uint32_t base) {  // base: first page of id_now's group
        const uint32_t i = issued / 2;
        const int id = i - base < 32 ? __shfl_sync(0xffffffffu, id_now, i - base)
                                     : __shfl_sync(0xffffffffu, id_next, i - base - 32);
        if (lane == 0) {
            const uint64_t at = (static_cast<uint64_t>(id < 0 ? 0 : id) * kv + g) * Shape::kItem;
            uint64_t* b = bar + issued % D;
            mbar_arrive_expect_tx(b, Shape::kItem);
            bulk_copy_g2s(ring + issued % D * Shape::kItem, (issued & 1 ? p.a.c.v : p.a.c.k) + at, Shape::kItem, b);
        }
        ++issued;
    };
    while (issued < 2 * mine && issued < D) issue(0);

    // query fragments: lane (g8, t4) of step (c, s) holds dims 64 c + 16 t4 + 4 s + 0..3 of head g8
    {
        const uint32_t h = tid / 16, piece = tid % 16;  // 16 threads a head, HD / 16 dims each
        constexpr int E = HD / 16;
        float x[E], m = 0.0f;
        const T* q = static_cast<const T*>(p.a.q) + static_cast<uint64_t>(seq) * p.a.q_stride +
                     static_cast<uint64_t>(g * R + h) * HD + piece * E;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] = h < R ? to_f32(q[e]) : 0.0f;
            m = fmaxf(m, fabsf(x[e]));
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float mul = kv8_row_unit(m);
        if (piece == 0) q_unit[h] = m < INFINITY ? 1.0f / mul : NAN;  // an infinity makes the row NaN, capped or not
        __half* f = reinterpret_cast<__half*>(qf);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int d = piece * E + e;
            const int step = d / 64 * 4 + d % 16 / 4, t = d % 64 / 16;
            const int at = ((step * 32 + static_cast<int>(h) * 4 + t) * 4) + d % 4;
            __half hi, lo;
            split_f16(x[e] * mul, hi, lo);
            if (kPacked) {
                if (h < 4) {
                    f[at] = hi;
                    f[at + 4 * 4 * 4] = lo;  // head h + 4
                }
            } else {
                f[at] = hi;
                if (SETS == 2) f[at + KS * 32 * 4] = lo;
            }
        }
    }
    __syncthreads();
    const int head0 = kPacked ? (2 * t4) % 4 : 2 * t4;  // heads of this lane's two columns
    const bool plain_cap = p.a.softcap > 0.0f, fast_cap = TERMS == 1 && plain_cap && p.a.softcap <= kKv8FastCap;
    const float unit = plain_cap ? 1.0f : kLog2e, inv_cap = plain_cap ? kv8_inv_cap(p.a.softcap) : 0.0f;
    const float sc[2] = {q_unit[head0] * (p.a.scale * unit), q_unit[head0 + 1] * (p.a.scale * unit)};

    float acc[KS][4];
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] = 0.0f;
    float mx[2] = {-INFINITY, -INFINITY}, m0[2] = {0.0f, 0.0f}, sum[2] = {0.0f, 0.0f};  // m0: what scores are weighed from
    bool ok = true;
    uint32_t used = 0;  // ring items consumed
    auto refill = [&](uint32_t base) {  // after a wait that gave up, in any lane: no more copies, and the page is the last
        ++used;
        ok = __all_sync(0xffffffffu, ok);
        __syncwarp();
        if (ok && issued < 2 * mine) issue(base);
    };

    for (uint32_t i = 0; i < mine && ok; ++i) {
        const uint32_t base = i & ~31u;
        if (i == base && i) {
            id_now = id_next;
            ks_now = ks_next;
            vs_now = vs_next;
            look_up(base + 32 + lane, id_next, ks_next, vs_next);
        }
        const float ks = __shfl_sync(0xffffffffu, ks_now, i & 31), vs = __shfl_sync(0xffffffffu, vs_now, i & 31);
        const bool there = __shfl_sync(0xffffffffu, id_now, i & 31) >= 0;
        const int64_t t0 = static_cast<int64_t>(span.page(j0 + warp + W * i)) * kKv8Page;

        // ---- scores: block b of 8 rows holds tokens 8 (row / 2) + row % 2 + 2 b
        ok &= mbar_wait_bounded(bar + used % D, (used / D) & 1);
        float s[2][4];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[m][e] = 0.0f;
        {
            const uint8_t* kp = ring + used % D * Shape::kItem + (8 * (g8 >> 1) + (g8 & 1)) * HD + t4 * 16;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
                uint32_t w[4][4];
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const uint4 u = *reinterpret_cast<const uint4*>(kp + 2 * b * HD + 64 * c);
                    w[b][0] = u.x ^ 0x80808080u;
                    w[b][1] = u.y ^ 0x80808080u;
                    w[b][2] = u.z ^ 0x80808080u;
                    w[b][3] = u.w ^ 0x80808080u;
                }
                // f32 rows: each 64 dims on their own, joined by rounding additions
                float part[2][4] = {};
                float (&z)[2][4] = TERMS == 2 ? part : s;
#pragma unroll
                for (int st = 0; st < 4; ++st) {
                    const uint2 q0 = qf[(c * 4 + st) * 32 + lane];
                    uint2 q1;
                    if (SETS == 2) q1 = qf[(KS + c * 4 + st) * 32 + lane];
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        const uint32_t a0 = codes_lo(w[2 * m][st]), a1 = codes_lo(w[2 * m + 1][st]);
                        const uint32_t a2 = codes_hi(w[2 * m][st]), a3 = codes_hi(w[2 * m + 1][st]);
                        if (SETS == 2) mma_f16(z[m], a0, a1, a2, a3, q1);
                        mma_f16(z[m], a0, a1, a2, a3, q0);
                    }
                }
                if (TERMS == 2) {
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[m][e] += part[m][e];
                }
            }
        }
        refill(base);
        if (kPacked) {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[m][e] += __shfl_xor_sync(0xffffffffu, s[m][e], 2);
        }
        // ---- softmax: s[m][2 r + h] is block 2 m + r, this lane's head h
        auto each = [&](auto f) {  // f(score, head)
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) s[b >> 1][2 * (b & 1) + h] = f(s[b >> 1][2 * (b & 1) + h], h);
        };
        each([&](float z, int h) { return z * (ks * sc[h]); });
        if (fast_cap) {
            each([&](float z, int) { return capped_fast(z, p.a.softcap, inv_cap); });
        } else if (plain_cap) {
            each([&](float z, int) { return capped_exact(z, p.a.softcap, inv_cap); });
        }
        float top[2] = {mx[0], mx[1]};
        const bool full = there && (t0 + 32 <= span.prefix || (t0 >= span.lo && t0 + 32 <= span.len));
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int64_t t = t0 + 8 * (g8 >> 1) + (g8 & 1) + 2 * b;
            const bool see = full || (there && (t < span.prefix || (t >= span.lo && t < span.len)));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float& z = s[b >> 1][2 * (b & 1) + h];
                if (!see) z = -INFINITY;
                top[h] = fmaxf(top[h], z);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], o));
        }
        if (__any_sync(0xffffffffu, top[0] != mx[0] || top[1] != mx[1])) {
            float f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                f[h] = mx[h] == -INFINITY ? 0.0f : ex2(mx[h] - top[h]);
                sum[h] *= f[h];
                mx[h] = top[h];
                m0[h] = mx[h] == -INFINITY ? 0.0f : kv8_base(mx[h]);
            }
#pragma unroll
            for (int q = 0; q < KS; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[q][e] *= f[e & 1];
        }
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            __half hi[2], lo[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // a score that was left out is -inf, whatever its scale: weight 0; a NaN stays
                const float w = ex2(s[b >> 1][2 * (b & 1) + h] - m0[h]);
                sum[h] += w;
                if (TERMS == 2) {
                    split_f16(w, hi[h], lo[h]);
                } else {
                    hi[h] = __float2half_rn(w);
                }
            }
            ph[b] = pack_half(hi[0], hi[1]);
            if (TERMS == 2) pl[b] = pack_half(lo[0], lo[1]);
            if (kPacked && t4 >= 2) ph[b] = pl[b];
            ph[b] = movmatrix(ph[b]);
            if (SETS == 2) pl[b] = movmatrix(pl[b]);
        }
        // ---- output
        ok &= mbar_wait_bounded(bar + used % D, (used / D) & 1);
        {
            const uint8_t* vp = ring + used % D * Shape::kItem + g8 * kKv8Page + t4 * 8;
#pragma unroll
            for (int q = 0; q < KS; ++q) {
                uint2 u0 = *reinterpret_cast<const uint2*>(vp + q * 16 * kKv8Page);
                uint2 u1 = *reinterpret_cast<const uint2*>(vp + (q * 16 + 8) * kKv8Page);
                u0.x ^= 0x80808080u;
                u0.y ^= 0x80808080u;
                u1.x ^= 0x80808080u;
                u1.y ^= 0x80808080u;
                float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                const uint32_t a0 = value_codes_lo(u0.x), a1 = value_codes_lo(u1.x), a2 = value_codes_hi(u0.x), a3 = value_codes_hi(u1.x);
                const uint32_t c0 = value_codes_lo(u0.y), c1 = value_codes_lo(u1.y), c2 = value_codes_hi(u0.y), c3 = value_codes_hi(u1.y);
                if (SETS == 2) {
                    mma_f16(o, a0, a1, a2, a3, make_uint2(pl[0], pl[1]));
                    mma_f16(o, c0, c1, c2, c3, make_uint2(pl[2], pl[3]));
                }
                mma_f16(o, a0, a1, a2, a3, make_uint2(ph[0], ph[1]));
                mma_f16(o, c0, c1, c2, c3, make_uint2(ph[2], ph[3]));
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[q][e] = fmaf(o[e], vs, acc[q][e]);
            }
        }
        refill(base);
    }
    if (!ok) {
        // the copies still under way, each slot's latest, land before their ring is used below
        for (uint32_t i = issued > D ? issued - D : 0; i < issued; ++i) mbar_wait_bounded(bar + i % D, (i / D) & 1);
        if (lane == 0) atomicOr(p.a.status, kStatusWaitTimeout);
    }

    // ---- join the warps: [warp][column][HD] outputs over the rings, then maxima and sums
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], o);
    }
    __syncthreads();
    float* wo = reinterpret_cast<float*>(sm);
    float* wm = reinterpret_cast<float*>(qf);  // [warp][8][2]
#pragma unroll
    for (int q = 0; q < KS; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) wo[(warp * 8 + 2 * t4 + (e & 1)) * HD + q * 16 + g8 + 8 * (e >> 1)] = acc[q][e];
    if (g8 == 0 && (!kPacked || t4 < 2)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            wm[(warp * 8 + 2 * t4 + h) * 2] = kv8_base(mx[h]);  // as the sums are weighed
            wm[(warp * 8 + 2 * t4 + h) * 2 + 1] = sum[h];
        }
    }
    __syncthreads();
    const bool alone = used_splits == 1;
    for (uint32_t r = warp; r < R; r += W) {
        float m = -INFINITY, l = 0.0f, f[W];
#pragma unroll
        for (int w = 0; w < W; ++w) m = fmaxf(m, wm[(w * 8 + r) * 2]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            // a warp without pages has maximum -inf and sum 0; one whose scores are NaN has sum NaN
            f[w] = wm[(w * 8 + r) * 2] == -INFINITY ? 1.0f : ex2(wm[(w * 8 + r) * 2] - m);
            l += wm[(w * 8 + r) * 2 + 1] * f[w];
        }
        const uint64_t row = static_cast<uint64_t>(seq) * p.a.H + g * R + r;
        float* part = p.part + (row * p.splits + split) * HD;
        T* out = static_cast<T*>(p.a.out) + static_cast<uint64_t>(seq) * p.a.out_stride + static_cast<uint64_t>(g * R + r) * HD;
        const float inv = l == 0.0f ? 0.0f : kKv8Unlift / l;
        for (int d = lane; d < HD; d += 32) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                float x = wo[(w * 8 + r) * HD + d];
                if (kPacked) x += wo[(w * 8 + r + 4) * HD + d];
                v = fmaf(x, f[w], v);
            }
            if (alone) {
                out[d] = from_f32<T>(v * inv);
            } else {
                part[d] = v * inv;
            }
        }
        if (lane == 0) {
            if (alone) {
                if (p.a.lse) p.a.lse[row] = kv8_lse(m, l);
            } else {
                p.part_ml[(row * p.splits + split) * 2] = m;
                p.part_ml[(row * p.splits + split) * 2 + 1] = l;
            }
        }
    }
}

// ------------------------------------------------------------------- host

static uint64_t kd_cap(int sms, uint32_t kv, uint32_t count) {
    const uint64_t want = 12ull * sms / (static_cast<uint64_t>(kv) * std::max(1u, count));
    return std::min<uint64_t>(std::max<uint64_t>(1, want), kKv8MaxSplits);
}

// Pages of a split and splits of a sequence that sees `pages` pages.  About three rounds of
// the 4 CTAs that an SM holds, so that sequences of unlike length even out;
// at least a page a warp, below which starting a CTA costs more than its
// pages.
static void kd_plan(int sms, uint32_t kv, uint32_t count, uint64_t pages, uint32_t& chunk, uint32_t& splits) {
    const uint64_t cap = kd_cap(sms, kv, count);
    uint64_t c = std::max<uint64_t>((pages + cap - 1) / cap, kKdWarps);
    c = (c + kKdWarps - 1) / kKdWarps * kKdWarps;
    chunk = static_cast<uint32_t>(c);
    splits = static_cast<uint32_t>((pages + c - 1) / c);
}

// For any number of visible pages up to max_len's: no plan has more splits
// than its cap, nor than one for each kKdWarps pages.
uint64_t kv8_decode_workspace(int sms, uint32_t hd, uint32_t kv, uint32_t heads, uint32_t count, uint32_t max_len) {
    const uint64_t pages = (static_cast<uint64_t>(max_len) + kKv8Page - 1) / kKv8Page;
    const uint64_t splits = std::min<uint64_t>(kd_cap(sms, kv, count), (pages + kKdWarps - 1) / kKdWarps);
    return splits > 1 ? static_cast<uint64_t>(count) * heads * splits * (hd + 2) * 4 : 0;
}

template <typename T, int HD, int TERMS, int SETS>
static cudaError_t kd_launch(const Kv8Split& p, cudaStream_t s) {
    using Shape = KdShape<HD>;
    constexpr uint32_t smem = Shape::kRing + SETS * Shape::kSteps * 32 * 8 + kKdWarps * Shape::kItems * 8 + 8 * 4;
    static std::mutex mu;
    static uint64_t done = 0;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    {
        std::lock_guard<std::mutex> lock(mu);
        const uint64_t bit = dev < 64 ? 1ull << dev : 0ull;
        if (!(done & bit)) {
            e = cudaFuncSetAttribute(kv8_decode_kernel<T, HD, TERMS, SETS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
            if (e != cudaSuccess) return e;
            done |= bit;
        }
    }
    e = launch(kv8_decode_kernel<T, HD, TERMS, SETS>, dim3(p.splits, p.a.c.kv, p.a.count), dim3(kKdThreads), smem, s, false, p);
    if (e != cudaSuccess || p.splits == 1) return e;
    return kv8_join(p, HD, p.a.dtype, s);
}

cudaError_t kv8_decode(const Kv8Attn& a, uint32_t hd, int sms, void* workspace, cudaStream_t s) {
    Kv8Split p{};
    p.a = a;
    p.tile = 1;
    const int dtype = a.dtype;
    uint64_t pages = (static_cast<uint64_t>(a.max_len) + kKv8Page - 1) / kKv8Page;
    // a window's tokens lie in one page more than they fill; a prefix adds its own
    if (a.window && !a.prefix) pages = std::min<uint64_t>(pages, (static_cast<uint64_t>(a.window) + kKv8Page - 2) / kKv8Page + 1);
    kd_plan(sms, a.c.kv, a.count, pages, p.chunk, p.splits);
    p.part = static_cast<float*>(workspace);
    p.part_ml = p.part + static_cast<uint64_t>(a.count) * a.H * p.splits * hd;
    const bool wide = a.H / a.c.kv > 4;
#define VRT_KD(HD)                                                                              \
    if (hd == HD) {                                                                             \
        if (dtype == VRT_F16) return kd_launch<__half, HD, 1, 1>(p, s);                         \
        if (dtype == VRT_BF16) return kd_launch<__nv_bfloat16, HD, 1, 1>(p, s);                 \
        return wide ? kd_launch<float, HD, 2, 2>(p, s) : kd_launch<float, HD, 2, 1>(p, s);      \
    }
    VRT_KD(64) VRT_KD(128) VRT_KD(256)
#undef VRT_KD
    return cudaErrorInvalidValue;
}

}  // namespace vrt
