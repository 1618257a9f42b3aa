// Prompt attention over the paged 8-bit KV cache on the 5th-generation tensor
// cores (tcgen05), for 16-bit rows.  The general form is in kv8_prefill.cu.
//
// One CTA an SM holds MT tiles of 128 rows (128 / R query tokens of the R
// heads that share a KV head) and walks the visible pages in key tiles of KT
// tokens:
//   S = Q K^T      tcgen05.mma, both from shared memory, fp32 in TMEM
//   P = exp2(...)  one thread a row: TMEM -> registers -> fp16 P over S's columns
//   O += P V       tcgen05.mma, P from TMEM, V from shared memory, fp32 in TMEM
// Warp roles:
//   warps 0..4MT-1  softmax: a warpgroup a tile; it also brings the query rows
//                   into shared memory, rescales O and writes the output;
//   next 4 warps    bring the pages: codes from global memory into registers
//                   one tile ahead, as fp16 (exact) into the 128B-swizzled
//                   K-major operand tiles; value pages lie [dim][token], which
//                   is V^T, the K-major form of the second product;
//   last warp       one lane issues the MMAs: S of a tile's next keys goes out
//                   behind its P V, so the tensor cores work on one tile while
//                   the other is in its softmax (MT = 1: on the other S buffer).
//
// Scales: a page's key scale and the row's factor are one FMA in front of the
// exponential.  A page's value scale cannot be taken out of O, which sums over
// pages: the weight is multiplied by v_scale / (largest v_scale that the CTA
// sees) in the same FMA, as an addend to the exponent, so that the codes stay
// exact and a weight is rounded once.  The sum of weights is kept by page in
// fp32 and divided by that ratio again, one FMA for 32 keys.
// The running maximum moves only when it grows by more than kTcSlack (base 2):
// weights are then up to 2^(kTcLift + kTcSlack), within fp16, and O is seldom
// rescaled.  What falls under fp16's smallest step is 2^-36 of the largest
// weight times the largest value.
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>

#include "gemm_q8t.cuh"
#include "kv8.cuh"

namespace vrt {

constexpr float kTcSlack = 4.0f, kTcLift = 11.0f;

template <int HD>
struct TcShape {
    static constexpr int MT = HD == 256 ? 1 : 2;          // row tiles
    static constexpr int KT = HD == 256 ? 64 : 128;       // keys of a tile
    static constexpr int PG = KT / static_cast<int>(kKv8Page);  // pages of a tile
    static constexpr int kStages = 2;
    static constexpr int kThreads = (4 * MT + 4 + 1) * 32;
    static constexpr uint32_t kQTile = 128 * HD * 2, kKTile = KT * HD * 2;  // bytes; K and V alike
    static constexpr uint32_t kTiles = MT * kQTile + 2 * kStages * kKTile;
    // at least 120 KB: one CTA an SM, which may then take all of TMEM
    static constexpr uint32_t kBytes = 1024 + (kTiles > 120 * 1024 ? kTiles : 120 * 1024) + 1024;
    static constexpr uint32_t kSCols = KT, kOCol = 2 * KT;  // TMEM columns: two S buffers, then O of each tile
};

struct TcMeta {  // what the softmax knows of a page
    float k_scale;
    float v_log;  // log2(v_scale / reference), 0 for a page of zeros
    float v_inv;  // 2^-v_log
    int there;
};

// D[tmem] (+)= A[tmem] * B[smem]^T
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// (a0, a1) * b + c and (a0, a1) + (b0, b1), two fp32 at once
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

template <typename T>
__device__ __forceinline__ uint32_t pack_rows(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack_rows<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack_rows<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// 16 codes as fp16 into two 16-byte pieces of a swizzled tile row; `swap`
// writes the second first, so that the lanes of a quarter warp meet all banks.
__device__ __forceinline__ void store_codes(uint8_t* a, uint8_t* b, uint4 u, bool swap) {
    const uint32_t w[4] = {u.x ^ 0x80808080u, u.y ^ 0x80808080u, u.z ^ 0x80808080u, u.w ^ 0x80808080u};
    const uint4 x = make_uint4(codes_lo(w[0]), codes_hi(w[0]), codes_lo(w[1]), codes_hi(w[1]));
    const uint4 y = make_uint4(codes_lo(w[2]), codes_hi(w[2]), codes_lo(w[3]), codes_hi(w[3]));
    *reinterpret_cast<uint4*>(swap ? b : a) = swap ? y : x;
    *reinterpret_cast<uint4*>(swap ? a : b) = swap ? x : y;
}

template <typename T, int HD>
__global__ void __launch_bounds__(TcShape<HD>::kThreads, 1) kv8_prefill_tc_kernel(const Kv8Split p) {
    using Shape = TcShape<HD>;
    constexpr int MT = Shape::MT, KT = Shape::KT, PG = Shape::PG, ST = Shape::kStages;
    constexpr int kLook = MT == 2 ? 1 : 2;  // key tiles that S runs ahead of P V
    constexpr uint32_t kIdescS = (1u << 4) | (static_cast<uint32_t>(KT >> 3) << 17) | (128u >> 4 << 24);
    constexpr uint32_t kIdescO = (1u << 4) | (static_cast<uint32_t>(HD >> 3) << 17) | (128u >> 4 << 24);
    extern __shared__ uint8_t tc_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tc_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sq = sm;                              // [MT][HD / 64][128 rows][128 bytes]
    uint8_t* sk = sq + MT * Shape::kQTile;         // [ST][HD / 64][KT rows][128]
    uint8_t* sv = sk + ST * Shape::kKTile;         // [ST][KT / 64][HD rows][128]
    uint64_t* k_full = reinterpret_cast<uint64_t*>(sm + Shape::kBytes - 2048);
    uint64_t* k_empty = k_full + ST;
    uint64_t* v_full = k_empty + ST;
    uint64_t* v_empty = v_full + ST;
    uint64_t* q_full = v_empty + ST;
    uint64_t* s_full = q_full + 1;   // [2] S buffer computed
    uint64_t* p_full = s_full + 2;   // [2] P in its place
    uint64_t* o_full = p_full + 2;   // [MT] P V added
    uint64_t* drained = o_full + 2;  // after a wait gave up: the MMAs in flight are done
    TcMeta* meta = reinterpret_cast<TcMeta*>(drained + 1);           // [4][PG]
    float* reference = reinterpret_cast<float*>(meta + 4 * PG);     // [4 warps], then the value scale that O counts in
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(reference + 5);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t R = p.a.H / p.a.c.kv, g = blockIdx.y, seq = blockIdx.z / p.splits, split = blockIdx.z % p.splits;
    pdl_trigger();
    int64_t r0;
    const uint32_t n = kv8_rows(p.a.cu, seq, p.a.max_new, p.a.status, r0);
    const uint32_t blocks = (p.a.max_new + p.tile - 1) / p.tile, i0 = (blocks - 1 - blockIdx.x) * p.tile;
    if (i0 >= n) return;
    const uint32_t tokens = min(p.tile, n - i0), per = 128u / R;  // query tokens of the CTA, of a row tile
    const Kv8Span span = kv8_span(p.a, seq, n, i0, i0 + tokens - 1);
    const uint32_t all = span.count(), used = kv8_used(all, p.chunk), share = kv8_share(all, used);
    if (split >= used) return;
    const uint32_t j0 = min(all, split * share), j1 = min(all, j0 + share);
    const int64_t pos0 = span.len - n + i0;
    // key tiles that row tile t needs: pages up to its own last token's
    int need[2] = {0, 0};
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        if (t * per >= tokens) continue;
        const int64_t last = pos0 + min((t + 1) * per, tokens) - 1;
        const uint32_t end = last < 0 ? 0u : static_cast<uint32_t>(last / kKv8Page) + 1;
        const uint32_t pages = min(max(span.a + max(span.b0, min(end, span.b1)) - span.b0, j0), j1) - j0;
        need[t] = static_cast<int>((pages + PG - 1) / PG);
    }
    const int J = max(need[0], need[1]);

    if (tid == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(k_full + s, 4);
            mbar_init(k_empty + s, 1);
            mbar_init(v_full + s, 4);
            mbar_init(v_empty + s, 1);
        }
        mbar_init(q_full, 4 * MT);
        mbar_init(drained, 1);
        for (int b = 0; b < 2; ++b) {
            mbar_init(s_full + b, 1);
            mbar_init(p_full + b, 4);
            mbar_init(o_full + b, 1);
        }
        fence_mbar_init();
    }
    if (warp == 4 * MT + 4) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool ok = true;

    if (warp < 4 * MT) {
        // --------------------------------------------------------- softmax
        const int t = warp >> 2, row = tid & 127;
        const uint32_t token = t * per + row / R, h = g * R + row % R;
        const bool live = row < static_cast<int>(per * R) && token < tokens;
        const int64_t pos = pos0 + token, lo = kv8_window_lo(pos, p.a.window);
        const uint64_t at = static_cast<uint64_t>(r0 + i0 + (live ? token : 0));
        float unit = 0.0f;  // score units of a row
        {
            const T* q = static_cast<const T*>(p.a.q) + at * p.a.q_stride + static_cast<uint64_t>(live ? h : g * R) * HD;
            float m = 0.0f;
#pragma unroll 4
            for (int d = 0; d < HD; d += 8) {
                float x[8];
                load_row<T, 8>(q + d, x);
                m = fmaxf(m, max_abs(x));
            }
            const float mul = kv8_row_unit(m);
            unit = 1.0f / mul * fabsf(p.a.scale);
            const float sign = live ? (p.a.scale < 0.0f ? -mul : mul) : 0.0f;
#pragma unroll 4
            for (int d = 0; d < HD; d += 8) {
                float x[8];
                load_row<T, 8>(q + d, x);
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[e] = live ? pack_half(__float2half_rn(x[2 * e] * sign), __float2half_rn(x[2 * e + 1] * sign)) : 0u;
                }
                *reinterpret_cast<uint4*>(sq + t * Shape::kQTile + d / 64 * (128 * 128) + sw128_offset(row, d % 64)) =
                    make_uint4(w[0], w[1], w[2], w[3]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        const bool cap = p.a.softcap > 0.0f;
        const float factor = cap ? unit : unit * kLog2e, inv_cap = cap ? 1.0f / p.a.softcap : 0.0f;
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // this warp's 32 TMEM lanes
        const int64_t tile0 = pos0 + t * per, tile1 = pos0 + min((t + 1) * per, tokens) - 1;
        const int64_t lo1 = kv8_window_lo(tile1, p.a.window);
        float mx = -INFINITY, sum = 0.0f;
        const int mine = need[t];
        for (int j = 0; j < mine; ++j) {
            const int buf = MT == 2 ? t : j & 1, phase = (MT == 2 ? j : j >> 1) & 1;
            const uint32_t s_col = tmem + lanes + buf * Shape::kSCols;
            ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(s_full + buf, phase));
            if (!ok) break;
            tc_fence_after();
            const TcMeta* mt = meta + (j & 3) * PG;
            uint32_t see[PG];  // keys of a page that the row sees
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < PG; ++c) {
                const uint32_t at_page = j0 + j * PG + c;
                const int64_t t0 = static_cast<int64_t>(span.page(at_page)) * kKv8Page;
                const bool there = mt[c].there;
                const bool full = there && (t0 + 32 <= span.prefix || (t0 + 31 <= tile0 && t0 >= lo1 && t0 + 32 <= span.len));
                see[c] = 0xffffffffu;
                if (!full) {
                    // bits [a, b) of the window, and those below the prefix
                    const int64_t e = min(pos + 1, span.len) - t0;
                    const int a = static_cast<int>(max(static_cast<int64_t>(0), min(lo - t0, static_cast<int64_t>(32))));
                    const int b = static_cast<int>(max(static_cast<int64_t>(0), min(e, static_cast<int64_t>(32))));
                    const int f = static_cast<int>(max(static_cast<int64_t>(0), min(span.prefix - t0, static_cast<int64_t>(32))));
                    auto below = [](int x) { return x >= 32 ? 0xffffffffu : (1u << x) - 1u; };
                    see[c] = there ? ((below(b) & ~below(a)) | below(f)) : 0u;
                }
                uint32_t v[32];
                tmem_ld32(s_col + 32 * c, v);
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (full) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) m4[e & 3] = fmaxf(m4[e & 3], __uint_as_float(v[e]));
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) m4[e & 3] = fmaxf(m4[e & 3], see[c] >> e & 1 ? __uint_as_float(v[e]) : -INFINITY);
                }
                float z = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                if (z != -INFINITY) {
                    z *= mt[c].k_scale * factor;
                    if (cap) z = capped<false>(z, p.a.softcap, inv_cap);
                    top = fmaxf(top, z);
                }
            }
            const bool grown = top > mx + kTcSlack;  // also from -inf
            if (__any_sync(0xffffffffu, grown)) {
                const float f = grown ? (mx == -INFINITY ? 0.0f : ex2(mx - top)) : 1.0f;
                if (grown) mx = top;
                sum *= f;
                if (j > 0) {
                    ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(o_full + t, (j - 1) & 1));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int d = 0; d < HD; d += 32) {
                        uint32_t v[32];
                        const uint32_t o = tmem + lanes + Shape::kOCol + t * HD + d;
                        tmem_ld32(o, v);
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
                        tmem_st32(o, v);
                    }
                    tmem_wait_st();
                }
            }
            const float base = kTcLift - (mx == -INFINITY ? 0.0f : mx);
#pragma unroll
            for (int c = 0; c < PG; ++c) {
                uint32_t v[32], w[16];
                tmem_ld32(s_col + 32 * c, v);
                const float a = mt[c].k_scale * factor, b = base + mt[c].v_log;
                const uint64_t a2 = pair(a, a), b2 = pair(b, b);
                uint64_t part[2] = {0, 0};
                if (cap) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        v[e] = __float_as_uint(capped<false>(__uint_as_float(v[e]) * a, p.a.softcap, inv_cap) + b);
                    }
                }
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    float x = __uint_as_float(v[e]), y = __uint_as_float(v[e + 1]);
                    if (!cap) unpair(fma2(pair(x, y), a2, b2), x, y);
                    x = ex2(x);
                    y = ex2(y);
                    if (see[c] != 0xffffffffu) {
                        if (!(see[c] >> e & 1)) x = 0.0f;
                        if (!(see[c] >> (e + 1) & 1)) y = 0.0f;
                    }
                    part[e >> 1 & 1] = add2(part[e >> 1 & 1], pair(x, y));
                    const __half2 hh = __floats2half2_rn(x, y);
                    w[e / 2] = *reinterpret_cast<const uint32_t*>(&hh);
                }
                float x, y;
                unpair(add2(part[0], part[1]), x, y);
                if (see[c]) sum = fmaf(x + y, mt[c].v_inv, sum);
                tmem_st16(s_col + 16 * c, w);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + buf);
        }
        // ---- output
        if (mine > 0) {
            ok = ok && mbar_wait_bounded(o_full + t, (mine - 1) & 1);
            tc_fence_after();
        }
        const float ref = mine > 0 ? reference[4] : 0.0f;
        const float mul = used == 1 ? (sum == 0.0f ? 0.0f : ref / sum) : ref;
        T* out = static_cast<T*>(p.a.out) + at * p.a.out_stride + static_cast<uint64_t>(h) * HD;
        const uint64_t prow = ((static_cast<uint64_t>(seq) * p.a.max_new + i0 + token) * p.a.H + h) * p.splits + split;
#pragma unroll 1
        for (int d = 0; d < HD; d += 32) {
            uint32_t v[32];
            if (mine > 0) {
                tmem_ld32(tmem + lanes + Shape::kOCol + t * HD + d, v);
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = 0u;
            }
            if (!live) continue;
            if (used == 1) {
                uint32_t x[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = pack_rows<T>(__uint_as_float(v[2 * e]) * mul, __uint_as_float(v[2 * e + 1]) * mul);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    reinterpret_cast<uint4*>(out + d)[e] = make_uint4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) p.part[prow * HD + d + e] = __uint_as_float(v[e]) * mul;
            }
        }
        if (live) {
            if (used == 1) {
                if (p.a.lse) p.a.lse[at * p.a.H + h] = kv8_lse(mx - kTcLift, sum);
            } else {
                p.part_ml[prow * 2] = mx - kTcLift;
                p.part_ml[prow * 2 + 1] = sum;
            }
        }
        tc_fence_before();
    } else if (warp < 4 * MT + 4) {
        // ----------------------------------------------------------- pages
        const int c0 = tid - 128 * MT;
        constexpr int C = PG * HD * 2 / 128;  // 16-byte pieces of a key tile that a thread brings, keys and values each
        constexpr int PP = HD * 2;            // pieces of a page
        // the largest value scale among the CTA's pages
        float m = 0.0f;
        for (uint32_t i = j0 + c0; i < j1; i += 128) {
            const int id = kv8_page(p.a.c, seq, span.page(i), p.a.status);
            const float s = id < 0 ? 0.0f : p.a.c.v_scale[static_cast<uint64_t>(id) * p.a.c.kv + g];
            if (s < INFINITY) m = fmaxf(m, s);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (lane == 0) reference[warp - 4 * MT] = m;
        named_bar_sync(1, 128);
        m = fmaxf(fmaxf(reference[0], reference[1]), fmaxf(reference[2], reference[3]));
        const float ref = m > 0.0f ? m : 1.0f;
        if (c0 == 0) reference[4] = ref;

        uint4 kr[C], vr[C];
        int ids[PG];
        auto page_ids = [&](int j) {
#pragma unroll
            for (int c = 0; c < PG; ++c) {
                const uint32_t i = j0 + j * PG + c;
                ids[c] = j < J && i < j1 ? kv8_page(p.a.c, seq, span.page(i), p.a.status) : -1;
            }
        };
        auto fetch = [&](uint4(&r)[C], const int8_t* from) {
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const int c = c0 + 128 * i, pg = c / PP;
                // a page that is not there is zeros: its weights are 0 and must meet finite values
                r[i] = make_uint4(0, 0, 0, 0);
                int id = -1;
#pragma unroll
                for (int x = 0; x < PG; ++x) id = x == pg ? ids[x] : id;
                if (id >= 0) {
                    r[i] = __ldg(reinterpret_cast<const uint4*>(from + (static_cast<uint64_t>(id) * p.a.c.kv + g) * (kKv8Page * HD)) + c % PP);
                }
            }
        };
        // value pieces are dealt so that a quarter warp's stores meet all banks
        auto v_piece = [](int c) {
            const int q = c / 2 % 4, d = c / 16 * 8 + c / 8 % 2 * 2 + (q & 1) + (q >> 1) * 4;
            return d * 2 + c % 2;
        };
        auto fetch_v = [&]() {
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const int c = c0 + 128 * i, pg = c / PP;
                vr[i] = make_uint4(0, 0, 0, 0);
                int id = -1;
#pragma unroll
                for (int x = 0; x < PG; ++x) id = x == pg ? ids[x] : id;
                if (id >= 0) {
                    vr[i] = __ldg(reinterpret_cast<const uint4*>(p.a.c.v + (static_cast<uint64_t>(id) * p.a.c.kv + g) * (kKv8Page * HD)) + v_piece(c % PP));
                }
            }
        };
        page_ids(0);
        fetch(kr, p.a.c.k);
        fetch_v();
        for (int j = 0; j < J; ++j) {
            const int s = j % ST;
            if (j >= ST) ok = ok && mbar_wait_bounded(k_empty + s, ((j / ST) - 1) & 1);
            if (!ok) break;
            if (c0 < PG) {
                int id = -1;
#pragma unroll
                for (int x = 0; x < PG; ++x) id = x == c0 ? ids[x] : id;
                const uint64_t head = static_cast<uint64_t>(id < 0 ? 0 : id) * p.a.c.kv + g;
                TcMeta e{0.0f, 0.0f, 1.0f, id >= 0};
                if (id >= 0) {
                    e.k_scale = p.a.c.k_scale[head];
                    const float vs = p.a.c.v_scale[head];
                    if (vs != 0.0f) {
                        e.v_log = vs < INFINITY ? fmaxf(log2f(vs / ref), -60.0f) : NAN;
                        e.v_inv = exp2f(-e.v_log);
                    }
                }
                meta[(j & 3) * PG + c0] = e;
            }
            uint8_t* kt = sk + s * Shape::kKTile;
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const int c = c0 + 128 * i, key = c / (HD / 16), d = c % (HD / 16) * 16;
                uint8_t* sub = kt + d / 64 * (KT * 128);
                store_codes(sub + sw128_offset(key, d % 64), sub + sw128_offset(key, d % 64 + 8), kr[i], (d / 64) & 1);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(k_full + s);
            page_ids(j + 1);
            if (j + 1 < J) fetch(kr, p.a.c.k);
            if (j >= ST) ok = ok && mbar_wait_bounded(v_empty + s, ((j / ST) - 1) & 1);
            if (!ok) break;
            uint8_t* vt = sv + s * Shape::kKTile;
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const int c = c0 + 128 * i, piece = v_piece(c % PP), d = piece / 2, key = c / PP * 32 + piece % 2 * 16;
                uint8_t* sub = vt + key / 64 * (HD * 128);
                store_codes(sub + sw128_offset(d, key % 64), sub + sw128_offset(d, key % 64 + 8), vr[i], false);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(v_full + s);
            if (j + 1 < J) fetch_v();
        }
    } else if (lane == 0) {
        // ------------------------------------------------------------- MMA
        auto wait = [&](uint64_t* bar, int phase) { ok = ok && mbar_wait_bounded(bar, phase & 1); };
        int k_seen = -1, v_seen = -1;
        auto issue_s = [&](int t, int j) {
            if (j > k_seen) {
                wait(k_full + j % ST, j / ST);
                k_seen = j;
            }
            if (!ok) return;
            tc_fence_after();
            const int buf = MT == 2 ? t : j & 1;
            const uint32_t qa = smem_addr(sq + t * Shape::kQTile), ka = smem_addr(sk + j % ST * Shape::kKTile);
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
                umma_f16(tmem + buf * Shape::kSCols, sw128_desc(qa + k / 4 * (128 * 128) + k % 4 * 32),
                         sw128_desc(ka + k / 4 * (KT * 128) + k % 4 * 32), kIdescS, k > 0);
            }
            umma_commit(s_full + buf);
            if (t == MT - 1 || j >= need[MT - 1]) umma_commit(k_empty + j % ST);  // no other tile reads these keys
        };
        if (J > 0) wait(q_full, 0);
        for (int l = 0; l < kLook; ++l)
            for (int t = 0; t < MT; ++t)
                if (l < need[t]) issue_s(t, l);
        for (int j = 0; j < J && ok; ++j) {
            for (int t = 0; t < MT && ok; ++t) {
                if (j >= need[t]) continue;
                const int buf = MT == 2 ? t : j & 1;
                wait(p_full + buf, MT == 2 ? j : j >> 1);
                if (j > v_seen) {
                    wait(v_full + j % ST, j / ST);
                    v_seen = j;
                }
                if (!ok) break;
                tc_fence_after();
                const uint32_t va = smem_addr(sv + j % ST * Shape::kKTile);
#pragma unroll
                for (int k = 0; k < KT / 16; ++k) {
                    umma_f16_ts(tmem + Shape::kOCol + t * HD, tmem + buf * Shape::kSCols + k * 8,
                                sw128_desc(va + k / 4 * (HD * 128) + k % 4 * 32), kIdescO, j > 0 || k > 0);
                }
                umma_commit(o_full + t);
                if (t == MT - 1 || j >= need[MT - 1]) umma_commit(v_empty + j % ST);
                if (j + kLook < need[t]) issue_s(t, j + kLook);
            }
        }
        if (!ok) {
            umma_commit(drained);
            mbar_wait_bounded(drained, 0);
        }
    }
    if (!ok) atomicOr(p.a.status, kStatusWaitTimeout);
    __syncthreads();
    if (warp == 4 * MT + 4) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// -------------------------------------------------------------------- host

template <typename T, int HD>
static cudaError_t tc_launch(const Kv8Split& p, cudaStream_t s) {
    using Shape = TcShape<HD>;
    static std::mutex mu;
    static uint64_t done = 0;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    {
        std::lock_guard<std::mutex> lock(mu);
        const uint64_t bit = dev < 64 ? 1ull << dev : 0ull;
        if (!(done & bit)) {
            e = cudaFuncSetAttribute(kv8_prefill_tc_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kBytes);
            if (e != cudaSuccess) return e;
            done |= bit;
        }
    }
    const dim3 grid((p.a.max_new + p.tile - 1) / p.tile, p.a.c.kv, p.a.count * p.splits);
    e = launch(kv8_prefill_tc_kernel<T, HD>, grid, dim3(Shape::kThreads), Shape::kBytes, s, false, p);
    if (e != cudaSuccess || p.splits == 1) return e;
    return kv8_join(p, HD, p.a.dtype, s);
}

uint32_t kv8_prefill_tc_rows(uint32_t hd) { return hd == 256 ? 128u : 256u; }

cudaError_t kv8_prefill_tc(const Kv8Split& p, uint32_t hd, cudaStream_t s) {
#define VRT_TC(HD)                                                              \
    if (hd == HD) {                                                             \
        if (p.a.dtype == VRT_F16) return tc_launch<__half, HD>(p, s);           \
        if (p.a.dtype == VRT_BF16) return tc_launch<__nv_bfloat16, HD>(p, s);   \
    }
    VRT_TC(64) VRT_TC(128) VRT_TC(256)
#undef VRT_TC
    return cudaErrorInvalidValue;
}

}  // namespace vrt
