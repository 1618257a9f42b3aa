// Prompt attention over the paged 8-bit KV cache on the 5th-generation tensor
// cores (tcgen05), for 16-bit rows.  The general form is in kv8_prefill.cu.
//
// One CTA an SM holds MT tiles of 128 rows (128 / R query tokens of the R
// heads that share a KV head) and walks the visible pages in tiles of 64 keys:
//   S = Q K^T      tcgen05.mma, both from shared memory, fp32 in TMEM
//   P = exp2(...)  one thread a row: TMEM -> registers -> fp16 P over S's columns
//   O += P V       tcgen05.mma, P from TMEM, V from shared memory, fp32 in TMEM
// Each row tile has two S buffers: the scores of the next keys are there when
// its softmax, which sets the pace, is done with the present ones.
// Warp roles:
//   warps 0..4MT-1  softmax: a warpgroup a tile; it also brings the query rows
//                   into shared memory, rescales O and writes the output;
//   next 4 + 4      bring the keys and the values, KB tokens at a time: codes
//                   from global memory into registers one block ahead, as fp16
//                   (exact) into the 128B-swizzled K-major operand tiles; value
//                   pages lie [dim][token], which is V^T, the K-major form of
//                   the second product;
//   last warpgroup  a warp for each row tile issues its MMAs.
//
// Scales: a page's key scale and the row's factor are one FMA in front of the
// exponential.  A page's value scale cannot be taken out of O, which sums over
// pages: it is 2^e f with f in [1/sqrt 2, sqrt 2).  The codes are stored times 2^e, counted
// from the largest value scale of the CTA's pages, which fp16 holds exactly down
// to 2^-28 of that (8 bits of code on its smallest step, 2^-24); the weight is
// multiplied by f in the FMA in front of its exponential, as an addend, and is
// rounded once.  So how large the values are that a row does not see, or hardly
// weighs, costs its own no bit.  The sum of weights is kept by page in fp32 and
// divided by f again, one FMA for 32 keys.  Pages whose value scales lie further
// apart than 2^28, or close to fp32's ends, take the form that follows below:
// scores and products of a row on its thread's fp32 pipes, O still in TMEM
// (8192 tokens in such a cache: 39 ms instead of 0.74).  A page with a NaN among
// its values counts as zeros; the outputs that see it are made NaN in the end,
// and no weight and no lse.
// The running maximum moves only when it grows by more than kTcSlack (base 2):
// weights are then up to 2^(kTcLift + kTcSlack), with f within fp16, and O is seldom
// rescaled (a rescale waits for the tensor cores: 2500 cycles).  Beyond kTcFar
// the FMA, which does not round the score, would part from the maximum, which
// is a rounded score, by whole numbers: there scores are rounded first.  What falls
// under fp16's smallest step is 2^-28 of a row's largest weight, times values that
// the row sees, each its own: far below half a step of a 16-bit output.
// O: the tensor core cuts the sum that it adds 16 keys to, always towards 0, by
// some 2^-24 of it: 1e-4 after 32,768 keys and 4e-4 after 131,072 (measured; an
// f16 output is rounded by 4.9e-4 at most).  So every kTcRun key tiles O is added
// to a sum in fp32 in the thread's local memory, by rounding additions, and
// starts again from 0.  A form of its own (RUNS) for calls that may see so many
// keys: its code made 8192 tokens 757 us instead of 740, 4x2048 capped 99
// instead of 94.
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "gemm_q8t.cuh"
#include "kv8.cuh"

namespace vrt {

constexpr float kTcSlack = 11.5f, kTcLift = 3.5f;
constexpr int kTcRun = 256;  // key tiles of a run: 16,384 keys
constexpr float kTcFar = 1048576.0f;  // scores (base 2) whose fp32 step is an eighth

// Value scales by the exponent field of their fp32: the largest of a CTA's
// pages within [kTcScaleLow, kTcScaleHigh], all others but zeros at most
// kTcScaleSpan below.
constexpr int kTcScaleLow = 40, kTcScaleHigh = 250, kTcScaleSpan = 28;
constexpr int kTcCodeUp = 4;  // codes of the largest are stored times 2^4 or 2^5: 1152 * 2^5, their offset, is within fp16
__device__ __forceinline__ int scale_exponent(float s) { return static_cast<int>(__float_as_uint(s) >> 23 & 255u); }
// The exponent field of the power of two that a scale is within [1/sqrt 2, sqrt 2) of, and how many times that it is.
__device__ __forceinline__ int scale_power(float s) { return static_cast<int>(__float_as_uint(s) + 0x4afb0du >> 23); }
__device__ __forceinline__ float scale_rest(float s) { return __uint_as_float(__float_as_uint(s) - (static_cast<uint32_t>(scale_power(s) - 127) << 23)); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

template <int HD>
struct TcShape {
    static constexpr int MT = HD == 256 ? 1 : 2;    // row tiles
    static constexpr int KT = 64;                   // keys of a tile: of one S buffer
    static constexpr int KB = HD == 256 ? 64 : 128; // keys of a block: of one operand stage
    static constexpr int SUB = KB / KT;
    static constexpr int PG = KB / static_cast<int>(kKv8Page);  // pages of a block
    static constexpr int kStages = 2;
    static constexpr int kThreads = (4 * MT + 8 + 4) * 32;  // whole warpgroups, for the register split
    // registers of a thread at launch, and as the warpgroups share them out: softmax, pages, MMA
    static constexpr int kRegs = MT == 2 ? 96 : 128;
    static constexpr int kRegsSoft = MT == 2 ? 144 : 200, kRegsPage = MT == 2 ? 64 : 104, kRegsMma = MT == 2 ? 64 : 104;
    static_assert(128 * (MT * kRegsSoft + 2 * kRegsPage + kRegsMma) <= kThreads * kRegs && kThreads * kRegs <= 65536,
                  "the shares come out of what the block was launched with");
    static constexpr uint32_t kQTile = 128 * HD * 2, kKTile = KB * HD * 2;  // bytes; K and V alike
    static constexpr uint32_t kTiles = MT * kQTile + 2 * kStages * kKTile;
    // at least 120 KB: one CTA an SM, which may then take all of TMEM
    static constexpr uint32_t kBytes = 1024 + (kTiles > 120 * 1024 ? kTiles : 120 * 1024) + 1024;
    static constexpr uint32_t kOCol = 2 * MT * KT;  // TMEM columns: two S buffers of each tile, then O of each tile
    static_assert(kOCol + MT * HD <= 512, "TMEM");
};

struct TcMeta {  // what the softmax knows of a page
    float k_scale;
    float v_log;  // log2 of f, what the value scale is of its power of two; 0 for a page of zeros
    float v_inv;  // 1 / f
    int there;
};

// MMA and commit for a whole warp whose lanes all pass the same operands: one
// elected lane issues.  A warp that stays together keeps the operands in
// uniform registers (one lane alone in a branch took 195 cycles an MMA).
// D[tmem] (+)= A[smem] * B[smem]^T
__device__ __forceinline__ void warp_mma_ss(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]^T
__device__ __forceinline__ void warp_mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void warp_commit(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar))
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
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int c = 0; c < 16; ++c) asm volatile("" : "+r"(v[c]));
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

// 2^x of two x <= 100 on the FMA pipe: 2^x = 2^n 2^f with n the nearest whole
// number (the low bits of x + 1.5 * 2^23) and f in [-1/2, 1/2], 2^f by the
// polynomial of degree 4 with the smallest relative error there (2^-18.5; a
// Lawson fit), n added to the exponent field.  From -126 down (-inf too) the
// result is some 2^-126, and NaN is lost.  For capped scores, which take two
// special functions (8 cycles a warp each) before their exponential: 4x2048
// capped 176 -> 98 us.  For plain scores a quarter or half of the exponentials
// done so changed nothing or cost 5%.
__device__ __forceinline__ void ex2_fma(float& x, float& y) {
    const uint64_t v = pair(fmaxf(x, -126.0f), fmaxf(y, -126.0f));
    const uint64_t r = add2(v, pair(12582912.0f, 12582912.0f));
    const uint64_t f = fma2(add2(r, pair(-12582912.0f, -12582912.0f)), pair(-1.0f, -1.0f), v);
    uint64_t q = fma2(f, pair(0.009570101276040077f, 0.009570101276040077f), pair(0.05591785907745361f, 0.05591785907745361f));
    q = fma2(f, q, pair(0.240247443318367f, 0.240247443318367f));
    q = fma2(f, q, pair(0.6931217908859253f, 0.6931217908859253f));
    q = fma2(f, q, pair(0.9999992847442627f, 0.9999992847442627f));
    float r0, r1, q0, q1;
    unpair(r, r0, r1);
    unpair(q, q0, q1);
    x = __uint_as_float((__float_as_uint(r0) << 23) + __float_as_uint(q0));
    y = __uint_as_float((__float_as_uint(r1) << 23) + __float_as_uint(q1));
}

__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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

// The largest magnitude of eight 16-bit values, as bits (ordered like the
// values), and what it stands for.
template <typename T>
__device__ __forceinline__ uint32_t row_top(const uint4& u) {
    const uint32_t w[4] = {u.x & 0x7fff7fffu, u.y & 0x7fff7fffu, u.z & 0x7fff7fffu, u.w & 0x7fff7fffu};
    const uint32_t m = __vmaxu2(__vmaxu2(w[0], w[1]), __vmaxu2(w[2], w[3]));
    return max(m & 0xffffu, m >> 16);
}
template <typename T>
__device__ __forceinline__ float row_magnitude(uint32_t top) {
    const unsigned short bits = static_cast<unsigned short>(top);
    return to_f32(*reinterpret_cast<const T*>(&bits));
}

// 16 codes as fp16 into two 16-byte pieces of a swizzled tile row.
__device__ __forceinline__ void store_codes(uint8_t* a, uint8_t* b, uint4 u) {
    const uint32_t w[4] = {u.x ^ 0x80808080u, u.y ^ 0x80808080u, u.z ^ 0x80808080u, u.w ^ 0x80808080u};
    *reinterpret_cast<uint4*>(a) = make_uint4(codes_lo(w[0]), codes_hi(w[0]), codes_lo(w[1]), codes_hi(w[1]));
    *reinterpret_cast<uint4*>(b) = make_uint4(codes_lo(w[2]), codes_hi(w[2]), codes_lo(w[3]), codes_hi(w[3]));
}

// The same times `mul`, a power of two in both halves; off is -1152 times it (codes_lo, in one FMA).
__device__ __forceinline__ uint32_t scaled_codes(uint32_t w, uint32_t bytes, __half2 mul, __half2 off) {
    const uint32_t b = __byte_perm(w, 0x64646464u, bytes);
    const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&b), mul, off);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void store_codes(uint8_t* a, uint8_t* b, uint4 u, __half2 mul, __half2 off) {
    const uint32_t w[4] = {u.x ^ 0x80808080u, u.y ^ 0x80808080u, u.z ^ 0x80808080u, u.w ^ 0x80808080u};
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[2 * i] = scaled_codes(w[i], 0x4140u, mul, off);
        h[2 * i + 1] = scaled_codes(w[i], 0x4342u, mul, off);
    }
    *reinterpret_cast<uint4*>(a) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(b) = make_uint4(h[4], h[5], h[6], h[7]);
}

// The four codes of a word whose bytes were offset by 128, as fp32: a byte under the exponent of 2^23.
__device__ __forceinline__ float code_f32(uint32_t w, int i) {
    return __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7550u + i)) - 8388736.0f;
}

template <int N>
__device__ __forceinline__ void more_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// 32 columns of this warp's lanes on their way into v; they are there after tmem_arrived.
__device__ __forceinline__ void tmem_fetch32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_arrived(uint32_t (&a)[32], uint32_t (&b)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    // the values exist from here on: no use of them may move in front of the wait
#pragma unroll
    for (int c = 0; c < 32; ++c) asm volatile("" : "+r"(a[c]), "+r"(b[c]));
}

// CAP: 0 plain scores, 1 capped up to kKv8FastCap, 2 capped above it (tanhf).  RUNS: more than kTcRun key tiles.
template <typename T, int HD, int CAP, bool RUNS>
__global__ void __launch_bounds__(TcShape<HD>::kThreads, 1) kv8_prefill_tc_kernel(const Kv8Split p) {
    using Shape = TcShape<HD>;
    constexpr int MT = Shape::MT, KT = Shape::KT, KB = Shape::KB, SUB = Shape::SUB, PG = Shape::PG, ST = Shape::kStages;
    constexpr int kLook = 2;  // key tiles that S runs ahead of P V
    constexpr uint32_t kIdescS = (1u << 4) | (static_cast<uint32_t>(KT >> 3) << 17) | (128u >> 4 << 24);
    constexpr uint32_t kIdescO = (1u << 4) | (static_cast<uint32_t>(HD >> 3) << 17) | (128u >> 4 << 24);
    extern __shared__ uint8_t tc_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(tc_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sq = sm;                              // [MT][HD / 64][128 rows][128 bytes]
    uint8_t* sk = sq + MT * Shape::kQTile;         // [ST][HD / 64][KB rows][128]
    uint8_t* sv = sk + ST * Shape::kKTile;         // [ST][KB / 64][HD rows][128]
    uint64_t* k_full = reinterpret_cast<uint64_t*>(sm + Shape::kBytes - 2048);
    uint64_t* k_empty = k_full + ST;
    uint64_t* v_full = k_empty + ST;
    uint64_t* v_empty = v_full + ST;
    uint64_t* q_full = v_empty + ST;
    uint64_t* s_full = q_full + 1;   // [tile][2] S buffer computed
    uint64_t* p_full = s_full + 4;   // [tile][2] P in its place
    uint64_t* o_last = p_full + 4;   // [tile][2] the last P V but one and the last are added
    uint64_t* drained = o_last + 4;  // [tile] after a wait gave up: the MMAs in flight are done
    TcMeta* meta = reinterpret_cast<TcMeta*>(drained + 2);           // [4][PG]
    float* unit_v = reinterpret_cast<float*>(meta + 4 * PG);  // what O counts in
    int* v_top = reinterpret_cast<int*>(unit_v + 1);          // [4 warps] the value scales' largest exponent field
    int* v_low = v_top + 4;                                   // [4 warps] and smallest, 0 if a scale is out of range
    volatile int* wide = reinterpret_cast<volatile int*>(v_low + 4);  // scales too far apart for fp16 codes
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_low + 5);
    volatile int* missing = reinterpret_cast<volatile int*>(tmem_slot + 1);  // a page was not in the pool
    volatile int* poisoned = missing + 1;                                    // a page has a NaN among its values

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t R = p.a.H / p.a.c.kv, g = blockIdx.x % p.a.c.kv;
    const uint32_t seq = blockIdx.z / p.splits, split = blockIdx.z % p.splits;
    pdl_trigger();
    int64_t r0;
    const uint32_t n = kv8_rows(p.a.cu, seq, p.a.max_new, p.a.status, r0);
    // all heads' latest tokens, which see the most, start first
    const uint32_t blocks = (p.a.max_new + p.tile - 1) / p.tile, i0 = (blocks - 1 - blockIdx.x / p.a.c.kv) * p.tile;
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
        need[t] = static_cast<int>((pages + 1) / 2);
    }
    const int J = max(need[0], need[1]), blocks_k = (J + SUB - 1) / SUB;

    if (tid == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(k_full + s, 4);
            mbar_init(k_empty + s, MT);
            mbar_init(v_full + s, 4);
            mbar_init(v_empty + s, MT);
        }
        mbar_init(q_full, 4 * MT);
        for (int b = 0; b < 4; ++b) {
            mbar_init(s_full + b, 1);
            mbar_init(p_full + b, 4);
            mbar_init(o_last + b, 1);
        }
        for (int t = 0; t < 2; ++t) mbar_init(drained + t, 1);
        *missing = 0;
        *poisoned = 0;
        *wide = 0;
        fence_mbar_init();
    }
    if (warp == 4 * MT + 8) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    bool ok = true;

    if (warp < 4 * MT) {
        // --------------------------------------------------------- softmax
        more_registers<Shape::kRegsSoft>();
        const int t = warp >> 2, row = tid & 127;
        const uint32_t token = t * per + row / R, h = g * R + row % R;
        const bool live = row < static_cast<int>(per * R) && token < tokens;
        const int64_t pos = pos0 + token;
        // what the row sees: keys [lo, end) and those below the prefix (lengths are below 2^31)
        const int lo = static_cast<int>(kv8_window_lo(pos, p.a.window)), end = static_cast<int>(min(pos + 1, span.len));
        const int prefix = static_cast<int>(span.prefix);
        const uint64_t at = static_cast<uint64_t>(r0 + i0 + (live ? token : 0));
        float unit = 0.0f;  // score units of a row
        {
            const T* q = static_cast<const T*>(p.a.q) + at * p.a.q_stride + static_cast<uint64_t>(live ? h : g * R) * HD;
            // the whole row on its way at once: its latency is the CTA's start
            uint4 raw[HD / 8];
#pragma unroll
            for (int d = 0; d < HD / 8; ++d) raw[d] = reinterpret_cast<const uint4*>(q)[d];
            uint32_t top = 0;  // of the magnitudes' bits: infinities and NaN above all numbers
#pragma unroll
            for (int d = 0; d < HD / 8; ++d) top = max(top, row_top<T>(raw[d]));
            const float m = row_magnitude<T>(top);
            const bool finite = m < INFINITY;
            const float mul = kv8_row_unit(m);
            unit = finite ? 1.0f / mul * fabsf(p.a.scale) : NAN;
            const float sign = live ? (p.a.scale < 0.0f ? -mul : mul) : 0.0f;
#pragma unroll
            for (int d = 0; d < HD / 8; ++d) {
                const T* x = reinterpret_cast<const T*>(&raw[d]);
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[e] = live ? pack_half(__float2half_rn(to_f32(x[2 * e]) * sign), __float2half_rn(to_f32(x[2 * e + 1]) * sign)) : 0u;
                }
                *reinterpret_cast<uint4*>(sq + t * Shape::kQTile + d / 8 * (128 * 128) + sw128_offset(row, d % 8 * 8)) =
                    make_uint4(w[0], w[1], w[2], w[3]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        const float factor = CAP ? unit : unit * kLog2e, inv_cap = CAP ? kv8_inv_cap(p.a.softcap) : 0.0f;
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // this warp's 32 TMEM lanes
        const int64_t tile0 = pos0 + t * per, tile1 = pos0 + min((t + 1) * per, tokens) - 1;
        const int64_t lo1 = kv8_window_lo(tile1, p.a.window);
        // list indexes of the pages that all rows of the tile see whole: below whole_a, and from whole_b to whole_c
        const int stop = static_cast<int>(j1), whole_a = min(stop, static_cast<int>(span.prefix / kKv8Page));
        const int whole_b = static_cast<int>(span.a) + max(0, static_cast<int>((lo1 + kKv8Page - 1) / kKv8Page) - static_cast<int>(span.b0));
        const int whole_c = min(stop, static_cast<int>(span.a) - static_cast<int>(span.b0) +
                                          static_cast<int>(max(static_cast<int64_t>(0), min(tile0 + 1, span.len)) / kKv8Page));
        float mx = -INFINITY, sum = 0.0f;
        bool far = false;  // a row of the warp has its maximum beyond kTcFar
        const int mine = need[t];
        // the keys of a page at t0 that the row sees, a bit each
        auto visible = [&](int t0) {
            auto below = [](int x) { return x >= 32 ? 0xffffffffu : x <= 0 ? 0u : (1u << x) - 1u; };
            return (below(end - t0) & ~below(lo - t0)) | below(prefix - t0);
        };
        bool slow = false;
        if (J > 0) {
            named_bar_sync(2, Shape::kThreads);  // the value scales have been looked through
            slow = *wide;
        }
        bool poison = false;  // the row sees a page with a NaN among its values
        if (mine > 0 && *poisoned) {
#pragma unroll 1
            for (uint32_t i = j0; i < min(j0 + 2 * mine, j1); ++i) {
                const uint32_t page = span.page(i);
                const int id = kv8_page(p.a.c, seq, page, p.a.status);
                const float v = id < 0 ? 0.0f : p.a.c.v_scale[static_cast<uint64_t>(id) * p.a.c.kv + g];
                if (v != v && visible(static_cast<int>(page * kKv8Page))) poison = true;
            }
        }
        float kept[HD], kept_mx = -INFINITY;  // O of the runs before, weighed from kept_mx
        if (__builtin_expect(slow, 0)) {
            const uint32_t at_o = tmem + lanes + Shape::kOCol + t * HD;
            const int pages = min(2 * mine, static_cast<int>(j1 - j0));
#pragma unroll 1
            for (int i = 0; i < pages; ++i) {
                const uint32_t page = span.page(j0 + i);
                const int id = kv8_page(p.a.c, seq, page, p.a.status);
                const uint64_t head = static_cast<uint64_t>(max(id, 0)) * p.a.c.kv + g;
                const uint32_t see = id < 0 ? 0u : visible(static_cast<int>(page * kKv8Page));
                const float kf = p.a.c.k_scale[head] * factor, vf = see ? p.a.c.v_scale[head] : 0.0f;
                const uint8_t* kp = reinterpret_cast<const uint8_t*>(p.a.c.k + head * (kKv8Page * HD));
                const uint8_t* vp = reinterpret_cast<const uint8_t*>(p.a.c.v + head * (kKv8Page * HD));
                float w[kKv8Page];  // scores, then weights
#pragma unroll
                for (int k = 0; k < 32; ++k) w[k] = 0.0f;
#pragma unroll 1
                for (int d = 0; d < HD; d += 4) {
                    const uint2 q4 = *reinterpret_cast<const uint2*>(sq + t * Shape::kQTile + d / 64 * (128 * 128) + sw128_offset(row, d % 64));
                    const float2 q01 = __half22float2(*reinterpret_cast<const __half2*>(&q4.x));
                    const float2 q23 = __half22float2(*reinterpret_cast<const __half2*>(&q4.y));
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        const uint32_t c = __ldg(reinterpret_cast<const uint32_t*>(kp + k * HD + d)) ^ 0x80808080u;
                        w[k] = fmaf(q01.x, code_f32(c, 0), w[k]);
                        w[k] = fmaf(q01.y, code_f32(c, 1), w[k]);
                        w[k] = fmaf(q23.x, code_f32(c, 2), w[k]);
                        w[k] = fmaf(q23.y, code_f32(c, 3), w[k]);
                    }
                }
                float top = mx;
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    float z = w[k] * kf;
                    if (CAP == 1) z = capped_fast(z, p.a.softcap, inv_cap);
                    if (CAP == 2) z = capped_exact(z, p.a.softcap, inv_cap);
                    w[k] = see >> k & 1 ? z : -INFINITY;
                    top = fmaxf(top, w[k]);
                }
                const float f = mx == -INFINITY ? 0.0f : ex2(mx - top), from = top == -INFINITY ? 0.0f : top;
                mx = top;
                sum *= f;
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    w[k] = ex2(w[k] - from);
                    sum += w[k];
                }
#pragma unroll 1
                for (int d = 0; d < HD; d += 16) {
                    uint32_t o[16] = {};
                    if (i > 0) tmem_ld16(at_o + d, o);
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const uint8_t* from_v = vp + (d + e) * static_cast<int>(kKv8Page);
                        float x = 0.0f;
#pragma unroll
                        for (int k = 0; k < 32; k += 4) {
                            const uint32_t c = __ldg(reinterpret_cast<const uint32_t*>(from_v + k)) ^ 0x80808080u;
#pragma unroll
                            for (int b = 0; b < 4; ++b) x = fmaf(w[k + b], code_f32(c, b), x);
                        }
                        o[e] = __float_as_uint(fmaf(x, vf, __uint_as_float(o[e]) * f));
                    }
                    tmem_st16(at_o + d, o);
                    tmem_wait_st();
                }
            }
        }
        for (int j = 0; j < mine && !slow; ++j) {
            const int buf = 2 * t + (j & 1);
            const uint32_t s_col = tmem + lanes + buf * KT;
            ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(s_full + buf, (j >> 1) & 1));
            if (!ok) break;
            tc_fence_after();
            uint32_t va[32], vb[32];  // scores of the tile's two pages
            tmem_fetch32(s_col, va);
            tmem_fetch32(s_col + 32, vb);
            const TcMeta* mt = meta + (j / SUB & 3) * PG + j % SUB * 2;
            float a0 = mt[0].k_scale * factor, a1 = mt[1].k_scale * factor, b0 = mt[0].v_log, b1 = mt[1].v_log;
            // a score times a plus b is the exponent of its weight times the value scale, inv takes that back for the
            // sum; a NaN (of a page's keys, or of the query in `factor`) reaches the sum, and so the row, through inv
            float i0v = mt[0].v_inv, i1v = mt[1].v_inv;
            const int i0p = static_cast<int>(j0) + 2 * j;
            const bool whole = (i0p + 1 < whole_a || (i0p >= whole_b && i0p + 1 < whole_c)) && !*missing;
            tmem_arrived(va, vb);
            if (!whole) {
                // Takes a page's scores to what the row sees: the rest is -inf, so the factor is kept above 0, and a NaN
                // key scale of a page that the row does not see is left out.
                auto mask = [&](int c, uint32_t(&v)[32], float& a, float& inv) {
                    const int t0 = static_cast<int>(span.page(j0 + 2 * j + c) * kKv8Page);
                    const uint32_t see = mt[c].there ? visible(t0) : 0u;
                    const bool bad = !(a < INFINITY);
                    a = bad ? 1.0f : fmaxf(a, 1e-37f);
                    inv = bad ? (see ? NAN : 1.0f) : inv;
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = see >> i & 1 ? v[i] : 0xff800000u;
                };
                mask(0, va, a0, i0v);
                mask(1, vb, a1, i1v);
            } else {
                i0v = a0 < INFINITY ? i0v : NAN;
                i1v = a1 < INFINITY ? i1v : NAN;
            }
            auto highest = [&](const uint32_t(&v)[32], float a) {
                float m4[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) m4[i] = fmaxf(__uint_as_float(v[i]), __uint_as_float(v[i + 4]));
#pragma unroll
                for (int i = 8; i < 32; i += 8) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) m4[q] = fmaxf(m4[q], fmaxf(__uint_as_float(v[i + q]), __uint_as_float(v[i + q + 4])));
                }
                const float z = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                if (CAP == 0 || z == -INFINITY) return z == -INFINITY ? z : z * a;
                return CAP == 1 ? capped_fast(z * a, p.a.softcap, inv_cap) : capped_exact(z * a, p.a.softcap, inv_cap);
            };
            const float top = fmaxf(highest(va, a0), highest(vb, a1));
            const bool grown = top > mx + kTcSlack;  // also from -inf
            if (__any_sync(0xffffffffu, grown)) {
                const float f = grown ? (mx == -INFINITY ? 0.0f : ex2(mx - top)) : 1.0f;
                if (grown) mx = top;
                far = __any_sync(0xffffffffu, mx > kTcFar || (mx < -kTcFar && mx != -INFINITY));
                sum *= f;
                if (j > 0) {
                    // P V of key tile j - 1 is done when S of j + 1, issued behind it, is
                    uint64_t* added = j + 1 < mine ? s_full + 2 * t + ((j + 1) & 1) : o_last + 2 * t;
                    ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(added, j + 1 < mine ? ((j + 1) >> 1) & 1 : 0));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int d = 0; d < HD; d += 32) {
                        uint32_t o[32];
                        const uint32_t at_o = tmem + lanes + Shape::kOCol + t * HD + d;
                        tmem_ld32(at_o, o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            asm volatile("" : "+r"(o[e]));
                            o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        }
                        tmem_st32(at_o, o);
                    }
                    tmem_wait_st();
                }
            }
            if (RUNS && j > 0 && j % kTcRun == 0) {
                uint64_t* added = j + 1 < mine ? s_full + 2 * t + ((j + 1) & 1) : o_last + 2 * t;
                ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(added, j + 1 < mine ? ((j + 1) >> 1) & 1 : 0));
                if (!ok) break;
                tc_fence_after();
                const float f = kept_mx == -INFINITY ? 0.0f : ex2(kept_mx - mx);
                kept_mx = mx;
#pragma unroll 1
                for (int d = 0; d < HD; d += 16) {
                    uint32_t o[16];
                    const uint32_t at_o = tmem + lanes + Shape::kOCol + t * HD + d;
                    tmem_ld16(at_o, o);
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        kept[d + e] = j == kTcRun ? __uint_as_float(o[e]) : fmaf(kept[d + e], f, __uint_as_float(o[e]));
                        o[e] = 0u;
                    }
                    tmem_st16(at_o, o);
                }
                tmem_wait_st();
            }
            const float seen = mx == -INFINITY ? 0.0f : mx, base = kTcLift - seen;
            // kHidden: scores of -inf among them, which a tanh would make finite; kFar: scores beyond kTcFar
            auto weigh = [&](int c, const uint32_t(&v)[32], float a, float b, float inv, auto kHidden, auto kFar) {
                uint32_t w[16];
                const float lifted = b + kTcLift;
                b += base;
                // CAP 1: cap * tanh(y) = cap - 2 cap / (e^2y + 1)
                const float ca = fminf(a * (inv_cap * 2.0f * kLog2e), 3e38f), c1 = p.a.softcap * kLog2e + b, c2 = -2.0f * kLog2e * p.a.softcap;
                const uint64_t a2 = pair(a, a), b2 = pair(b, b);
                uint64_t part[2] = {0, 0};
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    float x = __uint_as_float(v[e]), y = __uint_as_float(v[e + 1]);
                    if (CAP) {
                        const float s0 = x, s1 = y;
                        if (CAP == 1) {
                            x = fmaf(rcp_approx(ex2(x * ca) + 1.0f), c2, c1);
                            y = fmaf(rcp_approx(ex2(y * ca) + 1.0f), c2, c1);
                        } else {
                            // scores up to the cap, and beyond kTcFar: cut, as tanhf of a lower score may round higher
                            x = fminf(__fsub_rn(capped_exact(x * a, p.a.softcap, inv_cap), seen), kTcSlack) + lifted;
                            y = fminf(__fsub_rn(capped_exact(y * a, p.a.softcap, inv_cap), seen), kTcSlack) + lifted;
                        }
                        if (decltype(kHidden)::value) {
                            x = s0 == -INFINITY ? s0 : x;
                            y = s1 == -INFINITY ? s1 : y;
                        }
                    } else {
                        if (decltype(kFar)::value) {
                            x = __fsub_rn(__fmul_rn(x, a), seen) + lifted;
                            y = __fsub_rn(__fmul_rn(y, a), seen) + lifted;
                        } else {
                            unpair(fma2(pair(x, y), a2, b2), x, y);
                        }
                    }
                    if (CAP == 1) {  // two special functions are spent on the tanh already
                        ex2_fma(x, y);
                    } else {
                        x = ex2(x);
                        y = ex2(y);
                    }
                    part[e >> 1 & 1] = add2(part[e >> 1 & 1], pair(x, y));
                    const __half2 hh = __floats2half2_rn(x, y);
                    w[e / 2] = *reinterpret_cast<const uint32_t*>(&hh);
                }
                float x, y;
                unpair(add2(part[0], part[1]), x, y);
                sum = fmaf(x + y, inv, sum);
                tmem_st16(s_col + 16 * c, w);
            };
            if (CAP && !whole) {
                weigh(0, va, a0, b0, i0v, std::true_type{}, std::false_type{});
                weigh(1, vb, a1, b1, i1v, std::true_type{}, std::false_type{});
            } else if (!CAP && __builtin_expect(far, 0)) {
                weigh(0, va, a0, b0, i0v, std::false_type{}, std::true_type{});
                weigh(1, vb, a1, b1, i1v, std::false_type{}, std::true_type{});
            } else {
                weigh(0, va, a0, b0, i0v, std::false_type{}, std::false_type{});
                weigh(1, vb, a1, b1, i1v, std::false_type{}, std::false_type{});
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + buf);
        }
        // ---- output
        if (mine > 0 && !slow) {
            ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(o_last + 2 * t + 1, 0));
            tc_fence_after();
        }
        if (mx == -INFINITY && sum < INFINITY) sum = 0.0f;  // nothing seen: what ex2_fma makes of -inf
        const float ref = mine > 0 ? (slow ? 1.0f : *unit_v) : 0.0f, base = mx - (slow ? 0.0f : kTcLift);
        const float mul = poison ? NAN : sum == 0.0f ? 0.0f : ref / sum;
        T* out = static_cast<T*>(p.a.out) + at * p.a.out_stride + static_cast<uint64_t>(h) * HD;
        const uint64_t prow = ((static_cast<uint64_t>(seq) * p.a.max_new + i0 + token) * p.a.H + h) * p.splits + split;
        const bool more = RUNS && !slow && mine > kTcRun;
        const float f_kept = kept_mx == -INFINITY ? 0.0f : ex2(kept_mx - mx);
#pragma unroll 2
        for (int d = 0; d < HD; d += 16) {
            uint32_t v[16] = {};
            if (mine > 0) tmem_ld16(tmem + lanes + Shape::kOCol + t * HD + d, v);
            if (more) {
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(fmaf(kept[d + e], f_kept, __uint_as_float(v[e])));
            }
            if (live && used == 1) {
                uint32_t x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = pack_rows<T>(__uint_as_float(v[2 * e]) * mul, __uint_as_float(v[2 * e + 1]) * mul);
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    reinterpret_cast<uint4*>(out + d)[e] = make_uint4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
            } else if (live) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    reinterpret_cast<float4*>(p.part + prow * HD + d)[e] =
                        make_float4(__uint_as_float(v[4 * e]) * mul, __uint_as_float(v[4 * e + 1]) * mul,
                                    __uint_as_float(v[4 * e + 2]) * mul, __uint_as_float(v[4 * e + 3]) * mul);
                }
            }
        }
        if (live) {
            if (used == 1) {
                if (p.a.lse) p.a.lse[at * p.a.H + h] = kv8_lse(base, sum);
            } else {
                p.part_ml[prow * 2] = base;
                p.part_ml[prow * 2 + 1] = sum;
            }
        }
        tc_fence_before();
    } else if (warp < 4 * MT + 8) {
        // ----------------------------------------------------------- pages
        fewer_registers<Shape::kRegsPage>();
        const bool keys = warp < 4 * MT + 4;
        const int c0 = tid - 128 * (keys ? MT : MT + 1);
        constexpr int C = PG * HD * 2 / 128;  // 16-byte pieces of a block that a thread brings
        constexpr int kPieces = HD * 2 / 128; // of them in a page
        // Piece i of a thread is 128 pieces behind piece i - 1: a whole number of the periods below, so its page, its
        // offset in the page and in the operand tile are constants away.  Pieces are dealt so that a quarter warp's
        // stores meet all banks: 64 dims of two keys; 4 dims of values from both halves of a swizzle period.
        const int pairs = c0 / 8, k_key = pairs / (HD / 64) * 2 + c0 / 4 % 2, k_dim = (pairs % (HD / 64) * 4 + c0 % 4) * 16;
        const int q4 = c0 / 2 % 4, v_dim = c0 / 16 * 8 + c0 / 8 % 2 * 2 + (q4 & 1) + (q4 >> 1) * 4, v_key = c0 % 2 * 16;
        const int8_t* pool = (keys ? p.a.c.k + (k_key * HD + k_dim) : p.a.c.v + (v_dim * static_cast<int>(kKv8Page) + v_key)) +
                             static_cast<uint64_t>(g) * (kKv8Page * HD);
        const uint32_t to = keys ? k_dim / 64 * (KB * 128) + sw128_offset(k_key, k_dim % 64) : sw128_offset(v_dim, v_key);
        uint8_t* stages = keys ? sk : sv;
        uint64_t* full = keys ? k_full : v_full;
        uint64_t* empty = keys ? k_empty : v_empty;
        uint4 r[C];
        // pool index of each page of the block at hand and of the next: looked up a block ahead of the codes
        int ids[PG], ids_next[PG] = {};
        const int mine_c = keys ? c0 : lane;  // the page of a block whose scales this thread knows, if below PG
        float ks = 0.0f, vs = 0.0f;
        int v_exp = 0;  // the CTA's largest value scale, its exponent field
        for (int j = -2; j < blocks_k; ++j) {  // store block j, ask for block j + 1, look block j + 2 up
            if (j >= 0) {
                const int s = j % ST;
                // as one warp: lanes that gave up alone would leave the others in the warp barrier below
                if (j >= ST) ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(empty + s, ((j / ST) - 1) & 1));
                if (!ok) break;
                uint8_t* at = stages + s * Shape::kKTile;
                if (keys) {
                    if (c0 < PG) {
                        int id = ids[0];
#pragma unroll
                        for (int x = 1; x < PG; ++x) id = x == c0 ? ids[x] : id;
                        TcMeta e{0.0f, 0.0f, 1.0f, id >= 0};
                        if (e.there) {
                            e.k_scale = ks;
                            if (vs != 0.0f && vs == vs) {
                                const float f = scale_rest(vs);
                                e.v_log = log2f(f);
                                e.v_inv = 1.0f / f;
                            }
                        }
                        meta[(j & 3) * PG + c0] = e;
                    }
#pragma unroll
                    for (int i = 0; i < C; ++i) {
                        constexpr uint32_t step = 128 / (HD / 16) * 128;  // keys of 128 pieces
                        store_codes(at + to + i * step, at + (to ^ 16u) + i * step, r[i]);
                    }
                } else {
                    // the power of two that the codes of page `lane` are stored times; 0 for a page of zeros or NaN
                    const float up = vs > 0.0f ? power_of_two(scale_power(vs) - v_exp + kTcCodeUp) : 0.0f;
                    const __half2 up2 = __float2half2_rn(up);
                    const uint32_t mul_l = *reinterpret_cast<const uint32_t*>(&up2);
                    uint32_t mul = 0;
#pragma unroll
                    for (int i = 0; i < C; ++i) {
                        if (i % kPieces == 0) mul = __shfl_sync(0xffffffffu, mul_l, i / kPieces);
                        const __half2 m2 = *reinterpret_cast<const __half2*>(&mul), off = __hmul2(m2, __float2half2_rn(-1152.0f));
                        // 64 dims of 128 pieces; a page's keys are half a swizzled row, two pages a row
                        const uint32_t v_to = to ^ (i / kPieces % 2 * 64u);
                        const uint32_t place = i / kPieces / 2 * (HD * 128) + i % kPieces * (64 * 128);
                        store_codes(at + v_to + place, at + (v_to ^ 16u) + place, r[i], m2, off);
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(full + s);
            }
#pragma unroll
            for (int c = 0; c < PG; ++c) {
                ids[c] = ids_next[c];
                const uint32_t i = j0 + (j + 2) * PG + c;
                ids_next[c] = -1;
                if (j + 2 < blocks_k && i < j1) {
                    ids_next[c] = kv8_page(p.a.c, seq, span.page(i), p.a.status);
                    if (ids_next[c] < 0) *missing = 1;
                }
            }
            if (j < -1 || j + 1 >= blocks_k) continue;
            // a page that is not there is zeros: its weights are 0 and must meet finite values
#pragma unroll
            for (int c = 0; c < PG; ++c) {
                const int8_t* from = pool + static_cast<uint64_t>(max(ids[c], 0)) * p.a.c.kv * (kKv8Page * HD);
#pragma unroll
                for (int i = 0; i < kPieces; ++i) {
                    r[c * kPieces + i] = make_uint4(0, 0, 0, 0);
                    if (ids[c] >= 0) r[c * kPieces + i] = __ldg(reinterpret_cast<const uint4*>(from + i * 2048));
                }
            }
            if (mine_c < PG) {
                int id = ids[0];
#pragma unroll
                for (int x = 1; x < PG; ++x) id = x == mine_c ? ids[x] : id;
                const uint64_t head = static_cast<uint64_t>(max(id, 0)) * p.a.c.kv + g;
                ks = __ldg(p.a.c.k_scale + head);
                vs = id < 0 ? 0.0f : __ldg(p.a.c.v_scale + head);  // a page that is not there is zeros
            }
            if (j == -1) {
                if (keys) {
                    // the value scales of the CTA's pages, while the first block's codes travel
                    int top = 0, low = 255;
                    for (uint32_t i = j0 + c0; i < j1; i += 128) {
                        const int id = kv8_page(p.a.c, seq, span.page(i), p.a.status);
                        const float v = id < 0 ? 0.0f : p.a.c.v_scale[static_cast<uint64_t>(id) * p.a.c.kv + g];
                        if (v != v) *poisoned = 1;
                        if (v == 0.0f || v != v) continue;
                        top = max(top, scale_exponent(v));
                        low = min(low, v > 0.0f ? scale_exponent(v) : 0);
                    }
                    top = __reduce_max_sync(0xffffffffu, top);
                    low = __reduce_min_sync(0xffffffffu, low);
                    if (lane == 0) v_top[warp - 4 * MT] = top, v_low[warp - 4 * MT] = low;
                    named_bar_sync(1, 128);
                    if (c0 == 0) {
                        top = max(max(v_top[0], v_top[1]), max(v_top[2], v_top[3]));
                        low = min(min(v_low[0], v_low[1]), min(v_low[2], v_low[3]));
                        const bool some = low < 255;  // a scale that is not 0
                        *wide = some && (top < kTcScaleLow || top > kTcScaleHigh || low < top - kTcScaleSpan);
                        *unit_v = some ? power_of_two(min(max(top, kTcScaleLow), kTcScaleHigh) - 127 - kTcCodeUp) : 1.0f;
                    }
                }
                named_bar_sync(2, Shape::kThreads);
                if (*wide) break;
                v_exp = max(max(v_top[0], v_top[1]), max(v_top[2], v_top[3]));
            }
        }
    } else {
        // -------------------------------------------- MMA, as a whole warp: see warp_mma_ss
        fewer_registers<Shape::kRegsMma>();
        const int t = warp - (4 * MT + 8);
        if (t < MT) {
            if (J > 0) named_bar_sync(2, Shape::kThreads);
            auto wait = [&](uint64_t* bar, int phase) { ok = __all_sync(0xffffffffu, ok && mbar_wait_bounded(bar, phase & 1)); };
            const bool none = J == 0 || *wide;  // no key tile, or none for the tensor cores
            const int mine = none ? 0 : t ? need[1] : need[0];
            int k_seen = -1, v_seen = -1;  // blocks waited for
            const uint64_t qa = sw128_desc(smem_addr(sq + t * Shape::kQTile));
            if (mine > 0) wait(q_full, 0);
            // j < 0: only S of the first key tiles
#pragma unroll 1
            for (int j = -kLook; j < mine && ok; ++j) {
                if (j >= 0) {
                    const int buf = 2 * t + (j & 1), blk = j / SUB;
                    wait(p_full + buf, j >> 1);
                    if (blk > v_seen) {
                        wait(v_full + blk % ST, blk / ST);
                        v_seen = blk;
                    }
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t va = sw128_desc(smem_addr(sv + blk % ST * Shape::kKTile) + j % SUB * (HD * 128));
#pragma unroll
                    for (int k = 0; k < KT / 16; ++k) {
                        warp_mma_ts(tmem + Shape::kOCol + t * HD, tmem + buf * KT + k * 8, va + k * 2, kIdescO, j > 0 || k > 0);
                    }
                    if (j + 2 >= mine) warp_commit(o_last + 2 * t + (j + 1 == mine));
                    if (j + 1 == mine || j % SUB == SUB - 1) warp_commit(v_empty + blk % ST);
                }
                const int next = j + kLook;
                if (next < mine) {
                    const int buf = 2 * t + (next & 1), blk = next / SUB;
                    if (blk > k_seen) {
                        wait(k_full + blk % ST, blk / ST);
                        k_seen = blk;
                    }
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t ka = sw128_desc(smem_addr(sk + blk % ST * Shape::kKTile) + next % SUB * (KT * 128));
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {  // descriptors count in 16 bytes
                        warp_mma_ss(tmem + buf * KT, qa + (k / 4 * (128 * 128) + k % 4 * 32) / 16,
                                    ka + (k / 4 * (KB * 128) + k % 4 * 32) / 16, kIdescS, k > 0);
                    }
                    warp_commit(s_full + buf);
                    if (next + 1 == mine || next % SUB == SUB - 1) warp_commit(k_empty + blk % ST);
                }
            }
            // blocks that only the other row tile reads: given back as they come, so that each counts in its own phase
            for (int blk = (mine + SUB - 1) / SUB; blk < blocks_k && ok && !none; ++blk) {
                wait(k_full + blk % ST, blk / ST);
                if (lane == 0) mbar_arrive(k_empty + blk % ST);
                wait(v_full + blk % ST, blk / ST);
                if (lane == 0) mbar_arrive(v_empty + blk % ST);
            }
            if (!ok) {
                warp_commit(drained + t);
                mbar_wait_bounded(drained + t, 0);
            }
        } else if (J > 0) {
            named_bar_sync(2, Shape::kThreads);
        }
    }
    if (!ok) atomicOr(p.a.status, kStatusWaitTimeout);
    __syncthreads();
    if (warp == 4 * MT + 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// -------------------------------------------------------------------- host

template <typename T, int HD, int CAP, bool RUNS>
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
            e = cudaFuncSetAttribute(kv8_prefill_tc_kernel<T, HD, CAP, RUNS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kBytes);
            if (e != cudaSuccess) return e;
            done |= bit;
        }
    }
    const dim3 grid((p.a.max_new + p.tile - 1) / p.tile * p.a.c.kv, 1, p.a.count * p.splits);
    e = launch(kv8_prefill_tc_kernel<T, HD, CAP, RUNS>, grid, dim3(Shape::kThreads), Shape::kBytes, s, false, p);
    if (e != cudaSuccess || p.splits == 1) return e;
    return kv8_join(p, HD, p.a.dtype, s);
}

uint32_t kv8_prefill_tc_rows(uint32_t hd) { return hd == 256 ? 128u : 256u; }

template <typename T, int HD>
static cudaError_t tc_form(const Kv8Split& p, cudaStream_t s) {
    const bool runs = p.chunk > 2 * kTcRun;  // two pages a key tile
    if (p.a.softcap > kKv8FastCap) return tc_launch<T, HD, 2, true>(p, s);
    if (p.a.softcap > 0.0f) return runs ? tc_launch<T, HD, 1, true>(p, s) : tc_launch<T, HD, 1, false>(p, s);
    return runs ? tc_launch<T, HD, 0, true>(p, s) : tc_launch<T, HD, 0, false>(p, s);
}

cudaError_t kv8_prefill_tc(const Kv8Split& p, uint32_t hd, cudaStream_t s) {
#define VRT_TC(HD)                                                              \
    if (hd == HD) {                                                             \
        if (p.a.dtype == VRT_F16) return tc_form<__half, HD>(p, s);             \
        if (p.a.dtype == VRT_BF16) return tc_form<__nv_bfloat16, HD>(p, s);     \
    }
    VRT_TC(64) VRT_TC(128) VRT_TC(256)
#undef VRT_TC
    return cudaErrorInvalidValue;
}

}  // namespace vrt
