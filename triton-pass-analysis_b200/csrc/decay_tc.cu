// Decay attention of 16-bit inputs on the tensor cores (formulas: decay.cu).
//
// A chunk of 128 tokens, a head's dk <= 128 columns of q and k and 64 of v are four products:
//
//   scores  Q K^T            128 x 128 x dk    -> P = scores . L, as two terms
//   P V                      128 x 64 x 128    P from tensor memory, where its scores were
//   Q S                      128 x 64 x dk     S as two terms, side by side in N
//   K^T (w V)                dk x 64 x 128     w_j = decay^(C-1-j); w V as terms, side by side in N
//
// The state S stays in registers, float32, and takes the last product as S <- decay^C S + it (the power
// as two floats: it compounds over the chunks).  The factors w have 24 bits, so bfloat16's w V is cut
// into three terms of 8 bits, exactly; float16's is rounded to two of 11, which leaves 22.  (Two
// bfloat16 terms of w V would leave errors of 2.5e-6 in the state; these leave 3e-7.)  P and S are rounded to
// two terms for their products: 16 bits of bfloat16, 22 of float16, so that an output is as good as a
// float32 sum that is rounded once.  (P as one term: the error of bfloat16 outputs was 1.25 times that, of
// one head's 64 tokens 1.7 times; 16 x 2048 x 16 heads of 64 took 69 us, and takes 79.)  float16's range is far
// below what scores and states take: see its exponents below.
//
// Tensor memory holds 512 columns: scores 128, Q S 2 x 64, P V 64 (float16: 2 x 64), K^T (w V) 3 x 64 (2 x 64).
// Terms lie side by side because such narrow products are bound by shared memory: 128 x 64 x 16 reads 6 KB of
// operands, 48 cycles, where the tensor pipe needs 16; the other operand is read once for all terms.
//
// Warps have one role each, and each walks the block's items (a segment of a sequence, a head, 64 columns
// of v) and their chunks; what bounds a chunk is the chain scores -> P -> P V -> the next scores, which
// share their columns, and beside it instruction issue (49% of the slots taken, the tensor pipe
// 42%; DRAM 34%).  The code is kept short on purpose: with every loop unrolled it had 150 KB and
// ran at half the speed, waiting for instructions.  16 x 2048 tokens x 16 heads of 64, bf16: 79 us,
// 3.4 TB/s of 6.5 (float16: 110); 64 x 2048 x 8 of 128: 352 us, 3.1 TB/s; one sequence of 16384 x 32 of 128:
// 262 us (346), of which a third is the pass before, over k and v, that leaves the state of its first half.
//
// Waits are bounded as elsewhere (tc_common.cuh).
#include "decay.cuh"
#include "tc_common.cuh"

namespace snnb {
namespace decay {
namespace {

constexpr int C = 128;             // tokens of a chunk
constexpr int DV = 64;             // columns of v, and of the state, that a thread block takes

// STATES: no q, scores or outputs.
template <int DK, bool STATES, bool HALF> struct Smem {
    static constexpr int KB = DK / 64;                         // 64-column blocks of q and k
    static constexpr int BLOCK = C * 128;                      // 128 rows of 128 bytes
    static constexpr int QK_STAGES = DK == 64 || STATES ? 3 : 2, V_STAGES = STATES ? 3 : 2;
    static constexpr int K_IN_STAGE = STATES ? 0 : KB * BLOCK; // q, then k
    static constexpr int QK_STAGE = K_IN_STAGE + KB * BLOCK;
    static constexpr int V_OFF = QK_STAGES * QK_STAGE;
    static constexpr int S_OFF = V_OFF + V_STAGES * BLOCK;     // state: high and low terms
    static constexpr int S_TERM = STATES ? 0 : DK * 128;
    // the scaled v's three terms: both halves of a chunk where there is room, else one at a time
    static constexpr int VT_HALVES = DK == 64 || STATES ? 2 : 1;
    static constexpr int TERMS = HALF ? 2 : 3;
    static constexpr int VT_OFF = S_OFF + 2 * S_TERM, VT_TERM = BLOCK / 2, VT_HALF = TERMS * VT_TERM;
    static constexpr bool STAGED = DK == 64 && !STATES;                   // outputs leave by bulk copies
    static constexpr int O_OFF = VT_OFF + VT_HALVES * VT_HALF;         // 32 rows for each warp
    static constexpr int PW_OFF = O_OFF + (STAGED ? BLOCK : 0);  // 0 (31 times), decay^0 .. ^127
    static constexpr int RW_OFF = PW_OFF + 160 * 4;            // decay^31 .. decay^0
    static constexpr int WV_OFF = RW_OFF + 32 * 4;             // the factors of v's rows
    static constexpr int BAD_OFF = WV_OFF + C * 4;             // [4][DV] rows, [4] chunk numbers
    static constexpr int TOP_OFF = BAD_OFF + (4 * DV + 4) * 4; // [8][2] largest v, state
    // float16: the powers of two of P's rows [4 chunks][C], and what they come from: each row's largest
    // q and k [2][C]
    static constexpr int PROW_OFF = TOP_OFF + 8 * 2 * 4;
    static constexpr int TOP_ROW_OFF = PROW_OFF + (HALF ? 4 * C * 4 : 0);
    static constexpr int BAR_OFF = TOP_ROW_OFF + (HALF ? 2 * C * 4 : 0);
    static constexpr int NBARS = 2 * QK_STAGES + 2 * V_STAGES + 16;
    static constexpr int TMEM_OFF = BAR_OFF + NBARS * 8;
    static constexpr int DYN = TMEM_OFF + 8 + 1024;
    static_assert(DYN <= 227 * 1024, "shared memory");
    static_assert(BAR_OFF % 8 == 0 && RW_OFF % 16 == 0 && PROW_OFF % 16 == 0, "alignment");
};

// TMEM columns: scores (and over their first half P), q times the state's two terms, P V, K^T
// times the scaled v's two or three terms.
constexpr int T_QK = 0, T_QS = 128, T_PV = 256, T_KV = 320, T_COLS = 512;
constexpr int T_PV_LOW = 448;      // float16's second term of P times v, behind its two of the scaled v

// Warps 0-3 scores to P, 4 copies, 5 MMAs, 6 and 7 with warps 2 and 3, whose rows have the most
// scores; 8-11 outputs, 12-15 the state, 16-19 and 20-23 scaled v, a half of each chunk.
constexpr int THREADS = 24 * 32;
// Registers a thread of each group of four warps, each of which sets its own before its role: no
// more than 80 on the average, the launch's, or the state's warps would wait for theirs forever.
constexpr int REGS_P = 72, REGS_O = 72, REGS_S = 120, REGS_V = 72;
static_assert(2 * REGS_P + REGS_O + REGS_S + 2 * REGS_V <= 6 * 80, "registers");
template <int N> __device__ __forceinline__ void fewer_regs() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> __device__ __forceinline__ void more_regs() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

struct TcArgs {
    Args a;
    int tiles;                     // of DV columns
    int segs, cps;                 // segments of each sequence, chunks of a segment
    uint32_t items;                // of this launch
    float* work;                   // [segs][B H tiles][DK][DV] states (slot segs - 1: the start)
    int* status;
    bool out32;                    // the output's rows are 32-byte aligned
};

// A thread block's unit of work: a segment of a sequence, a head, DV columns.
struct Item {
    int64_t len;
    int b, h, hk, bht, tile, seg;
    int c0, n, last;               // first chunk, chunks, tokens of the last one
    bool end;                      // of the sequence
    float lam;
    __device__ __forceinline__ Item(const TcArgs& p, uint32_t it) {
        const Args& a = p.a;
        const uint32_t H = (uint32_t)a.H, tiles = p.tiles, rest = it / tiles;
        tile = (int)(it - rest * tiles);
        const uint32_t sb = rest / H;                          // segment and sequence
        h = (int)(rest - sb * H);
        seg = (int)(sb / (uint32_t)a.B);
        b = (int)(sb - (uint32_t)seg * (uint32_t)a.B);
        bht = (int)(it - (uint32_t)seg * (uint32_t)a.B * H * tiles);
        hk = (int)((uint32_t)h / (uint32_t)(a.H / a.Hk));
        len = a.length(b);
        lam = a.decay[h];
        const int all = (int)((len + C - 1) / C);
        c0 = min(seg * p.cps, all);
        n = min(p.cps, all - c0);
        end = c0 + n == all && (n > 0 || seg == 0);
        last = n > 0 && c0 + n == all ? (int)(len - (int64_t)(all - 1) * C) : C;
    }
};

// Operand with its rows (128 bytes, 128-byte swizzle) along K: `mn` bytes to the next 64 of M or N.
__device__ __forceinline__ uint64_t sdesc_mn_sw128(uint32_t saddr, uint32_t mn) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(mn >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
constexpr uint32_t A_MN = 1u << 15, B_MN = 1u << 16;           // instruction descriptor bits

// D (+)= A [TMEM, bf16 pairs] * B [smem].
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15, %16};" ::"r"(t),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z),
                 "r"(v.w)
                 : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(a)
                 : "memory");
    return v;
}
// Tables: written between barriers that the compiler does not move these across.
__device__ __forceinline__ float lds_f(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ float4 lds_f4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(a));
    return v;
}
__device__ __forceinline__ void sts_f(uint32_t a, float v) {
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}
// Byte offset of 16-byte piece `piece` of row `row` in a tile of 128-byte rows.
__device__ __forceinline__ uint32_t swizzled(int row, int piece) {
    return (uint32_t)(row * 128 + ((piece ^ (row & 7)) << 4));
}
template <bool HALF> __device__ __forceinline__ uint32_t pair(float a, float b) {
    if constexpr (HALF) return mx::round_pair(a, b, (const __half*)nullptr);
    else return mx::round_pair(a, b, (const __nv_bfloat16*)nullptr);
}
template <bool HALF> __device__ __forceinline__ float2 floats(uint32_t u) {
    if constexpr (HALF) return mx::pair_f32(u, (const __half*)nullptr);
    else return mx::pair_f32(u, (const __nv_bfloat16*)nullptr);
}
// Exponents.  float16 operands are brought below 2^15 by powers of two, exactly: its largest value
// is 65504, and scores, states and sums can be any.  bfloat16 has float's range and needs none.
//   P    each row by itself: |P_ij| < 2^7 |q_i| |k_j| with the largest |k| of j <= i, so that no later token
//        costs an earlier row its bits (one power for the chunk left scores of small rows beside large
//        ones few bits or none)
//   w V  by the largest of the chunk's 64 columns of v; S by the largest of the state's
// What a first term leaves, 2^-25 of the scaled range at most for values that are float16's
// subnormals there, is multiplied by LOW before it is rounded to the second, whose products are summed
// by themselves: a value is held to 2^-22 of itself or 2^-50 of the largest in that range, whichever is more.
// Rows' largest values and second terms of P: 8 x 2048 x 16 of 64 57 us (48 with one power for all).
__device__ __forceinline__ float pow2(int n) { return __int_as_float((n + 127) << 23); }
// b with |x| < 2^b for the largest magnitude's bits.
__device__ __forceinline__ int above_half(uint32_t bits) { return (int)max(bits >> 10, 1u) - 14; }
__device__ __forceinline__ int above_float(uint32_t bits) { return max((int)(bits >> 23) - 126, -100); }
constexpr float LOW = 2048.0f;
// 1 / x of a power of two.
__device__ __forceinline__ float over_pow2(float x) { return __int_as_float(0x7F000000 - __float_as_int(x)); }
constexpr uint32_t idesc16(bool half, int M, int N) {
    return tc::idesc_bf16_f32(M, N) & (half ? ~((1u << 7) | (1u << 10)) : ~0u);
}
// 16 outputs of a row, the first `cols` (a multiple of 8) inside.
__device__ __forceinline__ void store16(uint16_t* o, const uint32_t (&w)[8], int cols, bool al32) {
    if (al32) {                                      // then cols is a multiple of 16
        if (cols > 0)
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(o), "r"(w[0]),
                         "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
        return;
    }
    if (cols > 0) reinterpret_cast<uint4*>(o)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    if (cols > 8) reinterpret_cast<uint4*>(o)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}
// The upper halves of two floats as bf16 (cut, not rounded), and a float's upper half as a float.
__device__ __forceinline__ uint32_t tops(float a, float b) {
    return __byte_perm((uint32_t)__float_as_int(a), (uint32_t)__float_as_int(b), 0x7632);
}
// The largest magnitudes' bits of 16-bit values, in pairs.
__device__ __forceinline__ uint32_t largest(uint32_t top, uint4 r) {
    const uint32_t m = 0x7FFF7FFFu;
    return __vmaxu2(__vmaxu2(top, __vmaxu2(r.x & m, r.y & m)), __vmaxu2(r.z & m, r.w & m));
}
// The same without infinities and NaN, of float16.
__device__ __forceinline__ uint32_t largest_finite(uint32_t top, uint4 r) {
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
    for (int i = 0; i < 8; ++i) {
        const uint32_t x = u[i >> 1] >> (16 * (i & 1)) & 0x7FFFu;
        if (x < 0x7C00u) top = max(top, x);
    }
    return top;
}
__device__ __forceinline__ float top_f(float a) {
    return __int_as_float(__float_as_int(a) & (int)0xFFFF0000u);
}

// STATES: only the states that the segments leave, each from zero (the first: from state_in).
template <int DK, bool STATES, bool HALF>
__global__ void __launch_bounds__(THREADS, 1)
decay_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO,
                const __grid_constant__ TcArgs p) {
    using L = Smem<DK, STATES, HALF>;
    constexpr int NQ = L::QK_STAGES, NV = L::V_STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = tc::smem_u32(smem);
    const uint32_t pw = sbase + L::PW_OFF, rw = sbase + L::RW_OFF, wv = sbase + L::WV_OFF;
    const uint32_t prow = sbase + L::PROW_OFF;
    uint32_t* tops8 = reinterpret_cast<uint32_t*>(smem + L::TOP_OFF);       // of chunk g: 2 (g & 7)
    // of a chunk's columns, the first row that is not finite: 256 times the chunk's number + 255 - row
    uint32_t* bad_row = reinterpret_cast<uint32_t*>(smem + L::BAD_OFF);
    volatile int* bad_chunk = reinterpret_cast<int*>(bad_row + 4 * DV);
    const uint32_t bar0 = sbase + L::BAR_OFF;
    auto qk_full = [&](uint32_t s) { return bar0 + 8u * s; };
    auto qk_empty = [&](uint32_t s) { return bar0 + 8u * (NQ + s); };
    auto v_full = [&](uint32_t s) { return bar0 + 8u * (2 * NQ + s); };
    auto v_empty = [&](uint32_t s) { return bar0 + 8u * (2 * NQ + NV + s); };
    const uint32_t misc = bar0 + 8u * (2 * NQ + 2 * NV);
    const uint32_t qk_ready = misc, p_ready = misc + 8, o_ready = misc + 16, o_free = misc + 24,
                   kv_ready = misc + 40, kv_read = misc + 48,
                   s_ready = misc + 56, qs_done = misc + 64, vt_free = misc + 72,
                   done = misc + 80;
    auto vt_ready = [&](int half) { return misc + (half ? 88u : 32u); };
    auto top_ready = [&](uint32_t i) { return misc + 96u + 8u * i; };       // float16: four in turn
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::TMEM_OFF);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Args& a = p.a;

    if (threadIdx.x == 0) {
        for (int s = 0; s < NQ; ++s) {
            tc::mbar_init(qk_full(s), 1);
            tc::mbar_init(qk_empty(s), 1);
        }
        for (int s = 0; s < NV; ++s) {
            tc::mbar_init(v_full(s), 1);
            tc::mbar_init(v_empty(s), 1);
        }
        tc::mbar_init(qk_ready, 1);
        tc::mbar_init(p_ready, 6);
        tc::mbar_init(o_ready, 1);
        tc::mbar_init(o_free, 4);
        tc::mbar_init(vt_ready(0), 4);
        tc::mbar_init(vt_ready(1), 4);
        tc::mbar_init(kv_ready, 1);
        tc::mbar_init(kv_read, 4);
        tc::mbar_init(qs_done, 1);
        tc::mbar_init(vt_free, 1);
        for (int i = 0; i < 4; ++i) tc::mbar_init(top_ready(i), 4);
        tc::mbar_init(s_ready, 4);
        tc::mbar_init(done, 1);
        tc::fence_mbar_init();
        tc::prefetch_tmap(&tmQ);
        tc::prefetch_tmap(&tmK);
        tc::prefetch_tmap(&tmV);
        for (int i = 0; i < 4; ++i) bad_chunk[i] = -1;
    }
    if (threadIdx.x < 4 * DV) bad_row[threadIdx.x] = 0;
    else if (threadIdx.x < 4 * DV + 16) tops8[threadIdx.x - 4 * DV] = 0;
    if (warp == 5) {
        tc::tmem_alloc(sbase + L::TMEM_OFF, T_COLS);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_trigger();
    pdl_wait();

    // Every role walks the block's items and their chunks; g counts the chunks of all.
    uint32_t failed = 0, g = 0;
    if (warp < 8) {
        fewer_regs<REGS_P>();
        if (warp == 4) {
            // ------------------------------------------------ copies
            uint32_t issued_qk = 0, issued_v = 0;
            for (uint32_t it = blockIdx.x; it < p.items; it += gridDim.x) {
                const Item x(p, it);
                for (int c = 0; c < x.n; ++c, ++g) {
                    const uint32_t s = g % NQ, sv = g % NV;
                    const int n0 = (x.c0 + c) * C;
                    failed |= 1u - tc::mbar_wait_warp(qk_empty(s), ((g / NQ) & 1u) ^ 1u, failed);
                    if (!failed && tc::elect_one()) {
                        const uint32_t q = sbase + s * L::QK_STAGE, k = q + L::K_IN_STAGE;
                        tc::mbar_expect_tx(qk_full(s), (uint32_t)L::QK_STAGE);
#pragma unroll
                        for (int i = 0; i < L::KB; ++i) {
                            if (!STATES)
                                tc::tma_load_4d(q + i * L::BLOCK, &tmQ, qk_full(s), 64 * i, x.h, n0, x.b);
                            tc::tma_load_4d(k + i * L::BLOCK, &tmK, qk_full(s), 64 * i, x.hk, n0, x.b);
                        }
                    }
                    __syncwarp();
                    if (!failed) ++issued_qk;
                    failed |= 1u - tc::mbar_wait_warp(v_empty(sv), ((g / NV) & 1u) ^ 1u, failed);
                    if (!failed && tc::elect_one()) {
                        tc::mbar_expect_tx(v_full(sv), (uint32_t)L::BLOCK);
                        tc::tma_load_4d(sbase + L::V_OFF + sv * L::BLOCK, &tmV, v_full(sv), DV * x.tile,
                                        x.hk, n0, x.b);
                    }
                    __syncwarp();
                    if (!failed) ++issued_v;
                }
            }
            // copies in flight land before the block ends, whoever has given up waiting for them
            for (uint32_t k = 0; k < issued_qk && k < (uint32_t)NQ; ++k) {
                const uint32_t i = issued_qk - 1 - k;
                tc::mbar_wait_warp<true>(qk_full(i % NQ), (i / NQ) & 1u, 0);
            }
            for (uint32_t k = 0; k < issued_v && k < (uint32_t)NV; ++k) {
                const uint32_t i = issued_v - 1 - k;
                tc::mbar_wait_warp<true>(v_full(i % NV), (i / NV) & 1u, 0);
            }
        } else if (warp == 5) {
            // ------------------------------------------------ MMAs
            if (tc::elect_one()) {
                auto wait = [&](uint32_t bar, uint32_t parity) {
                    failed |= 1u - tc::mbar_wait_lane(bar, parity, failed);
                    tc::tc_fence_after();
                };
                uint32_t chunks = 0;
                for (uint32_t it = blockIdx.x; it < p.items; it += gridDim.x) chunks += Item(p, it).n;
                auto issue_qk = [&](uint32_t c) {
                    const uint32_t q = sbase + (c % NQ) * L::QK_STAGE, k = q + L::K_IN_STAGE;
                    wait(qk_full(c % NQ), (c / NQ) & 1u);
                    // products of different shapes are in no order of their own: P V of the chunk
                    // before, whose P the scores overwrite, has to be done
                    if (c && !STATES) wait(o_ready, (c - 1) & 1u);
                    if (failed || STATES) return;
#pragma unroll
                    for (int i = 0; i < 4 * L::KB; ++i)
                        tc::umma_bf16(tmem + T_QK, tc::sdesc_k_sw128(q + i / 4 * L::BLOCK) + 2 * (i % 4),
                                      tc::sdesc_k_sw128(k + i / 4 * L::BLOCK) + 2 * (i % 4),
                                      idesc16(HALF, 128, 128), i != 0);
                    tc::umma_commit(qk_ready);
                };
#pragma unroll 1
                for (g = 0; g < chunks && !failed; ++g) {
                    const uint32_t ph = g & 1u, s = g % NQ, sv = g % NV;
                    const uint32_t q = sbase + s * L::QK_STAGE, k = q + L::K_IN_STAGE;
                    issue_qk(g);
                    if (g) wait(kv_read, ph ^ 1u);
                    // k^T times the three terms of the scaled v, side by side, by half chunks
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        wait(vt_ready(half), ph);
                        if (failed) break;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            tc::umma_bf16(tmem + T_KV,
                                          sdesc_mn_sw128(k, DK == 64 ? 0 : L::BLOCK) + 128 * (4 * half + i),
                                          sdesc_mn_sw128(sbase + L::VT_OFF + (L::VT_HALVES - 1) * half * L::VT_HALF,
                                                         L::VT_TERM) + 128 * i,
                                          idesc16(HALF, 128, 64 * L::TERMS) | A_MN | B_MN, (half | i) != 0);
                        tc::umma_commit(half ? kv_ready : vt_free);
                    }
                    // No stage is handed back before its copies have landed, which those that scale v
                    // may have given up waiting for: its barrier's phase would still be open.
                    wait(v_full(sv), (g / NV) & 1u);
                    if (failed) break;
                    if (!STATES) {
                        wait(s_ready, ph);
                        if (g) wait(o_free, ph ^ 1u);
                        if (failed) break;
                        // q times both terms of the state, side by side
#pragma unroll
                        for (int i = 0; i < DK / 16; ++i)
                            tc::umma_bf16(tmem + T_QS, tc::sdesc_k_sw128(q + i / 4 * L::BLOCK) + 2 * (i % 4),
                                          sdesc_mn_sw128(sbase + L::S_OFF, L::S_TERM) + 128 * i,
                                          idesc16(HALF, 128, 128) | B_MN, i != 0);
                        tc::umma_commit(qs_done);
                    }
                    tc::umma_commit(qk_empty(s));
                    if (!STATES) {
                        wait(p_ready, ph);
                        if (failed) break;
#pragma unroll
                        for (int i = 0; i < 16; ++i)   // first terms, then second ones
                            umma_ts(tmem + (HALF && i >= 8 ? T_PV_LOW : T_PV),
                                    tmem + T_QK + 32 * (i % 8 / 2) + 8 * (i % 2) + i / 8 * 16,
                                    sdesc_mn_sw128(sbase + L::V_OFF + sv * L::BLOCK, 0) + 128 * (i % 8),
                                    idesc16(HALF, 128, 64) | B_MN, HALF ? i % 8 != 0 : i != 0);
                        tc::umma_commit(o_ready);
                    }
                    tc::umma_commit(v_empty(sv));
                }
                tc::umma_commit(done);
            }
            __syncwarp();
            failed = __any_sync(0xffffffffu, failed);
            failed |= 1u - tc::mbar_wait_warp<true>(done, 0, 0);
        } else {
            // ------------------------------------------------ scores to P
            // Blocks of 32 x 32: a warp has those of its rows (its lanes of TMEM) up to the
            // diagonal one; the third and the fourth of the last two warps' rows go to warps 6
            // and 7.  A block's P lies over its scores: 16 columns of first terms, 16 of second ones.
            const int q = warp & 3, first = warp >= 6 ? 2 : 0, row = 32 * q + lane;
            const bool two = q == 3 || (q >= 1 && first == 0);     // of these two blocks
            const int diag = q >= 2 && first == 0 ? -1 : q - first;     // which of the two, if any
            const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16) + T_QK;
            const uint64_t minus = mx::pack2(-1.0f, -1.0f), low2 = mx::pack2(LOW, LOW);
            auto clear = [&](uint32_t at) {
                const uint32_t zero[16] = {};
                tmem_st16(at, zero);
                tmem_st16(at + 16, zero);
            };
            for (uint32_t it = blockIdx.x; !STATES && it < p.items; it += gridDim.x) {
                const Item x(p, it);
                if (x.n == 0) continue;
                tc::named_bar_sync(2, 6 * 32);       // the last item's table has been read
                if (warp < 4) {
                    const float f = (float)power(x.lam, row);
                    sts_f(pw + 4 * (31 + row), f);
                    if (row < 32) sts_f(rw + 4 * (31 - row), f);
                    if (row < 31) sts_f(pw + 4 * row, 0.0f);
                }
                tc::named_bar_sync(2, 6 * 32);
                const float f0 = diag == 0 ? 0.0f : lds_f(pw + 4 * (row - 32 * first)),
                            f1 = diag == 1 || !two ? 0.0f : lds_f(pw + 4 * (row - 32 * first - 32));
#pragma unroll 1
                for (int c = 0; c < x.n; ++c, ++g) {
                    failed |= 1u - tc::mbar_wait_warp(qk_ready, g & 1u, failed);
                    tc::tc_fence_after();
                    float down = 1.0f;
                    if constexpr (HALF) {
                        failed |= 1u - tc::mbar_wait_warp(top_ready(g & 3), (g >> 2) & 1u, failed);
                        down = lds_f(prow + 4 * ((g & 3) * C + row));
                    }
#pragma unroll 1
                    for (int blk = 0; blk < 2; ++blk) {
                        const uint32_t at = tl + (first + blk) * 32;      // P takes its scores' place
                        uint32_t w[16], low[16];
                        if (blk && !two) {           // blocks of later tokens
                            clear(at);
                            continue;
                        }
                        float s[32];
                        tc::tmem_ld32(at, s);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(s[i]));
                        if (blk == diag) {
                            // later tokens count nothing, whatever their scores
                            const uint32_t d = pw + 4 * (31 + lane);
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                const float y = s[i] * (HALF ? lds_f(d - 4 * i) * down : lds_f(d - 4 * i));
                                s[i] = i <= lane ? y : 0.0f;
                            }
                        } else {
                            const float f = HALF ? (blk ? f1 : f0) * down : blk ? f1 : f0;
                            const uint64_t ff = mx::pack2(f, f);
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                const float4 r = lds_f4(rw + 4 * i);
                                mx::unpack2(mx::mul2(mx::pack2(s[i], s[i + 1]),
                                                     mx::mul2(ff, mx::pack2(r.x, r.y))), s[i], s[i + 1]);
                                mx::unpack2(mx::mul2(mx::pack2(s[i + 2], s[i + 3]),
                                                     mx::mul2(ff, mx::pack2(r.z, r.w))), s[i + 2], s[i + 3]);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 16; ++i) {         // the first terms, and what they leave
                            w[i] = pair<HALF>(s[2 * i], s[2 * i + 1]);
                            const float2 h = floats<HALF>(w[i]);
                            uint64_t yz = mx::fma2(mx::pack2(h.x, h.y), minus, mx::pack2(s[2 * i], s[2 * i + 1]));
                            if constexpr (HALF) yz = mx::mul2(low2, yz);
                            float y, z;
                            mx::unpack2(yz, y, z);
                            low[i] = pair<HALF>(y, z);
                        }
                        tmem_st16(at, w);
                        tmem_st16(at + 16, low);
                    }
                    if (q < 2) {
                        clear(tl + 64);
                        clear(tl + 96);
                    }
                    tmem_wait_st();
                    tc::tc_fence_before();
                    if (lane == 0) tc::mbar_arrive(p_ready);
                    __syncwarp();
                }
            }
        }
    } else if (warp < 12) {
        // ---------------------------------------------------- outputs
        fewer_regs<REGS_O>();
        const int q = warp & 3, row = 32 * q + lane;
        const uint32_t tl = tmem + ((uint32_t)(32 * q) << 16);
        const uint32_t stage = sbase + L::O_OFF + q * 32 * 128;
        for (uint32_t it = blockIdx.x; !STATES && it < p.items; it += gridDim.x) {
            const Item x(p, it);
            // a small scale and a power of the decay apart: their product may be less than float holds
            const float fq = (float)power(x.lam, row + 1);
            uint64_t fq2 = mx::pack2(fq, fq);
            const uint64_t sc2 = mx::pack2(a.scale, a.scale), up2 = mx::pack2(1.0f / LOW, 1.0f / LOW);
            const int cols = min(DV, a.dv - x.tile * DV);
            const int64_t ld = a.H * a.dv;
            uint16_t* out = static_cast<uint16_t*>(a.out) +
                                 ((int64_t)x.b * a.N * a.H + x.h) * a.dv + x.tile * DV +
                                 ((int64_t)x.c0 * C + row) * ld;
#pragma unroll 1
            for (int c = 0; c < x.n; ++c, ++g, out += C * ld) {
                const int64_t n = (int64_t)(x.c0 + c) * C + row;
                if (L::STAGED) {                     // the last copy has read its rows
                    if (lane == 0) tc::bulk_wait_group_read<0>();
                    __syncwarp();
                }
                failed |= 1u - tc::mbar_wait_warp(o_ready, g & 1u, failed);
                tc::tc_fence_after();
                uint64_t row2 = 0;
                if constexpr (HALF) {                // the powers of two of q S and of P's row undone
                    const float fs = fq * pow2(above_float(tops8[2 * (g & 7) + 1]) - 15);
                    const float f = over_pow2(lds_f(prow + 4 * ((g & 3) * C + row)));
                    fq2 = mx::pack2(fs, fs);
                    row2 = mx::pack2(f, f);
                }
                const bool spoiled = bad_chunk[g & 3] == (int)g, alive = n < x.len;
                const bool write = n < a.N && !failed && SNNB_IN_BOUNDS(n, a.N, p.status);
#pragma unroll 1
                for (int i = 0; i < DV; i += 16) {
                    float s[16], l[16], v[16];
                    tc::tmem_ld16(tl + T_QS + i, s);
                    tc::tmem_ld16(tl + T_QS + 64 + i, l);
                    if constexpr (HALF) {            // registers for two of the four
                        tc::tmem_wait_ld();
                        tc::reg_fence16(s);
                        tc::reg_fence16(l);
#pragma unroll
                        for (int j = 0; j < 16; j += 2)
                            mx::unpack2(mx::mul2(fq2, mx::fma2(mx::pack2(l[j], l[j + 1]), up2,
                                                               mx::pack2(s[j], s[j + 1]))), s[j], s[j + 1]);
                        tc::tmem_ld16(tl + T_PV_LOW + i, l);
                    }
                    tc::tmem_ld16(tl + T_PV + i, v);
                    tc::tmem_wait_ld();
                    if constexpr (!HALF) tc::reg_fence16(s);
                    tc::reg_fence16(l);
                    tc::reg_fence16(v);
                    if (i + 16 == DV) {
                        tc::tc_fence_before();
                        if (lane == 0) tc::mbar_arrive(o_free);
                        __syncwarp();
                    }
                    uint32_t w[8];
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        if constexpr (HALF) {
                            const uint64_t y = mx::fma2(mx::pack2(l[j], l[j + 1]), up2, mx::pack2(v[j], v[j + 1]));
                            mx::unpack2(mx::mul2(sc2, mx::fma2(row2, y, mx::pack2(s[j], s[j + 1]))), v[j], v[j + 1]);
                        } else {
                            const uint64_t y = mx::add2(mx::pack2(s[j], s[j + 1]), mx::pack2(l[j], l[j + 1]));
                            mx::unpack2(mx::mul2(sc2, mx::fma2(fq2, y, mx::pack2(v[j], v[j + 1]))), v[j],
                                        v[j + 1]);
                        }
                    }
                    if (spoiled) {
                        const uint32_t* rows = bad_row + (g & 3) * DV + i;
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (rows[j] >= (g << 8 | (255u - row))) v[j] = __int_as_float(0x7fffffff);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = alive ? pair<HALF>(v[2 * j], v[2 * j + 1]) : 0u;
                    if (L::STAGED) {
                        sts128(stage + swizzled(lane, i / 8), make_uint4(w[0], w[1], w[2], w[3]));
                        sts128(stage + swizzled(lane, i / 8 + 1), make_uint4(w[4], w[5], w[6], w[7]));
                    } else if (write) {
                        store16(out + i, w, cols - i, p.out32);
                    }
                    __syncwarp();
                }
                if (L::STAGED) {
                    tc::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0 && write) {        // rows behind N are not written
                        asm volatile(
                            "cp.async.bulk.tensor.4d.global.shared::cta.bulk_group "
                            "[%0, {%2, %3, %4, %5}], [%1];" ::"l"(&tmO),
                            "r"(stage), "r"(DV * x.tile), "r"(x.h), "r"((int)n), "r"(x.b)
                            : "memory");
                        tc::bulk_commit_group();
                    }
                }
            }
            if (x.end) {                             // rows behind the last chunk
                const uint32_t zero[8] = {};
#pragma unroll 1
                for (int64_t n = (int64_t)(x.c0 + x.n) * C + row; n < a.N; n += C, out += C * ld)
#pragma unroll 1
                    for (int i = 0; i < cols; i += 16) store16(out + i, zero, cols - i, p.out32);
            }
        }
        if (lane == 0) tc::bulk_wait_group<0>();     // the copies have left shared memory
    } else if (warp < 16) {
        // ---------------------------------------------------- the state
        // This thread's row and columns: DK = 64 products have 128 rows, the second 64 the
        // first's copy, so that each half of the threads takes half of the columns.
        more_regs<REGS_S>();
        const int t = threadIdx.x - 384;
        constexpr int W = DK == 64 ? 32 : 64;
        const int row = t % DK, col = DK == 64 ? t / 64 * 32 : 0;
        const uint32_t tl = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + T_KV + col;
        for (uint32_t it = blockIdx.x; it < p.items; it += gridDim.x) {
            const Item x(p, it);
            if (x.n == 0 && (STATES ? x.seg > 0 : !x.end)) continue;
            const int64_t at = (((int64_t)x.b * a.H + x.h) * a.dk + row) * a.dv + x.tile * DV + col;
            const int cols = row < a.dk ? min(W, a.dv - x.tile * DV - col) : 0;
            const int64_t slot = a.B * a.H * p.tiles * (DK * DV);
            float* work = p.work + (int64_t)x.bht * (DK * DV) + row * DV + col;
            float S[W];
            // what there is before the first chunk
            const bool segs = !STATES && p.segs > 1;
            const float* from = x.seg > 0 ? (segs ? work : nullptr)
                                : !a.state_in ? nullptr
                                : segs        ? work + (p.segs - 1) * slot
                                              : a.state_in + at;
            const int have = segs ? W : cols;
#pragma unroll
            for (int i = 0; i < W; i += 4) {
                const float4 y = from && i < have ? *reinterpret_cast<const float4*>(from + i)
                                                  : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                S[i] = y.x; S[i + 1] = y.y; S[i + 2] = y.z; S[i + 3] = y.w;
            }
            if (segs && x.seg > 1) {
                const double d = power(x.lam, p.cps * C);
                const float fh = (float)d, fl = (float)(d - (double)fh);
#pragma unroll 1
                for (int s = 1; s < x.seg; ++s) {
#pragma unroll
                    for (int i = 0; i < W; i += 4) {
                        const float4 y = *reinterpret_cast<const float4*>(work + s * slot + i);
                        S[i] = fmaf(S[i], fh, fmaf(S[i], fl, y.x));
                        S[i + 1] = fmaf(S[i + 1], fh, fmaf(S[i + 1], fl, y.y));
                        S[i + 2] = fmaf(S[i + 2], fh, fmaf(S[i + 2], fl, y.z));
                        S[i + 3] = fmaf(S[i + 3], fh, fmaf(S[i + 3], fl, y.w));
                    }
                }
            }
            auto put = [&](float* to, int n) {
#pragma unroll
                for (int i = 0; i < W; i += 4)
                    if (i < n)
                        *reinterpret_cast<float4*>(to + i) =
                            make_float4(S[i], S[i + 1], S[i + 2], S[i + 3]);
            };
            if (STATES && x.seg == 0 && a.state_in)  // state_out may be state_in
                put(work + (p.segs - 1) * slot, W);
            const double dc = power(x.lam, C), dl = power(x.lam, x.last);
            const float ch = (float)dc, cl = (float)(dc - (double)ch), lh = (float)dl,
                        ll = (float)(dl - (double)lh);
#pragma unroll 1
            for (int c = 0; c < x.n; ++c, ++g) {
                if (!STATES) {
                    // the state before this chunk, once q times the last one is done
                    if (g) failed |= 1u - tc::mbar_wait_warp(qs_done, (g - 1) & 1u, failed);
                    float up = 1.0f;
                    if constexpr (HALF) {
                        volatile uint32_t* top = tops8 + 2 * (g & 7) + 1;
                        float m = 0.0f;
#pragma unroll
                        for (int i = 0; i < W; ++i) m = fmaxf(m, fabsf(S[i]));
                        uint32_t bits = __reduce_max_sync(0xffffffffu, (uint32_t)__float_as_int(m));
                        if (lane == 0) atomicMax(&tops8[2 * (g & 7) + 1], bits);
                        if (t == 0) tops8[2 * ((g + 1) & 7) + 1] = 0;
                        tc::named_bar_sync(8, 128);
                        if (*top >= 0x7F800000u) {   // of the finite ones
                            tc::named_bar_sync(8, 128);
                            if (t == 0) *top = 0;
                            m = 0.0f;
#pragma unroll
                            for (int i = 0; i < W; ++i)
                                if (fabsf(S[i]) <= 3.4028235e38f) m = fmaxf(m, fabsf(S[i]));
                            bits = __reduce_max_sync(0xffffffffu, (uint32_t)__float_as_int(m));
                            tc::named_bar_sync(8, 128);
                            if (lane == 0) atomicMax(&tops8[2 * (g & 7) + 1], bits);
                            tc::named_bar_sync(8, 128);
                        }
                        up = pow2(15 - above_float(*top));
                    }
#pragma unroll
                    for (int i = 0; i < W; i += 8) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float y = S[i + 2 * j] * up, z = S[i + 2 * j + 1] * up;
                            hi[j] = pair<HALF>(y, z);
                            const float2 h = floats<HALF>(hi[j]);
                            lo[j] = HALF ? pair<HALF>((y - h.x) * LOW, (z - h.y) * LOW) : pair<HALF>(y - h.x, z - h.y);
                        }
                        const uint32_t o = sbase + L::S_OFF + swizzled(row, (col + i) / 8);
                        sts128(o, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                        sts128(o + L::S_TERM, make_uint4(lo[0], lo[1], lo[2], lo[3]));
                    }
                    tc::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(s_ready);
                }
                failed |= 1u - tc::mbar_wait_warp(kv_ready, g & 1u, failed);
                tc::tc_fence_after();
                const bool end = c + 1 == x.n;
                const float fh = end ? lh : ch, fl = end ? ll : cl;
                const uint64_t fh2 = mx::pack2(fh, fh), fl2 = mx::pack2(fl, fl);
                const uint64_t up2 = mx::pack2(1.0f / LOW, 1.0f / LOW);
                uint64_t back = 0;
                if constexpr (HALF) {
                    const float f = pow2(above_half(tops8[2 * (g & 7)]) - 15);
                    back = mx::pack2(f, f);
                }
#pragma unroll
                for (int i = 0; i < W; i += 16) {
                    float y[16], z[16], u[16];
                    tc::tmem_ld16(tl + i, y);
                    tc::tmem_ld16(tl + 64 + i, z);
                    if constexpr (!HALF) tc::tmem_ld16(tl + 128 + i, u);
                    tc::tmem_wait_ld();
                    tc::reg_fence16(y);
                    tc::reg_fence16(z);
                    if constexpr (!HALF) tc::reg_fence16(u);
                    if (i + 16 == W) {
                        tc::tc_fence_before();
                        if (lane == 0) tc::mbar_arrive(kv_read);
                        __syncwarp();
                    }
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const uint64_t old = mx::pack2(S[i + j], S[i + j + 1]);
                        uint64_t sum = mx::pack2(z[j], z[j + 1]);
                        if constexpr (HALF) {
                            sum = mx::fma2(sum, up2, mx::pack2(y[j], y[j + 1]));
                            sum = mx::fma2(sum, back, mx::mul2(old, fl2));
                        } else {
                            sum = mx::add2(sum, mx::pack2(u[j], u[j + 1]));
                            sum = mx::add2(mx::pack2(y[j], y[j + 1]), sum);
                            sum = mx::fma2(old, fl2, sum);
                        }
                        mx::unpack2(mx::fma2(old, fh2, sum), S[i + j], S[i + j + 1]);
                    }
                }
            }
            if (!failed && (STATES || (x.end && a.state_out)))
                put(STATES ? work + x.seg * slot : a.state_out + at, STATES ? W : cols);
        }
    } else {
        // ---------------------------------------------------- v scaled, as three bf16 terms
        fewer_regs<REGS_V>();
        const int t = threadIdx.x - 512, half = t >> 7;        // of each chunk
        const int piece = t & 7, r0 = (t >> 3) & 15, first = 64 * half + r0;
        const uint32_t vt = sbase + L::VT_OFF + (L::VT_HALVES == 2 ? half * L::VT_HALF : 0) +
                            swizzled(r0, piece);
        const uint64_t minus = mx::pack2(-1.0f, -1.0f), low2 = mx::pack2(LOW, LOW);
        for (uint32_t it = blockIdx.x; it < p.items; it += gridDim.x) {
            const Item x(p, it);
            int held = -1;                           // tokens that the factors are for
#pragma unroll 1
            for (int c = 0; c < x.n; ++c, ++g) {
                const uint32_t s = g % NV, sq = g % NQ;
                const int m = c + 1 == x.n ? x.last : C;
                if (m != held) {
                    tc::named_bar_sync(1, 256);
                    if (t < C) sts_f(wv + 4 * t, t < m ? (float)power(x.lam, m - 1 - t) : 0.0f);
                    held = m;
                    tc::named_bar_sync(1, 256);
                }
                failed |= 1u - tc::mbar_wait_warp(v_full(s), (g / NV) & 1u, failed);
                const uint32_t vs = sbase + L::V_OFF + s * L::BLOCK + swizzled(first, piece);
                if (m < C) {
                    // rows behind the sequence, whatever they hold (beyond the tensor: zeros)
                    failed |= 1u - tc::mbar_wait_warp(qk_full(sq), (g / NQ) & 1u, failed);
                    const uint32_t ks = sbase + sq * L::QK_STAGE + L::K_IN_STAGE + swizzled(first, piece);
                    const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll 1
                    for (int i = 0; i < 4; ++i)
                        if (first + 16 * i >= m) {
                            sts128(vs + 2048 * i, zero);
#pragma unroll
                            for (int k = 0; k < L::KB; ++k) {
                                sts128(ks + k * L::BLOCK + 2048 * i, zero);
                                if (HALF && !STATES) sts128(ks - L::K_IN_STAGE + k * L::BLOCK + 2048 * i, zero);
                            }
                        }
                }
                if constexpr (HALF && !STATES) {
                    // of each row the largest magnitudes of q (upper half) and of k
                    uint32_t* rows = reinterpret_cast<uint32_t*>(smem + L::TOP_ROW_OFF) + (g & 1) * C;
                    failed |= 1u - tc::mbar_wait_warp(qk_full(sq), (g / NQ) & 1u, failed);
                    const uint32_t qs = sbase + sq * L::QK_STAGE + swizzled(first, piece);
                    uint32_t y[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t tq = 0, tk = 0;
#pragma unroll
                        for (int k = 0; k < L::KB; ++k) {
                            tq = largest(tq, lds128(qs + k * L::BLOCK + 2048 * i));
                            tk = largest(tk, lds128(qs + L::K_IN_STAGE + k * L::BLOCK + 2048 * i));
                        }
                        y[i] = __vmaxu2(__byte_perm(tq, tk, 0x1054), __byte_perm(tq, tk, 0x3276));
                    }
#pragma unroll
                    for (int o = 1; o < 8; o *= 2)
#pragma unroll
                        for (int i = 0; i < 4; ++i) y[i] = __vmaxu2(y[i], __shfl_xor_sync(0xffffffffu, y[i], o));
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (piece == 0) rows[first + 16 * i] = y[i];
                }
                constexpr uint32_t INF = HALF ? 0x7C00u : 0x7F80u;
                uint32_t top = 0, hi[4][4], mid[4][4], low[4][4];
                uint4 raw[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    raw[i] = lds128(vs + 2048 * i);
                    top = largest(top, raw[i]);
                }
                float up = 1.0f;
                if constexpr (HALF) {
                    uint32_t* tops = tops8 + 2 * (g & 7);
                    uint32_t tv = max(top & 0xFFFFu, top >> 16);
                    if (tv >= INF) {
                        tv = 0;
#pragma unroll 1
                        for (int i = 0; i < 4; ++i) tv = largest_finite(tv, lds128(vs + 2048 * i));
                    }
                    tv = __reduce_max_sync(0xffffffffu, tv);
                    if (lane == 0) atomicMax(&tops[0], tv);
                    if (t == 0) tops8[2 * ((g + 1) & 7)] = 0;
                    tc::named_bar_sync(1, 256);
                    up = pow2(15 - above_half(tops[0]));
                    if (!STATES && half == 1) {
                        // P of row i is below 2^7 |q_i| |k_j|, j <= i: the rows' largest |k| so far
                        const uint32_t* rows = reinterpret_cast<uint32_t*>(smem + L::TOP_ROW_OFF) + (g & 1) * C;
                        const int r = t - 128;
                        const uint32_t own = rows[r];
                        uint32_t before = 0, most = own & 0xFFFFu;
#pragma unroll
                        for (int i = 0; i < 3; ++i)
                            if (i < r >> 5) before = max(before, rows[32 * i + lane] & 0xFFFFu);
#pragma unroll
                        for (int o = 1; o < 32; o *= 2) most = max(most, __shfl_up_sync(0xffffffffu, most, o));
                        most = max(most, __reduce_max_sync(0xffffffffu, before));
                        sts_f(prow + 4 * ((g & 3) * C + r), pow2(8 - above_half(own >> 16) - above_half(most)));
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(top_ready(g & 3));
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                    const float f = HALF ? lds_f(wv + 4 * (first + 16 * i)) * up : lds_f(wv + 4 * (first + 16 * i));
                    const uint64_t ff = mx::pack2(f, f);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 v = floats<HALF>(u[j]);
                        uint64_t yz = mx::mul2(mx::pack2(v.x, v.y), ff);
                        float y, z;
                        mx::unpack2(yz, y, z);
                        if constexpr (HALF) {
                            // 22 of 24 bits, in two terms
                            hi[i][j] = pair<HALF>(y, z);
                            const float2 h = floats<HALF>(hi[i][j]);
                            mx::unpack2(mx::mul2(low2, mx::fma2(mx::pack2(h.x, h.y), minus, yz)), y, z);
                            mid[i][j] = pair<HALF>(y, z);
                        } else {
                            // 24 bits, cut into three times 8: exact
                            hi[i][j] = tops(y, z);
                            yz = mx::fma2(mx::pack2(top_f(y), top_f(z)), minus, yz);
                            mx::unpack2(yz, y, z);
                            mid[i][j] = tops(y, z);
                            yz = mx::fma2(mx::pack2(top_f(y), top_f(z)), minus, yz);
                            mx::unpack2(yz, y, z);
                            low[i][j] = tops(y, z);
                        }
                    }
                }
                // the products have read what was there
                if (half && L::VT_HALVES == 1)
                    failed |= 1u - tc::mbar_wait_warp(vt_free, g & 1u, failed);
                else if (g)
                    failed |= 1u - tc::mbar_wait_warp(kv_ready, (g - 1) & 1u, failed);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t o = vt + 2048 * i;
                    sts128(o, make_uint4(hi[i][0], hi[i][1], hi[i][2], hi[i][3]));
                    sts128(o + L::VT_TERM, make_uint4(mid[i][0], mid[i][1], mid[i][2], mid[i][3]));
                    if constexpr (!HALF)
                        sts128(o + 2 * L::VT_TERM, make_uint4(low[i][0], low[i][1], low[i][2], low[i][3]));
                }
                if (__any_sync(0xffffffffu, (top & 0xFFFFu) >= INF || (top >> 16) >= INF)) {
                    // Values that are not finite: 0 * inf in the product of P and v would reach
                    // the chunk's earlier rows.  There they become zero, and the outputs of their
                    // columns NaN from their row on.
                    if (lane == 0) bad_chunk[g & 3] = (int)g;
                    uint32_t* rows = bad_row + (g & 3) * DV + 8 * piece;
#pragma unroll 1
                    for (int i = 0; i < 4; ++i) {
                        const uint4 r4 = lds128(vs + 2048 * i);
                        uint32_t u[4] = {r4.x, r4.y, r4.z, r4.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if ((u[j] & INF) == INF) {
                                atomicMax(&rows[2 * j], g << 8 | (255u - (first + 16 * i)));
                                u[j] &= 0xFFFF0000u;
                            }
                            if ((u[j] & (INF << 16)) == INF << 16) {
                                atomicMax(&rows[2 * j + 1], g << 8 | (255u - (first + 16 * i)));
                                u[j] &= 0xFFFFu;
                            }
                        }
                        sts128(vs + 2048 * i, make_uint4(u[0], u[1], u[2], u[3]));
                    }
                }
                tc::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(vt_ready(half));
            }
        }
    }
    if (failed && lane == 0) atomicExch(p.status, SNNB_ERR_TIMEOUT);
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 5) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, T_COLS);
    }
}

// [B, N, heads, d] as a tensor map with boxes of 128 tokens x 64 columns of one head.
int encode(CUtensorMap* m, const void* base, const int64_t* s, int64_t B, int64_t N, int64_t heads,
           int64_t d, bool half, int rows = C) {
    const uint64_t dims[4] = {(uint64_t)d, (uint64_t)heads, (uint64_t)N, (uint64_t)B};
    const uint64_t st[3] = {heads > 1 ? (uint64_t)s[2] * 2 : 16, N > 1 ? (uint64_t)s[1] * 2 : 16,
                            B > 1 ? (uint64_t)s[0] * 2 : 16};
    const uint32_t box[4] = {64, 1, (uint32_t)rows, 1};
    return encode_tmap(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, dims, st, box,
                       CU_TENSOR_MAP_SWIZZLE_128B);
}
bool mappable(const void* base, const int64_t* s, int64_t B, int64_t N, int64_t heads) {
    auto ok = [](int64_t st, int64_t n) {
        return n <= 1 || (st > 0 && st % 8 == 0 && st < (int64_t(1) << 39));
    };
    return aligned16(base) && ok(s[2], heads) && ok(s[1], N) && ok(s[0], B);
}

// SMs of the current device.
int sm_count() {
    static int counts[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (!counts[dev] &&
        cudaDeviceGetAttribute(&counts[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return 148;
    return counts[dev];
}

template <int DK, bool STATES, bool HALF>
int launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& o,
           TcArgs p, cudaStream_t s) {
    using L = Smem<DK, STATES, HALF>;
    if (const int st = allow_smem<decay_tc_kernel<DK, STATES, HALF>>(L::DYN)) return st;
    p.items = (uint32_t)(p.a.B * p.a.H * p.tiles * (STATES ? p.segs - 1 : p.segs));
    const int sms = sm_count();
    return launch_k(decay_tc_kernel<DK, STATES, HALF>, dim3(p.items < (uint32_t)sms ? p.items : sms), dim3(THREADS),
                    L::DYN, s, q, k, v, o, p);
}
template <int DK, bool HALF>
int launches(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
             const CUtensorMap& o, const TcArgs& p, cudaStream_t s) {
    if (p.segs > 1)
        if (const int st = launch<DK, true, HALF>(q, k, v, o, p, s)) return st;
    return launch<DK, false, HALF>(q, k, v, o, p, s);
}

// Segments of each sequence: more of them where the items leave SMs idle, for the price of a pass over
// k and v that leaves each segment's state.  In 0.1 us, measured with every SM busy: 24 for a chunk
// (16 to 26), 13 for one of the pass before, 30 for an item's start, 60 for the second launch.
int segments(int64_t items, int64_t chunks) {
    const int64_t sms = sm_count();
    int best = 1;
    int64_t least = 0;
    for (int n = 1; n <= 16 && (n == 1 || (chunks >= 2 * n && items <= sms)); ++n) {
        const int64_t cps = (chunks + n - 1) / n;
        if ((n - 1) * cps >= chunks) continue;
        const int64_t rounds = (items * n + sms - 1) / sms, before = (items * (n - 1) + sms - 1) / sms;
        const int64_t t = rounds * (cps * 24 + 30) + before * (cps * 13 + 30) + (n > 1 ? 60 : 0);
        if (n == 1 || t < least) {
            best = n;
            least = t;
        }
    }
    return best;
}

}  // namespace

bool tc_takes(const Args& a, int dtype) {
    return (dtype == SNNB_BF16 || dtype == SNNB_F16) && a.N > 0 && a.dk <= 128 && a.dk % 8 == 0 &&
           a.dv % 8 == 0 && aligned16(a.out) && aligned16(a.state_in) && aligned16(a.state_out) &&
           mappable(a.q, a.qs, a.B, a.N, a.H) &&
           mappable(a.k, a.ks, a.B, a.N, a.Hk) && mappable(a.v, a.vs, a.B, a.N, a.Hk);
}

int64_t tc_workspace(int dtype, int64_t B, int64_t N, int64_t H, int64_t dk, int64_t dv) {
    if ((dtype != SNNB_BF16 && dtype != SNNB_F16) || dk > 128 || dk % 8 || dv % 8 || B == 0 || N == 0) return 0;
    const int64_t items = B * H * ((dv + DV - 1) / DV);
    const int segs = segments(items, (N + C - 1) / C);
    return segs > 1 ? segs * items * (dk <= 64 ? 64 : 128) * DV * 4 : 0;
}

int tc_run(const Args& a, int dtype, void* work, int64_t bytes, cudaStream_t s) {
    const bool half = dtype == SNNB_F16;
    CUtensorMap q, k, v, o = {};
    int rc = encode(&q, a.q, a.qs, a.B, a.N, a.H, a.dk, half);
    if (!rc) rc = encode(&k, a.k, a.ks, a.B, a.N, a.Hk, a.dk, half);
    if (!rc) rc = encode(&v, a.v, a.vs, a.B, a.N, a.Hk, a.dv, half);
    const int64_t os[3] = {a.N * a.H * a.dv, a.H * a.dv, a.dv};
    if (!rc && a.dk <= 64) rc = encode(&o, a.out, os, a.B, a.N, a.H, a.dv, half, 32);
    if (rc) return rc;
    const int chunks = (int)((a.N + C - 1) / C), tiles = (a.dv + DV - 1) / DV;
    int segs = segments(a.B * a.H * tiles, chunks);
    const int cps = (chunks + segs - 1) / segs;
    TcArgs p = {a, tiles, segs, cps, 0, static_cast<float*>(work), device_status_ptr(),
                a.dv % 16 == 0 && reinterpret_cast<uintptr_t>(a.out) % 32 == 0};
    if (!p.status) return SNNB_ERR_CUDA;
    if (segs > 1 && (!work || !aligned16(work) ||
                     bytes < tc_workspace(dtype, a.B, a.N, a.H, a.dk, a.dv)))
        return SNNB_ERR_ARG;
    if (half) return a.dk <= 64 ? launches<64, true>(q, k, v, o, p, s) : launches<128, true>(q, k, v, o, p, s);
    return a.dk <= 64 ? launches<64, false>(q, k, v, o, p, s) : launches<128, false>(q, k, v, o, p, s);
}

}  // namespace decay
}  // namespace snnb
