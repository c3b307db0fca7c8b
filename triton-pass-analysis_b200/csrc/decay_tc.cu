// Decay attention of 16-bit inputs on the tensor cores (formulas: decay.cu).
#include "decay.cuh"
#include "tc_common.cuh"

namespace snnb {
namespace decay {
namespace {

constexpr int C = 128;             // tokens of a chunk
constexpr int DV = 64;             // columns of v, and of the state, that a thread block takes

template <int DK> struct Smem {
    static constexpr int STAGES = DK == 64 ? 1 : 2;
    static constexpr int QKB = DK == 64 ? 1 : 2;               // score buffers in TMEM
    static constexpr int KB = DK / 64;                         // 64-column blocks of q and k
    static constexpr int BLOCK = C * 128;                      // 128 rows of 128 bytes
    static constexpr int Q = 0, K = KB * BLOCK, V = 2 * KB * BLOCK, STAGE = (2 * KB + 1) * BLOCK;
    static constexpr int S_OFF = STAGES * STAGE;               // state: high and low terms
    static constexpr int S_TERM = DK * 128;
    static constexpr int VT_OFF = S_OFF + 2 * S_TERM;          // two slots for the scaled v's terms
    static constexpr int PW_OFF = VT_OFF + 2 * BLOCK;          // decay^0 .. decay^C
    static constexpr int RW_OFF = PW_OFF + 132 * 4;            // decay^31 .. decay^0
    static constexpr int CP_OFF = RW_OFF + 32 * 4;             // decay^C, decay^last as two floats
    static constexpr int BAD_OFF = CP_OFF + 16;                // [2][DV] rows, [2] chunk numbers
    static constexpr int BAR_OFF = BAD_OFF + (2 * DV + 2) * 4;
    static constexpr int NBARS = 2 * STAGES + 2 * QKB + 8;
    static constexpr int TMEM_OFF = BAR_OFF + NBARS * 8;
    static constexpr int DYN = TMEM_OFF + 8 + 1024;
    // TMEM columns: scores (and over their first half the rounded scores), q S, scores V, K^T V
    static constexpr int COLS = DK == 64 ? 256 : 512;
    static constexpr int T_QS = QKB * 128, T_PV = T_QS + 64, T_KV = DK == 64 ? 64 : T_PV + 64;
    static constexpr int CTAS_PER_SM = DK == 64 ? 2 : 1;
    static_assert(DYN <= 227 * 1024 && (DYN + 1024) * CTAS_PER_SM <= 228 * 1024, "shared memory");
    static_assert(BAR_OFF % 8 == 0 && RW_OFF % 16 == 0, "alignment");
};

constexpr int THREADS = 14 * 32;   // scores and outputs, state, scaled v: 4 warps each; copies; MMAs

struct TcArgs {
    Args a;
    int tiles;                     // of DV columns
    int* status;
    bool al_state, al_out;         // 16-byte aligned rows
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
// Byte offset of 16-byte piece `piece` of row `row` in a tile of 128-byte rows.
__device__ __forceinline__ uint32_t swizzled(int row, int piece) {
    return (uint32_t)(row * 128 + ((piece ^ (row & 7)) << 4));
}
__device__ __forceinline__ uint32_t bf2(float a, float b) {
    return mx::round_pair(a, b, (const __nv_bfloat16*)nullptr);
}
__device__ __forceinline__ float lo_f(uint32_t u) { return __int_as_float((int)(u << 16)); }
__device__ __forceinline__ float hi_f(uint32_t u) { return __int_as_float((int)(u & 0xFFFF0000u)); }

template <int DK>
__global__ void __launch_bounds__(THREADS, Smem<DK>::CTAS_PER_SM)
decay_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TcArgs p) {
    using L = Smem<DK>;
    constexpr int ST = L::STAGES, QKB = L::QKB;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = tc::smem_u32(smem);
    float* pw = reinterpret_cast<float*>(smem + L::PW_OFF);
    float* rw = reinterpret_cast<float*>(smem + L::RW_OFF);
    float* cp = reinterpret_cast<float*>(smem + L::CP_OFF);
    int* bad_row = reinterpret_cast<int*>(smem + L::BAD_OFF);
    volatile int* bad_chunk = bad_row + 2 * DV;
    const uint32_t bar0 = sbase + L::BAR_OFF;
    auto full = [&](int s) { return bar0 + 8u * s; };
    auto empty = [&](int s) { return bar0 + 8u * (ST + s); };
    auto qk_ready = [&](int i) { return bar0 + 8u * (2 * ST + i); };
    auto p_ready = [&](int i) { return bar0 + 8u * (2 * ST + QKB + i); };
    const uint32_t misc = bar0 + 8u * (2 * ST + 2 * QKB);
    const uint32_t o_ready = misc, o_free = misc + 8, vt_ready = misc + 16, vt_free = misc + 24,
                   vt3_ready = misc + 32, kv_ready = misc + 40, s_ready = misc + 48,
                   done = misc + 56;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::TMEM_OFF);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Args& a = p.a;

    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; ++s) {
            tc::mbar_init(full(s), 1);
            tc::mbar_init(empty(s), 1);
        }
        for (int i = 0; i < QKB; ++i) {
            tc::mbar_init(qk_ready(i), 1);
            tc::mbar_init(p_ready(i), 4);
        }
        tc::mbar_init(o_ready, 1);
        tc::mbar_init(o_free, 4);
        tc::mbar_init(vt_ready, 4);
        tc::mbar_init(vt_free, 1);
        tc::mbar_init(vt3_ready, 4);
        tc::mbar_init(kv_ready, 1);
        tc::mbar_init(s_ready, 4);
        tc::mbar_init(done, 1);
        tc::fence_mbar_init();
        tc::prefetch_tmap(&tmQ);
        tc::prefetch_tmap(&tmK);
        tc::prefetch_tmap(&tmV);
        bad_chunk[0] = bad_chunk[1] = -1;
    }
    if (warp == 13) {
        tc::tmem_alloc(sbase + L::TMEM_OFF, L::COLS);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_trigger();
    pdl_wait();

    const int tile = (int)(blockIdx.x % (uint32_t)p.tiles);
    const int64_t bh = blockIdx.x / (uint32_t)p.tiles;
    const int64_t b = bh / a.H, h = bh - b * a.H, hk = h / (a.H / a.Hk);
    const int64_t len = a.length(b);
    const int nc = (int)((len + C - 1) / C);
    const int last = nc ? (int)(len - (int64_t)(nc - 1) * C) : 0;     // tokens of the last chunk
    if (warp < 12) {
        const float lam = a.decay[h];
        const int t = threadIdx.x;
        if (t <= C) {
            const float x = power(lam, t);
            pw[t] = x;
            if (t < 32) rw[31 - t] = x;
        } else if (t >= 192 && t < 194) {
            const int n = t == 192 ? C : last;
            const double d = n == 0 ? 1.0 : exp((double)n * log((double)lam));
            cp[2 * (t - 192)] = (float)d;
            cp[2 * (t - 192) + 1] = (float)(d - (double)(float)d);
        }
        tc::named_bar_sync(2, 12 * 32);
    }
    uint32_t failed = 0;

    if (warp < 4) {
        // ---------------------------------------------------- scores to P, outputs
        const int row = threadIdx.x;                 // of the chunk, and lane of TMEM
        const uint32_t tl = tmem + ((uint32_t)(32 * warp) << 16);
        auto scores = [&](int c) {
            const int buf = c % QKB;
            failed |= 1u - tc::mbar_wait_warp(qk_ready(buf), (uint32_t)(c / QKB) & 1u, failed);
            tc::tc_fence_after();
            const uint32_t t = tl + buf * 128;
#pragma unroll 1
            for (int blk = 0; blk < 4; ++blk) {
                uint32_t w[16];
                if (blk > warp) {                    // later tokens
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[i] = 0;
                } else {
                    float x[32];
                    tc::tmem_ld32(t + blk * 32, x);
                    tc::tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) asm volatile("" : "+f"(x[i]));
                    if (blk == warp) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            x[i] = i <= lane ? x[i] * pw[lane - i] : 0.0f;
                    } else {
                        const float f = pw[row - 32 * blk - 31];
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 r = *reinterpret_cast<const float4*>(rw + i);
                            x[i] *= f * r.x;
                            x[i + 1] *= f * r.y;
                            x[i + 2] *= f * r.z;
                            x[i + 3] *= f * r.w;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[i] = bf2(x[2 * i], x[2 * i + 1]);
                }
                tmem_st16(t + blk * 16, w);
            }
            tmem_wait_st();
            tc::tc_fence_before();
            if (lane == 0) tc::mbar_arrive(p_ready(buf));
            __syncwarp();
        };
        const float fq = pw[row + 1];
        const int cols = min(DV, a.dv - tile * DV);
        __nv_bfloat16* out =
            static_cast<__nv_bfloat16*>(a.out) + (b * a.N * a.H + h) * a.dv + tile * DV;
        const int64_t ld = a.H * a.dv;
        auto store_row = [&](int64_t n, const uint32_t (&w)[32]) {
            __nv_bfloat16* o = out + n * ld;
            if (!SNNB_IN_BOUNDS(n, a.N, p.status)) return;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (8 * i < cols) {                  // dv is a multiple of 8
                    if (p.al_out) {
                        reinterpret_cast<uint4*>(o)[i] =
                            make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            reinterpret_cast<uint16_t*>(o)[8 * i + e] =
                                (uint16_t)(w[4 * i + e / 2] >> (16 * (e & 1)));
                    }
                }
        };
        auto outputs = [&](int c) {
            failed |= 1u - tc::mbar_wait_warp(o_ready, (uint32_t)c & 1u, failed);
            tc::tc_fence_after();
            uint32_t w[32];
            const bool spoiled = bad_chunk[c & 1] == c;
#pragma unroll
            for (int i = 0; i < DV; i += 16) {
                float s[16], v[16];
                tc::tmem_ld16(tl + L::T_QS + i, s);
                tc::tmem_ld16(tl + L::T_PV + i, v);
                tc::tmem_wait_ld();
                tc::reg_fence16(s);
                tc::reg_fence16(v);
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = (v[j] + fq * s[j]) * a.scale;
                if (spoiled) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (row >= bad_row[(c & 1) * DV + i + j]) v[j] = __int_as_float(0x7fffffff);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) w[i / 2 + j] = bf2(v[2 * j], v[2 * j + 1]);
            }
            tc::tc_fence_before();
            if (lane == 0) tc::mbar_arrive(o_free);
            __syncwarp();
            const int64_t n = (int64_t)c * C + row;
            if (n >= len) {
#pragma unroll
                for (int j = 0; j < 32; ++j) w[j] = 0;
            }
            if (n < a.N && !failed) store_row(n, w);
        };
        if (nc) {
            scores(0);
            for (int c = 0; c < nc; ++c) {
                if (QKB == 2 && c + 1 < nc) scores(c + 1);
                outputs(c);
                if (QKB == 1 && c + 1 < nc) scores(c + 1);
            }
        }
        // rows behind the last chunk
        const uint32_t zero[32] = {};
        for (int64_t n = (int64_t)nc * C + row; n < a.N; n += C) store_row(n, zero);
    } else if (warp < 8) {
        // ---------------------------------------------------- the state
        // This thread's row and columns: DK = 64 products have 128 rows, the second 64 the
        // first's copy, so that each half of the threads takes half of the columns.
        const int t = threadIdx.x - 128;
        constexpr int W = DK == 64 ? 32 : 64;
        const int row = t % DK, c0 = DK == 64 ? t / 64 * 32 : 0;
        const uint32_t tl = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + L::T_KV + c0;
        const int64_t at = (bh * a.dk + row) * a.dv + tile * DV + c0;
        const int cols = row < a.dk ? min(W, a.dv - tile * DV - c0) : 0;
        float S[W];
#pragma unroll
        for (int i = 0; i < W; ++i) S[i] = 0.0f;
        if (a.state_in) {
#pragma unroll
            for (int i = 0; i < W; i += 4)
                if (i < cols) {
                    if (p.al_state) {
                        const float4 x = *reinterpret_cast<const float4*>(a.state_in + at + i);
                        S[i] = x.x; S[i + 1] = x.y; S[i + 2] = x.z; S[i + 3] = x.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) S[i + e] = a.state_in[at + i + e];
                    }
                }
        }
        auto publish = [&]() {
#pragma unroll
            for (int i = 0; i < W; i += 8) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = S[i + 2 * j], y = S[i + 2 * j + 1];
                    hi[j] = bf2(x, y);
                    lo[j] = bf2(x - lo_f(hi[j]), y - hi_f(hi[j]));
                }
                const uint32_t o = sbase + L::S_OFF + swizzled(row, (c0 + i) / 8);
                sts128(o, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                sts128(o + L::S_TERM, make_uint4(lo[0], lo[1], lo[2], lo[3]));
            }
            tc::fence_proxy_async_smem();
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(s_ready);
        };
        publish();
        for (int c = 0; c < nc; ++c) {
            failed |= 1u - tc::mbar_wait_warp(kv_ready, (uint32_t)c & 1u, failed);
            tc::tc_fence_after();
            const float2 f = reinterpret_cast<const float2*>(cp)[c + 1 == nc];
#pragma unroll
            for (int i = 0; i < W; i += 16) {
                float x[16];
                tc::tmem_ld16(tl + i, x);
                tc::tmem_wait_ld();
                tc::reg_fence16(x);
#pragma unroll
                for (int j = 0; j < 16; ++j) S[i + j] = fmaf(S[i + j], f.x, fmaf(S[i + j], f.y, x[j]));
            }
            if (c + 1 < nc) publish();
        }
        if (a.state_out && !failed) {
#pragma unroll
            for (int i = 0; i < W; i += 4)
                if (i < cols) {
                    if (p.al_state) {
                        *reinterpret_cast<float4*>(a.state_out + at + i) =
                            make_float4(S[i], S[i + 1], S[i + 2], S[i + 3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) a.state_out[at + i + e] = S[i + e];
                    }
                }
        }
    } else if (warp < 12) {
        // ---------------------------------------------------- v scaled, as three bf16 terms
        const int t = threadIdx.x - 256, piece = t & 7, r0 = t >> 3;
        const uint32_t slot0 = sbase + L::VT_OFF, slot1 = slot0 + L::BLOCK;
        for (int c = 0; c < nc; ++c) {
            const int s = c % ST, m = c + 1 == nc ? last : C;
            failed |= 1u - tc::mbar_wait_warp(full(s), (uint32_t)(c / ST) & 1u, failed);
            const uint32_t stage = sbase + s * L::STAGE, vs = stage + L::V;
            uint32_t low[8][4], top = 0;
            // the slots' last readers
            if (c) failed |= 1u - tc::mbar_wait_warp(kv_ready, (uint32_t)(c - 1) & 1u, failed);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = r0 + 16 * i;
                const uint32_t o = swizzled(r, piece);
                uint4 raw = lds128(vs + o);
                const float w = r < m ? pw[m - 1 - r] : 0.0f;
                if (r >= m) {
                    // rows behind the sequence, whatever they hold (beyond the tensor: zeros)
                    raw = make_uint4(0, 0, 0, 0);
                    sts128(vs + o, raw);
#pragma unroll
                    for (int k = 0; k < L::KB; ++k) sts128(stage + L::K + k * L::BLOCK + o, raw);
                }
                const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
                uint32_t hi[4], mid[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    top = __vmaxu2(top, u[j] & 0x7FFF7FFFu);
                    float x = lo_f(u[j]) * w, y = hi_f(u[j]) * w;
                    hi[j] = bf2(x, y);
                    x -= lo_f(hi[j]);
                    y -= hi_f(hi[j]);
                    mid[j] = bf2(x, y);
                    low[i][j] = bf2(x - lo_f(mid[j]), y - hi_f(mid[j]));
                }
                sts128(slot0 + o, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                sts128(slot1 + o, make_uint4(mid[0], mid[1], mid[2], mid[3]));
            }
            if (tc::named_bar_any(1, 128, (top & 0xFFFFu) >= 0x7F80u || (top >> 16) >= 0x7F80u)) {
                // Values that are not finite: 0 * inf in the product of scores and v would reach
                // the chunk's earlier rows.  There they become zero, and the outputs of their
                // columns NaN from their row on.
                if (t < DV) bad_row[(c & 1) * DV + t] = C;
                tc::named_bar_sync(1, 128);
#pragma unroll 1
                for (int r = r0; r < C; r += 16) {
                    const uint32_t o = swizzled(r, piece);
                    uint4 raw = lds128(vs + o);
                    uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if ((u[j] & 0x7F80u) == 0x7F80u) {
                            atomicMin(&bad_row[(c & 1) * DV + 8 * piece + 2 * j], r);
                            u[j] &= 0xFFFF0000u;
                        }
                        if ((u[j] & 0x7F800000u) == 0x7F800000u) {
                            atomicMin(&bad_row[(c & 1) * DV + 8 * piece + 2 * j + 1], r);
                            u[j] &= 0xFFFFu;
                        }
                    }
                    sts128(vs + o, make_uint4(u[0], u[1], u[2], u[3]));
                }
                if (t == 0) bad_chunk[c & 1] = c;
            }
            tc::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(vt_ready);
            failed |= 1u - tc::mbar_wait_warp(vt_free, (uint32_t)c & 1u, failed);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                sts128(slot0 + swizzled(r0 + 16 * i, piece),
                       make_uint4(low[i][0], low[i][1], low[i][2], low[i][3]));
            tc::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(vt3_ready);
        }
    } else if (warp == 12) {
        // ---------------------------------------------------- copies
        uint32_t issued = 0;
        for (int c = 0; c < nc; ++c) {
            const int s = c % ST;
            failed |= 1u - tc::mbar_wait_warp(empty(s), ((uint32_t)(c / ST) & 1u) ^ 1u, failed);
            const uint32_t stage = sbase + s * L::STAGE;
            if (!failed && tc::elect_one()) {
                tc::mbar_expect_tx(full(s), (uint32_t)L::STAGE);
                const int n0 = c * C;
#pragma unroll
                for (int k = 0; k < L::KB; ++k) {
                    tc::tma_load_4d(stage + L::Q + k * L::BLOCK, &tmQ, full(s), 64 * k, (int)h, n0, (int)b);
                    tc::tma_load_4d(stage + L::K + k * L::BLOCK, &tmK, full(s), 64 * k, (int)hk, n0, (int)b);
                }
                tc::tma_load_4d(stage + L::V, &tmV, full(s), DV * tile, (int)hk, n0, (int)b);
            }
            __syncwarp();
            if (!failed) ++issued;
        }
        if (failed) {                                // copies in flight land before the block ends
            for (uint32_t k = 0; k < issued && k < (uint32_t)ST; ++k) {
                const int c = (int)issued - 1 - (int)k;
                tc::mbar_wait_warp<true>(full(c % ST), (uint32_t)(c / ST) & 1u, 0);
            }
        }
    } else {
        // ---------------------------------------------------- MMAs
        if (tc::elect_one()) {
            constexpr uint32_t I_QK = tc::idesc_bf16_f32(128, 128), I_64 = tc::idesc_bf16_f32(128, 64);
            auto wait = [&](uint32_t bar, uint32_t parity) {
                failed |= 1u - tc::mbar_wait_lane(bar, parity, failed);
                tc::tc_fence_after();
            };
            auto issue_qk = [&](int c) {
                const int s = c % ST, buf = c % QKB;
                wait(full(s), (uint32_t)(c / ST) & 1u);
                const uint32_t stage = sbase + s * L::STAGE;
                if (failed) return;
#pragma unroll
                for (int k = 0; k < L::KB; ++k) {
                    const uint64_t da = tc::sdesc_k_sw128(stage + L::Q + k * L::BLOCK);
                    const uint64_t db = tc::sdesc_k_sw128(stage + L::K + k * L::BLOCK);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        tc::umma_bf16(tmem + buf * 128, da + 2 * i, db + 2 * i, I_QK, (k | i) != 0);
                }
                tc::umma_commit(qk_ready(buf));
            };
            if (nc) issue_qk(0);
            for (int c = 0; c < nc && !failed; ++c) {
                const int s = c % ST, buf = c % QKB;
                const uint32_t stage = sbase + s * L::STAGE, ph = (uint32_t)c & 1u;
                if (QKB == 2 && c + 1 < nc) issue_qk(c + 1);
                if (QKB == 2 || c == 0) wait(s_ready, ph);
                if (c) wait(o_free, ph ^ 1u);
                if (failed) break;
                // q S
#pragma unroll
                for (int term = 0; term < 2; ++term)
#pragma unroll
                    for (int k = 0; k < DK / 16; ++k)
                        tc::umma_bf16(tmem + L::T_QS,
                                      tc::sdesc_k_sw128(stage + L::Q + k / 4 * L::BLOCK) + 2 * (k % 4),
                                      sdesc_mn_sw128(sbase + L::S_OFF + term * L::S_TERM, 0) + 128 * k,
                                      I_64 | B_MN, (term | k) != 0);
                if (QKB == 1) wait(p_ready(buf), (uint32_t)(c / QKB) & 1u);
                wait(vt_ready, ph);
                if (failed) break;
                auto kv = [&](uint32_t slot, bool first) {
                    const uint64_t da = sdesc_mn_sw128(stage + L::K, DK == 64 ? 0 : L::BLOCK);
                    const uint64_t db = sdesc_mn_sw128(sbase + L::VT_OFF + slot * L::BLOCK, 0);
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        tc::umma_bf16(tmem + L::T_KV, da + 128 * k, db + 128 * k, I_64 | A_MN | B_MN,
                                      !first || k != 0);
                };
                kv(0, true);
                tc::umma_commit(vt_free);
                kv(1, false);
                if (QKB == 2) wait(p_ready(buf), (uint32_t)(c / QKB) & 1u);
                if (failed) break;
                const uint64_t dv = sdesc_mn_sw128(stage + L::V, 0);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    umma_ts(tmem + L::T_PV, tmem + buf * 128 + 8 * k, dv + 128 * k, I_64 | B_MN, k != 0);
                tc::umma_commit(o_ready);
                wait(vt3_ready, ph);
                if (failed) break;
                kv(0, false);
                tc::umma_commit(kv_ready);
                tc::umma_commit(empty(s));
                if (QKB == 1 && c + 1 < nc) {
                    wait(s_ready, ph ^ 1u);          // K^T V has been read: its columns are scores'
                    if (!failed) issue_qk(c + 1);
                }
            }
            tc::umma_commit(done);
        }
        __syncwarp();
        failed = __any_sync(0xffffffffu, failed);
        failed |= 1u - tc::mbar_wait_warp<true>(done, 0, 0);
    }
    if (failed && lane == 0) atomicExch(p.status, SNNB_ERR_TIMEOUT);
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 13) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, L::COLS);
    }
}

// [B, N, heads, d] as a tensor map with boxes of 128 tokens x 64 columns of one head.
int encode(CUtensorMap* m, const void* base, const int64_t* s, int64_t B, int64_t N, int64_t heads,
           int64_t d) {
    const uint64_t dims[4] = {(uint64_t)d, (uint64_t)heads, (uint64_t)N, (uint64_t)B};
    const uint64_t st[3] = {heads > 1 ? (uint64_t)s[2] * 2 : 16, N > 1 ? (uint64_t)s[1] * 2 : 16,
                            B > 1 ? (uint64_t)s[0] * 2 : 16};
    const uint32_t box[4] = {64, 1, C, 1};
    return encode_tmap(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, dims, st, box,
                       CU_TENSOR_MAP_SWIZZLE_128B);
}
bool mappable(const void* base, const int64_t* s, int64_t B, int64_t N, int64_t heads) {
    auto ok = [](int64_t st, int64_t n) {
        return n <= 1 || (st > 0 && st % 8 == 0 && st < (int64_t(1) << 39));
    };
    return aligned16(base) && ok(s[2], heads) && ok(s[1], N) && ok(s[0], B);
}

template <int DK>
int launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const TcArgs& p,
           cudaStream_t s) {
    using L = Smem<DK>;
    if (const int st = allow_smem<decay_tc_kernel<DK>>(L::DYN)) return st;
    return launch_k(decay_tc_kernel<DK>, dim3((unsigned)(p.a.B * p.a.H * p.tiles)), dim3(THREADS),
                    L::DYN, s, q, k, v, p);
}

}  // namespace

bool tc_takes(const Args& a, int dtype) {
    return dtype == SNNB_BF16 && a.N > 0 && a.N < 0x7fffff00 && a.dk <= 128 && a.dk % 8 == 0 &&
           a.dv % 8 == 0 && a.H <= 0x7fffffff / 8 && mappable(a.q, a.qs, a.B, a.N, a.H) &&
           mappable(a.k, a.ks, a.B, a.N, a.Hk) && mappable(a.v, a.vs, a.B, a.N, a.Hk);
}

int tc_run(const Args& a, cudaStream_t s) {
    CUtensorMap q, k, v;
    int rc = encode(&q, a.q, a.qs, a.B, a.N, a.H, a.dk);
    if (!rc) rc = encode(&k, a.k, a.ks, a.B, a.N, a.Hk, a.dk);
    if (!rc) rc = encode(&v, a.v, a.vs, a.B, a.N, a.Hk, a.dv);
    if (rc) return rc;
    TcArgs p = {a, (a.dv + DV - 1) / DV, device_status_ptr(),
                aligned16(a.state_in) && aligned16(a.state_out), aligned16(a.out)};
    if (!p.status) return SNNB_ERR_CUDA;
    return a.dk <= 64 ? launch<64>(q, k, v, p, s) : launch<128>(q, k, v, p, s);
}

}  // namespace decay
}  // namespace snnb
