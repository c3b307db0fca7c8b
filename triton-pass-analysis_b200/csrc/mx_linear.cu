// Product of microscaled operands (formats: mx.cuh): out[r, n] = sum_k a[r, k] w[n, k] + bias[n],
// a [rows, K] in E2M1 or E4M3, w [N, K] in E2M1, on the tensor cores' block-scaled kinds: the
// scales multiply inside the MMA, sums are float32 in TMEM, rounded once on the way out.
//
// The product is taken transposed, D^T = W A^T: 128 output features are the 128 TMEM lanes of a
// tile and BN tokens its columns, so that one form serves one token (BN = 16, the weights stream
// through once) and thousands (BN = 256), a warp's stores are 32 consecutive features of one
// token, and the bias is one register.
//
// Operands, per stage of the ring (128 bytes of K a row, 128-byte swizzle):
//   a in E2M1: both operands by TMA as packed 4-bit codes, K = 256 a stage, kind::mxf4 (K = 64
//              an MMA, two scales a row each)
//   a in E4M3: the tokens by TMA, K = 128 a stage, kind::mxf8f6f4 (K = 32 an MMA, one scale a
//              row), which wants 16 4-bit codes as 8 bytes in a 16-byte slot: the packed weight
//              rows come by TMA into a second ring, and four warps, a stage each in turn, move
//              their 8-byte pieces into the slots
//   scales     512-byte groups (128 rows x 4 blocks) as they lie in memory; the MMA thread
//              copies them on to TMEM (tcgen05.cp), a slot per ring stage
//
//   warps 0-3  one kind of load each: tokens, their scales, the weights' scales, weights
//   warp 4     MMA issuer
//   warps 5-   epilogue (4 per 64 tokens), thread = TMEM lane = feature; then, for E4M3, the 4
//              warps that place the weight pieces
#include "mx.cuh"
#include "tc_common.cuh"

namespace snnb {
namespace {

struct MxParams {
    int rows, N, groups;             // tokens, features, 128-wide groups of K
    int tiles_w, tiles;              // feature tiles (of 128, or 256 a pair), tiles in all
    const float* bias;
    void* out;
    int out_dtype;
    int pairs, odd_pairs;            // 16-bit outputs may be stored two features at a time: N even, odd
    int* status;
};

// ---- block-scaled MMA ------------------------------------------------------------------
// Instruction descriptor: A type [7,10), B type [10,13), N / 8 [17,23), E8M0 scales bit 23,
// M / 128 [27,29); which byte of the 32-bit scale columns the MMA uses: B [4,6), A [29,31).
__host__ __device__ constexpr uint32_t idesc_mx(int a_type, int b_type, int M, int N) {
    return ((uint32_t)a_type << 7) | ((uint32_t)b_type << 10) | ((uint32_t)(N >> 3) << 17) |
           (1u << 23) | ((uint32_t)(M >> 7) << 27);
}
__device__ __forceinline__ uint32_t idesc_scale_byte(uint32_t byte) {
    return (byte << 4) | (byte << 29);
}
// PAIR: M = 256 over the two CTAs of a cluster, issued by one thread of the even CTA.
#define SNNB_MX_MMA(group, kind, vec)                                                        \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                           \
                 "tcgen05.mma.cta_group::" group ".kind::" kind ".block_scale.scale_vec::" vec \
                 " [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),                        \
                 "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)       \
                 : "memory")
template <int FMT, bool PAIR>
__device__ __forceinline__ void umma_mx(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t sa, uint32_t sb, uint32_t accumulate) {
    if constexpr (FMT == SNNB_MXFP4 && PAIR) SNNB_MX_MMA("2", "mxf4", "2X");
    else if constexpr (FMT == SNNB_MXFP4) SNNB_MX_MMA("1", "mxf4", "2X");
    else if constexpr (PAIR) SNNB_MX_MMA("2", "mxf8f6f4", "1X");
    else SNNB_MX_MMA("1", "mxf8f6f4", "1X");
}
#undef SNNB_MX_MMA
// One 512-byte scale group (32 rows of 16 bytes, unswizzled) to 4 TMEM columns, the same 32
// lanes in each of the four lane quarters.  PAIR: in both CTAs, each from its own memory.
template <bool PAIR>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t saddr) {
    uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(128 >> 4) << 32;                 // 8 rows to the next 8: 128 bytes
    d |= (uint64_t)1 << 46;
    if constexpr (PAIR)
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d)
                     : "memory");
    else
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d)
                     : "memory");
}
// Tiled loads completing on `bar`; PAIR: a barrier of the even CTA (a shared::cluster address).
template <bool PAIR>
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int c0,
                                        int c1) {
    if constexpr (PAIR)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(c0), "r"(c1)
            : "memory");
    else
        tc::tma_load_2d(dst, tm, bar, c0, c1);
}
template <bool PAIR>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* tm, uint32_t bar, int c0,
                                        int c1, int c2) {
    if constexpr (PAIR) tc::tma_load_3d_pair(dst, tm, bar, c0, c1, c2);
    else tc::tma_load_3d(dst, tm, bar, c0, c1, c2);
}
// Arrival on a barrier of the pair's even CTA, relaxed: it reports TMEM reads that have completed
// (tcgen05.wait::ld, fence::before_thread_sync) and no data in memory crosses the CTAs with it.  A
// release at cluster scope would wait for every earlier write of the SM instead (~1900 cycles,
// where a stage takes 540), the epilogue's stores among them.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr)
                 : "memory");
}

// ---- shared memory -----------------------------------------------------------------------
template <int FMT, int BN, int STAGES, bool PAIR, int PACKED_STAGES>
struct MxSmem {
    static constexpr int GROUPS = FMT == SNNB_MXFP4 ? 2 : 1;     // 128-wide groups of K a stage
    static constexpr int TOKEN_TILES = (BN + 127) / 128;         // scale tiles of the tokens
    static constexpr int A_ROWS = PAIR ? BN / 2 : BN;            // a pair: half the tokens a CTA
    static constexpr int W_TILE = 128 * 128;
    static constexpr int A_TILE = A_ROWS * 128;
    static constexpr int W_SCALES = GROUPS * mx::GROUP_BYTES;
    static constexpr int A_SCALES = TOKEN_TILES * GROUPS * mx::GROUP_BYTES;
    static constexpr int STAGE = W_TILE + A_TILE;                // operand tiles, 1024-aligned
    static constexpr int SCALES_OFF = STAGES * STAGE;
    static constexpr int SCALES = W_SCALES + A_SCALES;           // per stage
    static constexpr int PACKED = PACKED_STAGES > 0 ? 128 * 64 : 0;  // packed weights, per stage
    static constexpr int PACKED_OFF = SCALES_OFF + STAGES * SCALES;
    static constexpr int BAR_OFF = PACKED_OFF + PACKED_STAGES * PACKED;
    static constexpr int ACCS = BN <= 128 ? 2 : 1;               // accumulators in TMEM
    static constexpr int NBARS = 2 * STAGES + 2 * ACCS + 1 + 2 * PACKED_STAGES;
    static constexpr int TMEM_OFF = BAR_OFF + NBARS * 8;
    static constexpr int TOTAL = TMEM_OFF + 8;
    static constexpr int DYN = TOTAL + 1024;
    // TMEM: the accumulators, then per ring stage 4 columns per scale group
    static constexpr int SCALE_COLS = 4 * GROUPS * (1 + TOKEN_TILES);
    static constexpr int COLS_USED = ACCS * BN + STAGES * SCALE_COLS;
    static constexpr int COLS = COLS_USED <= 128 ? 128 : (COLS_USED <= 256 ? 256 : 512);
    static constexpr int CTAS_PER_SM = COLS <= 256 && (DYN + 1024) * 2 <= 228 * 1024 ? 2 : 1;
    static_assert(COLS_USED <= 512, "tensor memory");
    static_assert(DYN <= 227 * 1024, "shared memory");
};

constexpr int MX_PRODUCERS = 4;
template <int BN> constexpr int mx_epilogue_warps() { return BN <= 64 ? 4 : BN / 16; }
// Warps that place one stage's weight pieces (4 stages in turn): 2 where a block has an SM for
// itself and threads to spare.
template <int BN, int PACKED_STAGES> constexpr int mx_placers() {
    return PACKED_STAGES == 0 ? 0 : BN <= 128 ? 2 : 1;
}
template <int BN, int PACKED_STAGES> constexpr int mx_threads() {
    return 32 * (MX_PRODUCERS + 1 + mx_epilogue_warps<BN>() + 4 * mx_placers<BN, PACKED_STAGES>());
}

// One accumulator column pair (tokens i, i + 1) of a feature, rounded, as one word.
__device__ __forceinline__ uint32_t pack16(const MxParams& p, float a, float b) {
    return p.out_dtype == SNNB_F16 ? mx::round_pair(a, b, (const __half*)nullptr)
                                   : mx::round_pair(a, b, (const __nv_bfloat16*)nullptr);
}
__device__ __forceinline__ void store_one(const MxParams& p, int64_t i, float v) {
    if (!SNNB_IN_BOUNDS(i, (int64_t)p.rows * p.N, p.status)) return;
    if (p.out_dtype == SNNB_F32)
        static_cast<float*>(p.out)[i] = v;
    else if (p.out_dtype == SNNB_F16)
        static_cast<__half*>(p.out)[i] = __float2half_rn(v);
    else
        static_cast<__nv_bfloat16*>(p.out)[i] = __float2bfloat16_rn(v);
}
// N accumulator columns of this thread's lane; complete on return.
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t t, float (&r)[N]) {
    constexpr int STEP = N < 32 ? 16 : 32;
    static_assert(N % STEP == 0, "columns");
    float part[N / STEP][STEP];
#pragma unroll
    for (int i = 0; i < N / STEP; ++i) {
        if constexpr (STEP == 32) tc::tmem_ld32(t + i * STEP, part[i]);
        else tc::tmem_ld16(t + i * STEP, part[i]);
    }
    tc::tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        asm volatile("" : "+f"(part[i / STEP][i % STEP]));       // no use moves before the wait
        r[i] = part[i / STEP][i % STEP];
    }
}

// The accumulator columns [0, CW) at TMEM address t: tokens r0 .., the first `cols` of them
// inside; this lane's feature is n.  `release` hands the accumulator back, as soon as it has been
// read.  16-bit outputs with an even N go out two features at a time: a column pair is rounded
// into one word, neighbouring lanes exchange their words, and the even lane stores both features
// of token i, the odd lane of token i + 1.
template <int CW, bool ODD_PAIRS, typename Release>
__device__ __forceinline__ void store_tile(const MxParams& p, uint32_t t, float bias, int n,
                                           int64_t r0, int cols, Release release) {
    float r[CW];
    tmem_load(t, r);
    release();
    if (p.pairs) {
        const int odd = threadIdx.x & 1;
        const uint32_t pick = odd ? 0x3276u : 0x5410u;
        uint32_t* o = reinterpret_cast<uint32_t*>(
            static_cast<uint16_t*>(p.out) + (r0 + odd) * p.N + (n & ~1));
        const bool in = n < p.N;
        const int64_t step = p.N;                    // two rows of 16-bit values, in words
#pragma unroll
        for (int i = 0; i < CW; i += 2) {
            const uint32_t v = pack16(p, r[i] + bias, r[i + 1] + bias);
            const uint32_t w = __byte_perm(v, __shfl_xor_sync(0xffffffffu, v, 1), pick);
            if (in && i + odd < cols &&
                SNNB_IN_BOUNDS((r0 + odd + i) * p.N + n, (int64_t)p.rows * p.N, p.status))
                *o = w;
            o += step;
        }
    } else if (ODD_PAIRS && p.odd_pairs) {
        // N is odd, r0 + i even: token i's words begin at even features, token i + 1's at odd
        // ones, so either half takes the next lane's value.  Lanes 0 and 31 hold halves of token
        // i + 1's words that neighbouring warps share, the last feature half of token i's.
        // (4096 x 8191 x 512: 35 us, 47 by single values; 4223 x 14243 x 33: 69, 91.  Tiles of 256
        // tokens have 16 warps for it, whose registers this would spill: 4096 x 4097 x 4096 33 us
        // by single values, 35 to 37 so.)
        uint32_t v[CW / 2];
#pragma unroll
        for (int i = 0; i < CW / 2; ++i) v[i] = pack16(p, r[2 * i] + bias, r[2 * i + 1] + bias);
        const int lane = threadIdx.x & 31, odd = lane & 1;
        const uint32_t pick = odd ? 0x7632u : 0x5410u;
        uint16_t* o = static_cast<uint16_t*>(p.out) + (r0 + odd) * p.N + n;
        const bool pair = lane < 31 && n + 1 < p.N, last = n == p.N - 1;
        const bool half = (lane == 0 || lane == 31) && n < p.N;
#pragma unroll
        for (int i = 0; i < CW; i += 2) {
            const uint32_t x = v[i / 2];
            const uint32_t w = __byte_perm(x, __shfl_down_sync(0xffffffffu, x, 1), pick);
            if (pair && i + odd < cols &&
                SNNB_IN_BOUNDS((r0 + i + odd) * p.N + n + 1, (int64_t)p.rows * p.N, p.status))
                *reinterpret_cast<uint32_t*>(o) = w;
            if (half && i + 1 < cols &&
                SNNB_IN_BOUNDS((r0 + i + 1) * p.N + n, (int64_t)p.rows * p.N, p.status))
                o[(1 - odd) * p.N] = (uint16_t)(x >> 16);
            if (last && i < cols && SNNB_IN_BOUNDS((r0 + i) * p.N + n, (int64_t)p.rows * p.N, p.status))
                *o = (uint16_t)x;
            o += 2 * (int64_t)p.N;
        }
    } else {
#pragma unroll
        for (int i = 0; i < CW; ++i)
            if (n < p.N && i < cols) store_one(p, (r0 + i) * p.N + n, r[i] + bias);
    }
}

// The cluster's partial sums [column][128 features] at `part` of every CTA, added in rank order:
// CTA `rank` finishes BN / SPLITS of the columns (tokens), four features a thread.  Every load of
// a thread is in flight before the first sum: read one column after the other, the join took
// 4 us of a 64 x 2048 x 2048 product's 9.5.
template <int BN, int SPLITS>
__device__ __forceinline__ void join_splits(const MxParams& p, uint32_t part, int rank, int n0,
                                            int64_t r0) {
    constexpr int COLS = BN / SPLITS;
    constexpr int AHEAD = 16 / SPLITS;                           // units in flight
    uint32_t from[SPLITS];
#pragma unroll
    for (int r = 0; r < SPLITS; ++r) from[r] = tc::map_to_rank(part, (uint32_t)r);
    for (int u0 = threadIdx.x; u0 < COLS * 32; u0 += AHEAD * blockDim.x) {
        float4 x[AHEAD][SPLITS];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int u = u0 + i * blockDim.x;
            if (u < COLS * 32 && r0 + rank * COLS + (u >> 5) < p.rows) {
                const uint32_t at = (uint32_t)(((rank * COLS + (u >> 5)) * 32 + (u & 31)) * 16);
#pragma unroll
                for (int r = 0; r < SPLITS; ++r) x[i][r] = tc::ld_dsmem_f4(from[r] + at);
            }
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int u = u0 + i * blockDim.x;
            const int64_t row = r0 + rank * COLS + (u >> 5);
            const int n = n0 + (u & 31) * 4;
            if (u >= COLS * 32 || row >= p.rows || n >= p.N) continue;
            float v[4] = {x[i][0].x, x[i][0].y, x[i][0].z, x[i][0].w};
#pragma unroll
            for (int r = 1; r < SPLITS; ++r) {
                v[0] += x[i][r].x; v[1] += x[i][r].y; v[2] += x[i][r].z; v[3] += x[i][r].w;
            }
            const int have = p.N - n < 4 ? p.N - n : 4;
            if (p.bias) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < have) v[e] += __ldg(p.bias + n + e);
            }
            if (p.pairs) {                                       // 16 bits, N even
                uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + row * p.N + n);
                if (SNNB_IN_BOUNDS(row * p.N + n + have - 1, (int64_t)p.rows * p.N, p.status)) {
                    o[0] = pack16(p, v[0], v[1]);
                    if (have > 2) o[1] = pack16(p, v[2], v[3]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < have) store_one(p, row * p.N + n + e, v[e]);
            }
        }
    }
}

// The stages of K of CTA `rank` of `splits`: from its first to the next rank's first.  Its MMA
// thread waits for at least one.
__host__ __device__ constexpr int first_stage(int nstages, int rank, int splits) {
    return (int)((int64_t)nstages * rank / splits);
}
// Whether 2^log ways save 6 stages of ~0.25 us, which pay for the join (1.4 us), and leave every
// CTA a stage.
constexpr bool split_pays(int nstages, int log) {
    return (nstages >> log) >= 1 && nstages - (nstages >> log) >= 6;
}
constexpr bool every_rank_has_stages() {
    for (int n = 1; n <= 64; ++n)
        for (int log = 0; log <= 3; ++log)
            for (int r = 0; r < 1 << log; ++r)
                if ((log == 0 || split_pays(n, log)) &&
                    first_stage(n, r, 1 << log) >= first_stage(n, r + 1, 1 << log))
                    return false;
    return true;
}
static_assert(every_rank_has_stages(), "a CTA without a stage would wait for one");

// PAIR: two CTAs share a 256-feature x BN-token tile (each stages its own 128 features and half
// of the tokens) and walk whole tiles.  Otherwise: one tile, its K range split over the CTAs of
// a cluster, their float32 partial sums joined in rank order through distributed shared memory.
// PACKED_STAGES: of the packed weights' ring (E4M3 tokens), 0 for E2M1.
template <int FMT, int BN, int STAGES, bool PAIR, int PACKED_STAGES>
__global__ void __launch_bounds__(mx_threads<BN, PACKED_STAGES>(),
                                  MxSmem<FMT, BN, STAGES, PAIR, PACKED_STAGES>::CTAS_PER_SM)
mx_linear_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA,
                 const __grid_constant__ CUtensorMap tmWS, const __grid_constant__ CUtensorMap tmAS,
                 const MxParams p) {
    using S = MxSmem<FMT, BN, STAGES, PAIR, PACKED_STAGES>;
    constexpr int NP = MX_PRODUCERS, EW = mx_epilogue_warps<BN>(), PLACERS = mx_placers<BN, PACKED_STAGES>();
    constexpr int CTAS = PAIR ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = tc::smem_u32(smem);
    const uint32_t bar0 = sbase + S::BAR_OFF;
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (STAGES + s); };
    auto accf_bar = [&](int b) { return bar0 + 8u * (2 * STAGES + b); };
    auto acce_bar = [&](int b) { return bar0 + 8u * (2 * STAGES + S::ACCS + b); };
    const uint32_t done_bar = bar0 + 8u * (2 * STAGES + 2 * S::ACCS);
    auto w_tile = [&](int s) { return sbase + (uint32_t)(s * S::STAGE); };
    auto a_tile = [&](int s) { return sbase + (uint32_t)(s * S::STAGE + S::W_TILE); };
    auto scales_at = [&](int s) { return sbase + (uint32_t)(S::SCALES_OFF + s * S::SCALES); };
    // the packed weights' own ring (E4M3 tokens)
    auto packed = [&](int s) { return sbase + (uint32_t)(S::PACKED_OFF + s * S::PACKED); };
    auto pfull_bar = [&](int s) { return done_bar + 8u * (1 + s); };
    auto pempty_bar = [&](int s) { return done_bar + 8u * (1 + PACKED_STAGES + s); };
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + S::TMEM_OFF);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int crank = PAIR ? (int)tc::cluster_rank() : 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            // four loads, or three and the warps of each CTA that placed the weights
            tc::mbar_init(full_bar(s), PACKED_STAGES == 0 ? 4 : 3 + PLACERS * CTAS);
            tc::mbar_init(empty_bar(s), 1);
        }
        for (int s = 0; s < PACKED_STAGES; ++s) {
            tc::mbar_init(pfull_bar(s), 1);
            tc::mbar_init(pempty_bar(s), PLACERS);
        }
        for (int b = 0; b < S::ACCS; ++b) {
            tc::mbar_init(accf_bar(b), 1);
            tc::mbar_init(acce_bar(b), EW * CTAS);
        }
        tc::mbar_init(done_bar, 1);
        tc::fence_mbar_init();
        tc::prefetch_tmap(&tmW);
        tc::prefetch_tmap(&tmA);
        tc::prefetch_tmap(&tmWS);
        tc::prefetch_tmap(&tmAS);
    }
    if (warp == NP) {
        if constexpr (PAIR) {
            tc::tmem_alloc_pair(sbase + S::TMEM_OFF, S::COLS);
            tc::tmem_relinquish_pair();
        } else {
            tc::tmem_alloc(sbase + S::TMEM_OFF, S::COLS);
            tc::tmem_relinquish();
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) tc::cluster_sync();          // the even CTA's barriers are initialised
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_trigger();
    pdl_wait();

    // this CTA's tiles and, within a tile, its stages of K
    const int splits = PAIR ? 1 : (int)gridDim.x / p.tiles;
    const int rank = PAIR ? 0 : (int)blockIdx.x % splits;
    const int tile0 = PAIR ? (int)blockIdx.x / 2 : (int)blockIdx.x / splits;
    const int tile_step = PAIR ? (int)gridDim.x / 2 : p.tiles;
    const int nstages = (p.groups + S::GROUPS - 1) / S::GROUPS;
    const int k0 = first_stage(nstages, rank, splits), k1 = first_stage(nstages, rank + 1, splits);
    uint32_t failed = 0, issued = 0;                 // issued: a producer warp's copies

    if (warp < NP) {
        // ------------------------------------------------------------- copies
        // Issuing a tiled copy holds its thread for ~250 cycles, so each kind has a warp of its
        // own.  All bytes of a stage, a pair's both halves, complete the (even CTA's) full
        // barrier; packed weights their own ring's.
        // (an unpacking copy counts the packed bytes)
        constexpr uint32_t BYTES[4] = {S::A_TILE, S::A_SCALES, S::W_SCALES,
                                       FMT == SNNB_MXFP4 ? S::W_TILE : S::W_TILE / 2};
        const uint32_t mine = (warp == 0 ? BYTES[0] : warp == 1 ? BYTES[1] : warp == 2 ? BYTES[2]
                                                                                      : BYTES[3]) *
                              (uint32_t)CTAS;
        const bool own_ring = S::PACKED > 0 && warp == 3;
        const int ring = own_ring ? PACKED_STAGES : STAGES;
        uint32_t it = 0;
        for (int tile = tile0; tile < p.tiles && !failed; tile += tile_step) {
            const int tw = (tile % p.tiles_w) * CTAS + crank, tt = tile / p.tiles_w;
            for (int ks = k0; ks < k1; ++ks, ++it) {
                const int s = (int)(it % ring);
                failed |= 1u - tc::mbar_wait_warp(own_ring ? pempty_bar(s) : empty_bar(s),
                                                  ((it / ring) & 1u) ^ 1u, failed);
                if (failed) break;
                if (own_ring) {
                    if (tc::elect_one()) {
                        tc::mbar_expect_tx(pfull_bar(s), (uint32_t)S::PACKED);
                        tc::tma_load_2d(packed(s), &tmW, pfull_bar(s), ks * 64, tw * 128);
                    }
                } else if (tc::elect_one()) {
                    if (crank == 0) tc::mbar_expect_tx(full_bar(s), mine);
                    const uint32_t fb = PAIR ? tc::map_to_rank(full_bar(s), 0) : full_bar(s);
                    if (warp == 0)
                        load_2d<PAIR>(a_tile(s), &tmA, fb, ks * 128, tt * BN + crank * S::A_ROWS);
                    else if (warp == 1)
                        load_3d<PAIR>(scales_at(s) + S::W_SCALES, &tmAS, fb, 0, ks * S::GROUPS,
                                      tt * S::TOKEN_TILES);
                    else if (warp == 2)
                        load_3d<PAIR>(scales_at(s), &tmWS, fb, 0, ks * S::GROUPS, tw);
                    else
                        // E2M1: bytes; unpacked: elements (128 of either a stage)
                        load_2d<PAIR>(w_tile(s), &tmW, fb, ks * 128, tw * 128);
                }
                __syncwarp();
                ++issued;
            }
        }
    } else if (warp == NP) {
        // ------------------------------------------------------------- MMA issuer
        constexpr uint32_t IDESC = FMT == SNNB_MXFP4 ? idesc_mx(1, 1, 128 * CTAS, BN)
                                                     : idesc_mx(5, 0, 128 * CTAS, BN);
        auto commit = [&](uint32_t bar) {
            if constexpr (PAIR) tc::umma_commit_pair(bar, 3);
            else tc::umma_commit(bar);
        };
        auto wait_full = [&](uint32_t it) {
            const uint32_t bar = full_bar((int)(it % STAGES)), ph = (it / STAGES) & 1u;
            // the odd CTA's warps arrive here as well once they have placed weight pieces
            if constexpr (PAIR && PACKED_STAGES > 0)
                failed |= 1u - tc::mbar_wait_lane_cluster(bar, ph, failed);
            else
                failed |= 1u - tc::mbar_wait_lane(bar, ph, failed);
            tc::tc_fence_after();
        };
        if (crank == 0) {
            if (tc::elect_one()) {
                uint32_t it = 0, local = 0;
                for (int tile = tile0; tile < p.tiles && !failed; tile += tile_step, ++local) {
                    const int b = (int)(local % S::ACCS);
                    failed |= 1u - tc::mbar_wait_lane(acce_bar(b), ((local / S::ACCS) & 1u) ^ 1u, failed);
                    tc::tc_fence_after();
                    wait_full(it);
                    const uint32_t d = tmem + (uint32_t)(b * BN);
                    // after a wait that ran out: no more MMAs and nothing handed on, so that
                    // every other role's wait runs out too
                    for (int ks = k0; ks < k1 && !failed; ++ks, ++it) {
                        const int s = (int)(it % STAGES);
                        const uint32_t sw = tmem + (uint32_t)(S::ACCS * BN + s * S::SCALE_COLS);
                        const uint32_t sa = sw + 4 * S::GROUPS;
                        const uint32_t sc = scales_at(s);
                        const uint64_t dw = tc::sdesc_k_sw128(w_tile(s));
                        const uint64_t da = tc::sdesc_k_sw128(a_tile(s));
                        constexpr int PER_GROUP = 4 / S::GROUPS;     // MMAs per 128 of K
#pragma unroll
                        for (int g = 0; g < S::GROUPS; ++g) {
                            if (g > 0 && ks * S::GROUPS + g >= p.groups) break;
                            copy_scales<PAIR>(sw + 4 * g, sc + g * mx::GROUP_BYTES);
#pragma unroll
                            for (int h = 0; h < S::TOKEN_TILES; ++h)
                                copy_scales<PAIR>(sa + 4 * (g * S::TOKEN_TILES + h),
                                                  sc + S::W_SCALES +
                                                      (h * S::GROUPS + g) * mx::GROUP_BYTES);
#pragma unroll
                            for (int m = 0; m < PER_GROUP; ++m) {
                                const int k = g * PER_GROUP + m;
                                umma_mx<FMT, PAIR>(d, dw + 2 * k, da + 2 * k,
                                                   IDESC | idesc_scale_byte(m * S::GROUPS),
                                                   sw + 4 * g, sa + 4 * g * S::TOKEN_TILES,
                                                   (ks != k0) || (k != 0));
                            }
                        }
                        // the next stage before this one's commit: a wait behind a commit
                        // returns only once the tensor pipe has drained
                        if (ks + 1 < k1) wait_full(it + 1);
                        if (!failed) commit(empty_bar(s));
                    }
                    if (!failed) commit(accf_bar(b));
                }
                commit(done_bar);
            }
            __syncwarp();
            failed = __any_sync(0xffffffffu, (int)failed);
        }
        // every MMA of this CTA's (or its pair's) has completed
        failed |= 1u - tc::mbar_wait_warp<true>(done_bar, 0, 0);
    } else if (warp < NP + 1 + EW) {
        // ------------------------------------------------------------- epilogue
        const int q = warp & 3;
        constexpr int CW = BN / (EW / 4);            // columns of a warp
        const int c0 = (warp - NP - 1) / 4 * CW;
        uint32_t local = 0;
        for (int tile = tile0; tile < p.tiles; tile += tile_step, ++local) {
            const int tw = (tile % p.tiles_w) * CTAS + crank, tt = tile / p.tiles_w;
            const int b = (int)(local % S::ACCS);
            const int n = tw * 128 + 32 * q + lane;
            const float bias = p.bias && n < p.N ? __ldg(p.bias + n) : 0.0f;
            failed |= 1u - tc::mbar_wait_warp(accf_bar(b), (local / S::ACCS) & 1u, failed);
            tc::tc_fence_after();
            if (failed) break;
            const uint32_t t = tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(b * BN + c0);
            auto release = [&] {
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (PAIR) mbar_arrive_cluster_relaxed(tc::map_to_rank(acce_bar(b), 0));
                    else tc::mbar_arrive(acce_bar(b));
                }
            };
            if (!PAIR && splits > 1) {
                // partial sums [column][lane] in the drained ring
                float* part = reinterpret_cast<float*>(smem) + c0 * 128 + 32 * q + lane;
#pragma unroll 1
                for (int c = 0; c < CW; c += 16) {
                    float r[16];
                    tmem_load(t + c, r);
#pragma unroll
                    for (int i = 0; i < 16; ++i) part[(c + i) * 128] = r[i];
                }
                release();
            } else {
                const int64_t r0 = (int64_t)tt * BN + c0;
                const int64_t left = (int64_t)p.rows - r0;
                store_tile<CW, BN != 256>(p, t, bias, n, r0, (int)(left < CW ? left : CW), release);
            }
        }
    } else {
        // ------------------------------------------------------------- weight pieces (E4M3)
        // The warps w, w + 4 take the stages w, w + 4, ... (each a part of the rows): 16 codes
        // (8 bytes) to the low half of a 16-byte slot, slot c of row r at c ^ (r % 8).
        // A wait by parity needs the phase before to have completed, and a slot's phase before is
        // another warp's stage, whose copy may land after a later one.  So the stage's release
        // is waited for first: every MMA up to stage it - STAGES is done, hence every copy up to
        // there has landed, which covers the packed slot's last use.
        static_assert(PACKED_STAGES == 0 || (STAGES >= 4 && PACKED_STAGES >= STAGES),
                      "a wait of a warp that takes every fourth stage is at most one phase ahead");
        constexpr int ROWS = PLACERS > 0 ? 16 / PLACERS : 0;         // groups of 8 rows a warp
        const uint32_t w = (uint32_t)(warp - NP - 1 - EW) & 3u;
        const int part = (warp - NP - 1 - EW) >> 2;
        uint32_t it = 0;
        for (int tile = tile0; tile < p.tiles && !failed; tile += tile_step) {
            for (int ks = k0; ks < k1; ++ks, ++it) {
                if ((it & 3u) != w) continue;
                const int s = (int)(it % STAGES), ps = PLACERS > 0 ? (int)(it % PACKED_STAGES) : 0;
                failed |= 1u - tc::mbar_wait_warp(empty_bar(s), ((it / STAGES) & 1u) ^ 1u, failed);
                failed |= 1u - tc::mbar_wait_warp(pfull_bar(ps), PLACERS > 0 ? (it / PACKED_STAGES) & 1u : 0,
                                                  failed);
                if (failed) break;
                const uint8_t* src = smem + S::PACKED_OFF + ps * S::PACKED + part * ROWS * 512 + lane * 16;
                uint8_t* dst = smem + s * S::STAGE + part * ROWS * 1024 + (lane >> 2) * 128;
                const int c = (lane & 3) * 2, x = lane >> 2;         // row u * 8 + x
#pragma unroll
                for (int h = 0; h < ROWS; h += 8) {
                    uint4 v[8];                      // loads ahead of the stores
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        v[u] = *reinterpret_cast<const uint4*>(src + (h + u) * 512);
#pragma unroll
                    for (int u = 0; u < 8; ++u) {
                        uint8_t* d = dst + (h + u) * 1024;
                        *reinterpret_cast<uint2*>(d + ((c ^ x) << 4)) = make_uint2(v[u].x, v[u].y);
                        *reinterpret_cast<uint2*>(d + (((c + 1) ^ x) << 4)) = make_uint2(v[u].z, v[u].w);
                    }
                }
                tc::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    tc::mbar_arrive(pempty_bar(ps));
                    // the even CTA's thread issues the MMA that reads the odd CTA's pieces: the
                    // one thing that orders it after their stores is a release at cluster scope.
                    // (It costs 4096 x 8192 x 4000 128 us against 111 with a relaxed arrival, 2300
                    // x 2304 x 1100 16.4 against 14.5, 6523 x 4000 x 32 24.0 against 22.0; tiles of
                    // one CTA, which need none, take 215, 21.9 and 57.)
                    if (crank) tc::mbar_arrive_cluster(tc::map_to_rank(full_bar(s), 0));
                    else tc::mbar_arrive(full_bar(s));
                }
            }
        }
    }
    if (failed && lane == 0) atomicExch(p.status, SNNB_ERR_TIMEOUT);
    if (!PAIR && splits > 1) {
        tc::cluster_sync();                          // every CTA's partial sums are in place
        const int tw = tile0 % p.tiles_w, tt = tile0 / p.tiles_w;
        if (splits == 2) join_splits<BN, 2>(p, sbase, rank, tw * 128, (int64_t)tt * BN);
        else if (splits == 4) join_splits<BN, 4>(p, sbase, rank, tw * 128, (int64_t)tt * BN);
        else join_splits<BN, 8>(p, sbase, rank, tw * 128, (int64_t)tt * BN);
    }
    tc::tc_fence_before();
    if (__syncthreads_or((int)failed)) {
        // copies still in flight land before the CTA may exit: waits on the full barrier, or for
        // the odd CTA of a pair (whose copies complete the even CTA's) on the stage's release,
        // with the limit that outlasts any copy.  The newest copy first: once that limit has run
        // out, which it does where a stage is never handed on, it has done so for the older ones.
        if (warp < NP) {
            const bool own_ring = S::PACKED > 0 && warp == 3;
            const uint32_t ring = own_ring ? PACKED_STAGES : STAGES;
            for (uint32_t k = 0; k < issued && k < ring; ++k) {
                const uint32_t g = issued - 1 - k;
                const int s = (int)(g % ring);
                if (!tc::mbar_wait_warp<true>(own_ring ? pfull_bar(s) : crank ? empty_bar(s) : full_bar(s),
                                              (g / ring) & 1u, 0))
                    break;
            }
        }
        __syncthreads();
    }
    // neither CTA of a pair leaves while the other may signal its barriers or have its memory
    // read by the tensor pipe; nor one of a split cluster while its partial sums are read
    if (PAIR || splits > 1) tc::cluster_sync();
    if (warp == NP) {
        tc::tc_fence_after();
        if constexpr (PAIR) tc::tmem_dealloc_pair(tmem, S::COLS);
        else tc::tmem_dealloc(tmem, S::COLS);
    }
}

struct MxMaps {
    CUtensorMap w, a, ws, as;
};

// One instantiation's launch settings on the current device, asked for once: the shared-memory
// opt-in, and how many clusters of 1, 2, 4, 8 CTAs are resident at once.
struct MxDevice {
    bool ready;
    int clusters[4];
};
template <typename Kernel>
int mx_device(Kernel k, int threads, int smem, bool pair, MxDevice (&cache)[64], const MxDevice*& out) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (dev < 0 || dev >= 64) return SNNB_ERR_UNSUPPORTED;
    MxDevice& d = cache[dev];
    if (!__atomic_load_n(&d.ready, __ATOMIC_ACQUIRE)) {
        e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return record_cuda_error(e);
        for (int i = 0; i < 4 && !pair; ++i) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(1u << i);
            cfg.blockDim = dim3((unsigned)threads);
            cfg.dynamicSmemBytes = (size_t)smem;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 1u << i;
            attr[0].val.clusterDim.y = 1;
            attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int n = 0;
            e = cudaOccupancyMaxActiveClusters(&n, k, &cfg);
            if (e != cudaSuccess) return record_cuda_error(e);
            __atomic_store_n(&d.clusters[i], n, __ATOMIC_RELAXED);
        }
        __atomic_store_n(&d.ready, true, __ATOMIC_RELEASE);
    }
    out = &d;
    return SNNB_OK;
}

// Launches one form.  min_split > 0: only if the K range can be split at least that much with
// every cluster resident at once, else SNNB_ERR_UNSUPPORTED.
template <int FMT, int BN, int STAGES, bool PAIR, int PACKED_STAGES>
int launch_mx(const void* a, const void* as, const void* w, const void* ws, int64_t K, MxParams p,
              cudaStream_t s, int min_split = 0) {
    using S = MxSmem<FMT, BN, STAGES, PAIR, PACKED_STAGES>;
    static MxDevice cache[64];
    auto k = mx_linear_kernel<FMT, BN, STAGES, PAIR, PACKED_STAGES>;
    const MxDevice* dev = nullptr;
    int rc = mx_device(k, mx_threads<BN, PACKED_STAGES>(), S::DYN, PAIR, cache, dev);
    if (rc != SNNB_OK) return rc;
    const int64_t width = PAIR ? 256 : 128;
    p.tiles_w = (int)((p.N + width - 1) / width);
    const int64_t tiles = p.tiles_w * (((int64_t)p.rows + BN - 1) / BN);
    if (tiles > 0x7fffffff / 8) return SNNB_ERR_ARG;
    p.tiles = (int)tiles;
    unsigned grid, cluster;
    if (PAIR) {
        grid = 2 * (unsigned)(tiles < 74 ? tiles : 74);
        cluster = 2;
    } else {
        // The largest split that leaves every cluster resident at once (the occupancy call counts
        // one CTA an SM) and pays; none where the tiles alone nearly fill the SMs, unless K is
        // long.  Tokens x features x K in 4 bits: 1 x 16384 x 4096: 9.3 us, 9.8 split in 2; 1 x
        // 8192 x 8192: 12.7, 10.6 in 2, 9.2 in 4; 64 x 2048 x 2048: 5.2, 6.4 in 4; with tokens in
        // 8 bits 16 x 16384 x 4096: 12.7, 11.9 in 2; 1 x 2048 x 2048: 6.4, 5.3 in 4, 4.6 in 8.
        const int nstages = (p.groups + S::GROUPS - 1) / S::GROUPS;
        int log = 0;
        for (int l = 1; l <= 3 && (tiles < 100 || nstages >= 24); ++l)
            if (tiles <= (int64_t)dev->clusters[l] * S::CTAS_PER_SM && split_pays(nstages, l))
                log = l;
        if ((1 << log) < min_split) return SNNB_ERR_UNSUPPORTED;
        grid = (unsigned)(tiles << log);
        cluster = 1u << log;
    }
    const uint64_t nb = (uint64_t)mx::blocks_of(K), groups = (uint64_t)p.groups;
    MxMaps m;
    const uint64_t wrow = nb * 16, arow = nb * mx::Fmt<FMT>::BLOCK_BYTES;
    const uint64_t wdims[2] = {wrow, (uint64_t)p.N}, adims[2] = {arow, (uint64_t)p.rows};
    const uint32_t wbox[2] = {PACKED_STAGES > 0 ? 64u : 128u, 128}, abox[2] = {128, (uint32_t)S::A_ROWS};
    rc = encode_tmap(&m.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, a, adims, &arow, abox,
                         CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != SNNB_OK) return rc;
    if (FMT == SNNB_MXFP8 && PACKED_STAGES == 0) {
        // 16 codes to the low half of a 16-byte slot, by the copy itself
        const uint64_t wels[2] = {wrow * 2, (uint64_t)p.N};
        rc = encode_tmap(&m.w, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, 2, w, wels, &wrow, wbox,
                         CU_TENSOR_MAP_SWIZZLE_128B);
    } else {
        rc = encode_tmap(&m.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, w, wdims, &wrow, wbox,
                         PACKED_STAGES > 0 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B);
    }
    if (rc != SNNB_OK) return rc;
    // scale groups as [row tile][group][128 words]
    const uint64_t str[2] = {512, groups * 512};
    const uint64_t asdims[3] = {128, groups, (uint64_t)(p.rows + 127) / 128};
    const uint64_t wsdims[3] = {128, groups, (uint64_t)(p.N + 127) / 128};
    const uint32_t asbox[3] = {128, S::GROUPS, S::TOKEN_TILES}, wsbox[3] = {128, S::GROUPS, 1};
    rc = encode_tmap(&m.as, CU_TENSOR_MAP_DATA_TYPE_INT32, 3, as, asdims, str, asbox,
                     CU_TENSOR_MAP_SWIZZLE_NONE);
    if (rc != SNNB_OK) return rc;
    rc = encode_tmap(&m.ws, CU_TENSOR_MAP_DATA_TYPE_INT32, 3, ws, wsdims, str, wsbox,
                     CU_TENSOR_MAP_SWIZZLE_NONE);
    if (rc != SNNB_OK) return rc;
    return launch_kc(k, dim3(grid), dim3(mx_threads<BN, PACKED_STAGES>()), S::DYN, s, cluster, m.w, m.a, m.ws,
                     m.as, p);
}

// UNPACK: the copies unpack the weights beside E4M3 tokens.
template <int FMT, bool UNPACK>
int pick_mx(const void* a, const void* as, const void* w, const void* ws, int64_t rows, int64_t N,
            int64_t K, const MxParams& p, cudaStream_t s) {
    constexpr bool F4 = FMT == SNNB_MXFP4, P = !F4 && !UNPACK;      // P: a packed ring
    // Up to 128 tokens: one token tile, K split.  Two CTAs an SM, or one whose packed ring covers
    // the latency of HBM.
    if (rows <= 16) return launch_mx<FMT, 16, P ? 4 : 5, false, P ? 16 : 0>(a, as, w, ws, K, p, s);
    if (rows <= 32) return launch_mx<FMT, 32, 4, false, P ? 14 : 0>(a, as, w, ws, K, p, s);
    if (rows <= 64) return launch_mx<FMT, 64, 4, false, P ? 12 : 0>(a, as, w, ws, K, p, s);
    if (rows <= 128) return launch_mx<FMT, 128, P ? 4 : 6, false, P ? 8 : 0>(a, as, w, ws, K, p, s);
    // Pairs, 74 at once.  128 tokens a tile where that still fits one round, and for short K,
    // where the second accumulator hides the stores (8192 x 8192, K = 512: 35 us against 43 with
    // 256; K = 2048: 78 against 68); 256 otherwise.
    const int64_t pw = (N + 255) / 256, nstages = (p.groups + (F4 ? 1 : 0)) / (F4 ? 2 : 1);
    if (pw * ((rows + 127) / 128) <= 74) {
        // One round that leaves SMs idle over a long K: split K instead (200 x 512 x 16384 in 4
        // bits: 8.5 us against 20; 1024 x 1024 x 1024: 10 against 4.4).  Only 2 ways fit: from 24
        // stages (256 x 2304 x 8192: 10.1 against 11.8; x 4096: 8.1 against 7.5; 512 x 2048 x
        // 5632 with tokens in 8 bits: 11.5 against 14.2; x 2048: 8.2 against 7.3; with a packed
        // ring 256 x 2304 x 4000: 14.3 against 17.4; x 1936: 11.5 against 10.9).
        if (nstages >= 12) {
            const int rc = launch_mx<FMT, 128, P ? 4 : 6, false, P ? 8 : 0>(
                a, as, w, ws, K, p, s, nstages >= 24 ? 2 : 4);
            if (rc != SNNB_ERR_UNSUPPORTED) return rc;
        }
        return launch_mx<FMT, 128, P ? 6 : 7, true, P ? 6 : 0>(a, as, w, ws, K, p, s);
    }
    if (K <= 768 && pw * ((rows + 255) / 256) > 74)
        return launch_mx<FMT, 128, P ? 6 : 7, true, P ? 6 : 0>(a, as, w, ws, K, p, s);
    return launch_mx<FMT, 256, P ? 5 : 6, true, P ? 5 : 0>(a, as, w, ws, K, p, s);
}

int run_mx(const void* a, const void* as, int a_fmt, int64_t rows, int64_t K, const void* w,
           const void* ws, int64_t N, const float* bias, void* out, int out_dtype, cudaStream_t s) {
    MxParams p = {};
    p.status = device_status_ptr();
    if (!p.status) return SNNB_ERR_CUDA;
    p.rows = (int)rows; p.N = (int)N; p.groups = (int)mx::groups_of(K);
    p.bias = bias; p.out = out; p.out_dtype = out_dtype;
    const bool words = out_dtype != SNNB_F32 && reinterpret_cast<uintptr_t>(out) % 4 == 0;
    p.pairs = words && N % 2 == 0;
    p.odd_pairs = words && N % 2 == 1;
    if (a_fmt == SNNB_MXFP4) return pick_mx<SNNB_MXFP4, false>(a, as, w, ws, rows, N, K, p, s);
    // an unpacking copy wants whole groups of 128 elements a row and a base on 32 bytes
    if (mx::blocks_of(K) % 4 == 0 && reinterpret_cast<uintptr_t>(w) % 32 == 0)
        return pick_mx<SNNB_MXFP8, true>(a, as, w, ws, rows, N, K, p, s);
    return pick_mx<SNNB_MXFP8, false>(a, as, w, ws, rows, N, K, p, s);
}

}  // namespace
}  // namespace snnb

using namespace snnb;

extern "C" int snnb_mx_linear(const void* a, const void* a_scales, int a_fmt, int64_t rows,
                              int64_t K, const void* w, const void* w_scales, int64_t N,
                              const float* bias, void* out, int out_dtype, snnb_stream_t stream) {
    if (const int inj = take_injected_status()) return inj;
    if (a_fmt != SNNB_MXFP4 && a_fmt != SNNB_MXFP8) return SNNB_ERR_ARG;
    if (out_dtype != SNNB_F32 && out_dtype != SNNB_F16 && out_dtype != SNNB_BF16)
        return SNNB_ERR_ARG;
    if (N < 1 || !mx::sizes_ok(rows, K) || !mx::sizes_ok(N, K)) return SNNB_ERR_ARG;
    if (rows == 0) return SNNB_OK;
    if (!a || !a_scales || !w || !w_scales || !out || !aligned16(a) || !aligned16(a_scales) ||
        !aligned16(w) || !aligned16(w_scales))
        return SNNB_ERR_ARG;
    const uintptr_t es = out_dtype == SNNB_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(out) % es || reinterpret_cast<uintptr_t>(bias) % 4)
        return SNNB_ERR_ARG;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return run_mx(a, a_scales, a_fmt, rows, K, w, w_scales, N, bias, out, out_dtype, s);
}
