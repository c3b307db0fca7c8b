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
//              row), which wants 16 4-bit codes as 8 bytes in a 16-byte slot: four warps copy the
//              weights' 8-byte pieces there with cp.async
//   scales     512-byte groups (128 rows x 4 blocks) as they lie in memory, by bulk copies; the
//              MMA thread copies them on to TMEM (tcgen05.cp), a slot per ring stage
//
//   warp 0     TMA and bulk copies        warps 2-5  epilogue, thread = TMEM lane = feature
//   warp 1     MMA issuer                 warps 6-9  (E4M3 only) weight pieces
#include "mx.cuh"
#include "tc_common.cuh"

namespace snnb {
namespace {

struct MxParams {
    int rows, N, groups;             // tokens, features, 128-wide groups of K
    int tiles_w, tiles;              // feature tiles, tiles in all
    int64_t w_row_bytes;
    const uint8_t *w, *w_scales, *a_scales;
    const float* bias;
    void* out;
    int out_dtype;
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
template <int FMT>
__device__ __forceinline__ void umma_mx(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t sa, uint32_t sb, uint32_t accumulate) {
    if constexpr (FMT == SNNB_MXFP4)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X"
            " [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X"
            " [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)
            : "memory");
}
// One 512-byte scale group (32 rows of 16 bytes, unswizzled) to 4 TMEM columns, the same 32
// lanes in each of the four lane quarters.
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t saddr) {
    uint64_t d = (uint64_t)((saddr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(128 >> 4) << 32;                 // 8 rows to the next 8: 128 bytes
    d |= (uint64_t)1 << 46;
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
        : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait_group() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
    asm volatile("cp.async.commit_group;" ::: "memory");
}

// ---- shared memory -----------------------------------------------------------------------
template <int FMT, int BN, int STAGES>
struct MxSmem {
    static constexpr int GROUPS = FMT == SNNB_MXFP4 ? 2 : 1;     // 128-wide groups of K a stage
    static constexpr int TOKEN_TILES = (BN + 127) / 128;
    static constexpr int W_TILE = 128 * 128;
    static constexpr int A_TILE = BN * 128;
    static constexpr int W_SCALES = GROUPS * mx::GROUP_BYTES;
    static constexpr int A_SCALES = TOKEN_TILES * GROUPS * mx::GROUP_BYTES;
    static constexpr int STAGE = W_TILE + A_TILE;                // operand tiles, 1024-aligned
    static constexpr int SCALES_OFF = STAGES * STAGE;
    static constexpr int SCALES = W_SCALES + A_SCALES;           // per stage
    static constexpr int BAR_OFF = SCALES_OFF + STAGES * SCALES;
    static constexpr int ACCS = BN <= 128 ? 2 : 1;               // accumulators in TMEM
    static constexpr int NBARS = 2 * STAGES + 2 * ACCS + 1;
    static constexpr int TMEM_OFF = BAR_OFF + NBARS * 8;
    static constexpr int TOTAL = TMEM_OFF + 8;
    static constexpr int DYN = TOTAL + 1024;
    // TMEM: the accumulators, then per ring stage 4 columns per scale group
    static constexpr int SCALE_COLS = 4 * GROUPS * (1 + TOKEN_TILES);
    static constexpr int COLS_USED = ACCS * BN + STAGES * SCALE_COLS;
    static constexpr int COLS = COLS_USED <= 128 ? 128 : (COLS_USED <= 256 ? 256 : 512);
    static_assert(COLS_USED <= 512, "tensor memory");
    static_assert(DYN <= 227 * 1024, "shared memory");
};

template <int FMT> constexpr int mx_threads() { return FMT == SNNB_MXFP4 ? 192 : 320; }

__device__ __forceinline__ void store_out(const MxParams& p, int64_t i, float v) {
    if (!SNNB_IN_BOUNDS(i, (int64_t)p.rows * p.N, p.status)) return;
    if (p.out_dtype == SNNB_F32)
        static_cast<float*>(p.out)[i] = v;
    else if (p.out_dtype == SNNB_F16)
        static_cast<__half*>(p.out)[i] = __float2half_rn(v);
    else
        static_cast<__nv_bfloat16*>(p.out)[i] = __float2bfloat16_rn(v);
}

// SPLIT: the K range of one tile over a cluster of CTAs, their float32 partial sums joined in
// rank order through distributed shared memory; otherwise a CTA walks whole tiles.
template <int FMT, int BN, int STAGES, bool SPLIT>
__global__ void __launch_bounds__(mx_threads<FMT>(), 1)
mx_linear_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA,
                 const MxParams p) {
    using S = MxSmem<FMT, BN, STAGES>;
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
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + S::TMEM_OFF);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            tc::mbar_init(full_bar(s), FMT == SNNB_MXFP4 ? 1 : 5);
            tc::mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < S::ACCS; ++b) {
            tc::mbar_init(accf_bar(b), 1);
            tc::mbar_init(acce_bar(b), 4);
        }
        tc::mbar_init(done_bar, 1);
        tc::fence_mbar_init();
        tc::prefetch_tmap(&tmW);
        tc::prefetch_tmap(&tmA);
    }
    if (warp == 1) {
        tc::tmem_alloc(sbase + S::TMEM_OFF, S::COLS);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_trigger();
    pdl_wait();

    // this CTA's tiles and, within a tile, its stages of K
    const int splits = SPLIT ? (int)gridDim.x / p.tiles : 1;
    const int rank = SPLIT ? (int)blockIdx.x % splits : 0;
    const int tile0 = SPLIT ? (int)blockIdx.x / splits : (int)blockIdx.x;
    const int tile_step = SPLIT ? p.tiles : (int)gridDim.x;
    const int nstages = (p.groups + S::GROUPS - 1) / S::GROUPS;
    const int k0 = (int)((int64_t)nstages * rank / splits);
    const int k1 = (int)((int64_t)nstages * (rank + 1) / splits);
    uint32_t failed = 0;

    if (warp == 0) {
        // ------------------------------------------------------------- copies
        uint32_t it = 0, issued = 0;
        for (int tile = tile0; tile < p.tiles; tile += tile_step) {
            const int tw = tile % p.tiles_w, tt = tile / p.tiles_w;
            for (int ks = k0; ks < k1; ++ks, ++it) {
                const int s = (int)(it % STAGES);
                failed |= 1u - tc::mbar_wait_warp(empty_bar(s), ((it / STAGES) & 1u) ^ 1u, failed);
                if (failed) break;
                if (tc::elect_one()) {
                    const int g0 = ks * S::GROUPS;
                    const uint32_t gb = (uint32_t)(min(S::GROUPS, p.groups - g0) * mx::GROUP_BYTES);
                    // token tiles of 128 rows that exist (the others' scales are not read)
                    const int tiles128 = min(S::TOKEN_TILES, (p.rows + 127) / 128 - tt * S::TOKEN_TILES);
                    const uint32_t bytes = (uint32_t)S::A_TILE + gb * (uint32_t)(1 + tiles128) +
                                           (FMT == SNNB_MXFP4 ? (uint32_t)S::W_TILE : 0u);
                    tc::mbar_expect_tx(full_bar(s), bytes);
                    if (FMT == SNNB_MXFP4)
                        tc::tma_load_2d(w_tile(s), &tmW, full_bar(s), ks * 128, tw * 128);
                    tc::tma_load_2d(a_tile(s), &tmA, full_bar(s), ks * 128, tt * BN);
                    const uint32_t sc = scales_at(s);
                    bulk_load(sc, p.w_scales + ((int64_t)tw * p.groups + g0) * mx::GROUP_BYTES, gb,
                              full_bar(s));
                    for (int h = 0; h < tiles128; ++h)
                        bulk_load(sc + S::W_SCALES + h * S::GROUPS * mx::GROUP_BYTES,
                                  p.a_scales + ((int64_t)(tt * S::TOKEN_TILES + h) * p.groups + g0) *
                                                   mx::GROUP_BYTES,
                                  gb, full_bar(s));
                }
                __syncwarp();
                ++issued;
            }
            if (failed) break;
        }
        if (failed) {
            // copies still in flight land before the CTA may exit
            for (uint32_t k = 0; k < issued && k < (uint32_t)STAGES; ++k) {
                const uint32_t g = issued - 1 - k;
                tc::mbar_wait_warp<true>(full_bar((int)(g % STAGES)), (g / STAGES) & 1u, 0);
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------- MMA issuer
        constexpr uint32_t IDESC = FMT == SNNB_MXFP4 ? idesc_mx(1, 1, 128, BN)
                                                     : idesc_mx(5, 0, 128, BN);
        if (tc::elect_one()) {
            uint32_t it = 0, local = 0;
            for (int tile = tile0; tile < p.tiles; tile += tile_step, ++local) {
                const int b = (int)(local % S::ACCS);
                failed |= 1u - tc::mbar_wait_lane(acce_bar(b), ((local / S::ACCS) & 1u) ^ 1u, failed);
                tc::tc_fence_after();
                const uint32_t d = tmem + (uint32_t)(b * BN);
                for (int ks = k0; ks < k1; ++ks, ++it) {
                    const int s = (int)(it % STAGES);
                    failed |= 1u - tc::mbar_wait_lane(full_bar(s), (it / STAGES) & 1u, failed);
                    tc::tc_fence_after();
                    if (!failed) {
                        const uint32_t sw = tmem + (uint32_t)(S::ACCS * BN + s * S::SCALE_COLS);
                        const uint32_t sa = sw + 4 * S::GROUPS;
                        const uint32_t sc = scales_at(s);
                        const int ng = min(S::GROUPS, p.groups - ks * S::GROUPS);
                        for (int g = 0; g < ng; ++g) {
                            copy_scales(sw + 4 * g, sc + g * mx::GROUP_BYTES);
#pragma unroll
                            for (int h = 0; h < S::TOKEN_TILES; ++h)
                                copy_scales(sa + 4 * (g * S::TOKEN_TILES + h),
                                            sc + S::W_SCALES + (h * S::GROUPS + g) * mx::GROUP_BYTES);
                        }
                        const uint64_t dw = tc::sdesc_k_sw128(w_tile(s));
                        const uint64_t da = tc::sdesc_k_sw128(a_tile(s));
                        constexpr int PER_GROUP = 4 / S::GROUPS;     // MMAs per 128 of K
                        for (int g = 0; g < ng; ++g) {
#pragma unroll
                            for (int m = 0; m < PER_GROUP; ++m) {
                                const int k = g * PER_GROUP + m;
                                umma_mx<FMT>(d, dw + 2 * k, da + 2 * k,
                                             IDESC | idesc_scale_byte(m * S::GROUPS), sw + 4 * g,
                                             sa + 4 * g * S::TOKEN_TILES, (ks != k0) || (k != 0));
                            }
                        }
                    }
                    tc::umma_commit(empty_bar(s));
                }
                tc::umma_commit(accf_bar(b));
            }
            tc::umma_commit(done_bar);
        }
        __syncwarp();
        failed = __shfl_sync(0xffffffffu, failed, 0);
        failed |= 1u - tc::mbar_wait_warp<true>(done_bar, 0, 0);
    } else if (warp < 6) {
        // ------------------------------------------------------------- epilogue
        const int q = warp & 3;
        uint32_t local = 0;
        for (int tile = tile0; tile < p.tiles; tile += tile_step, ++local) {
            const int tw = tile % p.tiles_w, tt = tile / p.tiles_w;
            const int b = (int)(local % S::ACCS);
            failed |= 1u - tc::mbar_wait_warp(accf_bar(b), (local / S::ACCS) & 1u, failed);
            tc::tc_fence_after();
            if (failed) break;
            const uint32_t t = tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)(b * BN);
            const int n = tw * 128 + 32 * q + lane;
            constexpr int STEP = BN < 32 ? 16 : 32;
            if (SPLIT && splits > 1) {
                // partial sums [column][lane] in the drained ring
                float* part = reinterpret_cast<float*>(smem) + 32 * q + lane;
#pragma unroll 1
                for (int c = 0; c < BN; c += 16) {
                    float r[16];
                    tc::tmem_ld16(t + c, r);
                    tc::tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) part[(c + i) * 128] = r[i];
                }
            } else {
                const float bias = p.bias && n < p.N ? __ldg(p.bias + n) : 0.0f;
                const int64_t left = (int64_t)p.rows - (int64_t)tt * BN;
                const int cols = (int)(left < BN ? left : BN);
                int64_t o = (int64_t)tt * BN * p.N + n;
#pragma unroll 1
                for (int c = 0; c < cols; c += STEP) {
                    float r[STEP];
                    if constexpr (STEP == 32) tc::tmem_ld32(t + c, r);
                    else tc::tmem_ld16(t + c, r);
                    tc::tmem_wait_ld();
                    if (n < p.N) {
#pragma unroll
                        for (int i = 0; i < STEP; ++i)
                            if (c + i < cols) store_out(p, o + (int64_t)(c + i) * p.N, r[i] + bias);
                    }
                }
            }
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(acce_bar(b));
        }
    } else {
        // ------------------------------------------------------------- weight pieces (E4M3)
        // 16 codes (8 bytes) to the low half of a 16-byte slot; slot c of row r at c ^ (r % 8)
        constexpr int AHEAD = STAGES - 2;
        const int i = (warp - 6) * 32 + lane;
        const int c = i & 7;
        uint32_t it = 0;
        for (int tile = tile0; tile < p.tiles; tile += tile_step) {
            const int64_t n0 = (int64_t)(tile % p.tiles_w) * 128;
            for (int ks = k0; ks < k1; ++ks, ++it) {
                const int s = (int)(it % STAGES);
                failed |= 1u - tc::mbar_wait_warp(empty_bar(s), ((it / STAGES) & 1u) ^ 1u, failed);
                if (failed) break;
                const int64_t kb = (int64_t)ks * 64 + c * 8;
                const uint32_t dst = w_tile(s);
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int r = u * 16 + (i >> 3);
                    const bool in = n0 + r < p.N && kb < p.w_row_bytes;
                    tc::cp_async_8(dst + r * 128 + ((c ^ (r & 7)) << 4),
                                   p.w + (in ? (n0 + r) * p.w_row_bytes + kb : 0), in ? 8u : 0u);
                }
                cp_async_commit();
                if (it >= (uint32_t)AHEAD) {
                    cp_async_wait_group<AHEAD>();
                    tc::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(full_bar((int)((it - AHEAD) % STAGES)));
                }
            }
            if (failed) break;
        }
        tc::cp_async_wait_all();
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (!failed && lane == 0)
            for (uint32_t g = it > (uint32_t)AHEAD ? it - AHEAD : 0; g < it; ++g)
                tc::mbar_arrive(full_bar((int)(g % STAGES)));
    }
    if (failed && lane == 0) atomicExch(p.status, SNNB_ERR_TIMEOUT);
    if (SPLIT && splits > 1) {
        tc::cluster_sync();                          // every CTA's partial sums are in place
        if (warp >= 2 && warp < 6) {
            const int q = warp & 3;
            const int tw = tile0 % p.tiles_w, tt = tile0 / p.tiles_w;
            const int n = tw * 128 + 32 * q + lane;
            const float bias = p.bias && n < p.N ? __ldg(p.bias + n) : 0.0f;
            const int64_t left = (int64_t)p.rows - (int64_t)tt * BN;
            const int cols = (int)(left < BN ? left : BN);
            const uint32_t mine = sbase + (uint32_t)(32 * q + lane) * 4u;
            for (int c = rank; c < cols; c += splits) {
                float v = 0.0f;
                for (int r = 0; r < splits; ++r) {
                    float x;
                    asm volatile("ld.shared::cluster.f32 %0, [%1];"
                                 : "=f"(x)
                                 : "r"(tc::map_to_rank(mine + (uint32_t)c * 512u, (uint32_t)r)));
                    v += x;
                }
                if (n < p.N) store_out(p, ((int64_t)tt * BN + c) * p.N + n, v + bias);
            }
        }
        tc::cluster_sync();                          // nobody reads this CTA's memory any more
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, S::COLS);
    }
}

template <int FMT, int BN, int STAGES, bool SPLIT>
int launch_mx(const CUtensorMap& tw, const CUtensorMap& ta, const MxParams& p, int splits,
              cudaStream_t s) {
    using S = MxSmem<FMT, BN, STAGES>;
    auto k = mx_linear_kernel<FMT, BN, STAGES, SPLIT>;
    const cudaError_t e =
        cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, S::DYN);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (SPLIT)
        return launch_kc(k, dim3((unsigned)(p.tiles * splits)), dim3(mx_threads<FMT>()), S::DYN, s,
                         (unsigned)splits, tw, ta, p);
    const int grid = p.tiles < 148 ? p.tiles : 148;
    return launch_k(k, dim3((unsigned)grid), dim3(mx_threads<FMT>()), S::DYN, s, tw, ta, p);
}

template <int FMT>
int run_mx(const void* a, const void* as, int64_t rows, int64_t K, const void* w, const void* ws,
           int64_t N, const float* bias, void* out, int out_dtype, cudaStream_t s) {
    int* status = device_status_ptr();
    if (!status) return SNNB_ERR_CUDA;
    const int64_t nb = mx::blocks_of(K);
    const int BN = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
    CUtensorMap tw = {}, ta = {};
    const uint64_t wrow = (uint64_t)nb * 16, arow = (uint64_t)nb * mx::Fmt<FMT>::BLOCK_BYTES;
    const uint64_t wdims[2] = {wrow, (uint64_t)N}, adims[2] = {arow, (uint64_t)rows};
    const uint32_t wbox[2] = {128, 128}, abox[2] = {128, (uint32_t)BN};
    int rc = encode_tmap(&ta, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, a, adims, &arow, abox,
                         CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != SNNB_OK) return rc;
    rc = encode_tmap(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, w, wdims, &wrow, wbox,
                     CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != SNNB_OK) return rc;
    MxParams p = {};
    p.rows = (int)rows; p.N = (int)N; p.groups = (int)mx::groups_of(K);
    p.tiles_w = (int)((N + 127) / 128);
    const int64_t tiles = p.tiles_w * ((rows + BN - 1) / BN);
    if (tiles > 0x7fffffff / 8) return SNNB_ERR_ARG;
    p.tiles = (int)tiles;
    p.w_row_bytes = (int64_t)wrow;
    p.w = static_cast<const uint8_t*>(w);
    p.w_scales = static_cast<const uint8_t*>(ws);
    p.a_scales = static_cast<const uint8_t*>(as);
    p.bias = bias; p.out = out; p.out_dtype = out_dtype; p.status = status;
    const int per = FMT == SNNB_MXFP4 ? 2 : 1;
    const int nstages = (p.groups + per - 1) / per;
    int splits = 1;
    while (splits < 8 && tiles * splits * 2 <= 296 && splits * 2 <= nstages) splits *= 2;
    if (BN == 16) return launch_mx<FMT, 16, 5, true>(tw, ta, p, splits, s);
    if (BN == 32) return launch_mx<FMT, 32, 4, true>(tw, ta, p, splits, s);
    if (BN == 64) return launch_mx<FMT, 64, 4, true>(tw, ta, p, splits, s);
    if (BN == 128) return launch_mx<FMT, 128, 5, true>(tw, ta, p, splits, s);
    return launch_mx<FMT, 256, 4, false>(tw, ta, p, 1, s);
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
    if (rows < 0 || N < 1 || K < 1 || rows > 0x7fffffff || N > 0x7fffffff || K > 0x7fffffff)
        return SNNB_ERR_ARG;
    if (rows == 0) return SNNB_OK;
    if (!a || !a_scales || !w || !w_scales || !out || !aligned16(a) || !aligned16(a_scales) ||
        !aligned16(w) || !aligned16(w_scales))
        return SNNB_ERR_ARG;
    const uintptr_t es = out_dtype == SNNB_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(out) % es || reinterpret_cast<uintptr_t>(bias) % 4)
        return SNNB_ERR_ARG;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return a_fmt == SNNB_MXFP4
               ? run_mx<SNNB_MXFP4>(a, a_scales, rows, K, w, w_scales, N, bias, out, out_dtype, s)
               : run_mx<SNNB_MXFP8>(a, a_scales, rows, K, w, w_scales, N, bias, out, out_dtype, s);
}
