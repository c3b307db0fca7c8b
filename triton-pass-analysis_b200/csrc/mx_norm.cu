// Root-mean-square norm of x + residual with a microscaled output (formats: mx.cuh):
//   h = x + residual                        float32; also stored, rounded to x's type
//   y = (h / sqrt(mean(h^2) + eps)) * weight
//   codes, scales = y in E2M1 or E4M3, one scale per 32 values
//
// Rounding.  The norm is taken of the unrounded sum h.  Squares are summed in float32 within 8
// values and in float64 beyond, and 1 / sqrt is float64, so that rstd is good to ~1e-9: an error
// of one float32 ulp (6e-8) in y already moves ~7e-7 of the codes to a neighbour.  y itself is
// float32 unless it lies within 4 ulp of a value that a code boundary could be (its low 19 bits
// zero: 3 mantissa bits and the half step), where it is formed again in float64 and rounded to
// odd, which keeps it on its side of the boundary.
//
// Two forms.  Many aligned rows: a team of LANES threads walks rows, whose x and residual come
// by bulk copies into a ring in shared memory while earlier rows are worked on; both passes over
// a row (squares, output) read it there.  Few rows, unaligned rows or rows too long for the ring:
// a row's values stay in registers between the passes (or are read twice past 1024 threads x 32).
// Four neighbouring lanes hold one block of 32, as in the quantisation kernel.
//
// Bound: HBM for many rows; for few, the latency of one load, one sum over the block, one store.
#include "mx.cuh"
#include "tc_common.cuh"

namespace snnb {
namespace {

struct NormParams {
    const void* weight;
    int w_f32;                   // weight is float32 (else of x's type)
    int fmt;
    float eps;
    double inv_k;
    uint32_t rows, K, nb, groups;
    int64_t ldx, ldr;
    uint8_t* data;
    uint32_t* scales;
    int* status;
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
// Sum of 8 squares.
__device__ __forceinline__ float squares8(const float (&h)[8]) {
    const float a = fmaf(h[0], h[0], h[1] * h[1]), b = fmaf(h[2], h[2], h[3] * h[3]);
    const float c = fmaf(h[4], h[4], h[5] * h[5]), d = fmaf(h[6], h[6], h[7] * h[7]);
    return (a + b) + (c + d);
}
// ... in float64 where float32 overflows or loses it: squares of values past 2^63 or below 2^-50.
__device__ __forceinline__ double squares8_exact(const float (&h)[8]) {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fma((double)h[i], (double)h[i], s);
    return s;
}
__device__ __forceinline__ double add_squares(const float (&h)[8]) {
    const float s = squares8(h);
    return s > 1e-30f && s < 1e38f ? (double)s : squares8_exact(h);
}
__device__ __forceinline__ double rstd_of(const NormParams& p, double sum) {
    return rsqrt(fma(sum, p.inv_k, (double)p.eps));
}

template <typename T, bool ALIGNED>
__device__ __forceinline__ void weights8(const NormParams& p, uint32_t k, int n, float (&w)[8]) {
    if (p.w_f32) {
        const float* q = static_cast<const float*>(p.weight);
        mx::Raw8<float> r = mx::zero8<float>();
        if (n > 0) {
            if (ALIGNED) {
#pragma unroll
                for (int i = 0; i < 2; ++i) r.v[i] = __ldg(reinterpret_cast<const uint4*>(q + k) + i);
            } else {
                r = mx::load_any8(q + k, n, q, (int64_t)p.K);
            }
        }
        mx::to_floats(r, w);
    } else {
        const T* q = static_cast<const T*>(p.weight);
        mx::Raw8<T> r = mx::zero8<T>();
        if (n > 0) {
            if (ALIGNED) {
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                    r.v[i] = __ldg(reinterpret_cast<const uint4*>(q + k) + i);
            } else {
                r = mx::load_any8(q + k, n, q, (int64_t)p.K);
            }
        }
        mx::to_floats(r, w);
    }
}

// y of 8 values (see the top); values past n, whose h and w are 0, give 0.
__device__ __forceinline__ void normed8(const float (&h)[8], const float (&w)[8], float rstd,
                                        double rstd64, float (&y)[8]) {
    uint32_t near = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        y[i] = __fmul_rn(__fmul_rn(h[i], rstd), w[i]);
        near = min(near, ((uint32_t)__float_as_int(y[i]) + 4u) & 0x7FFFFu);
    }
    if (near <= 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t bits = (uint32_t)__float_as_int(y[i]);
            if (((bits + 4u) & 0x7FFFFu) > 8 || (bits << 1) == 0) continue;
            const double d = (double)h[i] * rstd64 * (double)w[i];
            const float t = __double2float_rz(d);
            y[i] = (double)t != d && isfinite(t) ? __int_as_float(__float_as_int(t) | 1) : t;
        }
    }
}

// Codes and scale word of 8 values at column k of a row.  Every lane of the warp calls.
__device__ __forceinline__ void emit8(const NormParams& p, uint32_t row, uint32_t k, bool in_row,
                                      const float (&y)[8], int lane) {
    const uint32_t j = k >> 5, sub = lane & 3;
    const bool inside = in_row && j < p.nb;
    const uint32_t e = mx::top_exponent(y);
    const uint64_t block = (uint64_t)(row * p.nb + j);
    uint32_t byte;
    if (p.fmt == SNNB_MXFP4) {
        uint32_t c;
        byte = mx::quantise_block<SNNB_MXFP4>(y, e, c);
        if (inside) *reinterpret_cast<uint32_t*>(p.data + block * 16 + sub * 4) = c;
    } else {
        uint2 c;
        byte = mx::quantise_block<SNNB_MXFP8>(y, e, c);
        if (inside) *reinterpret_cast<uint2*>(p.data + block * 32 + sub * 8) = c;
    }
    const uint32_t word = mx::join_scales(byte, lane);
    if (in_row && (j >> 2) < p.groups && (lane & 15) == 0)
        p.scales[mx::scale_word(row, j >> 2, p.groups)] = word;
}

// ---- rows through registers --------------------------------------------------------------
template <typename T, bool ALIGNED>
__device__ __forceinline__ void take8(const NormParams& p, const T* x, const T* r, uint32_t row,
                                      uint32_t k, int n, float (&h)[8]) {
    mx::Raw8<T> a = mx::zero8<T>();
    const T* xr = x + (int64_t)row * p.ldx;
    if (n > 0) a = ALIGNED ? mx::load_aligned8(xr + k) : mx::load_any8(xr + k, n, xr, (int64_t)p.K);
    mx::to_floats(a, h);
    if (r) {
        mx::Raw8<T> b = mx::zero8<T>();
        const T* rr = r + (int64_t)row * p.ldr;
        if (n > 0) b = ALIGNED ? mx::load_aligned8(rr + k) : mx::load_any8(rr + k, n, rr, (int64_t)p.K);
        float f[8];
        mx::to_floats(b, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] += f[i];
    }
}
template <typename T, bool ALIGNED>
__device__ __forceinline__ void put_h8(const NormParams& p, T* h_out, uint32_t row, uint32_t k,
                                       int n, const float (&h)[8], int lane) {
    mx::Raw8<T> o;
    mx::from_floats(h, o);
    T* q = h_out + (n > 0 ? (uint64_t)row * p.K + k : 0);
    if (!ALIGNED) mx::store_any8(q, n, o, lane);
    else if (n > 0) mx::store_aligned8(q, o);
}

// LANES threads a row, CHUNKS x 8 values a thread: thread t holds columns (c * LANES + t) * 8 ..
// + 7 of chunk c.  CHUNKS == 0: rows of any length, read twice.
template <typename T, bool ALIGNED, int LANES, int CHUNKS>
__global__ void __launch_bounds__(LANES == 32 ? 256 : LANES)
rms_norm_mx_kernel(const T* __restrict__ x, const T* __restrict__ r, T* __restrict__ h_out,
                   const NormParams p) {
    constexpr uint32_t THREADS = LANES == 32 ? 256 : LANES;
    __shared__ double shared[32];
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const uint32_t t = LANES == 32 ? lane : threadIdx.x;
    const uint32_t row = LANES == 32 ? blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    const bool in_row = row < p.rows;
    auto valid = [&](uint32_t k) { return in_row && k < p.K ? (int)min(8u, p.K - k) : 0; };
    auto row_sum = [&](double v) {
        v = warp_sum(v);
        if (LANES == 32) return v;
        if (lane == 0) shared[threadIdx.x >> 5] = v;
        __syncthreads();
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < LANES / 32; ++i) s += shared[i];
        return s;
    };
    auto finish = [&](uint32_t k, const float (&h)[8], float rstd, double rstd64) {
        float w[8], y[8];
        weights8<T, ALIGNED>(p, k, valid(k), w);
        normed8(h, w, rstd, rstd64, y);
        emit8(p, row, k, in_row, y, lane);
    };
    double sum = 0.0;
    if constexpr (CHUNKS > 0) {
        float h[CHUNKS][8];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t k = (c * LANES + t) * 8;
            take8<T, ALIGNED>(p, x, r, row, k, valid(k), h[c]);
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t k = (c * LANES + t) * 8;
            if (h_out) put_h8<T, ALIGNED>(p, h_out, row, k, valid(k), h[c], lane);
            if (valid(k)) sum += add_squares(h[c]);
        }
        const double rstd64 = rstd_of(p, row_sum(sum));
        const float rstd = (float)rstd64;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            if ((c * LANES + (t & ~31u)) * 8 >= p.groups * 128) break;       // whole warps
            finish((c * LANES + t) * 8, h[c], rstd, rstd64);
        }
    } else {
        float h[8];
        for (uint32_t k = t * 8; (k & ~255u) < p.K; k += LANES * 8) {        // whole warps
            const int n = valid(k);
            take8<T, ALIGNED>(p, x, r, row, k, n, h);
            if (h_out) put_h8<T, ALIGNED>(p, h_out, row, k, n, h, lane);
            if (n) sum += add_squares(h);
        }
        const double rstd64 = rstd_of(p, row_sum(sum));
        const float rstd = (float)rstd64;
        for (uint32_t k = t * 8; (k & ~255u) < p.groups * 128; k += LANES * 8) {
            take8<T, ALIGNED>(p, x, r, row, k, valid(k), h);
            finish(k, h, rstd, rstd64);
        }
    }
    mx::zero_row_padding(p.scales, p.rows, p.groups, (uint64_t)blockIdx.x * THREADS + threadIdx.x,
                         (uint64_t)gridDim.x * THREADS);
}

// ---- rows through shared memory ----------------------------------------------------------
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
        : "memory");
}
template <typename T>
__device__ __forceinline__ mx::Raw8<T> smem8(const uint8_t* row, uint32_t k) {
    mx::Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        r.v[i] = reinterpret_cast<const uint4*>(row + k * sizeof(T))[i];
    return r;
}

constexpr int RING_MAX = 4;
constexpr int RING_HEAD = 1024;              // barriers and sums, before the ring

// Teams of LANES threads; team g of all walks the rows g, g + (number of teams), ...  A ring
// stage holds one row of x and, `half` bytes behind it, of the residual.
template <typename T, int LANES>
__global__ void __launch_bounds__(LANES < 256 ? 256 : LANES)
rms_norm_mx_ring_kernel(const T* __restrict__ x, const T* __restrict__ r, T* __restrict__ h_out,
                        const NormParams p, int stages, uint32_t half) {
    constexpr int THREADS = LANES < 256 ? 256 : LANES, TEAMS = THREADS / LANES, WARPS = LANES / 32;
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31;
    const int team = threadIdx.x / LANES;
    const uint32_t t = threadIdx.x % LANES;
    const uint32_t stage_bytes = half * (r ? 2 : 1);
    const uint32_t bars = tc::smem_u32(smem) + (uint32_t)team * RING_MAX * 8;
    double* sums = reinterpret_cast<double*>(smem + TEAMS * RING_MAX * 8) + team * 2 * WARPS;
    uint8_t* ring = smem + RING_HEAD + (size_t)team * stages * stage_bytes;
    const uint32_t ring32 = tc::smem_u32(ring);
    if (t == 0) {
        for (int s = 0; s < stages; ++s) tc::mbar_init(bars + 8 * s, 1);
        tc::fence_mbar_init();
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    const uint32_t row0 = blockIdx.x * TEAMS + team, step = gridDim.x * TEAMS;
    const uint32_t bytes = p.K * (uint32_t)sizeof(T);
    auto fetch = [&](uint32_t row, int s) {
        const uint32_t dst = ring32 + (uint32_t)s * stage_bytes;
        tc::mbar_expect_tx(bars + 8 * s, bytes * (r ? 2u : 1u));
        bulk_load(dst, x + (int64_t)row * p.ldx, bytes, bars + 8 * s);
        if (r) bulk_load(dst + half, r + (int64_t)row * p.ldr, bytes, bars + 8 * s);
    };
    auto team_sync = [&] {
        if constexpr (LANES == 32) __syncwarp();
        else tc::named_bar_sync(1 + team, LANES);
    };
    if (t == 0)
        for (int s = 0; s < stages; ++s)
            if (row0 + (uint64_t)s * step < p.rows) fetch(row0 + s * step, s);
    uint32_t failed = 0;
    int s = 0;
    uint32_t parity = 0, odd = 0;
    for (uint64_t row64 = row0; row64 < p.rows; row64 += step, odd ^= 1) {
        const uint32_t row = (uint32_t)row64;
        if (!failed && !tc::mbar_wait_warp(bars + 8 * s, parity, 0)) {
            // a wait ran out: this warp works on and stores nothing; the copies in flight land
            // before the block may exit
            failed = 1;
            int fs = s;
            uint32_t fp = parity;
            for (int i = 0; i < stages; ++i) {
                if (row64 + (uint64_t)i * step < p.rows) tc::mbar_wait_warp<true>(bars + 8 * fs, fp, 0);
                if (++fs == stages) {
                    fs = 0;
                    fp ^= 1;
                }
            }
            if (lane == 0) atomicExch(p.status, SNNB_ERR_TIMEOUT);
        }
        const uint8_t* xs = ring + (size_t)s * stage_bytes;
        const uint8_t* rs = xs + half;
        auto take = [&](uint32_t k, float (&h)[8]) {
            mx::to_floats(smem8<T>(xs, k), h);
            if (r) {
                float f[8];
                mx::to_floats(smem8<T>(rs, k), f);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[i] += f[i];
            }
        };
        double sum = 0.0;
        for (uint32_t k = t * 8; k < p.K; k += LANES * 8) {
            float h[8];
            take(k, h);
            if (h_out && !failed) {
                mx::Raw8<T> o;
                mx::from_floats(h, o);
                mx::store_aligned8(h_out + (uint64_t)row * p.K + k, o);
            }
            sum += add_squares(h);
        }
        sum = warp_sum(sum);
        if constexpr (LANES > 32) {
            if (lane == 0) sums[odd * WARPS + (t >> 5)] = sum;
            team_sync();
            sum = 0.0;
#pragma unroll
            for (int i = 0; i < WARPS; ++i) sum += sums[odd * WARPS + i];
        }
        const double rstd64 = rstd_of(p, sum);
        const float rstd = (float)rstd64;
        for (uint32_t k = t * 8; (k & ~255u) < p.groups * 128; k += LANES * 8) {
            float h[8] = {0, 0, 0, 0, 0, 0, 0, 0}, w[8], y[8];
            const int n = k < p.K ? 8 : 0;
            if (n) take(k, h);
            weights8<T, true>(p, k, n, w);
            normed8(h, w, rstd, rstd64, y);
            emit8(p, row, k, !failed, y, lane);
        }
        team_sync();                                  // the stage has been read by all
        const uint64_t next = row64 + (uint64_t)stages * step;
        if (t == 0 && !failed && next < p.rows) fetch((uint32_t)next, s);
        if (++s == stages) {
            s = 0;
            parity ^= 1;
        }
    }
    mx::zero_row_padding(p.scales, p.rows, p.groups, (uint64_t)blockIdx.x * THREADS + threadIdx.x,
                         (uint64_t)gridDim.x * THREADS);
}

// ---- host ------------------------------------------------------------------------------
template <typename T, bool ALIGNED, int LANES, int CHUNKS>
int launch_norm(const void* x, const void* r, void* h, const NormParams& p, cudaStream_t s) {
    const uint32_t per = LANES == 32 ? 8 : 1;
    return launch_k(rms_norm_mx_kernel<T, ALIGNED, LANES, CHUNKS>, dim3((p.rows + per - 1) / per),
                    dim3(LANES == 32 ? 256 : LANES), 0, s, static_cast<const T*>(x),
                    static_cast<const T*>(r), static_cast<T*>(h), p);
}

constexpr uint32_t RING_BUDGET = 100 * 1024;         // two blocks an SM

template <typename T, int LANES>
bool ring_fits(const NormParams& p, bool res, uint32_t budget, int& stages) {
    constexpr uint32_t TEAMS = LANES < 256 ? 256 / LANES : 1;
    const uint64_t stage = ((uint64_t)p.K * sizeof(T) + 127) / 128 * 128 * (res ? 2 : 1);
    const uint64_t fit = (budget - RING_HEAD) / (stage * TEAMS);
    stages = (int)(fit > RING_MAX ? RING_MAX : fit);
    return stages >= 2;
}
template <typename T, int LANES>
int launch_ring(const void* x, const void* r, void* h, const NormParams& p, int stages,
                int per_sm, cudaStream_t s) {
    constexpr uint32_t TEAMS = LANES < 256 ? 256 / LANES : 1;
    const uint32_t half = (p.K * (uint32_t)sizeof(T) + 127) / 128 * 128;
    const size_t smem = RING_HEAD + (size_t)TEAMS * stages * half * (r ? 2 : 1);
    auto k = rms_norm_mx_ring_kernel<T, LANES>;
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    const uint32_t need = (p.rows + TEAMS - 1) / TEAMS, most = 148u * per_sm;
    return launch_k(k, dim3(need < most ? need : most), dim3(LANES < 256 ? 256 : LANES), smem, s,
                    static_cast<const T*>(x), static_cast<const T*>(r), static_cast<T*>(h), p,
                    stages, half);
}

template <typename T>
int run_norm(const void* x, const void* r, void* h, const NormParams& p, cudaStream_t s) {
    const int64_t es = sizeof(T);
    const uint32_t K = p.K;
    const bool one = p.rows == 1;
    const bool aligned = K % 8 == 0 && aligned16(x) && (one || p.ldx * es % 16 == 0) &&
                         (!r || (aligned16(r) && (one || p.ldr * es % 16 == 0))) &&
                         (!h || aligned16(h)) && aligned16(p.weight);
    if (!aligned) {
        if (K <= 1024) return launch_norm<T, false, 32, 4>(x, r, h, p, s);
        if (K <= 8192) return launch_norm<T, false, 256, 4>(x, r, h, p, s);
        return launch_norm<T, false, 1024, 0>(x, r, h, p, s);
    }
    // Few rows (at most one per SM): as many threads as the row has groups of 8, for the shortest
    // chain of loads, sum and stores.
    if (p.rows <= 148) {
        if (K <= 256) return launch_norm<T, true, 32, 1>(x, r, h, p, s);
        if (K <= 2048) return launch_norm<T, true, 256, 1>(x, r, h, p, s);
        if (K <= 4096) return launch_norm<T, true, 512, 1>(x, r, h, p, s);
        if (K <= 8192) return launch_norm<T, true, 1024, 1>(x, r, h, p, s);
        return launch_norm<T, true, 1024, 0>(x, r, h, p, s);
    }
    int st;
    if (ring_fits<T, 32>(p, r, RING_BUDGET, st)) return launch_ring<T, 32>(x, r, h, p, st, 2, s);
    if (ring_fits<T, 128>(p, r, RING_BUDGET, st)) return launch_ring<T, 128>(x, r, h, p, st, 2, s);
    if (ring_fits<T, 256>(p, r, RING_BUDGET, st)) return launch_ring<T, 256>(x, r, h, p, st, 2, s);
    if (ring_fits<T, 512>(p, r, 2 * RING_BUDGET, st)) return launch_ring<T, 512>(x, r, h, p, st, 1, s);
    return launch_norm<T, true, 1024, 0>(x, r, h, p, s);
}

}  // namespace
}  // namespace snnb

using namespace snnb;

extern "C" int snnb_rms_norm_mx(const void* x, int64_t ldx, const void* residual, int64_t ldr,
                                int x_dtype, const void* weight, int weight_dtype, float eps,
                                int64_t rows, int64_t K, int fmt, void* data, void* scales,
                                void* h_out, snnb_stream_t stream) {
    if (const int inj = take_injected_status()) return inj;
    if (x_dtype != SNNB_F32 && x_dtype != SNNB_F16 && x_dtype != SNNB_BF16) return SNNB_ERR_ARG;
    if (weight_dtype != x_dtype && weight_dtype != SNNB_F32) return SNNB_ERR_ARG;
    if (fmt != SNNB_MXFP4 && fmt != SNNB_MXFP8) return SNNB_ERR_ARG;
    if (!mx::sizes_ok(rows, K) || !mx::stride_ok(rows, ldx) || !mx::stride_ok(rows, ldr) ||
        !(eps >= 0.0f))
        return SNNB_ERR_ARG;
    if (rows == 0) return SNNB_OK;
    if (!x || !weight || !data || !scales || !aligned16(data) || !aligned16(scales))
        return SNNB_ERR_ARG;
    const uintptr_t es = x_dtype == SNNB_F32 ? 4 : 2, ws = weight_dtype == SNNB_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(x) % es || reinterpret_cast<uintptr_t>(residual) % es ||
        reinterpret_cast<uintptr_t>(h_out) % es || reinterpret_cast<uintptr_t>(weight) % ws)
        return SNNB_ERR_ARG;
    NormParams p = {};
    p.status = device_status_ptr();
    if (!p.status) return SNNB_ERR_CUDA;
    p.weight = weight;
    p.w_f32 = weight_dtype == SNNB_F32;
    p.fmt = fmt;
    p.eps = eps;
    p.inv_k = 1.0 / (double)K;
    p.rows = (uint32_t)rows;
    p.K = (uint32_t)K;
    p.nb = (uint32_t)mx::blocks_of(K);
    p.groups = (uint32_t)mx::groups_of(K);
    p.ldx = ldx;
    p.ldr = ldr;
    p.data = static_cast<uint8_t*>(data);
    p.scales = static_cast<uint32_t*>(scales);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (x_dtype == SNNB_F32) return run_norm<float>(x, residual, h_out, p, s);
    if (x_dtype == SNNB_F16) return run_norm<__half>(x, residual, h_out, p, s);
    return run_norm<__nv_bfloat16>(x, residual, h_out, p, s);
}
