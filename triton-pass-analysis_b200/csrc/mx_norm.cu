// Root-mean-square norm of x + residual with a microscaled output (formats: mx.cuh):
//   h = x + residual                        float32; also stored, rounded to x's type
//   y = (h / sqrt(mean(h^2) + eps)) * weight
//   codes, scales = y in E2M1 or E4M3, one scale per 32 values
//
// Rounding.  The norm is taken of the float32 h, before it is rounded to x's type.  An error of one float32 ulp (6e-8) in y
// already moves ~7e-7 of the codes to a neighbour, so the squares are summed and 1 / sqrt is
// taken in float64.  y itself is float32 unless it lies within 4 ulp of a value that a code
// boundary could be (its low 19 bits zero: 3 mantissa bits and the half step), where it is formed
// again in float64 and rounded to odd, which keeps it on its side of the boundary.
//
// Two forms.  Many aligned rows of more than 1024 values: a team of LANES threads walks rows, whose
// x and residual come by bulk copies into a ring in shared memory while earlier rows are worked on.
// Others: teams of one row each, straight from memory.  In both a row's values stay in registers
// between the passes (squares, output); only rows that a team cannot hold are read twice: past 8192
// values where the aligned rows are few, past 16384 (aligned float32 with a residual: 12800)
// elsewhere.  Four neighbouring lanes hold one block of 32, as in the quantisation kernel.
//
// Bound: HBM for many wide aligned rows (16384 x 8192 bf16 with residual 165 us, 5.7 TB/s); for few
// rows the latency of one load, one sum over the block, one store.  Short rows (12544 x 384: 12.3
// us, 2.7 TB/s) wait for loads, as nothing is in flight while a team sums and stores; unaligned
// ones (8192 x 4096 at odd starts: 83 us, 2.8 TB/s) take 55% of the issue slots besides, for the
// shifts.
#include "mx.cuh"
#include "tc_common.cuh"

namespace snnb {
namespace {

struct NormParams {
    int fmt;
    float eps;
    double inv_k;
    uint32_t rows, K, nb, groups;
    int64_t ldx, ldr;
    uint8_t* data;
    uint32_t* scales;
    int* status;
    int stall;                   // test hook: the ring kernel's block 0 never fetches its second rows
};

__device__ __forceinline__ void add8(float (&a)[8], const float (&b)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2)
        mx::unpack2(mx::add2(mx::pack2(a[i], a[i + 1]), mx::pack2(b[i], b[i + 1])), a[i], a[i + 1]);
}
// Sum over aligned groups of LANES lanes of a warp.
template <int LANES>
__device__ __forceinline__ double lanes_sum(double v) {
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
// Sum of N x 8 squares, as if in float64 (~2^-40).  Two float32 sums start at a power of two M
// above all they will reach: t = fl(a a + s) is then a multiple of M 2^-23, s - t is exact, and
// fl(a a + (s - t)) is what t lost, summed apart; 4 operations for two squares (converting every
// value to float64 took 27 us more of a 16384 x 8192 launch's 197).  Values whose squares leave
// float32's range, infinities and NaN go through float64.
template <int N>
__device__ __forceinline__ double squares(const float (&h)[N][8]) {
    float m = 0.0f;
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
        for (int i = 0; i < 8; i += 2) m = mx::max_abs3(m, h[c][i], h[c][i + 1]);
    if (m == 0.0f) return 0.0;
    if (!(m > 1e-15f && m < 1e15f)) {
        double d = 0.0;
        for (int c = 0; c < N; ++c)
            for (int i = 0; i < 8; ++i) d = fma((double)h[c][i], (double)h[c][i], d);
        return d;
    }
    // 4 N squares a sum, each below 2^(2 e + 2) for e the exponent of m
    constexpr int UP = N <= 1 ? 5 : N <= 2 ? 6 : 7;
    const int e = (int)((uint32_t)__float_as_int(m) >> 23) - 127;
    const float M = __int_as_float((2 * e + UP + 127) << 23);
    const uint64_t minus = mx::pack2(-1.0f, -1.0f);
    uint64_t s = mx::pack2(M, M), lost = mx::pack2(0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const uint64_t a = mx::pack2(h[c][i], h[c][i + 1]);
            const uint64_t t = mx::fma2(a, a, s);
            lost = mx::add2(lost, mx::fma2(a, a, mx::fma2(t, minus, s)));
            s = t;
        }
    float s0, s1, l0, l1;
    mx::unpack2(s, s0, s1);
    mx::unpack2(lost, l0, l1);
    return (double)(s0 - M) + (double)(s1 - M) + (double)(l0 + l1);
}
// 1 / sqrt(sum / K + eps): one Newton step in float64 on the float32 approximation (2^-22, so
// ~2^-44 after it).
__device__ __forceinline__ double rstd_of(const NormParams& p, double sum) {
    const double m = fma(sum, p.inv_k, (double)p.eps);
    if (!(m > 1e-30 && m < 1e37)) return rsqrt(m);
    const double r = (double)rsqrtf((float)m);
    return fma(0.5 * r, fma(-m * r, r, 1.0), r);
}

// y of 8 values (see the top); values past n, whose h and w are 0, give 0.
__device__ __forceinline__ void normed8(const float (&h)[8], const float (&w)[8], float rstd,
                                        double rstd64, float (&y)[8]) {
    // two values' low halves at once (a carry out of the lower one only comes from a value that
    // is near itself)
    const uint64_t rr = mx::pack2(rstd, rstd);
    uint32_t pairs = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        mx::unpack2(mx::mul2(mx::mul2(mx::pack2(h[i], h[i + 1]), rr), mx::pack2(w[i], w[i + 1])), y[i],
                    y[i + 1]);
        pairs = __vminu2(pairs, __byte_perm((uint32_t)__float_as_int(y[i]),
                                            (uint32_t)__float_as_int(y[i + 1]), 0x5410) + 0x00040004u);
    }
    const uint32_t near = min(pairs & 0xffffu, pairs >> 16);
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

// Where a row's codes and scale words go (nullptr: nowhere).
struct RowOut {
    uint8_t* data;
    uint32_t* scales;
    __device__ __forceinline__ RowOut(const NormParams& p, uint32_t row, bool in_row) {
        data = in_row ? p.data + (uint64_t)(row * p.nb) * (p.fmt == SNNB_MXFP4 ? 16 : 32) : nullptr;
        scales = p.scales + mx::scale_word(row, 0, p.groups);
    }
};
// Codes and scale word of 8 values at column k of a row.  Every lane of the warp calls.
template <int LANES = 32>
__device__ __forceinline__ void emit8(const NormParams& p, const RowOut& o, uint32_t k,
                                      const float (&y)[8], int lane) {
    const uint32_t j = k >> 5;
    const bool inside = o.data && j < p.nb;
    const uint32_t e = mx::top_exponent(y);
    uint32_t byte;
    if (p.fmt == SNNB_MXFP4) {
        uint32_t c;
        byte = mx::quantise_block<SNNB_MXFP4>(y, e, c);
        if (inside) *reinterpret_cast<uint32_t*>(o.data + k / 2) = c;
    } else {
        uint2 c;
        byte = mx::quantise_block<SNNB_MXFP8>(y, e, c);
        if (inside) *reinterpret_cast<uint2*>(o.data + k) = c;
    }
    const uint32_t word = mx::join_scales<LANES>(byte, lane);
    if (o.data && (j >> 2) < p.groups && (lane & (LANES < 16 ? 7 : 15)) == 0)
        o.scales[(j >> 2) * (mx::GROUP_BYTES / 4)] = word;
}

// ---- rows through registers --------------------------------------------------------------
template <typename T, bool ALIGNED>
__device__ __forceinline__ void take8(const NormParams& p, const T* x, const T* r, uint32_t row,
                                      uint32_t k, int n, mx::RowEnds xs, mx::RowEnds rs,
                                      float (&h)[8]) {
    mx::Raw8<T> a = mx::zero8<T>();
    const T* xr = x + (int64_t)row * p.ldx;
    if (n > 0) a = ALIGNED ? mx::load_aligned8(xr + k) : mx::load_any8(xr, k, p.K, xs);
    mx::to_floats(a, h);
    if (r) {
        mx::Raw8<T> b = mx::zero8<T>();
        const T* rr = r + (int64_t)row * p.ldr;
        if (n > 0) b = ALIGNED ? mx::load_aligned8(rr + k) : mx::load_any8(rr, k, p.K, rs);
        float f[8];
        mx::to_floats(b, f);
        add8(h, f);
    }
}
template <typename T, bool ALIGNED, int LANES>
__device__ __forceinline__ void put_h8(const NormParams& p, T* h_out, uint32_t row, uint32_t k,
                                       int n, const float (&h)[8], int lane) {
    mx::Raw8<T> o;
    mx::from_floats(h, o);
    T* q = h_out + (n > 0 ? (uint64_t)row * p.K + k : 0);
    if (!ALIGNED) mx::store_any8<T, LANES < 32 ? LANES : 32>(q, n, o, lane);
    else if (n > 0) mx::store_aligned8(q, o);
}

template <typename W>
__device__ __forceinline__ mx::Raw8<W> weights8(const NormParams& p, const W* weight, uint32_t k) {
    if (k >= p.K) return mx::zero8<W>();
    if (k + 8 > p.K || (reinterpret_cast<uintptr_t>(weight) & 15)) return mx::load_any8(weight, k, p.K);
    mx::Raw8<W> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(W) / 2; ++i)
        r.v[i] = __ldg(reinterpret_cast<const uint4*>(weight + k) + i);
    return r;
}

// LANES threads a row, CHUNKS x 8 values a thread: thread t holds columns (c * LANES + t) * 8 ..
// + 7 of chunk c.  CHUNKS == 0: rows of any length, read twice.
constexpr int direct_threads(int lanes) { return lanes <= 32 ? 256 : lanes; }
template <typename T, typename W, bool ALIGNED, int LANES, int CHUNKS>
__global__ void __launch_bounds__(direct_threads(LANES))
rms_norm_mx_kernel(const T* __restrict__ x, const T* __restrict__ r, T* __restrict__ h_out,
                   const W* __restrict__ weight, const NormParams p) {
    constexpr uint32_t THREADS = direct_threads(LANES);
    __shared__ double shared[32];
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const uint32_t t = threadIdx.x % LANES;
    const uint32_t row = blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
    const bool in_row = row < p.rows;
    const RowOut out(p, row, in_row);
    mx::RowEnds xs, rs;
    if (!ALIGNED && LANES <= 128 && in_row) {           // longer rows: not worth the tests
        xs = mx::RowEnds(x, p.rows, p.ldx, p.K, row);
        if (r) rs = mx::RowEnds(r, p.rows, p.ldr, p.K, row);
    }
    auto valid = [&](uint32_t k) { return in_row && k < p.K ? (int)min(8u, p.K - k) : 0; };
    // whole warps: a chunk that begins past the row's end is left out
    auto past = [&](uint32_t k, uint32_t end) {
        return (k & ~(uint32_t)(LANES >= 32 ? 255 : LANES * 8 - 1)) >= end;
    };
    auto row_sum = [&](double v) {
        v = lanes_sum<LANES < 32 ? LANES : 32>(v);
        if (LANES <= 32) return v;
        if (lane == 0) shared[threadIdx.x >> 5] = v;
        __syncthreads();
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < LANES / 32; ++i) s += shared[i];
        return s;
    };
    auto finish = [&](uint32_t k, const float (&h)[8], float rstd, double rstd64) {
        float w[8], y[8];
        mx::to_floats(weights8<W>(p, weight, k), w);
        normed8(h, w, rstd, rstd64, y);
        emit8<LANES < 32 ? LANES : 32>(p, out, k, y, lane);
    };
    double sum = 0.0;
    if constexpr (CHUNKS > 0) {
        float h[CHUNKS][8];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t k = (c * LANES + t) * 8;
            take8<T, ALIGNED>(p, x, r, row, k, valid(k), xs, rs, h[c]);
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t k = (c * LANES + t) * 8;
            if (c > 0 && past(k, p.K)) break;
            if (h_out) put_h8<T, ALIGNED, LANES>(p, h_out, row, k, valid(k), h[c], lane);
        }
        sum = squares(h);
        const double rstd64 = rstd_of(p, row_sum(sum));
        const float rstd = (float)rstd64;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t k = (c * LANES + t) * 8;
            if (c > 0 && past(k, p.groups * 128)) break;
            finish(k, h[c], rstd, rstd64);
        }
    } else {
        float h1[1][8];
        float (&h)[8] = h1[0];
        for (uint32_t k = t * 8; !past(k, p.K); k += LANES * 8) {
            const int n = valid(k);
            take8<T, ALIGNED>(p, x, r, row, k, n, xs, rs, h);
            if (h_out) put_h8<T, ALIGNED, LANES>(p, h_out, row, k, n, h, lane);
            sum += squares(h1);
        }
        const double rstd64 = rstd_of(p, row_sum(sum));
        const float rstd = (float)rstd64;
        for (uint32_t k = t * 8; !past(k, p.groups * 128); k += LANES * 8) {
            take8<T, ALIGNED>(p, x, r, row, k, valid(k), xs, rs, h);
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
constexpr int RING_CHUNKS = 4;
constexpr int ring_threads(int lanes) { return lanes < 256 ? 256 : lanes; }
// Resident blocks to compile for: 80 registers a thread, 128 where values or weights are float32.
template <typename T, typename W> constexpr int ring_blocks(int lanes) {
    return (sizeof(T) == 4 || sizeof(W) == 4 ? 512 : 768) / ring_threads(lanes);
}

// Teams of LANES threads; team g of all walks the rows g, g + (number of teams), ...  A ring
// stage holds one row of x and, `half` bytes behind it, of the residual (RES).  A thread holds
// CHUNKS x 8 values of the row in registers, as in rms_norm_mx_kernel, and its columns' weights
// for all rows.
// FULL: K is all that a team holds, so that no value needs a bounds test (8192 x 8192 float32:
// 148 us with the tests, 130 without).
template <typename T, typename W, int LANES, bool RES, bool FULL>
__global__ void __launch_bounds__(ring_threads(LANES), ring_blocks<T, W>(LANES))
rms_norm_mx_ring_kernel(const T* __restrict__ x, const T* __restrict__ r, T* __restrict__ h_out,
                        const W* __restrict__ weight, const NormParams p, int stages,
                        uint32_t half) {
    constexpr int THREADS = ring_threads(LANES), TEAMS = THREADS / LANES, WARPS = LANES / 32;
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31;
    const int team = threadIdx.x / LANES;
    const uint32_t t = threadIdx.x % LANES;
    const uint32_t stage_bytes = half * (RES ? 2 : 1);
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
        tc::mbar_expect_tx(bars + 8 * s, bytes * (RES ? 2u : 1u));
        bulk_load(dst, x + (int64_t)row * p.ldx, bytes, bars + 8 * s);
        if (RES) bulk_load(dst + half, r + (int64_t)row * p.ldr, bytes, bars + 8 * s);
    };
    auto team_sync = [&] {
        if constexpr (LANES == 32) __syncwarp();
        else tc::named_bar_sync(1 + team, LANES);
    };
    if (t == 0)
        for (int s = 0; s < stages; ++s)
            if (row0 + (uint64_t)s * step < p.rows && !(p.stall && blockIdx.x == 0 && s == 1))
                fetch(row0 + s * step, s);
    mx::Raw8<W> w[RING_CHUNKS];
#pragma unroll
    for (int c = 0; c < RING_CHUNKS; ++c) w[c] = weights8<W>(p, weight, (c * LANES + t) * 8);
    uint32_t failed = 0;
    int s = 0;
    uint32_t parity = 0, odd = 0;
    for (uint64_t row64 = row0; row64 < p.rows; row64 += step, odd ^= 1) {
        const uint32_t row = (uint32_t)row64;
        if (!failed && !tc::mbar_wait_warp(bars + 8 * s, parity, 0)) {
            // a wait ran out: this warp works on and stores nothing.  The copies in flight, all of
            // them by the team's first warp, land before the block may exit; a wait of that limit
            // that runs out has outlasted those behind it as well
            failed = 1;
            int fs = s;
            uint32_t fp = parity;
            for (int i = 0; t < 32 && i < stages && row64 + (uint64_t)i * step < p.rows; ++i) {
                if (!tc::mbar_wait_warp<true>(bars + 8 * fs, fp, 0)) break;
                if (++fs == stages) {
                    fs = 0;
                    fp ^= 1;
                }
            }
            if (lane == 0) atomicExch(p.status, SNNB_ERR_TIMEOUT);
        }
        const uint8_t* xs = ring + (size_t)s * stage_bytes;
        T* hr = h_out ? h_out + (uint64_t)row * p.K : nullptr;
        if (failed) hr = nullptr;
        float h[RING_CHUNKS][8];
        double sum;
#pragma unroll
        for (int c = 0; c < RING_CHUNKS; ++c) {
            const uint32_t k = (c * LANES + t) * 8;
            const bool in = FULL || k < p.K;
            mx::to_floats(in ? smem8<T>(xs, k) : mx::zero8<T>(), h[c]);
            if (RES) {
                float f[8];
                mx::to_floats(in ? smem8<T>(xs + half, k) : mx::zero8<T>(), f);
                add8(h[c], f);
            }
            if (hr && in) {
                mx::Raw8<T> o;
                mx::from_floats(h[c], o);
                mx::store_aligned8(hr + k, o);
            }
        }
        sum = lanes_sum<32>(squares(h));
        if constexpr (LANES > 32) {
            if (lane == 0) sums[odd * WARPS + (t >> 5)] = sum;
        }
        team_sync();                                  // sums written, the stage read by all
        const uint64_t next = row64 + (uint64_t)stages * step;
        if (t == 0 && !failed && next < p.rows) fetch((uint32_t)next, s);
        if (++s == stages) {
            s = 0;
            parity ^= 1;
        }
        if constexpr (LANES > 32) {
            sum = 0.0;
#pragma unroll
            for (int i = 0; i < WARPS; ++i) sum += sums[odd * WARPS + i];
        }
        const double rstd64 = rstd_of(p, sum);
        const float rstd = (float)rstd64;
        const RowOut out(p, row, !failed);
#pragma unroll
        for (int c = 0; c < RING_CHUNKS; ++c) {
            const uint32_t k = (c * LANES + t) * 8;
            if (!FULL && c > 0 && (k & ~255u) >= p.groups * 128) break;       // whole warps
            float wf[8], y[8];
            mx::to_floats(w[c], wf);
            normed8(h[c], wf, rstd, rstd64, y);
            emit8(p, out, k, y, lane);
        }
    }
    mx::zero_row_padding(p.scales, p.rows, p.groups, (uint64_t)blockIdx.x * THREADS + threadIdx.x,
                         (uint64_t)gridDim.x * THREADS);
}

// ---- host ------------------------------------------------------------------------------
struct NormArgs {
    const void *x, *r, *weight;
    void* h;
    cudaStream_t s;
};

template <typename T, typename W, bool ALIGNED, int LANES, int CHUNKS>
int launch_norm(const NormArgs& a, const NormParams& p) {
    constexpr uint32_t THREADS = direct_threads(LANES), PER = THREADS / LANES;
    return launch_k(rms_norm_mx_kernel<T, W, ALIGNED, LANES, CHUNKS>,
                    dim3((p.rows + PER - 1) / PER), dim3(THREADS), 0, a.s,
                    static_cast<const T*>(a.x), static_cast<const T*>(a.r), static_cast<T*>(a.h),
                    static_cast<const W*>(a.weight), p);
}

// Shared memory of a ring of two stages sets the blocks per SM (as many as were compiled for at
// most), what that leaves the stages.
constexpr uint32_t RING_SM_BYTES = 224 * 1024;
// Lets `k` use as much shared memory as any ring asks for, once per device.  The setting is the
// kernel's, not the launch's: set to each call's own size, another host thread could lower it
// between this thread's setting and launch.
template <typename Kernel>
int allow_ring(Kernel k, bool (&ready)[64]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (dev < 0 || dev >= 64) return SNNB_ERR_UNSUPPORTED;
    if (__atomic_load_n(&ready[dev], __ATOMIC_ACQUIRE)) return SNNB_OK;
    e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)RING_SM_BYTES);
    if (e != cudaSuccess) return record_cuda_error(e);
    __atomic_store_n(&ready[dev], true, __ATOMIC_RELEASE);
    return SNNB_OK;
}

template <typename T, typename W, int LANES>
int launch_ring(const NormArgs& a, NormParams p) {
    constexpr uint32_t THREADS = ring_threads(LANES), TEAMS = THREADS / LANES;
    constexpr uint32_t BLOCKS = ring_blocks<T, W>(LANES);
    const uint32_t half = (p.K * (uint32_t)sizeof(T) + 127) / 128 * 128;
    const uint32_t stage = TEAMS * half * (a.r ? 2 : 1);
    uint32_t per_sm = RING_SM_BYTES / (2 * stage + RING_HEAD + 1024);
    if (per_sm < 1) return SNNB_ERR_UNSUPPORTED;
    if (per_sm > BLOCKS) per_sm = BLOCKS;
    uint32_t stages = (RING_SM_BYTES / per_sm - RING_HEAD - 1024) / stage;
    if (stages > RING_MAX) stages = RING_MAX;
    const size_t smem = RING_HEAD + (size_t)stages * stage;
    const bool full = p.K == 8 * LANES * RING_CHUNKS;
    auto k = a.r ? full ? rms_norm_mx_ring_kernel<T, W, LANES, true, true>
                        : rms_norm_mx_ring_kernel<T, W, LANES, true, false>
                 : full ? rms_norm_mx_ring_kernel<T, W, LANES, false, true>
                        : rms_norm_mx_ring_kernel<T, W, LANES, false, false>;
    static bool ready[4][64];
    const int rc = allow_ring(k, ready[(a.r ? 2 : 0) + full]);
    if (rc != SNNB_OK) return rc;
    const uint32_t need = (p.rows + TEAMS - 1) / TEAMS, most = 148u * per_sm;
    p.stall = take_injected_stall();
    return launch_k(k, dim3(need < most ? need : most), dim3(THREADS), smem, a.s,
                    static_cast<const T*>(a.x), static_cast<const T*>(a.r), static_cast<T*>(a.h),
                    static_cast<const W*>(a.weight), p, (int)stages, half);
}

template <typename T, typename W>
int run_norm(const NormArgs& a, const NormParams& p) {
    const int64_t es = sizeof(T);
    const uint32_t K = p.K;
    const bool one = p.rows == 1;
    const bool aligned = K % 8 == 0 && aligned16(a.x) && (one || p.ldx * es % 16 == 0) &&
                         (!a.r || (aligned16(a.r) && (one || p.ldr * es % 16 == 0))) &&
                         (!a.h || aligned16(a.h)) && aligned16(a.weight);
    if (!aligned) {
        // a team with as many lanes as the row needs: 63025 x 34 bf16 with residual 13 us (57 with
        // a warp a row), 15646 x 189 11 (16), 34225 x 404 45 (57; float32, 10000 x 500: 23, 21);
        // from 8192 columns on, one read instead of two: 3000 x 16001 123 us (175)
        if (K <= 64) return launch_norm<T, W, false, 8, 1>(a, p);
        if (K <= 128) return launch_norm<T, W, false, 16, 1>(a, p);
        if (K <= 256) return launch_norm<T, W, false, 16, 2>(a, p);
        if (K <= 512 && es == 2) return launch_norm<T, W, false, 16, 4>(a, p);
        if (K <= 1024) return launch_norm<T, W, false, 32, 4>(a, p);
        if (K <= 2048) return launch_norm<T, W, false, 64, 4>(a, p);
        if (K <= 4096) return launch_norm<T, W, false, 128, 4>(a, p);
        if (K <= 8192) return launch_norm<T, W, false, 256, 4>(a, p);
        if (K <= 16384) return launch_norm<T, W, false, 512, 4>(a, p);
        return launch_norm<T, W, false, 1024, 0>(a, p);
    }
    // short rows: the copies of a ring cost more than they hide (57885 x 32 bf16 with residual: 7.1
    // us with 8 lanes a row, 12.8 with 16)
    if (K <= 64) return launch_norm<T, W, true, 8, 1>(a, p);
    if (K <= 128) return launch_norm<T, W, true, 16, 1>(a, p);
    if (K <= 256) return launch_norm<T, W, true, 32, 1>(a, p);
    // Few rows (at most one per SM): as many threads as the row has groups of 8, for the shortest
    // chain of loads, sum and stores.
    if (p.rows <= 148) {
        if (K <= 2048) return launch_norm<T, W, true, 256, 1>(a, p);
        if (K <= 4096) return launch_norm<T, W, true, 512, 1>(a, p);
        if (K <= 8192) return launch_norm<T, W, true, 1024, 1>(a, p);
        return launch_norm<T, W, true, 1024, 0>(a, p);
    }
    // two rows a warp up to 512 (12544 x 384: 12.2 us, 14.8 with one), one up to 1024
    if (K <= 512) return launch_norm<T, W, true, 16, 4>(a, p);
    if (K <= 1024) return launch_norm<T, W, true, 32, 4>(a, p);
    // 32 values a thread; a ring of two rows (and residuals) has to fit the SM
    if (K <= 2048) return launch_ring<T, W, 64>(a, p);
    if (K <= 4096) return launch_ring<T, W, 128>(a, p);
    if (K <= 8192) return launch_ring<T, W, 256>(a, p);
    if (K <= 16384 && (uint64_t)K * es * (a.r ? 2 : 1) <= 100 * 1024)
        return launch_ring<T, W, 512>(a, p);
    return launch_norm<T, W, true, 1024, 0>(a, p);
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
    const NormArgs a = {x, residual, weight, h_out, s};
    if (x_dtype == SNNB_F32) return run_norm<float, float>(a, p);
    if (x_dtype == SNNB_F16)
        return weight_dtype == SNNB_F32 ? run_norm<__half, float>(a, p)
                                        : run_norm<__half, __half>(a, p);
    return weight_dtype == SNNB_F32 ? run_norm<__nv_bfloat16, float>(a, p)
                                    : run_norm<__nv_bfloat16, __nv_bfloat16>(a, p);
}
