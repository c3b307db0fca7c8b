// Root-mean-square norm of x + residual with a microscaled output (formats: mx.cuh):
//   h = x + residual                        kept in float32; also stored, rounded to x's type
//   y = (h / sqrt(mean(h^2) + eps)) * weight
//   codes, scales = y in E2M1 or E4M3, one scale per 32 values
// The norm is taken of the unrounded sum h, in float32 throughout; the stored h and the codes
// are the only roundings.
//
// A row is held in registers between its two uses (the sum of squares and the output), so x and
// the residual are read once: LANES threads a row, CHUNKS x 8 values a thread, thread t holding
// columns (c * LANES + t) * 8 .. + 7 of chunk c.  Four neighbouring lanes hold one block of 32,
// as in the quantisation kernel.  Rows longer than 1024 threads x 4 chunks hold are read twice
// (the second time mostly from L2).
//
// Bound: HBM for many rows, the latency of one load, one block-wide sum and one store for few.
#include "mx.cuh"

namespace snnb {
namespace {

struct NormParams {
    const void* weight;
    int w_f32;                   // weight is float32 (else of x's type)
    int fmt;
    float eps;
    int64_t rows, K, ldx, ldr;
    uint8_t* data;
    uint32_t* scales;
};

// Sum over the LANES threads of a row: warp shuffles, then one value per warp through shared
// memory, added in warp order by every thread.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* shared) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if (LANES == 32) return v;
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < LANES / 32; ++i) s += shared[i];
    return s;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load_weight(const NormParams& p, int64_t k, int n, float (&w)[8]) {
    if (p.w_f32)
        mx::load8<VEC>(static_cast<const float*>(p.weight) + (n > 0 ? k : 0), n, w);
    else
        mx::load8<VEC>(static_cast<const T*>(p.weight) + (n > 0 ? k : 0), n, w);
}

// One chunk's output: y from h, its codes and scale word.  Every lane of the warp calls.
template <typename T, bool VEC>
__device__ __forceinline__ void emit8(const NormParams& p, int64_t row, int64_t k, int n,
                                      const float (&h)[8], float rstd, int64_t nb,
                                      int64_t groups, int lane) {
    float w[8], y[8];
    load_weight<T, VEC>(p, k, n, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = n > i ? __fmul_rn(__fmul_rn(h[i], rstd), w[i]) : 0.0f;
    const int64_t j = k >> 5;
    const bool inside = row < p.rows && j < nb;
    const int sub = lane & 3;
    uint32_t byte;
    if (p.fmt == SNNB_MXFP4) {
        uint32_t c;
        byte = mx::quantise_block<SNNB_MXFP4>(y, c);
        if (inside) *reinterpret_cast<uint32_t*>(p.data + (row * nb + j) * 16 + sub * 4) = c;
    } else {
        uint2 c;
        byte = mx::quantise_block<SNNB_MXFP8>(y, c);
        if (inside) *reinterpret_cast<uint2*>(p.data + (row * nb + j) * 32 + sub * 8) = c;
    }
    const uint32_t word = mx::join_scales(byte, lane);
    if (row < p.rows && (j >> 2) < groups && (lane & 15) == 0)
        p.scales[mx::scale_word(row, j >> 2, groups)] = word;
}

// h of 8 columns; stores its rounded value where h_out is set.
template <typename T, bool VEC>
__device__ __forceinline__ void take8(const NormParams& p, const T* x, const T* r, int64_t row,
                                      int64_t k, int n, float (&h)[8]) {
    mx::load8<VEC>(x + (n > 0 ? row * p.ldx + k : 0), n, h);
    if (r) {
        float b[8];
        mx::load8<VEC>(r + (n > 0 ? row * p.ldr + k : 0), n, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] += b[i];
    }
}

// CHUNKS == 0: rows of any length, read twice.
template <typename T, bool VEC, int LANES, int CHUNKS>
__global__ void __launch_bounds__(LANES == 32 ? 256 : LANES)
rms_norm_mx_kernel(const T* __restrict__ x, const T* __restrict__ r, T* __restrict__ h_out,
                   const NormParams p) {
    constexpr int THREADS = LANES == 32 ? 256 : LANES;
    __shared__ float shared[32];
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int t = LANES == 32 ? lane : (int)threadIdx.x;
    const int64_t row = LANES == 32 ? (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5)
                                    : (int64_t)blockIdx.x;
    const int64_t nb = mx::blocks_of(p.K), groups = (nb + 3) / 4;
    auto inside = [&](int64_t k) {
        return row < p.rows ? (int)max((int64_t)0, min((int64_t)8, p.K - k)) : 0;
    };
    float sum = 0.0f;
    if constexpr (CHUNKS > 0) {
        float h[CHUNKS][8];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int64_t k = (int64_t)(c * LANES + t) * 8;
            take8<T, VEC>(p, x, r, row, k, inside(k), h[c]);
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int64_t k = (int64_t)(c * LANES + t) * 8;
            const int n = inside(k);
            if (h_out) mx::store8<VEC>(h_out + (n > 0 ? row * p.K + k : 0), n, h[c]);
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s = fmaf(h[c][i], h[c][i], s);
            sum += s;
        }
        sum = row_sum<LANES>(sum, shared);
        const float rstd = 1.0f / sqrtf(sum / (float)p.K + p.eps);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int64_t k = (int64_t)(c * LANES + t) * 8;
            if (c > 0 && (int64_t)(c * LANES + (t & ~31)) * 8 >= groups * 128) break;
            emit8<T, VEC>(p, row, k, inside(k), h[c], rstd, nb, groups, lane);
        }
    } else {
        float h[8];
        for (int64_t k = (int64_t)t * 8; k < p.K; k += LANES * 8) {
            const int n = inside(k);
            take8<T, VEC>(p, x, r, row, k, n, h);
            if (h_out) mx::store8<VEC>(h_out + row * p.K + k, n, h);
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s = fmaf(h[i], h[i], s);
            sum += s;
        }
        sum = row_sum<LANES>(sum, shared);
        const float rstd = 1.0f / sqrtf(sum / (float)p.K + p.eps);
        // whole warps: up to the end of the last group of 4 blocks
        for (int64_t k = (int64_t)t * 8; (k & ~int64_t(255)) < groups * 128; k += LANES * 8) {
            const int n = inside(k);
            take8<T, VEC>(p, x, r, row, k, n, h);
            emit8<T, VEC>(p, row, k, n, h, rstd, nb, groups, lane);
        }
    }
    mx::zero_row_padding(p.scales, p.rows, groups, (int64_t)blockIdx.x * THREADS + threadIdx.x,
                         (int64_t)gridDim.x * THREADS);
}

template <typename T, bool VEC, int LANES, int CHUNKS>
int launch_norm(const void* x, const void* r, void* h, const NormParams& p, cudaStream_t s) {
    const int64_t per = LANES == 32 ? 8 : 1;
    const int64_t grid = (p.rows + per - 1) / per;
    if (grid > 0x7fffffff) return SNNB_ERR_ARG;
    return launch_k(rms_norm_mx_kernel<T, VEC, LANES, CHUNKS>, dim3((unsigned)grid),
                    dim3(LANES == 32 ? 256 : LANES), 0, s, static_cast<const T*>(x),
                    static_cast<const T*>(r), static_cast<T*>(h), p);
}

// Threads per row and values per thread.  Many rows: enough values a thread that a row's loads
// overlap and its sum is a small part.  Few rows (at most one per SM): as many threads as the
// row has groups of 8, for the shortest chain.
template <typename T, bool VEC>
int pick_norm(const void* x, const void* r, void* h, const NormParams& p, cudaStream_t s) {
    const int64_t K = p.K;
    const bool few = p.rows <= 148;
    if (K <= 256) return launch_norm<T, VEC, 32, 1>(x, r, h, p, s);
    if (K <= 512 && !few) return launch_norm<T, VEC, 32, 2>(x, r, h, p, s);
    if (K <= 1024 && !few) return launch_norm<T, VEC, 32, 4>(x, r, h, p, s);
    if (K <= 2048 && few) return launch_norm<T, VEC, 256, 1>(x, r, h, p, s);
    if (K <= 4096 && few) return launch_norm<T, VEC, 512, 1>(x, r, h, p, s);
    if (K <= 8192 && few) return launch_norm<T, VEC, 1024, 1>(x, r, h, p, s);
    if (K <= 4096) return launch_norm<T, VEC, 128, 4>(x, r, h, p, s);
    if (K <= 8192) return launch_norm<T, VEC, 256, 4>(x, r, h, p, s);
    if (K <= 16384) return launch_norm<T, VEC, 512, 4>(x, r, h, p, s);
    if (K <= 32768) return launch_norm<T, VEC, 1024, 4>(x, r, h, p, s);
    return launch_norm<T, VEC, 1024, 0>(x, r, h, p, s);
}

template <typename T>
int run_norm(const void* x, const void* r, void* h, const NormParams& p, cudaStream_t s) {
    const int64_t es = sizeof(T);
    const bool vec = p.K % 8 == 0 && aligned16(x) && p.ldx * es % 16 == 0 &&
                     (!r || (aligned16(r) && p.ldr * es % 16 == 0)) && (!h || aligned16(h)) &&
                     aligned16(p.weight);
    return vec ? pick_norm<T, true>(x, r, h, p, s) : pick_norm<T, false>(x, r, h, p, s);
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
    const int64_t limit = int64_t(1) << 40;
    if (rows < 0 || K < 1 || K > 0x7fffffff || rows > limit / K || ldx < 0 || ldr < 0 ||
        (rows > 1 && (ldx > limit / rows || ldr > limit / rows)) || !(eps >= 0.0f))
        return SNNB_ERR_ARG;
    if (rows == 0) return SNNB_OK;
    if (!x || !weight || !data || !scales || !aligned16(data) || !aligned16(scales))
        return SNNB_ERR_ARG;
    const uintptr_t es = x_dtype == SNNB_F32 ? 4 : 2, ws = weight_dtype == SNNB_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(x) % es || reinterpret_cast<uintptr_t>(residual) % es ||
        reinterpret_cast<uintptr_t>(h_out) % es || reinterpret_cast<uintptr_t>(weight) % ws)
        return SNNB_ERR_ARG;
    NormParams p = {};
    p.weight = weight;
    p.w_f32 = weight_dtype == SNNB_F32;
    p.fmt = fmt;
    p.eps = eps;
    p.rows = rows; p.K = K; p.ldx = ldx; p.ldr = ldr;
    p.data = static_cast<uint8_t*>(data);
    p.scales = static_cast<uint32_t*>(scales);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (x_dtype == SNNB_F32) return run_norm<float>(x, residual, h_out, p, s);
    if (x_dtype == SNNB_F16) return run_norm<__half>(x, residual, h_out, p, s);
    return run_norm<__nv_bfloat16>(x, residual, h_out, p, s);
}
