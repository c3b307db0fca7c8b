// Product of microscaled operands (formats: mx.cuh): out[r, n] = sum_k a[r, k] w[n, k] + bias[n],
// a in E4M3 or E2M1, w in E2M1.  Float32 products and sums, rounded once to out's type.
//
// Simple form: 64 x 64 outputs a CTA, both operands' values of one block of 32 staged in shared
// memory, 4 x 4 outputs a thread.
#include "mx.cuh"

namespace snnb {
namespace {

constexpr int T = 64;

template <int FMT>
__device__ __forceinline__ void stage(const uint8_t* data, const uint8_t* scales, int64_t rows,
                                      int64_t r0, int64_t j, int64_t nb, int64_t groups,
                                      float (*dst)[T + 1]) {
    using F = mx::Fmt<FMT>;
    using Codes = typename F::Codes8;
    const int r = threadIdx.x >> 2, sub = threadIdx.x & 3;
    const int64_t row = r0 + r;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (row < rows) {
        const Codes c = *reinterpret_cast<const Codes*>(data + (row * nb + j) * F::BLOCK_BYTES +
                                                        sub * sizeof(Codes));
        mx::decode8(c, v);
        const float s = mx::scale_value(scales[mx::scale_word(row, j >> 2, groups) * 4 + (j & 3)]);
        for (int i = 0; i < 8; ++i) v[i] *= s;
    }
    for (int i = 0; i < 8; ++i) dst[sub * 8 + i][r] = v[i];
}

template <int FMT, typename O>
__global__ void __launch_bounds__(256)
mx_linear_kernel(const uint8_t* a, const uint8_t* as, int64_t rows, int64_t K, const uint8_t* w,
                 const uint8_t* ws, int64_t N, const float* bias, O* out) {
    __shared__ float A[32][T + 1], W[32][T + 1];
    pdl_wait();
    pdl_trigger();
    const int64_t nb = mx::blocks_of(K), groups = (nb + 3) / 4;
    const int64_t r0 = (int64_t)blockIdx.y * T, n0 = (int64_t)blockIdx.x * T;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (int64_t j = 0; j < nb; ++j) {
        stage<FMT>(a, as, rows, r0, j, nb, groups, A);
        stage<SNNB_MXFP4>(w, ws, N, n0, j, nb, groups, W);
        __syncthreads();
        for (int k = 0; k < 32; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    acc[i][c] = fmaf(A[k][ty + 16 * i], W[k][tx + 16 * c], acc[i][c]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int c = 0; c < 4; ++c) {
            const int64_t r = r0 + ty + 16 * i, n = n0 + tx + 16 * c;
            if (r < rows && n < N)
                mx::round_to(acc[i][c] + (bias ? bias[n] : 0.0f), out + r * N + n);
        }
}

template <int FMT, typename O>
int run(const void* a, const void* as, int64_t rows, int64_t K, const void* w, const void* ws,
        int64_t N, const float* bias, void* out, cudaStream_t s) {
    const int64_t gy = (rows + T - 1) / T;
    if (gy > 65535) return SNNB_ERR_ARG;
    return launch_k(mx_linear_kernel<FMT, O>, dim3((unsigned)((N + T - 1) / T), (unsigned)gy),
                    dim3(256), 0, s, static_cast<const uint8_t*>(a),
                    static_cast<const uint8_t*>(as), rows, K, static_cast<const uint8_t*>(w),
                    static_cast<const uint8_t*>(ws), N, bias, static_cast<O*>(out));
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
#define SNNB_MXL(fmt)                                                                            \
    if (a_fmt == fmt) {                                                                          \
        if (out_dtype == SNNB_F32)                                                               \
            return run<fmt, float>(a, a_scales, rows, K, w, w_scales, N, bias, out, s);          \
        if (out_dtype == SNNB_F16)                                                               \
            return run<fmt, __half>(a, a_scales, rows, K, w, w_scales, N, bias, out, s);         \
        return run<fmt, __nv_bfloat16>(a, a_scales, rows, K, w, w_scales, N, bias, out, s);      \
    }
    SNNB_MXL(SNNB_MXFP4)
    SNNB_MXL(SNNB_MXFP8)
#undef SNNB_MXL
    return SNNB_ERR_ARG;
}
