// Group norm of channels-last tensors x [B, S, C], C in G groups, then an activation:
//
//   y = act((x - mean) / sqrt(var + eps) * weight + bias),
//
// mean and var (biased) over the S * C / G values of a group of a sample.  The variance is that of
// the differences from the mean, in float32, not E[x^2] - mean^2, which a large mean cancels.
#include "common.cuh"
#include "mx.cuh"

namespace snnb {
namespace {

constexpr int GN_THREADS = 256;

template <int ACT>
__device__ __forceinline__ float activate(float y) {
    if (ACT == SNNB_ACT_SILU) return y / (1.0f + expf(-y));
    if (ACT == SNNB_ACT_RELU) return y < 0.0f ? 0.0f : y;      // a NaN stays one
    if (ACT == SNNB_ACT_GELU) return 0.5f * y * (1.0f + erff(y * 0.70710678118654752f));
    return y;
}

__device__ __forceinline__ float block_sum(float v, float* part) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.0f;
    for (int i = 0; i < GN_THREADS / 32; ++i) s += part[i];
    return s;
}

// One thread block per sample and group.
template <typename T, int ACT>
__global__ void __launch_bounds__(GN_THREADS)
group_norm_kernel(const T* __restrict__ x, int64_t xb, int64_t xs, uint32_t S, uint32_t C,
                  uint32_t G, const void* weight, const void* bias, int wf32, float eps, T* y) {
    __shared__ float part[GN_THREADS / 32];
    pdl_wait();
    pdl_trigger();
    const uint32_t b = blockIdx.x / G, g = blockIdx.x - b * G, cg = C / G;
    const uint64_t count = (uint64_t)S * cg;
    const T* in = x + b * xb + g * cg;
    T* out = y + (uint64_t)b * S * C + g * cg;
    float sum = 0.0f;
    for (uint64_t i = threadIdx.x; i < count; i += GN_THREADS)
        sum += to_f32(in[(int64_t)(i / cg) * xs + i % cg]);
    const float mean = block_sum(sum, part) / (float)count;
    float sq = 0.0f;
    for (uint64_t i = threadIdx.x; i < count; i += GN_THREADS) {
        const float v = to_f32(in[(int64_t)(i / cg) * xs + i % cg]) - mean;
        sq += v * v;
    }
    const float r = 1.0f / sqrtf(block_sum(sq, part) / (float)count + eps);
    for (uint64_t i = threadIdx.x; i < count; i += GN_THREADS) {
        const uint32_t row = (uint32_t)(i / cg), c = (uint32_t)(i % cg);
        float v = (to_f32(in[(int64_t)row * xs + c]) - mean) * r;
        const uint32_t ch = g * cg + c;
        if (weight)
            v *= wf32 ? static_cast<const float*>(weight)[ch] : to_f32(static_cast<const T*>(weight)[ch]);
        if (bias)
            v += wf32 ? static_cast<const float*>(bias)[ch] : to_f32(static_cast<const T*>(bias)[ch]);
        mx::round_to(activate<ACT>(v), out + (uint64_t)row * C + c);
    }
}

template <typename T, int ACT>
int run(const void* x, int64_t xb, int64_t xs, int64_t B, int64_t S, int64_t C, int64_t G,
        const void* w, const void* bias, int wf32, float eps, void* y, cudaStream_t s) {
    return launch_k(group_norm_kernel<T, ACT>, dim3((unsigned)(B * G)), dim3(GN_THREADS), 0, s,
                    static_cast<const T*>(x), xb, xs, (uint32_t)S, (uint32_t)C, (uint32_t)G, w,
                    bias, wf32, eps, static_cast<T*>(y));
}

}  // namespace
}  // namespace snnb

using namespace snnb;

#define SNNB_GN_ACT(T, ...)                                          \
    switch (act) {                                                   \
        case SNNB_ACT_NONE: return run<T, SNNB_ACT_NONE>(__VA_ARGS__); \
        case SNNB_ACT_SILU: return run<T, SNNB_ACT_SILU>(__VA_ARGS__); \
        case SNNB_ACT_RELU: return run<T, SNNB_ACT_RELU>(__VA_ARGS__); \
        default: return run<T, SNNB_ACT_GELU>(__VA_ARGS__);            \
    }

extern "C" int snnb_group_norm_act(const void* x, int64_t x_batch_stride, int64_t x_row_stride,
                                   int dtype, int64_t B, int64_t S, int64_t C, int64_t groups,
                                   const void* weight, const void* bias, int weight_dtype,
                                   float eps, int act, void* out, snnb_stream_t stream) {
    if (const int inj = take_injected_status()) return inj;
    if (dtype != SNNB_F32 && dtype != SNNB_F16 && dtype != SNNB_BF16) return SNNB_ERR_ARG;
    if (weight_dtype != SNNB_F32 && weight_dtype != dtype) return SNNB_ERR_ARG;
    if (act < SNNB_ACT_NONE || act > SNNB_ACT_GELU || !(eps >= 0.0f)) return SNNB_ERR_ARG;
    if (B < 0 || S < 0 || C < 1 || groups < 1 || C % groups) return SNNB_ERR_ARG;
    if (B > 0x7fffffff || S > 0x7fffffff || C > 0x7fffff || B * groups > 0x7fffffff)
        return SNNB_ERR_ARG;
    if (B == 0 || S == 0) return SNNB_OK;
    if (!x || !out || B > (int64_t(1) << 40) / S / C) return SNNB_ERR_ARG;
    const int size = dtype == SNNB_F32 ? 4 : 2, wsize = weight_dtype == SNNB_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(out) % size ||
        reinterpret_cast<uintptr_t>(weight) % wsize || reinterpret_cast<uintptr_t>(bias) % wsize)
        return SNNB_ERR_ARG;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int wf32 = weight_dtype == SNNB_F32;
#define SNNB_GN_ARGS x, x_batch_stride, x_row_stride, B, S, C, groups, weight, bias, wf32, eps, out, s
    if (dtype == SNNB_F32) { SNNB_GN_ACT(float, SNNB_GN_ARGS) }
    if (dtype == SNNB_F16) { SNNB_GN_ACT(__half, SNNB_GN_ARGS) }
    SNNB_GN_ACT(__nv_bfloat16, SNNB_GN_ARGS)
}
