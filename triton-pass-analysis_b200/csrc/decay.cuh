// Arguments of the decay attention's kernels (formulas: decay.cu).
#pragma once

#include "common.cuh"
#include "mx.cuh"

namespace snnb {
namespace decay {

constexpr int MAX_DIM = 256;       // of a head's keys and of its values
// Tokens of a sequence: the exponents below, whole chunks of them, are 32 bits (a negative one would
// not end).
constexpr int64_t MOST_TOKENS = 0x7fffff00;

struct Args {
    const void *q, *k, *v;         // [B, N, H or Hk, dk or dv], unit column stride
    void* out;                     // [B, N, H, dv] contiguous
    int64_t qs[3], ks[3], vs[3];   // strides of batch, token, head in elements
    int64_t B, N, H, Hk;
    int dk, dv;
    const float* decay;            // [H]
    float scale;
    const float* state_in;         // [B, H, dk, dv]
    float* state_out;
    const void* lengths;           // [B] int32 (lengths_dtype 0) or int64 (1)
    int lengths_dtype;

    // Tokens of sequence b, within [0, N].
    __device__ __forceinline__ int64_t length(int64_t b) const {
        if (!lengths) return N;
        const int64_t n = lengths_dtype ? static_cast<const int64_t*>(lengths)[b]
                                        : (int64_t) static_cast<const int32_t*>(lengths)[b];
        return n < 0 ? 0 : n > N ? N : n;
    }
};

// base^n for whole 0 <= n < 2^31, with 0^0 = 1, by squaring in float64: powers compound over the
// chunks.
__device__ __forceinline__ double power(float base, int n) {
    double r = 1.0, x = base;
#pragma unroll 1
    for (; n; n >>= 1, x *= x)
        if (n & 1) r *= x;
    return r;
}

// Allows `kernel` `bytes` of shared memory, once per device.
template <auto kernel>
int allow_smem(int bytes) {
    static bool done[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (dev >= 0 && dev < 64 && done[dev]) return SNNB_OK;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (dev >= 0 && dev < 64) done[dev] = true;
    return SNNB_OK;
}

// The tensor cores' form (decay_tc.cu): whether it takes these arguments, the workspace that it may
// need for them, and its launches.
bool tc_takes(const Args& a, int dtype);
int64_t tc_workspace(int dtype, int64_t B, int64_t N, int64_t H, int64_t dk, int64_t dv);
int tc_run(const Args& a, int dtype, void* work, int64_t bytes, cudaStream_t s);

}  // namespace decay
}  // namespace snnb
