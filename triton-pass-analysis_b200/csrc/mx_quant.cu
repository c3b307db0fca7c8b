// Quantisation to the microscaled formats and back (formats and layout: mx.cuh).
//
// Four neighbouring lanes hold one block of 32 values, 8 each: a 16-byte load of bf16 per lane,
// the block's largest magnitude by two shuffles, one hardware conversion per pair of elements,
// and the codes of a warp's 8 blocks as one contiguous store.  A row is padded to whole groups
// of 4 blocks, so that the 16 lanes of a group join their scale bytes into the one word that
// the group has in the scale layout.  The blocks of the whole tensor are numbered through, so
// short rows fill a warp as well as long ones do.
//
// Bound: HBM.  Every value is read once, its code written once; nothing is read again.
#include "mx.cuh"

namespace snnb {

int* device_status_ptr();

namespace {

constexpr int Q_THREADS = 256;
constexpr int Q_UNROLL = 4;                      // blocks per lane group in flight

template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(Q_THREADS)
mx_quantize_kernel(const T* __restrict__ x, int64_t rows, int64_t K, int64_t ldx,
                   uint8_t* __restrict__ data, uint32_t* __restrict__ scales) {
    using F = mx::Fmt<FMT>;
    using Codes = typename F::Codes8;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t nb = mx::blocks_of(K), groups = (nb + 3) / 4;
    const int64_t thread = (int64_t)blockIdx.x * Q_THREADS + threadIdx.x;
    const int64_t threads = (int64_t)gridDim.x * Q_THREADS;
    const int sub = lane & 3;
    mx::BlockWalk w(thread >> 2, threads >> 2, groups * 4);
    // the 32 lanes of a warp leave together: the loop ends on the warp's first block
    mx::BlockWalk first(thread >> 5 << 3, threads >> 2, groups * 4);
    while (first.row < rows) {
        float v[Q_UNROLL][8];
        int64_t row[Q_UNROLL], j[Q_UNROLL];
#pragma unroll
        for (int u = 0; u < Q_UNROLL; ++u) {
            row[u] = w.row;
            j[u] = w.j;
            const int64_t k = w.j * 32 + sub * 8;
            const int n = w.row < rows ? (int)max((int64_t)0, min((int64_t)8, K - k)) : 0;
            mx::load8<VEC>(x + (n > 0 ? w.row * ldx + k : 0), n, v[u]);
            w.next();
            first.next();
        }
#pragma unroll
        for (int u = 0; u < Q_UNROLL; ++u) {
            Codes c;
            const uint32_t byte = mx::quantise_block<FMT>(v[u], c);
            const uint32_t word = mx::join_scales(byte, lane);
            if (row[u] < rows) {
                if (j[u] < nb)
                    *reinterpret_cast<Codes*>(data + (row[u] * nb + j[u]) * F::BLOCK_BYTES +
                                              sub * sizeof(Codes)) = c;
                if ((lane & 15) == 0)
                    scales[mx::scale_word(row[u], j[u] >> 2, groups)] = word;
            }
        }
    }
    mx::zero_row_padding(scales, rows, groups, thread, threads);
}

template <typename T, int FMT, bool VEC>
__global__ void __launch_bounds__(Q_THREADS)
mx_dequantize_kernel(const uint8_t* __restrict__ data, const uint32_t* __restrict__ scales,
                     int64_t rows, int64_t K, T* __restrict__ out) {
    using F = mx::Fmt<FMT>;
    using Codes = typename F::Codes8;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t nb = mx::blocks_of(K), groups = (nb + 3) / 4;
    const int64_t thread = (int64_t)blockIdx.x * Q_THREADS + threadIdx.x;
    const int64_t threads = (int64_t)gridDim.x * Q_THREADS;
    const int sub = lane & 3;
    mx::BlockWalk w(thread >> 2, threads >> 2, nb);
    while (w.row < rows) {
        Codes c[Q_UNROLL];
        uint32_t word[Q_UNROLL];
        int64_t row[Q_UNROLL], j[Q_UNROLL];
#pragma unroll
        for (int u = 0; u < Q_UNROLL; ++u) {
            row[u] = w.row;
            j[u] = w.j;
            if (w.row < rows) {
                c[u] = __ldg(reinterpret_cast<const Codes*>(
                    data + (w.row * nb + w.j) * F::BLOCK_BYTES + sub * sizeof(Codes)));
                word[u] = __ldg(scales + mx::scale_word(w.row, w.j >> 2, groups));
            }
            w.next();
        }
#pragma unroll
        for (int u = 0; u < Q_UNROLL; ++u) {
            if (row[u] >= rows) continue;
            float v[8];
            mx::decode8(c[u], v);
            const float s = mx::scale_value((word[u] >> (8 * (j[u] & 3))) & 255u);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= s;
            const int64_t k = j[u] * 32 + sub * 8;
            const int n = (int)max((int64_t)0, min((int64_t)8, K - k));
            mx::store8<VEC>(out + row[u] * K + k, n, v);
        }
    }
}

// Blocks for `quads` lane groups of 4, a full round of resident blocks at most (8 of 256
// threads per SM).
unsigned grid_for(int64_t quads) {
    const int64_t need = (quads * 4 + Q_THREADS - 1) / Q_THREADS;
    return (unsigned)(need < 1 ? 1 : (need > 148 * 8 ? 148 * 8 : need));
}

template <typename T, int FMT>
int run_quantize(const void* x, int64_t rows, int64_t K, int64_t ldx, void* data, void* scales,
                 cudaStream_t s) {
    const bool vec = K % 8 == 0 && aligned16(x) && ldx * (int64_t)sizeof(T) % 16 == 0;
    const unsigned grid = grid_for(rows * mx::groups_of(K) * 4);
    auto k = vec ? mx_quantize_kernel<T, FMT, true> : mx_quantize_kernel<T, FMT, false>;
    return launch_k(k, dim3(grid), dim3(Q_THREADS), 0, s, static_cast<const T*>(x), rows, K, ldx,
                    static_cast<uint8_t*>(data), static_cast<uint32_t*>(scales));
}

template <typename T, int FMT>
int run_dequantize(const void* data, const void* scales, int64_t rows, int64_t K, void* out,
                   cudaStream_t s) {
    const bool vec = K % 8 == 0 && aligned16(out);
    const unsigned grid = grid_for(rows * mx::blocks_of(K));
    auto k = vec ? mx_dequantize_kernel<T, FMT, true> : mx_dequantize_kernel<T, FMT, false>;
    return launch_k(k, dim3(grid), dim3(Q_THREADS), 0, s, static_cast<const uint8_t*>(data),
                    static_cast<const uint32_t*>(scales), rows, K, static_cast<T*>(out));
}

}  // namespace
}  // namespace snnb

using namespace snnb;

#define SNNB_MX_DISPATCH(dtype, fmt, fn, ...)                                               \
    switch ((dtype) * 2 + (fmt)) {                                                          \
        case SNNB_F32 * 2 + SNNB_MXFP4: return fn<float, SNNB_MXFP4>(__VA_ARGS__);          \
        case SNNB_F32 * 2 + SNNB_MXFP8: return fn<float, SNNB_MXFP8>(__VA_ARGS__);          \
        case SNNB_F16 * 2 + SNNB_MXFP4: return fn<__half, SNNB_MXFP4>(__VA_ARGS__);         \
        case SNNB_F16 * 2 + SNNB_MXFP8: return fn<__half, SNNB_MXFP8>(__VA_ARGS__);         \
        case SNNB_BF16 * 2 + SNNB_MXFP4: return fn<__nv_bfloat16, SNNB_MXFP4>(__VA_ARGS__); \
        default: return fn<__nv_bfloat16, SNNB_MXFP8>(__VA_ARGS__);                         \
    }

// Largest extents: 2^40 elements a tensor keep every index and byte count far inside 64 bits.
static bool mx_sizes_ok(int64_t rows, int64_t K) {
    return rows >= 0 && K >= 1 && K <= 0x7fffffff && rows <= (int64_t(1) << 40) / K;
}
static bool mx_aligned(const void* data, const void* scales) {
    return aligned16(data) && aligned16(scales);
}

extern "C" int snnb_mx_quantize(const void* x, int x_dtype, int64_t rows, int64_t K, int64_t ldx,
                                int fmt, void* data, void* scales, snnb_stream_t stream) {
    if (const int inj = take_injected_status()) return inj;
    if (x_dtype != SNNB_F32 && x_dtype != SNNB_F16 && x_dtype != SNNB_BF16) return SNNB_ERR_ARG;
    if (fmt != SNNB_MXFP4 && fmt != SNNB_MXFP8) return SNNB_ERR_ARG;
    if (!mx_sizes_ok(rows, K) || ldx < 0 || (rows > 1 && ldx > (int64_t(1) << 40) / rows))
        return SNNB_ERR_ARG;
    if (rows == 0) return SNNB_OK;
    if (!x || !data || !scales || !mx_aligned(data, scales)) return SNNB_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(x) % (x_dtype == SNNB_F32 ? 4 : 2)) return SNNB_ERR_ARG;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    SNNB_MX_DISPATCH(x_dtype, fmt, run_quantize, x, rows, K, ldx, data, scales, s)
}

extern "C" int snnb_mx_dequantize(const void* data, const void* scales, int fmt, int64_t rows,
                                  int64_t K, void* out, int out_dtype, snnb_stream_t stream) {
    if (const int inj = take_injected_status()) return inj;
    if (out_dtype != SNNB_F32 && out_dtype != SNNB_F16 && out_dtype != SNNB_BF16)
        return SNNB_ERR_ARG;
    if (fmt != SNNB_MXFP4 && fmt != SNNB_MXFP8) return SNNB_ERR_ARG;
    if (!mx_sizes_ok(rows, K)) return SNNB_ERR_ARG;
    if (rows == 0) return SNNB_OK;
    if (!out || !data || !scales || !mx_aligned(data, scales)) return SNNB_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(out) % (out_dtype == SNNB_F32 ? 4 : 2)) return SNNB_ERR_ARG;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    SNNB_MX_DISPATCH(out_dtype, fmt, run_dequantize, data, scales, rows, K, out, s)
}
