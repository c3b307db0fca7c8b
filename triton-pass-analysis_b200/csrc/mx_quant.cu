// Quantisation to the microscaled formats and back (formats and layout: mx.cuh).
//
// Four neighbouring lanes hold one block of 32 values, 8 each: a 16-byte load of bf16 per lane,
// the block's largest exponent by two shuffles, one hardware conversion per pair of elements,
// and the codes of a warp's 8 blocks as one contiguous store.  A row is padded to whole groups
// of 4 blocks, so that the 16 lanes of a group join their scale bytes into the one word that
// the group has in the scale layout.
//
// Rows that are 16-byte aligned: the blocks of the whole tensor are numbered through, so short
// rows fill a warp as well as long ones do.  Others: a warp takes 256 consecutive values of one
// row, through aligned loads (or stores) around them that it shifts into place.
//
// Bound: HBM for aligned rows: every value is read once, its code written once.  Unaligned ones
// (8192 x 4099 bf16 -> E2M1: 26 us, 3.3 TB/s; back 29) are bound by instructions: the shifts leave
// two thirds of the issue slots taken and the integer pipe full.
#include "mx.cuh"

namespace snnb {
namespace {

constexpr int Q_THREADS = 256;

// A thread block takes U x 64 consecutive blocks of 32 (or U x 8 row pieces of 256), so that a
// thread has U loads in flight, and ends: with blocks resident for the whole launch that stride
// through the tensor, 16384 x 8192 bf16 took 69 us (E2M1; 63 in this form) and 68 back (52).
// U is 4 (2 for row pieces), or 1 for tensors too small for four (eight) such blocks an SM.

// FLAT: K % 128 == 0 and contiguous rows, so values and codes lie at their block's index.
template <typename T, int FMT, int U, bool FLAT>
__global__ void __launch_bounds__(Q_THREADS)
mx_quantize_kernel(const T* __restrict__ x, uint32_t rows, uint32_t K, int64_t ldx, uint32_t nb,
                   uint32_t groups, mx::FastDiv per_row, uint32_t total,
                   uint8_t* __restrict__ data, uint32_t* __restrict__ scales) {
    using F = mx::Fmt<FMT>;
    using Codes = typename F::Codes8;
    pdl_wait();
    pdl_trigger();
    const uint32_t lane = threadIdx.x & 31, sub = lane & 3;
    const uint64_t thread = (uint64_t)blockIdx.x * Q_THREADS + threadIdx.x;
    // of this warp; blocks past the last count as zeros
    constexpr uint32_t step = Q_THREADS / 4;
    const uint32_t first = blockIdx.x * (U * step) + (threadIdx.x >> 5) * 8;
    {
        mx::Raw8<T> raw[U];
        uint32_t row[U], j[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t q = first + u * step + (lane >> 2);
            if (FLAT) {
                raw[u] = q < total ? mx::load_aligned8(x + (uint64_t)q * 32 + sub * 8) : mx::zero8<T>();
            } else {
                row[u] = per_row.div(q);
                j[u] = q - row[u] * per_row.d;
                const uint32_t k = j[u] * 32 + sub * 8;
                raw[u] = q < total && k < K ? mx::load_aligned8(x + row[u] * ldx + k) : mx::zero8<T>();
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float v[8];
            mx::to_floats(raw[u], v);
            Codes c;
            const uint32_t byte = mx::quantise_block<FMT>(v, mx::top_exponent(raw[u], v), c);
            const uint32_t word = mx::join_scales(byte, lane);
            const uint32_t q = first + u * step + (lane >> 2);
            if (q >= total) continue;
            if (FLAT) {
                *reinterpret_cast<Codes*>(data + (uint64_t)q * F::BLOCK_BYTES + sub * sizeof(Codes)) = c;
                if ((lane & 15) == 0) {
                    const uint32_t r = per_row.div(q);
                    scales[mx::scale_word(r, (q - r * per_row.d) >> 2, groups)] = word;
                }
            } else {
                if (j[u] < nb)
                    *reinterpret_cast<Codes*>(data + (uint64_t)(row[u] * nb + j[u]) * F::BLOCK_BYTES +
                                              sub * sizeof(Codes)) = c;
                if ((lane & 15) == 0) scales[mx::scale_word(row[u], j[u] >> 2, groups)] = word;
            }
        }
    }
    mx::zero_row_padding(scales, rows, groups, thread, (uint64_t)gridDim.x * Q_THREADS);
}

// LANES threads a piece of 8 LANES values.  total: pieces, per_row.d of them a row (LANES = 8:
// rows of one piece).
template <typename T, int FMT, int U, int LANES>
__global__ void __launch_bounds__(Q_THREADS)
mx_quantize_any_kernel(const T* __restrict__ x, uint32_t rows, uint32_t K, int64_t ldx,
                       uint32_t nb, uint32_t groups, mx::FastDiv per_row, uint32_t total,
                       uint8_t* __restrict__ data, uint32_t* __restrict__ scales) {
    using F = mx::Fmt<FMT>;
    using Codes = typename F::Codes8;
    pdl_wait();
    pdl_trigger();
    const uint32_t lane = threadIdx.x & 31, sub = lane & 3;
    const uint64_t thread = (uint64_t)blockIdx.x * Q_THREADS + threadIdx.x;
    constexpr uint32_t step = Q_THREADS / LANES;
    const uint32_t first = blockIdx.x * (U * step) + threadIdx.x / LANES;
    {
        mx::Raw8<T> raw[U];
        uint32_t row[U], k[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t q = first + u * step;
            row[u] = per_row.div(q);
            k[u] = ((q - row[u] * per_row.d) * LANES + (lane & (LANES - 1))) * 8;
            // short rows are mostly ends; in longer ones the test costs more than it gives
            mx::RowEnds ends;
            if (LANES < 32 && q < total) ends = mx::RowEnds(x, rows, ldx, K, row[u]);
            raw[u] = q < total && k[u] < K ? mx::load_any8(x + row[u] * ldx, k[u], K, ends)
                                           : mx::zero8<T>();
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float v[8];
            mx::to_floats(raw[u], v);
            Codes c;
            const uint32_t byte = mx::quantise_block<FMT>(v, mx::top_exponent(raw[u], v), c);
            const uint32_t word = mx::join_scales<LANES>(byte, lane);
            const uint32_t j = k[u] >> 5;
            if (first + u * step < total) {
                if (j < nb)
                    *reinterpret_cast<Codes*>(data + (uint64_t)(row[u] * nb + j) * F::BLOCK_BYTES +
                                              sub * sizeof(Codes)) = c;
                if ((lane & (LANES < 16 ? 7 : 15)) == 0 && (j >> 2) < groups)
                    scales[mx::scale_word(row[u], j >> 2, groups)] = word;
            }
        }
    }
    mx::zero_row_padding(scales, rows, groups, thread, (uint64_t)gridDim.x * Q_THREADS);
}

template <typename T, int FMT>
__device__ __forceinline__ mx::Raw8<T> decode_scaled(typename mx::Fmt<FMT>::Codes8 c,
                                                     uint32_t byte) {
    float v[8];
    mx::decode8(c, v);
    mx::scale8(v, mx::scale_value(byte), v);
    mx::Raw8<T> r;
    mx::from_floats(v, r);
    return r;
}

// K % 8 == 0 and out 16-byte aligned; FLAT: K % 32 == 0, so values lie at their block's index.
// total: blocks, per_row.d = nb of them a row.
template <typename T, int FMT, int U, bool FLAT>
__global__ void __launch_bounds__(Q_THREADS)
mx_dequantize_kernel(const uint8_t* __restrict__ data, const uint8_t* __restrict__ scales,
                     uint32_t rows, uint32_t K, uint32_t groups, mx::FastDiv per_row,
                     uint32_t total, T* __restrict__ out) {
    using F = mx::Fmt<FMT>;
    using Codes = typename F::Codes8;
    pdl_wait();
    pdl_trigger();
    const uint32_t sub = threadIdx.x & 3;
    constexpr uint32_t step = Q_THREADS / 4;
    const uint32_t first = blockIdx.x * (U * step) + (threadIdx.x >> 2);
    {
        Codes c[U];
        uint32_t byte[U], row[U], j[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t q = first + u * step;
            row[u] = per_row.div(q);
            j[u] = q - row[u] * per_row.d;
            if (q < total) {
                c[u] = __ldg(reinterpret_cast<const Codes*>(data + (uint64_t)q * F::BLOCK_BYTES +
                                                            sub * sizeof(Codes)));
                byte[u] = __ldg(scales + 4 * (uint64_t)mx::scale_word(row[u], j[u] >> 2, groups) +
                                (j[u] & 3));
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t q = first + u * step, k = j[u] * 32 + sub * 8;
            if (q < total && (FLAT || k < K))
                mx::store_aligned8(out + (FLAT ? (uint64_t)q * 32 + sub * 8 : (uint64_t)row[u] * K + k),
                                   decode_scaled<T, FMT>(c[u], byte[u]));
        }
    }
}

// LANES threads a piece of 8 LANES values.  total: pieces, per_row.d of them a row.
template <typename T, int FMT, int U, int LANES>
__global__ void __launch_bounds__(Q_THREADS)
mx_dequantize_any_kernel(const uint8_t* __restrict__ data, const uint8_t* __restrict__ scales,
                         uint32_t rows, uint32_t K, uint32_t nb, uint32_t groups,
                         mx::FastDiv per_row, uint32_t total, T* __restrict__ out) {
    using F = mx::Fmt<FMT>;
    using Codes = typename F::Codes8;
    pdl_wait();
    pdl_trigger();
    const uint32_t lane = threadIdx.x & 31, sub = lane & 3;
    constexpr uint32_t step = Q_THREADS / LANES;
    const uint32_t first = blockIdx.x * (U * step) + threadIdx.x / LANES;
    {
        Codes c[U];
        uint32_t byte[U], row[U], k[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t q = first + u * step;
            row[u] = per_row.div(q);
            k[u] = ((q - row[u] * per_row.d) * LANES + (lane & (LANES - 1))) * 8;
            const uint32_t j = k[u] >> 5;
            c[u] = Codes{};
            byte[u] = 0;
            if (q < total && j < nb) {
                c[u] = __ldg(reinterpret_cast<const Codes*>(
                    data + (uint64_t)(row[u] * nb + j) * F::BLOCK_BYTES + sub * sizeof(Codes)));
                byte[u] = __ldg(scales + 4 * (uint64_t)mx::scale_word(row[u], j >> 2, groups) + (j & 3));
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = first + u * step < total && k[u] < K;
            mx::store_any8<T, LANES>(out + (in ? (uint64_t)row[u] * K + k[u] : 0),
                           in ? (int)min(8u, K - k[u]) : 0, decode_scaled<T, FMT>(c[u], byte[u]),
                           (int)lane);
        }
    }
}

// Whether U = 1: `units` (per thread block and unit of U: `per`) do not fill four blocks an SM at U
// = 4, eight at U = 2.
bool small(int64_t units, int64_t per) { return units <= 148 * 4 * 4 * per; }
// Lanes a piece of an unaligned row: what short rows fill (63025 x 34 bf16 -> E2M1: 5.0 us, 13.2
// with 32; 27336 x 113: 4.6, 6.6; 27997 x 344: 9.0, 12.2), 32 beyond (3000 x 16001: 34 us, 37
// with 16).
int any_lanes(int64_t K) { return K <= 64 ? 8 : K <= 128 || (K > 256 && K <= 512) ? 16 : 32; }
unsigned blocks_for(int64_t units, int64_t per) { return (unsigned)((units + per - 1) / per); }

template <typename T, int FMT>
int run_quantize(const void* x, int64_t rows, int64_t K, int64_t ldx, void* data, void* scales,
                 cudaStream_t s) {
    const uint32_t nb = (uint32_t)mx::blocks_of(K), groups = (uint32_t)mx::groups_of(K);
    const bool aligned = K % 8 == 0 && aligned16(x) && (rows == 1 || ldx * (int64_t)sizeof(T) % 16 == 0);
    const bool flat = K % 128 == 0 && (rows == 1 || ldx == K);
    const int lanes = aligned ? 4 : any_lanes(K);
    const uint32_t per = aligned ? groups * 4 : (uint32_t)((K + 8 * lanes - 1) / (8 * lanes));
    const int64_t total = rows * per, unit = Q_THREADS / lanes;
    const bool one = small(total, unit);
    auto k = lanes == 8  ? (one ? mx_quantize_any_kernel<T, FMT, 1, 8> : mx_quantize_any_kernel<T, FMT, 2, 8>)
             : lanes == 16 ? (one ? mx_quantize_any_kernel<T, FMT, 1, 16> : mx_quantize_any_kernel<T, FMT, 2, 16>)
             : lanes == 32 ? (one ? mx_quantize_any_kernel<T, FMT, 1, 32> : mx_quantize_any_kernel<T, FMT, 2, 32>)
             : flat   ? (one ? mx_quantize_kernel<T, FMT, 1, true> : mx_quantize_kernel<T, FMT, 4, true>)
                      : (one ? mx_quantize_kernel<T, FMT, 1, false> : mx_quantize_kernel<T, FMT, 4, false>);
    const int U = one ? 1 : aligned ? 4 : 2;
    return launch_k(k, dim3(blocks_for(total, U * unit)), dim3(Q_THREADS), 0, s,
                    static_cast<const T*>(x), (uint32_t)rows, (uint32_t)K, ldx, nb, groups,
                    mx::FastDiv(per), (uint32_t)total, static_cast<uint8_t*>(data),
                    static_cast<uint32_t*>(scales));
}

template <typename T, int FMT>
int run_dequantize(const void* data, const void* scales, int64_t rows, int64_t K, void* out,
                   cudaStream_t s) {
    const uint32_t nb = (uint32_t)mx::blocks_of(K), groups = (uint32_t)mx::groups_of(K);
    const uint8_t* d = static_cast<const uint8_t*>(data);
    const uint8_t* sc = static_cast<const uint8_t*>(scales);
    if (K % 8 == 0 && aligned16(out)) {
        const int64_t total = rows * nb, unit = Q_THREADS / 4;
        const bool one = small(total, unit), flat = K % 32 == 0;
        auto k = flat ? (one ? mx_dequantize_kernel<T, FMT, 1, true> : mx_dequantize_kernel<T, FMT, 4, true>)
                      : (one ? mx_dequantize_kernel<T, FMT, 1, false> : mx_dequantize_kernel<T, FMT, 4, false>);
        return launch_k(k, dim3(blocks_for(total, (one ? 1 : 4) * unit)), dim3(Q_THREADS), 0, s, d,
                        sc, (uint32_t)rows, (uint32_t)K, groups, mx::FastDiv(nb), (uint32_t)total,
                        static_cast<T*>(out));
    }
    const int lanes = any_lanes(K);
    const uint32_t per = (uint32_t)((K + 8 * lanes - 1) / (8 * lanes));
    const int64_t total = rows * per, unit = Q_THREADS / lanes;
    const bool one = small(total, unit);
    auto k = lanes == 8    ? (one ? mx_dequantize_any_kernel<T, FMT, 1, 8> : mx_dequantize_any_kernel<T, FMT, 2, 8>)
             : lanes == 16 ? (one ? mx_dequantize_any_kernel<T, FMT, 1, 16> : mx_dequantize_any_kernel<T, FMT, 2, 16>)
                           : (one ? mx_dequantize_any_kernel<T, FMT, 1, 32> : mx_dequantize_any_kernel<T, FMT, 2, 32>);
    return launch_k(k, dim3(blocks_for(total, (one ? 1 : 2) * unit)), dim3(Q_THREADS), 0, s, d, sc,
                    (uint32_t)rows, (uint32_t)K, nb, groups, mx::FastDiv(per), (uint32_t)total,
                    static_cast<T*>(out));
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

extern "C" int snnb_mx_quantize(const void* x, int x_dtype, int64_t rows, int64_t K, int64_t ldx,
                                int fmt, void* data, void* scales, snnb_stream_t stream) {
    if (const int inj = take_injected_status()) return inj;
    if (x_dtype != SNNB_F32 && x_dtype != SNNB_F16 && x_dtype != SNNB_BF16) return SNNB_ERR_ARG;
    if (fmt != SNNB_MXFP4 && fmt != SNNB_MXFP8) return SNNB_ERR_ARG;
    if (!mx::sizes_ok(rows, K) || !mx::stride_ok(rows, ldx)) return SNNB_ERR_ARG;
    if (rows == 0) return SNNB_OK;
    if (!x || !data || !scales || !aligned16(data) || !aligned16(scales)) return SNNB_ERR_ARG;
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
    if (!mx::sizes_ok(rows, K)) return SNNB_ERR_ARG;
    if (rows == 0) return SNNB_OK;
    if (!out || !data || !scales || !aligned16(data) || !aligned16(scales)) return SNNB_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(out) % (out_dtype == SNNB_F32 ? 4 : 2)) return SNNB_ERR_ARG;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    SNNB_MX_DISPATCH(out_dtype, fmt, run_dequantize, data, scales, rows, K, out, s)
}
