// Group norm of channels-last tensors x [B, S, C], C in G groups, then an activation:
//
//   y = act((x - mean) / sqrt(var + eps) * weight + bias),
//
// mean and var (biased) over the S * C / G values of a group of a sample.  The variance is that of
// the differences from the mean, in float32, not E[x^2] - mean^2, which a large mean cancels.
//
// Bound: HBM.  Two forms, both read x from memory once where it fits:
//   teams   groups of few values (a token's heads): a few lanes hold one group in registers
//   slabs   images: a slab of neighbouring groups (128 bytes of a row or more) of one sample, its
//           rows divided over the blocks of a cluster, which hold them in shared memory and join
//           their sums through it; larger samples are read again from L2
#include "common.cuh"
#include "mx.cuh"
#include "tc_common.cuh"

namespace snnb {
namespace {

constexpr int GN_THREADS = 256;

template <int BYTES> struct Bits;
template <> struct Bits<16> { typedef uint4 type; };
template <> struct Bits<8> { typedef uint2 type; };
template <> struct Bits<4> { typedef uint32_t type; };
template <> struct Bits<2> { typedef uint16_t type; };

struct GnArgs {
    const void* x;
    int64_t xb, xs;                // strides of sample and row
    uint32_t B, S, C, G, cg;       // cg: channels of a group
    const void *weight, *bias;
    int wf32;
    float eps;
    void* y;
};

// 16-bit outputs take the fast exponential and division (errors of 2^-21, far below their steps).
template <typename T, int ACT>
__device__ __forceinline__ float activate(float y) {
    if (ACT == SNNB_ACT_SILU)
        return sizeof(T) == 2 ? __fdividef(y, 1.0f + __expf(fminf(-y, 80.0f))) : y / (1.0f + expf(-y));
    if (ACT == SNNB_ACT_RELU) return y < 0.0f ? 0.0f : y;      // a NaN stays one
    if (ACT == SNNB_ACT_GELU) return 0.5f * y * (1.0f + erff(y * 0.70710678118654752f));
    return y;
}

template <typename T, int VEC>
__device__ __forceinline__ void unpack(typename Bits<VEC * sizeof(T)>::type r, float (&v)[VEC]) {
    const T* t = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_f32(t[i]);
}
// VEC parameters from channel c on (`missing` without any).
template <typename T, int VEC>
__device__ __forceinline__ void params(const void* p, int f32, uint32_t c, float missing, float (&v)[VEC]) {
    using P = typename Bits<VEC * sizeof(T)>::type;
    if (!p) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = missing;
    } else if (sizeof(T) == 2 && f32) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = __ldg(static_cast<const float*>(p) + c + i);
    } else if (reinterpret_cast<uintptr_t>(p) % (VEC * sizeof(T)) == 0) {
        unpack<T, VEC>(__ldg(reinterpret_cast<const P*>(static_cast<const T*>(p) + c)), v);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = to_f32(static_cast<const T*>(p)[c + i]);
    }
}
// (x - mean) * scale + shift, activated and rounded.
template <typename T, int VEC, int ACT>
__device__ __forceinline__ typename Bits<VEC * sizeof(T)>::type finish(const float (&x)[VEC], const float (&mean)[VEC],
                                                                       const float (&scale)[VEC],
                                                                       const float (&shift)[VEC]) {
    typename Bits<VEC * sizeof(T)>::type r;
    T* t = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        mx::round_to(activate<T, ACT>(fmaf(x[i] - mean[i], scale[i], shift[i])), t + i);
    return r;
}

// A team of P lanes holds one group of one sample: R pieces of VEC values a lane, a row's pieces
// next to one another.
template <typename T, int VEC, int P, int R, int ACT>
__global__ void __launch_bounds__(GN_THREADS) gn_team_kernel(GnArgs a, uint32_t per_row, uint32_t items) {
    using V = typename Bits<VEC * sizeof(T)>::type;
    pdl_wait();
    pdl_trigger();
    const uint32_t item = (blockIdx.x * GN_THREADS + threadIdx.x) / P, l = threadIdx.x % P;
    const bool in = item < items;
    const uint32_t b = item / a.G, g = item - b * a.G, pieces = a.S * per_row;
    const T* x = static_cast<const T*>(a.x) + b * a.xb + g * a.cg;
    float v[R][VEC];
    uint32_t row[R], c[R];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const uint32_t p = l + i * P;
        row[i] = p / per_row;
        c[i] = (p - row[i] * per_row) * VEC;
        if (in && p < pieces) {
            unpack<T, VEC>(__ldg(reinterpret_cast<const V*>(x + row[i] * a.xs + c[i])), v[i]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum += v[i][j];
        }
    }
#pragma unroll
    for (int o = P / 2; o; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float n = (float)(a.S * a.cg), mean = sum / n;
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (in && l + i * P < pieces) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) sq += (v[i][j] - mean) * (v[i][j] - mean);
        }
#pragma unroll
    for (int o = P / 2; o; o /= 2) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    const float r = 1.0f / sqrtf(sq / n + a.eps);
    T* y = static_cast<T*>(a.y) + (int64_t)b * a.S * a.C + g * a.cg;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (!in || l + i * P >= pieces) continue;
        float m[VEC], w[VEC], s[VEC];
        params<T, VEC>(a.weight, a.wf32, g * a.cg + c[i], 1.0f, w);
        params<T, VEC>(a.bias, a.wf32, g * a.cg + c[i], 0.0f, s);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            m[j] = mean;
            w[j] *= r;
        }
        *reinterpret_cast<V*>(y + (int64_t)row[i] * a.C + c[i]) = finish<T, VEC, ACT>(v[i], m, w, s);
    }
}

// part [n][w] floats: row 0 becomes the sum of the n rows.
__device__ __forceinline__ void add_rows(float* part, uint32_t n, uint32_t w) {
    while (n > 1) {
        const uint32_t half = (n + 1) / 2;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < (n - half) * w; i += GN_THREADS) part[i] += part[i + half * w];
        n = half;
    }
    __syncthreads();
}

// Of every group: the sum of its channels' sums in this block (own), then over the cluster's blocks in
// rank order (all).
__device__ __forceinline__ void join_groups(const float* part, uint32_t groups, uint32_t cg, uint32_t blocks,
                                            float* own, float* all) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (uint32_t g = warp; g < groups; g += GN_THREADS / 32) {
        float s = 0.0f;
        for (uint32_t c = lane; c < cg; c += 32) s += part[g * cg + c];
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) own[g] = s;
    }
    if (blocks == 1) {
        __syncthreads();
        for (uint32_t g = threadIdx.x; g < groups; g += GN_THREADS) all[g] = own[g];
    } else {
        tc::cluster_sync();
        for (uint32_t g = threadIdx.x; g < groups; g += GN_THREADS) {
            float s = 0.0f;
            for (uint32_t r = 0; r < blocks; ++r) {
                float v;
                asm volatile("ld.shared::cluster.f32 %0, [%1];"
                             : "=f"(v)
                             : "r"(tc::map_to_rank(tc::smem_u32(own + g), r)));
                s += v;
            }
            all[g] = s;
        }
    }
    __syncthreads();
}

// KEEP: the block's rows stay in shared memory.
struct SlabArgs {
    GnArgs a;
    uint32_t slabs, width, blocks;             // slabs of a sample, channels of one, blocks of a cluster
    mx::FastDiv per_group;                     // channel / cg
    uint32_t part_off, group_off;              // in shared memory, in bytes
};
template <typename T, int VEC, int ACT, bool KEEP>
__global__ void __launch_bounds__(GN_THREADS, 2) gn_slab_kernel(const __grid_constant__ SlabArgs s) {
    using V = typename Bits<VEC * sizeof(T)>::type;
    constexpr int U = 8;                       // rows in flight
    extern __shared__ uint8_t smem[];
    const GnArgs& a = s.a;
    V* tile = reinterpret_cast<V*>(smem);
    float* part = reinterpret_cast<float*>(smem + s.part_off);
    float* own1 = reinterpret_cast<float*>(smem + s.group_off);
    pdl_wait();
    pdl_trigger();
    const uint32_t rank = blockIdx.x % s.blocks, at = blockIdx.x / s.blocks;
    const uint32_t b = at / s.slabs, slab = at - b * s.slabs, c0 = slab * s.width;
    const uint32_t width = min(s.width, a.C - c0), groups = width / a.cg, most = s.width / a.cg;
    float *sum = own1 + most, *own2 = sum + most, *sq = own2 + most;
    const uint32_t r0 = (uint32_t)((uint64_t)a.S * rank / s.blocks);
    const uint32_t rows = (uint32_t)((uint64_t)a.S * (rank + 1) / s.blocks) - r0;
    const uint32_t nv = width / VEC, t = threadIdx.x;
    // a block's threads: whole rows of pieces, or a part of one row at a time (a narrower last slab
    // leaves some idle: `part` has room for this many rows)
    const uint32_t nc = min(s.width / VEC, (uint32_t)GN_THREADS), rp = GN_THREADS / nc;
    const bool in = t < rp * nc;
    const uint32_t vc = t % nc, rr = t / nc;
    const T* x = static_cast<const T*>(a.x) + b * a.xb + r0 * a.xs + c0;
    T* y = static_cast<T*>(a.y) + ((int64_t)b * a.S + r0) * a.C + c0;
    const float n = (float)a.S * (float)a.cg;

    // f(row, piece's raw bits) over a column of pieces
    auto walk = [&](uint32_t v, bool kept, auto f) {
        if (!in || v >= nv) return;
        for (uint32_t r = rr; r < rows; r += U * rp) {
            V raw[U];
#pragma unroll
            for (int i = 0; i < U; ++i)
                if (r + i * rp < rows)
                    raw[i] = kept ? tile[(r + i * rp) * nv + v]
                                  : *reinterpret_cast<const V*>(x + (int64_t)(r + i * rp) * a.xs + v * VEC);
#pragma unroll
            for (int i = 0; i < U; ++i)
                if (r + i * rp < rows) f(r + i * rp, raw[i]);
        }
    };
    auto to_part = [&](uint32_t v, const float (&acc)[VEC]) {
        if (!in || v >= nv) return;
#pragma unroll
        for (int j = 0; j < VEC; ++j) part[rr * width + v * VEC + j] = acc[j];
    };
    // with more pieces a row than threads, a row of `part` is filled in turns (rp is 1)
    const uint32_t turns = (nv + nc - 1) / nc;
    for (uint32_t i = 0, v = vc; i < turns; ++i, v += nc) {
        float acc[VEC] = {};
        walk(v, false, [&](uint32_t r, V raw) {
            if (KEEP) tile[r * nv + v] = raw;
            float f[VEC];
            unpack<T, VEC>(raw, f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] += f[j];
        });
        to_part(v, acc);
    }
    add_rows(part, rp, width);
    join_groups(part, groups, a.cg, s.blocks, own1, sum);
    for (uint32_t i = 0, v = vc; i < turns; ++i, v += nc) {
        float acc[VEC] = {}, mean[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            mean[j] = v < nv ? sum[s.per_group.div(v * VEC + j)] / n : 0.0f;
        walk(v, KEEP, [&](uint32_t, V raw) {
            float f[VEC];
            unpack<T, VEC>(raw, f);
#pragma unroll
            for (int j = 0; j < VEC; ++j) acc[j] = fmaf(f[j] - mean[j], f[j] - mean[j], acc[j]);
        });
        to_part(v, acc);
    }
    add_rows(part, rp, width);
    join_groups(part, groups, a.cg, s.blocks, own2, sq);
    // no block ends, and none overwrites its sums, while another reads them
    if (s.blocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    for (uint32_t i = 0, v = vc; i < turns; ++i, v += nc) {
        float mean[VEC], w[VEC], shift[VEC];
        if (in && v < nv) {
            params<T, VEC>(a.weight, a.wf32, c0 + v * VEC, 1.0f, w);
            params<T, VEC>(a.bias, a.wf32, c0 + v * VEC, 0.0f, shift);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const uint32_t g = s.per_group.div(v * VEC + j);
                mean[j] = sum[g] / n;
                w[j] *= 1.0f / sqrtf(sq[g] / n + a.eps);
            }
        }
        walk(v, KEEP, [&](uint32_t r, V raw) {
            float f[VEC];
            unpack<T, VEC>(raw, f);
            *reinterpret_cast<V*>(y + (int64_t)r * a.C + v * VEC) = finish<T, VEC, ACT>(f, mean, w, shift);
        });
    }
    if (s.blocks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

template <typename T, int VEC, int P, int R, int ACT>
int launch_team(const GnArgs& a, cudaStream_t s) {
    const int64_t items = (int64_t)a.B * a.G;
    return launch_k(gn_team_kernel<T, VEC, P, R, ACT>, dim3((unsigned)((items * P + GN_THREADS - 1) / GN_THREADS)),
                    dim3(GN_THREADS), 0, s, a, a.cg / VEC, (uint32_t)items);
}
template <typename T, int VEC, int ACT>
int run_team(const GnArgs& a, cudaStream_t s) {
    const uint32_t pieces = a.S * (a.cg / VEC);
    if (pieces <= 4) return launch_team<T, VEC, 4, 1, ACT>(a, s);
    if (pieces <= 8) return launch_team<T, VEC, 8, 1, ACT>(a, s);
    if (pieces <= 16) return launch_team<T, VEC, 16, 1, ACT>(a, s);
    if (pieces <= 32) return launch_team<T, VEC, 32, 1, ACT>(a, s);
    return launch_team<T, VEC, 32, 4, ACT>(a, s);
}

constexpr int SLAB_SMEM = 110 * 1024;          // of a block: two an SM

template <typename T, int VEC, int ACT, bool KEEP>
int launch_slab(const SlabArgs& p, int smem, cudaStream_t s) {
    auto k = gn_slab_kernel<T, VEC, ACT, KEEP>;
    static bool done[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (dev < 0 || dev >= 64 || !done[dev]) {
        e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SLAB_SMEM);
        if (e != cudaSuccess) return record_cuda_error(e);
        if (dev >= 0 && dev < 64) done[dev] = true;
    }
    return launch_kc(k, dim3(p.a.B * p.slabs * p.blocks), dim3(GN_THREADS), smem, s, p.blocks, p);
}
template <typename T, int VEC, int ACT>
int run_slab(const GnArgs& a, cudaStream_t s) {
    SlabArgs p;
    p.a = a;
    // whole groups and whole pieces, 128 bytes of a row or more
    uint32_t unit = a.cg;
    while (unit % VEC) unit += a.cg;
    p.width = unit;
    while (p.width < a.C && p.width * sizeof(T) < 128) p.width += unit;
    if (p.width > a.C) p.width = a.C;
    p.slabs = (a.C + p.width - 1) / p.width;
    p.per_group = mx::FastDiv(a.cg);
    const uint32_t groups = p.width / a.cg, nv = p.width / VEC;
    const uint32_t rp = nv < (uint32_t)GN_THREADS ? GN_THREADS / nv : 1;
    const int64_t part = (int64_t)rp * p.width * 4, sums = (int64_t)groups * 16;
    const int64_t room = SLAB_SMEM - part - sums - 32, row = (int64_t)p.width * sizeof(T);
    if (room < 0) return SNNB_ERR_UNSUPPORTED;
    // blocks of a cluster (8 are portable): until a block's rows fit, and until every SM has two
    p.blocks = 1;
    auto rows = [&] { return (int64_t)(a.S + p.blocks - 1) / p.blocks; };
    while (p.blocks < 8 && (rows() * row > room || ((int64_t)a.B * p.slabs * p.blocks < 296 && rows() >= 8 * rp)))
        p.blocks *= 2;
    if ((int64_t)a.B * p.slabs * p.blocks > 0x7fffffff) return SNNB_ERR_ARG;
    const bool keep = rows() * row <= room;
    const int64_t tile = keep ? (rows() * row + 15) / 16 * 16 : 0;
    p.part_off = (uint32_t)tile;
    p.group_off = (uint32_t)(tile + (part + 15) / 16 * 16);
    const int smem = (int)(p.group_off + sums);
    return keep ? launch_slab<T, VEC, ACT, true>(p, smem, s) : launch_slab<T, VEC, ACT, false>(p, smem, s);
}

template <typename T, int VEC, int ACT>
int run_vec(const GnArgs& a, bool team, cudaStream_t s) {
    return team ? run_team<T, VEC, ACT>(a, s) : run_slab<T, VEC, ACT>(a, s);
}
template <typename T, int ACT>
int run(const GnArgs& a, cudaStream_t s) {
    constexpr int MOST = 16 / (int)sizeof(T);
    // the widest piece that rows are made of, and for teams groups
    auto widest = [&](bool team) {
        int v = MOST;
        for (; v > 1; v /= 2)
            if (a.C % v == 0 && (!team || a.cg % v == 0) &&
                (reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y)) % (v * sizeof(T)) == 0 &&
                (a.B == 1 || a.xb % v == 0) && (a.S == 1 || a.xs % v == 0))
                break;
        return v;
    };
    // few values a group, in pieces of 16 bytes or single rows: a row's pieces are then neighbours'
    int v = widest(true);
    const bool team = (int64_t)a.S * (a.cg / v) <= 128 && (a.S == 1 || a.cg * sizeof(T) >= 32);
    if (!team) v = widest(false);
    if (v == MOST) return run_vec<T, MOST, ACT>(a, team, s);
    if constexpr (MOST == 8)
        if (v == 4) return run_vec<T, 4, ACT>(a, team, s);
    if (v == 2) return run_vec<T, 2, ACT>(a, team, s);
    return run_vec<T, 1, ACT>(a, team, s);
}

}  // namespace
}  // namespace snnb

using namespace snnb;

#define SNNB_GN_ACT(T)                                        \
    switch (act) {                                            \
        case SNNB_ACT_NONE: return run<T, SNNB_ACT_NONE>(a, s); \
        case SNNB_ACT_SILU: return run<T, SNNB_ACT_SILU>(a, s); \
        case SNNB_ACT_RELU: return run<T, SNNB_ACT_RELU>(a, s); \
        default: return run<T, SNNB_ACT_GELU>(a, s);            \
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
    if (B > 0x7fffffff || S > 0x7fffffff || C > 0x4000 || B * groups > 0x7ffffff) return SNNB_ERR_ARG;
    if (B == 0 || S == 0) return SNNB_OK;
    if (!x || !out || B > (int64_t(1) << 40) / S / C) return SNNB_ERR_ARG;
    const int size = dtype == SNNB_F32 ? 4 : 2, wsize = weight_dtype == SNNB_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(out) % size ||
        reinterpret_cast<uintptr_t>(weight) % wsize || reinterpret_cast<uintptr_t>(bias) % wsize)
        return SNNB_ERR_ARG;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const GnArgs a = {x, x_batch_stride, x_row_stride, (uint32_t)B, (uint32_t)S, (uint32_t)C, (uint32_t)groups,
                      (uint32_t)(C / groups), weight, bias, weight_dtype == SNNB_F32, eps, out};
    if (dtype == SNNB_F32) { SNNB_GN_ACT(float) }
    if (dtype == SNNB_F16) { SNNB_GN_ACT(__half) }
    SNNB_GN_ACT(__nv_bfloat16)
}
