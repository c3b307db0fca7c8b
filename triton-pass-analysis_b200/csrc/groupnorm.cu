// Group norm of channels-last tensors x [B, S, C], C in G groups, then an activation:
//
//   y = act((x - mean) / sqrt(var + eps) * weight + bias),
//
// mean and var (biased) over the S * C / G values of a group of a sample.  The variance is that of
// the differences from the mean, in float32, not E[x^2] - mean^2, which a large mean cancels.
//
// Bound: HBM.  Three forms; the first two read x from memory once:
//   teams   groups of few values (a token's heads): a few lanes hold one group in registers
//   slabs   images: a slab of neighbouring groups (128 bytes of a row or more) of one sample, its
//           rows divided over the blocks of a cluster, which hold them in shared memory and join
//           their sums through it
//   passes  large tensors: statistics of blocks of whole rows, then the outputs; what the second
//           pass finds in L2 is not read from memory again
//
// bf16, us (floor): 12544 x 384 in 8 groups 9.5 (2.9); 64 x 28 x 28 x 256 in 32 18.5 (7.8); 64 x 56 x 56 x 256
// 68 (31, or 47 when the second pass reads memory too, which it does: 27 for the statistics and 41,
// issue slots 45% taken in both).
#include "common.cuh"
#include "mx.cuh"
#include "tc_common.cuh"

namespace snnb {
namespace {

constexpr int GN_THREADS = 256;

// BYTES of values as they lie in memory, moved at once.
template <int BYTES> struct alignas(BYTES) Bits {
    uint32_t w[BYTES / 4];
};
template <> struct Bits<2> { uint16_t w[1]; };

// Rows that a thread has in flight: 64 bytes, or as many as registers allow of narrow pieces.
template <typename T, int VEC> constexpr int rows_ahead() {
    return VEC * (int)sizeof(T) >= 16 ? 4 : VEC * (int)sizeof(T) == 8 ? 8 : 16;
}

struct GnArgs {
    const void* x;
    int64_t xb, xs;                // strides of sample and row
    uint32_t B, S, C, G, cg;       // cg: channels of a group
    const void *weight, *bias;
    int wf32;
    float eps;
    void* y;
};

__device__ __forceinline__ float reciprocal(float a) {         // to 1 ulp; of infinity zero
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
    return r;
}
__device__ __forceinline__ float exp2_fast(float a) {          // to 2^-22
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
    return r;
}
// 16-bit outputs take the fast exponential and reciprocal (errors of 2^-21, far below their steps).
template <typename T, int ACT>
__device__ __forceinline__ float activate(float y) {
    if (ACT == SNNB_ACT_SILU)
        return sizeof(T) == 2 ? y * reciprocal(1.0f + exp2_fast(-1.44269504f * y)) : y / (1.0f + expf(-y));
    if (ACT == SNNB_ACT_RELU) return y < 0.0f ? 0.0f : y;      // a NaN stays one
    if (ACT == SNNB_ACT_GELU) return 0.5f * y * (1.0f + erff(y * 0.70710678118654752f));
    return y;
}

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Bits<VEC * sizeof(T)>& r, float (&v)[VEC]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = __int_as_float((int)r.w[i]);
    } else if constexpr (VEC == 1) {
        v[0] = mx::pair_f32(r.w[0], (const T*)nullptr).x;
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            const float2 f = mx::pair_f32(r.w[i / 2], (const T*)nullptr);
            v[i] = f.x;
            v[i + 1] = f.y;
        }
    }
}
// VEC parameters from channel c on (`missing` without any).
template <typename T, int VEC>
__device__ __forceinline__ void params(const void* p, int f32, uint32_t c, float missing, float (&v)[VEC]) {
    using P = Bits<VEC * (int)sizeof(T)>;
    if (!p) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = missing;
    } else if (sizeof(T) == 2 && f32) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = __ldg(static_cast<const float*>(p) + c + i);
    } else if (reinterpret_cast<uintptr_t>(p) % (VEC * sizeof(T)) == 0) {
        unpack<T, VEC>(*reinterpret_cast<const P*>(static_cast<const T*>(p) + c), v);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = to_f32(static_cast<const T*>(p)[c + i]);
    }
}
// (x - mean) * scale + shift, activated and rounded.  FOLDED: shift holds - mean * scale too.
template <typename T, int VEC, int ACT, bool FOLDED = false>
__device__ __forceinline__ Bits<VEC * sizeof(T)> finish(const float (&x)[VEC], const float (&mean)[VEC],
                                                        const float (&scale)[VEC], const float (&shift)[VEC]) {
    Bits<VEC * sizeof(T)> r;
    float f[VEC];
    if constexpr (VEC == 1) {
        f[0] = FOLDED ? fmaf(x[0], scale[0], shift[0]) : fmaf(x[0] - mean[0], scale[0], shift[0]);
    } else if constexpr (FOLDED) {
#pragma unroll
        for (int i = 0; i < VEC; i += 2)
            mx::unpack2(mx::fma2(mx::pack2(x[i], x[i + 1]), mx::pack2(scale[i], scale[i + 1]),
                                 mx::pack2(shift[i], shift[i + 1])), f[i], f[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            const uint64_t d = mx::add2(mx::pack2(x[i], x[i + 1]), mx::pack2(-mean[i], -mean[i + 1]));
            mx::unpack2(mx::fma2(d, mx::pack2(scale[i], scale[i + 1]), mx::pack2(shift[i], shift[i + 1])), f[i],
                        f[i + 1]);
        }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = activate<T, ACT>(f[i]);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) r.w[i] = (uint32_t)__float_as_int(f[i]);
    } else if constexpr (VEC == 1) {
        r.w[0] = (uint16_t)mx::round_pair(f[0], f[0], (const T*)nullptr);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) r.w[i / 2] = mx::round_pair(f[i], f[i + 1], (const T*)nullptr);
    }
    return r;
}

// A team of P lanes holds one group of one sample: R pieces of VEC values a lane, a row's pieces
// next to one another.
template <typename T, int VEC, int P, int R, int ACT>
__global__ void __launch_bounds__(GN_THREADS) gn_team_kernel(GnArgs a, mx::FastDiv per_row, uint32_t items) {
    using V = Bits<VEC * (int)sizeof(T)>;
    pdl_wait();
    pdl_trigger();
    const uint32_t item = (blockIdx.x * GN_THREADS + threadIdx.x) / P, l = threadIdx.x % P;
    const bool in = item < items;
    const uint32_t b = item / a.G, g = item - b * a.G, pieces = a.S * per_row.d;
    const T* x = static_cast<const T*>(a.x) + b * a.xb + g * a.cg;
    float v[R][VEC];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const uint32_t p = l + i * P, row = per_row.div(p), c = (p - row * per_row.d) * VEC;
        if (in && p < pieces) unpack<T, VEC>(*reinterpret_cast<const V*>(x + row * a.xs + c), v[i]);
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (in && l + i * P < pieces) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum += v[i][j];
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
        const uint32_t p = l + i * P, row = per_row.div(p), c = (p - row * per_row.d) * VEC;
        if (!in || p >= pieces) continue;
        float m[VEC], w[VEC], s[VEC];
        params<T, VEC>(a.weight, a.wf32, g * a.cg + c, 1.0f, w);
        params<T, VEC>(a.bias, a.wf32, g * a.cg + c, 0.0f, s);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            m[j] = mean;
            w[j] *= r;
        }
        *reinterpret_cast<V*>(y + (int64_t)row * a.C + c) = finish<T, VEC, ACT>(v[i], m, w, s);
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
// rank order, and what `f` makes of that (all).
template <typename F>
__device__ __forceinline__ void join_groups(const float* part, uint32_t groups, uint32_t cg, uint32_t blocks,
                                            float* own, float* all, F f) {
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
        for (uint32_t g = threadIdx.x; g < groups; g += GN_THREADS) all[g] = f(own[g]);
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
            all[g] = f(s);
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
__global__ void __launch_bounds__(GN_THREADS, 4) gn_slab_kernel(const __grid_constant__ SlabArgs s) {
    using V = Bits<VEC * (int)sizeof(T)>;
    constexpr int U = rows_ahead<T, VEC>();
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
    float *mean_of = own1 + most, *own2 = mean_of + most, *rstd_of = own2 + most;
    const uint32_t r0 = (uint32_t)((uint64_t)a.S * rank / s.blocks);
    const uint32_t rows = (uint32_t)((uint64_t)a.S * (rank + 1) / s.blocks) - r0;
    const uint32_t nv = width / VEC, t = threadIdx.x;
    // a block's threads: whole rows of pieces, or a part of one row at a time (a narrower last slab
    // leaves some idle: `part` has room for this many rows)
    const uint32_t nc = min(s.width / VEC, (uint32_t)GN_THREADS), rp = GN_THREADS / nc;
    const bool in = t < rp * nc, lanes = 32 % nc == 0;
    const uint32_t vc = t % nc, rr = t / nc, turns = (nv + nc - 1) / nc;
    const T* x = static_cast<const T*>(a.x) + b * a.xb + r0 * a.xs + c0;
    T* y = static_cast<T*>(a.y) + ((int64_t)b * a.S + r0) * a.C + c0;
    const float over_n = 1.0f / ((float)a.S * (float)a.cg);

    // f(piece's raw bits, its place in the tile, in the output) over a column of pieces
    auto walk = [&](uint32_t v, bool kept, auto f) {
        if (!in || v >= nv) return;
        const T* from = x + rr * a.xs + v * VEC;
        const int64_t step = rp * a.xs, ystep = (int64_t)rp * a.C;
        V* at = tile + rr * nv + v;
        T* to = y + (int64_t)rr * a.C + v * VEC;
        const uint32_t tstep = rp * nv;
        uint32_t left = rr < rows ? (rows - rr + rp - 1) / rp : 0;
        for (; left >= U; left -= U) {
            V raw[U];
#pragma unroll
            for (int i = 0; i < U; ++i) raw[i] = kept ? at[i * tstep] : *reinterpret_cast<const V*>(from + i * step);
#pragma unroll
            for (int i = 0; i < U; ++i) f(raw[i], at + i * tstep, to + i * ystep);
            from += U * step;
            at += U * tstep;
            to += U * ystep;
        }
        for (; left; --left, from += step, at += tstep, to += ystep)
            f(kept ? *at : *reinterpret_cast<const V*>(from), at, to);
    };
    // a thread's sums by channel: to its row of `part`, or to its warp's where lanes hold whole rows
    auto to_part = [&](uint32_t v, float (&acc)[VEC]) {
        if (lanes) {
            for (uint32_t o = nc; o < 32; o *= 2) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
            }
            if ((t & 31) >= nc) return;
        }
        if (!in || v >= nv) return;
#pragma unroll
        for (int j = 0; j < VEC; ++j) part[(lanes ? t >> 5 : rr) * width + v * VEC + j] = acc[j];
    };
    const uint32_t part_rows = lanes ? GN_THREADS / 32 : rp;

    // sums, and squares of the differences from the thread's first row, which is near enough to the
    // mean that they do not cancel
    float s1[VEC] = {}, s2[VEC] = {}, base[VEC] = {};
    for (uint32_t i = 0, v = vc; i < turns; ++i, v += nc) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) s1[j] = s2[j] = base[j] = 0.0f;
        if (in && v < nv && rr < rows)
            unpack<T, VEC>(*reinterpret_cast<const V*>(x + (int64_t)rr * a.xs + v * VEC), base);
        walk(v, false, [&](V raw, V* at, T*) {
            if (KEEP) *at = raw;
            float f[VEC];
            unpack<T, VEC>(raw, f);
            if constexpr (VEC == 1) {
                f[0] -= base[0];
                s1[0] += f[0];
                s2[0] = fmaf(f[0], f[0], s2[0]);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; j += 2) {
                    const uint64_t d = mx::add2(mx::pack2(f[j], f[j + 1]), mx::pack2(-base[j], -base[j + 1]));
                    mx::unpack2(mx::add2(d, mx::pack2(s1[j], s1[j + 1])), s1[j], s1[j + 1]);
                    mx::unpack2(mx::fma2(d, d, mx::pack2(s2[j], s2[j + 1])), s2[j], s2[j + 1]);
                }
            }
        });
        const float count = in && v < nv && rr < rows ? (float)((rows - rr + rp - 1) / rp) : 0.0f;
        float acc[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = fmaf(count, base[j], s1[j]);
        to_part(v, acc);
        if (count > 0.0f) {                    // the thread's own mean, and the squares around it
            const float over = 1.0f / count;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float m = s1[j] * over;
                s2[j] = fmaxf(fmaf(-m, s1[j], s2[j]), 0.0f);
                s1[j] = base[j] + m;
            }
        }
    }
    add_rows(part, part_rows, width);
    join_groups(part, groups, a.cg, s.blocks, own1, mean_of, [&](float v) { return v * over_n; });
    for (uint32_t i = 0, v = vc; i < turns; ++i, v += nc) {
        float acc[VEC] = {}, mean[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            mean[j] = v < nv ? mean_of[s.per_group.div(v * VEC + j)] : 0.0f;
        if (turns == 1) {
            const float count = in && v < nv && rr < rows ? (float)((rows - rr + rp - 1) / rp) : 0.0f;
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (count > 0.0f) acc[j] = fmaf(count * (s1[j] - mean[j]), s1[j] - mean[j], s2[j]);
        } else {
            walk(v, KEEP, [&](V raw, V*, T*) {
                float f[VEC];
                unpack<T, VEC>(raw, f);
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] = fmaf(f[j] - mean[j], f[j] - mean[j], acc[j]);
            });
        }
        to_part(v, acc);
    }
    add_rows(part, part_rows, width);
    join_groups(part, groups, a.cg, s.blocks, own2, rstd_of,
                [&](float v) { return 1.0f / sqrtf(fmaf(v, over_n, a.eps)); });
    // no block ends while another reads its sums
    if (s.blocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    for (uint32_t i = 0, v = vc; i < turns; ++i, v += nc) {
        float mean[VEC], w[VEC], shift[VEC];
        if (in && v < nv) {
            params<T, VEC>(a.weight, a.wf32, c0 + v * VEC, 1.0f, w);
            params<T, VEC>(a.bias, a.wf32, c0 + v * VEC, 0.0f, shift);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const uint32_t g = s.per_group.div(v * VEC + j);
                mean[j] = mean_of[g];
                w[j] *= rstd_of[g];
            }
        }
        walk(v, KEEP, [&](V raw, V*, T* to) {
            float f[VEC];
            unpack<T, VEC>(raw, f);
            *reinterpret_cast<V*>(to) = finish<T, VEC, ACT>(f, mean, w, shift);
        });
    }
    if (s.blocks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}

// Values of a group that a warp can hold.
constexpr uint32_t TEAM_VALUES = 2048;

template <typename T, int VEC, int P, int R, int ACT>
int launch_team(const GnArgs& a, cudaStream_t s) {
    const int64_t items = (int64_t)a.B * a.G;
    return launch_k(gn_team_kernel<T, VEC, P, R, ACT>, dim3((unsigned)((items * P + GN_THREADS - 1) / GN_THREADS)),
                    dim3(GN_THREADS), 0, s, a, mx::FastDiv(a.cg / VEC), (uint32_t)items);
}
template <typename T, int VEC, int ACT>
int run_team(const GnArgs& a, cudaStream_t s) {
    const uint32_t pieces = a.S * (a.cg / VEC);
    if (pieces <= 4) return launch_team<T, VEC, 4, 1, ACT>(a, s);
    if (pieces <= 8) return launch_team<T, VEC, 8, 1, ACT>(a, s);
    if (pieces <= 16) return launch_team<T, VEC, 16, 1, ACT>(a, s);
    if (pieces <= 32) return launch_team<T, VEC, 32, 1, ACT>(a, s);
    if (pieces <= 128) return launch_team<T, VEC, 32, 4, ACT>(a, s);
    if constexpr (VEC <= 4)
        if (pieces <= 512) return launch_team<T, VEC, 32, 16, ACT>(a, s);
    if constexpr (VEC == 1)
        if (pieces <= 1024) return launch_team<T, VEC, 32, 32, ACT>(a, s);
    return launch_team<T, VEC, 32, TEAM_VALUES / 32 / VEC, ACT>(a, s);
}

// Shared memory of a block: four an SM, or one, for groups of many channels.
constexpr int SLAB_SMEM = 55 * 1024, SLAB_SMEM_MOST = 110 * 1024;

template <typename T, int VEC, int ACT, bool KEEP>
int launch_slab(const SlabArgs& p, int smem, cudaStream_t s) {
    auto k = gn_slab_kernel<T, VEC, ACT, KEEP>;
    static bool done[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (dev < 0 || dev >= 64 || !done[dev]) {
        e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SLAB_SMEM_MOST);
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
    const uint32_t part_rows = nv <= 32 && 32 % nv == 0 ? GN_THREADS / 32 : rp;
    const int64_t part = (int64_t)part_rows * p.width * 4, sums = (int64_t)groups * 16;
    const int64_t most = part + sums < SLAB_SMEM / 2 ? SLAB_SMEM : SLAB_SMEM_MOST;
    const int64_t room = most - part - sums - 32, row = (int64_t)p.width * sizeof(T);
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


// ---- two passes over large tensors -----------------------------------------------------------
// Of every block of `chunk` rows of a sample, each part of a group's mean and sum of squares around it,
// then the outputs from those of the sample's blocks.  Slabs hold whole parts (a group is one, or
// several where it has more pieces than a block has threads), at most one piece a thread.
struct PassArgs {
    GnArgs a;
    uint32_t slabs, width, chunk, chunks;      // channels of a slab; rows of a block; blocks of a sample
    uint32_t parts, pc;                        // of a group; channels of one
    mx::FastDiv per_group, per_part;
    float2* stats;                             // [B][chunks][G parts]
};
template <typename T, int VEC>
__global__ void __launch_bounds__(GN_THREADS, 4) gn_stats_kernel(const __grid_constant__ PassArgs s) {
    using V = Bits<VEC * (int)sizeof(T)>;
    constexpr int U = rows_ahead<T, VEC>();    // at a time, as many ahead
    extern __shared__ float part[];            // [rows][width], then [groups] means
    const GnArgs& a = s.a;
    pdl_wait();
    pdl_trigger();
    const uint32_t slab = blockIdx.x % s.slabs, rest = blockIdx.x / s.slabs;
    const uint32_t b = rest / s.chunks, chunk = rest - b * s.chunks, c0 = slab * s.width;
    const uint32_t width = min(s.width, a.C - c0), groups = width / s.pc, nv = width / VEC, t = threadIdx.x;
    const uint32_t r0 = chunk * s.chunk, rows = min(s.chunk, a.S - r0);
    const uint32_t nc = s.width / VEC, rp = GN_THREADS / nc, vc = t % nc, rr = t / nc;
    const bool in = t < rp * nc && vc < nv && rr < rows;
    const T* x = static_cast<const T*>(a.x) + b * a.xb + (int64_t)(r0 + rr) * a.xs + c0 + vc * VEC;
    const int64_t step = rp * a.xs;
    float s1[VEC] = {}, s2[VEC] = {}, base[VEC] = {};
    uint32_t left = in ? (rows - rr + rp - 1) / rp : 0;
    const float count = (float)left;
    auto add = [&](V raw) {
        float f[VEC];
        unpack<T, VEC>(raw, f);
        if constexpr (VEC == 1) {
            f[0] -= base[0];
            s1[0] += f[0];
            s2[0] = fmaf(f[0], f[0], s2[0]);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; j += 2) {
                const uint64_t d = mx::add2(mx::pack2(f[j], f[j + 1]), mx::pack2(base[j], base[j + 1]));
                mx::unpack2(mx::add2(d, mx::pack2(s1[j], s1[j + 1])), s1[j], s1[j + 1]);
                mx::unpack2(mx::fma2(d, d, mx::pack2(s2[j], s2[j + 1])), s2[j], s2[j + 1]);
            }
        }
    };
    V raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
        if (i < left) raw[i] = *reinterpret_cast<const V*>(x + i * step);
    if (left) {                                // minus the first row: near enough to the mean that the
        unpack<T, VEC>(raw[0], base);          // squares do not cancel
        if constexpr (VEC > 1) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) base[j] = -base[j];
        }
    }
    for (; left >= 2 * U; left -= U) {         // the next rows in flight
        V now[U];
#pragma unroll
        for (int i = 0; i < U; ++i) now[i] = raw[i];
        x += U * step;
#pragma unroll
        for (int i = 0; i < U; ++i) raw[i] = *reinterpret_cast<const V*>(x + i * step);
#pragma unroll
        for (int i = 0; i < U; ++i) add(now[i]);
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
        if (i < left) add(raw[i]);
    for (uint32_t i = U; i < left; ++i) add(*reinterpret_cast<const V*>(x + i * step));
    // the thread's own means and squares around them
    const float over = count > 0.0f ? 1.0f / count : 0.0f;
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        if (VEC > 1) base[j] = -base[j];
        const float m = s1[j] * over;
        s2[j] = fmaxf(fmaf(-m, s1[j], s2[j]), 0.0f);
        acc[j] = fmaf(count, base[j], s1[j]);
        s1[j] = base[j] + m;
    }
    const bool lanes = 32 % nc == 0;
    float* mean = part + (lanes ? GN_THREADS / 32 : rp) * s.width;
    auto to_part = [&]() {
        if (lanes)
            for (uint32_t o = nc; o < 32; o *= 2) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
            }
        if (lanes ? (t & 31) < nc && vc < nv : t < rp * nc && vc < nv) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) part[(lanes ? t >> 5 : rr) * width + vc * VEC + j] = acc[j];
        }
        add_rows(part, lanes ? GN_THREADS / 32 : rp, width);
    };
    auto each_group = [&](auto f) {
        for (uint32_t g = t >> 5; g < groups; g += GN_THREADS / 32) {
            float v = 0.0f;
            for (uint32_t c = t & 31; c < s.pc; c += 32) v += part[g * s.pc + c];
#pragma unroll
            for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if ((t & 31) == 0) f(g, v);
        }
    };
    to_part();
    const float all = 1.0f / ((float)rows * (float)s.pc);
    each_group([&](uint32_t g, float v) { mean[g] = v * all; });
    __syncthreads();
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const float d = vc < nv ? s1[j] - mean[s.per_part.div(vc * VEC + j)] : 0.0f;
        acc[j] = count > 0.0f ? fmaf(count * d, d, s2[j]) : 0.0f;
    }
    to_part();
    float2* out = s.stats + ((int64_t)b * s.chunks + chunk) * (a.G * s.parts) + c0 / s.pc;
    each_group([&](uint32_t g, float v) { out[g] = make_float2(mean[g], v); });
}

template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(GN_THREADS, 4) gn_apply_kernel(const __grid_constant__ PassArgs s) {
    using V = Bits<VEC * (int)sizeof(T)>;
    constexpr int U = rows_ahead<T, VEC>();
    constexpr bool FOLDED = sizeof(T) == 2;
    extern __shared__ float groups_of[];       // [groups] mean, [groups] 1 / deviation
    const GnArgs& a = s.a;
    pdl_wait();
    pdl_trigger();
    // the last blocks first: their rows are the likeliest to be in L2 still
    const uint32_t at = gridDim.x - 1 - blockIdx.x, slab = at % s.slabs, rest = at / s.slabs;
    const uint32_t b = rest / s.chunks, chunk = rest - b * s.chunks, c0 = slab * s.width;
    const uint32_t width = min(s.width, a.C - c0), nv = width / VEC, t = threadIdx.x;
    const uint32_t g0 = c0 / a.cg, groups = (c0 + width - 1) / a.cg - g0 + 1;      // that the slab touches
    const uint32_t r0 = chunk * s.chunk, rows = min(s.chunk, a.S - r0);
    const uint32_t nc = s.width / VEC, rp = GN_THREADS / nc, vc = t % nc, rr = t / nc;
    const bool in = t < rp * nc && vc < nv && rr < rows;
    const T* x = static_cast<const T*>(a.x) + b * a.xb + (int64_t)(r0 + rr) * a.xs + c0 + vc * VEC;
    T* y = static_cast<T*>(a.y) + ((int64_t)b * a.S + r0 + rr) * a.C + c0 + vc * VEC;
    const int64_t step = rp * a.xs, ystep = (int64_t)rp * a.C;
    uint32_t left = in ? (rows - rr + rp - 1) / rp : 0;
    V raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
        if (i < left) raw[i] = *reinterpret_cast<const V*>(x + i * step);
    const uint32_t of = a.G * s.parts, all = s.chunks * s.parts;
    const float2* stats = s.stats + (int64_t)b * s.chunks * of + g0 * s.parts;
    const float over_n = 1.0f / ((float)a.S * (float)a.cg), pc = (float)s.pc;
    const float whole = (float)s.chunk * pc, last = (float)(a.S - (s.chunks - 1) * s.chunk) * pc;
    for (uint32_t g = t >> 5; g < groups; g += GN_THREADS / 32) {
        float sum = 0.0f, sq = 0.0f;
        for (uint32_t i = t & 31; i < all; i += 32) {
            const uint32_t c = i / s.parts;
            sum += stats[(int64_t)c * of + g * s.parts + i - c * s.parts].x * (c + 1 == s.chunks ? last : whole);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float mean = sum * over_n;
        for (uint32_t i = t & 31; i < all; i += 32) {
            const uint32_t c = i / s.parts;
            const float2 v = stats[(int64_t)c * of + g * s.parts + i - c * s.parts];
            const float d = v.x - mean;
            sq += fmaf((c + 1 == s.chunks ? last : whole) * d, d, v.y);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
        if ((t & 31) == 0) {
            groups_of[g] = mean;
            groups_of[groups + g] = 1.0f / sqrtf(fmaf(sq, over_n, a.eps));
        }
    }
    __syncthreads();
    if (!in) return;
    float mean[VEC], w[VEC], shift[VEC];
    params<T, VEC>(a.weight, a.wf32, c0 + vc * VEC, 1.0f, w);
    params<T, VEC>(a.bias, a.wf32, c0 + vc * VEC, 0.0f, shift);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const uint32_t g = s.per_group.div(c0 + vc * VEC + j) - g0;
        mean[j] = groups_of[g];
        w[j] *= groups_of[groups + g];
        // 16-bit values: a mean that is 2^k deviations leaves them 11 - k bits or fewer, and this 24 - k
        if (FOLDED) shift[j] = fmaf(-mean[j], w[j], shift[j]);
    }
    auto put = [&](const V& bits, T* to) {
        float f[VEC];
        unpack<T, VEC>(bits, f);
        *reinterpret_cast<V*>(to) = finish<T, VEC, ACT, FOLDED>(f, mean, w, shift);
    };
    for (; left >= 2 * U; left -= U) {         // the next rows in flight
        V now[U];
#pragma unroll
        for (int i = 0; i < U; ++i) now[i] = raw[i];
        x += U * step;
#pragma unroll
        for (int i = 0; i < U; ++i) raw[i] = *reinterpret_cast<const V*>(x + i * step);
#pragma unroll
        for (int i = 0; i < U; ++i) put(now[i], y + i * ystep);
        y += U * ystep;
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
        if (i < left) put(raw[i], y + i * ystep);
    for (uint32_t i = U; i < left; ++i) put(*reinterpret_cast<const V*>(x + i * step), y + i * ystep);
}

// Slabs and blocks of the two passes for pieces of `vec` values; false: no slab of whole
// groups has at most a piece a thread.
bool plan_passes(const GnArgs& a, uint32_t vec, PassArgs& p) {
    const uint32_t most = GN_THREADS * vec;
    // a group's parts, alike: whole pieces where it has several, and then whole parts a slab
    uint32_t parts = 1, unit = a.cg;
    while (unit % vec) unit += a.cg;
    if (unit > most) {
        for (parts = 2; parts < a.cg; ++parts)
            if (a.cg % parts == 0 && a.cg / parts <= most && a.cg / parts % vec == 0) break;
        unit = a.cg / parts;
        if (a.cg % parts || unit > most || unit % vec) return false;
    }
    p.a = a;
    p.parts = parts;
    p.pc = a.cg / parts;
    p.width = most / unit * unit;
    if (p.width > a.C) p.width = a.C;
    p.slabs = (a.C + p.width - 1) / p.width;
    p.width = (a.C / unit + p.slabs - 1) / p.slabs * unit;     // alike in width
    p.slabs = (a.C + p.width - 1) / p.width;
    p.per_group = mx::FastDiv(a.cg);
    p.per_part = mx::FastDiv(p.pc);
    const uint32_t rp = GN_THREADS / (p.width / vec);
    // one round of four blocks an SM where samples are few, 8 rows a thread or more: a thread's start
    // and end cost as much as some 10 rows (64 KB a block: 136 us for 64 x 3136 x 256, so 70)
    const int64_t room = 592 / ((int64_t)a.B * p.slabs);
    p.chunks = room > 1 ? (uint32_t)room : 1;
    p.chunk = (a.S + p.chunks - 1) / p.chunks;
    if (p.chunk < 8 * rp) p.chunk = 8 * rp;
    p.chunks = (a.S + p.chunk - 1) / p.chunk;
    return (int64_t)a.B * p.chunks * p.slabs <= 0x7fffffff;
}
// Bytes from which the two passes are faster (bf16: 64 x 784 x 256, 26 MB, 28 us and 19 in one pass;
// 64 x 3136 x 256, 103 MB, 72 and 81).
constexpr int64_t TWO_PASSES = int64_t(64) << 20;

template <typename T, int VEC, int ACT>
int run_passes(PassArgs p, cudaStream_t s) {
    const uint32_t nc = p.width / VEC, rp = GN_THREADS / nc, rows = 32 % nc == 0 ? GN_THREADS / 32 : rp;
    const uint32_t groups = p.width / p.pc;            // or more of either kind
    const dim3 grid(p.a.B * p.chunks * p.slabs);
    if (const int st = launch_k(gn_stats_kernel<T, VEC>, grid, dim3(GN_THREADS),
                                (rows * p.width + groups) * sizeof(float), s, p))
        return st;
    return launch_k(gn_apply_kernel<T, VEC, ACT>, grid, dim3(GN_THREADS), 2 * (groups + 2) * sizeof(float), s, p);
}

template <typename T, int VEC, int ACT>
int run_vec(const GnArgs& a, bool team, float2* work, cudaStream_t s) {
    if (team) return run_team<T, VEC, ACT>(a, s);
    PassArgs p;
    if (work && plan_passes(a, VEC, p)) {
        p.stats = work;
        return run_passes<T, VEC, ACT>(p, s);
    }
    return run_slab<T, VEC, ACT>(a, s);
}
// The widest piece that rows are made of, and for teams groups.
int widest(const GnArgs& a, int size, bool team) {
    int v = 16 / size;
    for (; v > 1; v /= 2)
        if (a.C % v == 0 && (!team || a.cg % v == 0) &&
            (reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y)) % (v * size) == 0 &&
            (a.B == 1 || a.xb % v == 0) && (a.S == 1 || a.xs % v == 0))
            break;
    return v;
}
// Few values a group, in pieces of 32 bytes or of single rows: a row's pieces are then neighbours'.
bool team_takes(const GnArgs& a, int size, int v) {
    return (int64_t)a.S * (a.cg / v) <= (a.S == 1 ? TEAM_VALUES / v : 128) && (a.S == 1 || a.cg * size >= 32);
}
template <typename T, int ACT>
int run(const GnArgs& a, float2* work, cudaStream_t s) {
    constexpr int MOST = 16 / (int)sizeof(T);
    int v = widest(a, sizeof(T), true);
    const bool team = team_takes(a, sizeof(T), v);
    if (!team) v = widest(a, sizeof(T), false);
    if (v == MOST) return run_vec<T, MOST, ACT>(a, team, work, s);
    if constexpr (MOST == 8)
        if (v == 4) return run_vec<T, 4, ACT>(a, team, work, s);
    if (v == 2) return run_vec<T, 2, ACT>(a, team, work, s);
    return run_vec<T, 1, ACT>(a, team, work, s);
}

}  // namespace
}  // namespace snnb

using namespace snnb;

#define SNNB_GN_ACT(T)                                              \
    switch (act) {                                                  \
        case SNNB_ACT_NONE: return run<T, SNNB_ACT_NONE>(a, work, s); \
        case SNNB_ACT_SILU: return run<T, SNNB_ACT_SILU>(a, work, s); \
        case SNNB_ACT_RELU: return run<T, SNNB_ACT_RELU>(a, work, s); \
        default: return run<T, SNNB_ACT_GELU>(a, work, s);            \
    }

static bool norm_sizes_ok(int dtype, int64_t B, int64_t S, int64_t C, int64_t groups) {
    return (dtype == SNNB_F32 || dtype == SNNB_F16 || dtype == SNNB_BF16) && B >= 0 && S >= 0 && C >= 1 &&
           groups >= 1 && C % groups == 0 && B <= 0x7fffffff && S <= 0x7fffffff && C <= 0x4000 &&
           B * groups <= 0x7ffffff && (B == 0 || S == 0 || B <= (int64_t(1) << 40) / S / C);
}

extern "C" int64_t snnb_group_norm_act_workspace_bytes(int dtype, int64_t B, int64_t S, int64_t C,
                                                       int64_t groups) {
    if (!norm_sizes_ok(dtype, B, S, C, groups)) return -1;
    const int size = dtype == SNNB_F32 ? 4 : 2;
    if (B == 0 || B * S * C * size < TWO_PASSES) return 0;
    GnArgs a = {};
    a.B = (uint32_t)B;
    a.S = (uint32_t)S;
    a.C = (uint32_t)C;
    a.G = (uint32_t)groups;
    a.cg = (uint32_t)(C / groups);
    // the most that pieces of any width ask for
    int64_t most = 0;
    for (int v = 16 / size; v >= 1; v /= 2) {
        PassArgs p;
        if (C % v == 0 && plan_passes(a, v, p)) {
            const int64_t n = B * p.chunks * groups * p.parts * (int64_t)sizeof(float2);
            most = n > most ? n : most;
        }
    }
    return S == 1 && a.cg <= TEAM_VALUES ? 0 : most;
}

extern "C" int snnb_group_norm_act(const void* x, int64_t x_batch_stride, int64_t x_row_stride,
                                   int dtype, int64_t B, int64_t S, int64_t C, int64_t groups,
                                   const void* weight, const void* bias, int weight_dtype,
                                   float eps, int act, void* out, void* workspace,
                                   int64_t workspace_bytes, snnb_stream_t stream) {
    if (const int inj = take_injected_status()) return inj;
    if (!norm_sizes_ok(dtype, B, S, C, groups)) return SNNB_ERR_ARG;
    if (weight_dtype != SNNB_F32 && weight_dtype != dtype) return SNNB_ERR_ARG;
    if (act < SNNB_ACT_NONE || act > SNNB_ACT_GELU || !(eps >= 0.0f)) return SNNB_ERR_ARG;
    if (B == 0 || S == 0) return SNNB_OK;
    if (!x || !out) return SNNB_ERR_ARG;
    const int size = dtype == SNNB_F32 ? 4 : 2, wsize = weight_dtype == SNNB_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(out) % size ||
        reinterpret_cast<uintptr_t>(weight) % wsize || reinterpret_cast<uintptr_t>(bias) % wsize)
        return SNNB_ERR_ARG;
    const int64_t need = snnb_group_norm_act_workspace_bytes(dtype, B, S, C, groups);
    if (need > 0 && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 8))
        return SNNB_ERR_ARG;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    float2* work = need > 0 ? static_cast<float2*>(workspace) : nullptr;
    const GnArgs a = {x, x_batch_stride, x_row_stride, (uint32_t)B, (uint32_t)S, (uint32_t)C, (uint32_t)groups,
                      (uint32_t)(C / groups), weight, bias, weight_dtype == SNNB_F32, eps, out};
    if (dtype == SNNB_F32) { SNNB_GN_ACT(float) }
    if (dtype == SNNB_F16) { SNNB_GN_ACT(__half) }
    SNNB_GN_ACT(__nv_bfloat16)
}
