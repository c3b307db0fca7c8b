// Rotary positions with several axes (time, height, width ...) for queries and keys.
//
//   pair i of a head, columns (i, i + R) or (2i, 2i + 1) of its first 2R, turns by the angle
//   t = positions[axis(i)] * f(i):   (a, b) -> (a cos t - b sin t, a sin t + b cos t)
//
// The angle is held in turns: positions are exact in float64 (up to 2^53), f / 2 pi comes in float64 and
// the product's whole turns are dropped there, so that an angle is good to 2^-50 of itself (in float32 a
// position of 2^20 would be off by 0.06 rad); what remains of it, in [-1/2, 1/2], is exact enough in
// float32 for the sine and the cosine.
//
// Bound: HBM (every value is read and written once).  A thread holds the sines and cosines of the
// pairs of one piece of 16 bytes (two pieces R columns apart, or one of neighbouring pairs) and takes
// that piece through about 20 heads (the sines and cosines cost as much as turning six), two heads at a
// time, the next two's loads in flight.  32768 tokens x 40 heads of 128, bf16: 117 us, 5.8 TB/s (a
// copy of the same bytes takes 109); 8 heads a thread and four at a time with no loads ahead took
// 164, 20 heads so 141.
#include "common.cuh"
#include "mx.cuh"

namespace snnb {
namespace {

constexpr int R_THREADS = 256;
constexpr int MAX_PAIRS = 256;

// The pairs' frequencies and axes, passed by value: a launch holds its own copy.
struct Ladder {
    double turns[MAX_PAIRS];       // frequency / 2 pi
    uint8_t axis[MAX_PAIRS];
};

struct Heads {                     // [B, N, heads, d], strides in elements, unit column stride
    const void* in;
    void* out;
    int64_t ib, in_, ih, ob, on, oh;
};

struct Positions {
    const void* p;
    int64_t sb, sn, sa;            // strides of batch, token, axis
    int type;                      // 0 int32, 1 int64, 2 float32
    __device__ __forceinline__ double at(int64_t b, int64_t n, int a) const {
        const int64_t i = b * sb + n * sn + a * sa;
        if (type == 0) return (double)static_cast<const int32_t*>(p)[i];
        if (type == 1) return (double)static_cast<const int64_t*>(p)[i];
        return (double)static_cast<const float*>(p)[i];
    }
};

// Rounded alike in every form.
__device__ __forceinline__ float turned0(float a, float b, float cs, float sn) {
    return fmaf(a, cs, -__fmul_rn(b, sn));
}
__device__ __forceinline__ float turned1(float a, float b, float cs, float sn) {
    return fmaf(a, sn, __fmul_rn(b, cs));
}

template <int BYTES> struct Piece;
template <> struct Piece<16> { typedef uint4 type; };
template <> struct Piece<8> { typedef uint2 type; };
template <> struct Piece<4> { typedef uint32_t type; };

// The angle of a pair.
__device__ __forceinline__ void sine(const Positions& pos, const Ladder& ladder, int64_t b, int64_t n,
                                     uint32_t pair, int inverse, int& axis, double& place, float& cs,
                                     float& sn) {
    if (ladder.axis[pair] != axis) {
        axis = ladder.axis[pair];
        place = pos.at(b, n, axis);
    }
    const double t = place * ladder.turns[pair];
    sincospif(2.0f * (float)(t - rint(t)), &sn, &cs);
    if (inverse) sn = -sn;
}

// Pieces of VEC columns of one token, taken through `per` heads.  Units of a token: the pairs'
// pieces, then those that are copied.  The thread's index: unit, token, group of heads.
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(R_THREADS, 4)
rotary_vec_kernel(Heads q, Heads k, uint32_t hq, uint32_t hk, uint32_t per, uint32_t N, uint32_t turned,
                  uint32_t units, uint32_t tokens_units, int64_t total, uint32_t pairs, int inverse,
                  Positions pos, const __grid_constant__ Ladder ladder) {
    using P = typename Piece<VEC * (int)sizeof(T)>::type;
    constexpr int NP = INTERLEAVED ? VEC / 2 : VEC;            // pairs of a thread
    constexpr int U = 2;                                       // heads at a time, as many ahead
    pdl_wait();
    pdl_trigger();
    const int64_t at = (int64_t)blockIdx.x * R_THREADS + threadIdx.x;
    if (at >= total) return;
    const uint32_t group = (uint32_t)(at / tokens_units), rest = (uint32_t)(at - (int64_t)group * tokens_units);
    const uint32_t token = rest / units, u = rest - token * units;
    const int64_t b = token / N, n = token - (uint32_t)b * N;
    const bool turn = u < turned;
    const uint32_t c0 = turn ? u * VEC : 2 * pairs + (u - turned) * VEC;
    float cs[NP], sn[NP];
    if (turn) {
        int axis = -1;
        double place = 0.0;
#pragma unroll
        for (int i = 0; i < NP; ++i) sine(pos, ladder, b, n, u * NP + i, inverse, axis, place, cs[i], sn[i]);
    }
    const uint32_t end = min(hq + hk, (group + 1) * per);
    auto at_head = [&](uint32_t h, bool out) {
        const Heads& t = h < hq ? q : k;
        const int64_t hh = h < hq ? h : h - hq;
        return out ? (T*)t.out + b * t.ob + n * t.on + hh * t.oh + c0
                   : (T*)t.in + b * t.ib + n * t.in_ + hh * t.ih + c0;
    };
    P x[U], y[U];
    auto load = [&](uint32_t h0) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (h0 + i >= end) continue;
            const T* in = at_head(h0 + i, false);
            x[i] = *reinterpret_cast<const P*>(in);
            if (!INTERLEAVED && turn) y[i] = *reinterpret_cast<const P*>(in + pairs);
        }
    };
    load(group * per);
    for (uint32_t h0 = group * per; h0 < end; h0 += U) {
        P x0[U], y0[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            x0[i] = x[i];
            y0[i] = y[i];
        }
        load(h0 + U);                                // a head is read before its piece is written
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (h0 + i >= end) continue;
            if (turn) {
                T* a = reinterpret_cast<T*>(&x0[i]);
                T* c = reinterpret_cast<T*>(&y0[i]);
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    T* p0 = INTERLEAVED ? a + 2 * j : a + j;
                    T* p1 = INTERLEAVED ? a + 2 * j + 1 : c + j;
                    const float v0 = to_f32(*p0), v1 = to_f32(*p1);
                    mx::round_to(turned0(v0, v1, cs[j], sn[j]), p0);
                    mx::round_to(turned1(v0, v1, cs[j], sn[j]), p1);
                }
            }
            T* out = at_head(h0 + i, true);
            *reinterpret_cast<P*>(out) = x0[i];
            if (!INTERLEAVED && turn) *reinterpret_cast<P*>(out + pairs) = y0[i];
        }
    }
}

// One thread per token and pair (or column that is not turned); it goes through the heads.
template <typename T>
__global__ void __launch_bounds__(R_THREADS)
rotary_kernel(Heads q, Heads k, uint32_t hq, uint32_t hk, uint32_t N, uint32_t units,
              int64_t total, uint32_t pairs, uint32_t d, int interleaved, int inverse,
              Positions pos, const __grid_constant__ Ladder ladder) {
    pdl_wait();
    pdl_trigger();
    const int64_t at = (int64_t)blockIdx.x * R_THREADS + threadIdx.x;
    if (at >= total) return;
    const int64_t token = at / units;
    const uint32_t u = (uint32_t)(at - token * units);
    const int64_t b = token / N, n = token - b * N;
    const bool turn = u < pairs;
    const uint32_t c0 = !turn ? u + pairs : interleaved ? 2 * u : u;
    const uint32_t c1 = !turn ? c0 : interleaved ? 2 * u + 1 : u + pairs;
    float cs = 1.0f, sn = 0.0f;
    if (turn) {
        const double t = pos.at(b, n, ladder.axis[u]) * ladder.turns[u];
        sincospif(2.0f * (float)(t - rint(t)), &sn, &cs);
        if (inverse) sn = -sn;
    }
    for (uint32_t h = 0; h < hq + hk; ++h) {
        const Heads& x = h < hq ? q : k;
        const uint32_t hh = h < hq ? h : h - hq;
        const T* in = static_cast<const T*>(x.in) + b * x.ib + n * x.in_ + hh * x.ih;
        T* out = static_cast<T*>(x.out) + b * x.ob + n * x.on + hh * x.oh;
        const float a0 = to_f32(in[c0]), a1 = to_f32(in[c1]);
        if (turn) {
            mx::round_to(turned0(a0, a1, cs, sn), out + c0);
            mx::round_to(turned1(a0, a1, cs, sn), out + c1);
        } else {
            out[c0] = in[c0];
        }
    }
}

// The widest piece that every row and both halves are made of, in elements; 1: none.
int piece(int size, int64_t d, int64_t pairs, int interleaved, const Heads& q, int64_t hq,
          const Heads& k, int64_t hk, int64_t B, int64_t N) {
    for (int v = 16 / size; v > 1; v /= 2) {
        if (d % v || (interleaved ? 2 * pairs : pairs) % v) continue;
        auto fits = [&](const Heads& x, int64_t heads) {
            if (!heads) return true;
            const uintptr_t ends = reinterpret_cast<uintptr_t>(x.in) | reinterpret_cast<uintptr_t>(x.out);
            return ends % (v * size) == 0 && (B == 1 || (x.ib | x.ob) % v == 0) &&
                   (N == 1 || (x.in_ | x.on) % v == 0) && (heads == 1 || (x.ih | x.oh) % v == 0);
        };
        if (fits(q, hq) && fits(k, hk)) return v;
    }
    return 1;
}

struct VecArgs {
    Heads q, k;
    uint32_t hq, hk, per, N, turned, units, tokens_units;
    int64_t total;
    uint32_t pairs;
    int inverse;
    Positions pos;
};
template <typename T, int VEC>
int run_vec(const VecArgs& a, int interleaved, const Ladder& ladder, cudaStream_t s) {
    auto kernel = interleaved ? rotary_vec_kernel<T, VEC, true> : rotary_vec_kernel<T, VEC, false>;
    return launch_k(kernel, dim3((unsigned)((a.total + R_THREADS - 1) / R_THREADS)), dim3(R_THREADS), 0,
                    s, a.q, a.k, a.hq, a.hk, a.per, a.N, a.turned, a.units, a.tokens_units, a.total,
                    a.pairs, a.inverse, a.pos, ladder);
}
template <typename T>
int run_vec(const VecArgs& a, int vec, int interleaved, const Ladder& ladder, cudaStream_t s) {
    constexpr int MOST = 16 / (int)sizeof(T);
    if (vec == MOST) return run_vec<T, MOST>(a, interleaved, ladder, s);
    if constexpr (MOST == 8)
        if (vec == 4) return run_vec<T, 4>(a, interleaved, ladder, s);
    return run_vec<T, 2>(a, interleaved, ladder, s);
}

}  // namespace
}  // namespace snnb

using namespace snnb;

extern "C" int snnb_rotary_axes(const void* q, void* q_out, int64_t q_heads,
                                const int64_t* q_strides, const void* k, void* k_out,
                                int64_t k_heads, const int64_t* k_strides, int dtype, int64_t B,
                                int64_t N, int64_t d, const void* positions, int positions_dtype,
                                const int64_t* positions_strides, const double* turns,
                                const uint8_t* axis, int pairs, int interleaved, int inverse,
                                snnb_stream_t stream) {
    if (const int inj = take_injected_status()) return inj;
    if (dtype != SNNB_F32 && dtype != SNNB_F16 && dtype != SNNB_BF16) return SNNB_ERR_ARG;
    if (positions_dtype < 0 || positions_dtype > 2) return SNNB_ERR_ARG;
    if (B < 0 || N < 0 || q_heads < 0 || k_heads < 0 || d < 1 || d > 0x7fffffff) return SNNB_ERR_ARG;
    if (pairs < 1 || pairs > MAX_PAIRS || 2 * (int64_t)pairs > d) return SNNB_ERR_ARG;
    if (q_heads > 0x3fffffff || k_heads > 0x3fffffff || N > 0x7fffffff) return SNNB_ERR_ARG;
    if (B == 0 || N == 0 || q_heads + k_heads == 0) return SNNB_OK;
    if (!positions || !positions_strides || !turns || !axis) return SNNB_ERR_ARG;
    if (q_heads && (!q || !q_out || !q_strides)) return SNNB_ERR_ARG;
    if (k_heads && (!k || !k_out || !k_strides)) return SNNB_ERR_ARG;
    const int size = dtype == SNNB_F32 ? 4 : 2, psize = positions_dtype == 1 ? 8 : 4;
    const void* ptrs[4] = {q_heads ? q : nullptr, q_heads ? q_out : nullptr,
                           k_heads ? k : nullptr, k_heads ? k_out : nullptr};
    for (const void* p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) % size) return SNNB_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(positions) % psize) return SNNB_ERR_ARG;
    const int64_t units = d - pairs;
    if (B > (int64_t(1) << 38) / N / units) return SNNB_ERR_ARG;
    Ladder ladder = {};
    for (int i = 0; i < pairs; ++i) {
        ladder.turns[i] = turns[i];
        ladder.axis[i] = axis[i];
    }
    auto heads = [](const void* in, void* out, const int64_t* s) {
        return s ? Heads{in, out, s[0], s[1], s[2], s[3], s[4], s[5]} : Heads{};
    };
    const Heads hq = heads(q, q_out, q_heads ? q_strides : nullptr);
    const Heads hk = heads(k, k_out, k_heads ? k_strides : nullptr);
    const Positions pos{positions, positions_strides[0], positions_strides[1],
                        positions_strides[2], positions_dtype};
    const int vec = piece(size, d, pairs, interleaved, hq, q_heads, hk, k_heads, B, N);
    const int64_t turned = (interleaved ? 2 * pairs : pairs) / vec, pieces = turned + (d - 2 * pairs) / vec;
    if (vec > 1 && B * N * pieces <= 0x7fffffff) {
        // about 20 heads a thread, fewer where that leaves less than 4 blocks an SM
        const int64_t heads = q_heads + k_heads, tokens_units = B * N * pieces, groups = (heads + 19) / 20;
        int64_t per = (heads + groups - 1) / groups;
        while (per > 1 && tokens_units * ((heads + per - 1) / per) < 148 * 4 * R_THREADS) per = (per + 1) / 2;
        const VecArgs a = {hq, hk, (uint32_t)q_heads, (uint32_t)k_heads, (uint32_t)per, (uint32_t)N,
                           (uint32_t)turned, (uint32_t)pieces, (uint32_t)tokens_units,
                           tokens_units * ((heads + per - 1) / per), (uint32_t)pairs, inverse, pos};
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        if (dtype == SNNB_F32) return run_vec<float>(a, vec, interleaved, ladder, st);
        if (dtype == SNNB_F16) return run_vec<__half>(a, vec, interleaved, ladder, st);
        return run_vec<__nv_bfloat16>(a, vec, interleaved, ladder, st);
    }
    const int64_t total = B * N * units;
    auto kernel = dtype == SNNB_F32   ? rotary_kernel<float>
                  : dtype == SNNB_F16 ? rotary_kernel<__half>
                                      : rotary_kernel<__nv_bfloat16>;
    return launch_k(kernel, dim3((unsigned)((total + R_THREADS - 1) / R_THREADS)), dim3(R_THREADS),
                    0, static_cast<cudaStream_t>(stream), hq, hk, (uint32_t)q_heads,
                    (uint32_t)k_heads, (uint32_t)N, (uint32_t)units, total, (uint32_t)pairs,
                    (uint32_t)d, interleaved, inverse, pos, ladder);
}
