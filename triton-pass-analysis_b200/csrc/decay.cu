// Linear attention with a decay for each head: whole sequences in chunks, and single tokens.
//
//   S_t = decay S_{t-1} + k_t v_t^T        state [dk, dv], float32
//   o_t = scale q_t S_t
//
// A chunk of C tokens with the state S before it, L_ij = decay^(i-j) for j <= i, else 0:
//
//   O  = scale ((Q K^T . L) V + diag(decay^(i+1)) Q S)
//   S' = decay^C S + K^T diag(decay^(C-1-j)) V
//
// Powers are formed in float64: they compound over the chunks.  This file has the form for every type
// and size on the CUDA cores, and the single token's; 16-bit inputs whose rows tensor maps can describe go
// to the tensor cores (decay_tc.cu).
#include "decay.cuh"

namespace snnb {
namespace {

using namespace decay;

constexpr int GC = 64;             // tokens of a chunk
constexpr int GV = 64;             // columns of the state that a thread block holds
constexpr int GP = GC + 4;         // floats of a row of a tile: 16-byte aligned, four banks on a row
constexpr int G_THREADS = 256;

struct AnyArgs {
    Args a;
    uint32_t tiles, items;         // of GV columns; of this launch
    int segs, cps;                 // segments of each sequence, chunks of a segment
    float* work;                   // [segs][B H tiles][dk][GV] states (slot segs - 1: the start)
};

__device__ __forceinline__ void fma44(float (&c)[4][4], const float4& a, const float4& b) {
    const float x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) c[i][j] = fmaf(x[i], y[j], c[i][j]);
}

// Every type, size and stride: products in float32 on the CUDA cores, 4 x 4 results a thread, from
// tiles in shared memory (two 16-byte loads for 16 products: bound by issue and shared memory, and by
// latency, at two blocks an SM).  A thread block takes a segment of a sequence, a head and GV
// columns.  3 x 1003 tokens x 6 heads of 64 and 96, float32: 56 us (with one result a thread at a time
// from chunks of 32 tokens 438; with fewer loads in flight, of the segments' states above all, 71; floor
// 1.9).  8 x 2048 x 16 of 64: 390 us, issue slots 61% busy, two thirds of them multiply-adds.
// STATES: only the states that the segments leave, each from zero (the first: from state_in).
template <typename T, bool STATES>
__global__ void __launch_bounds__(G_THREADS, 2) decay_any_kernel(const __grid_constant__ AnyArgs p) {
    extern __shared__ float4 sm4[];
    const Args& a = p.a;
    const int dk = a.dk, dkp = (dk + 3) / 4 * 4, t = threadIdx.x, warp = t >> 5, lane = t & 31;
    float* S = reinterpret_cast<float*>(sm4);      // [dkp][GP]
    float* k = S + dkp * GP;                       // [dkp][GP]: column-major, tokens along a row
    float* v = k + dkp * GP;                       // [GC][GP]
    float* q = v + GC * GP;                        // [dkp][GP], as k; then the scores, [GC][GP]
    float* pt = q;
    float* pw = q + (STATES ? 0 : max(dkp, GC) * GP);          // decay^0 .. decay^GC
    pdl_wait();
    pdl_trigger();
    const uint32_t rest = blockIdx.x / p.tiles, tile = blockIdx.x - rest * p.tiles;
    const uint32_t sb = rest / (uint32_t)a.H, h = rest - sb * (uint32_t)a.H;
    const uint32_t seg = sb / (uint32_t)a.B, b = sb - seg * (uint32_t)a.B, hk = h / (uint32_t)(a.H / a.Hk);
    const int c0 = tile * GV, nv = min(GV, a.dv - c0);
    const int64_t len = a.length(b), chunks = (len + GC - 1) / GC;
    const int64_t first = min((int64_t)seg * p.cps, chunks), count = min((int64_t)p.cps, chunks - first);
    const bool end = first + count == chunks && (count > 0 || seg == 0);
    const float lam = a.decay[h];
    const int last = count > 0 && first + count == chunks ? (int)(len - (chunks - 1) * GC) : GC;
    if (t <= GC) pw[t] = (float)power(lam, t);
    const int64_t bht = ((int64_t)b * a.H + h) * p.tiles + tile, slot = a.B * a.H * p.tiles * (int64_t)(dk * GV);
    float* work = p.work + bht * (dk * GV);
    const int64_t state = ((int64_t)b * a.H + h) * dk * a.dv + c0;
    // what there is before the first chunk
    {
        const double d = power(lam, p.cps * GC);
        const float fh = (float)d, fl = (float)(d - (double)fh);
        // AHEAD rows of a thread's column at a time, their loads in flight together
        constexpr int STEP = G_THREADS / GV, AHEAD = 16;
        const int c = t % GV;
        const bool own = seg == 0 && a.state_in;
        const float* from = !own ? work : !STATES && p.segs > 1 ? work + (p.segs - 1) * slot : a.state_in + state;
        const int64_t width = own && from == a.state_in + state ? a.dv : GV;
        for (int r0 = t / GV; r0 < dkp; r0 += AHEAD * STEP) {
            float x[AHEAD];
            auto get = [&](const float* at, int64_t width, float (&y)[AHEAD], bool any) {
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    const int r = r0 + i * STEP;
                    y[i] = any && r < dk && c < nv ? at[r * width + c] : 0.0f;
                }
            };
            get(from, width, x, own || (!STATES && seg > 0));
            for (uint32_t s = 1; !STATES && s < seg; ++s) {
                float y[AHEAD];
                get(work + s * slot, GV, y, true);
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) x[i] = fmaf(x[i], fh, fmaf(x[i], fl, y[i]));
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int r = r0 + i * STEP;
                if (r >= dkp) continue;
                // state_out may be state_in
                if (STATES && own && r < dk && c < nv) work[(p.segs - 1) * slot + r * GV + c] = x[i];
                S[r * GP + c] = x[i];
            }
        }
    }
    const double dc = power(lam, GC), dl = power(lam, last);
    const float ch = (float)dc, cl = (float)(dc - (double)ch), lh = (float)dl, ll = (float)(dl - (double)lh);
    const T* qg = static_cast<const T*>(a.q) + b * a.qs[0] + h * a.qs[2];
    const T* kg = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
    const T* vg = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2] + c0;
    T* og = static_cast<T*>(a.out) + ((int64_t)b * a.N * a.H + h) * a.dv + c0;
    const int64_t ld = a.H * a.dv;
    const int i0 = t / 16 * 4, j0 = t % 16 * 4;    // this thread's rows and columns
    const bool wide = a.dv % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % (4 * sizeof(T)) == 0;
    for (int64_t n = 0; n < count; ++n) {
        const int64_t n0 = (first + n) * GC;
        const int m = n + 1 == count ? last : GC;
        __syncthreads();
        bool bad = false;
        // a warp: eight tokens' rows, a column a lane, two columns of k and q in flight together with v's;
        // four tokens a store (single ones met four to a bank)
        const int mp = (m + 3) / 4 * 4;            // rows that are used
        constexpr int R = GC / (G_THREADS / 32);
        const T* kr = kg + n0 * a.ks[1];
        const T* qr = qg + n0 * a.qs[1];
        const T* vr = vg + n0 * a.vs[1];
        float z[GV / 32][R];
#pragma unroll
        for (int j = 0; j < GV / 32; ++j)
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int r = warp * R + i, c = lane + 32 * j;
                z[j][i] = r < m && c < nv ? to_f32(vr[r * a.vs[1] + c]) : 0.0f;
            }
        for (int l = lane; l < dkp; l += 64) {
            float x[2][R], y[2][R];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    const int r = warp * R + i, c = l + 32 * j;
                    const bool in = r < m && c < dk;
                    x[j][i] = in ? to_f32(kr[r * a.ks[1] + c]) : 0.0f;
                    if (!STATES) y[j][i] = in ? to_f32(qr[r * a.qs[1] + c]) * a.scale : 0.0f;
                }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int c = l + 32 * j;
                if (c >= dkp) continue;
#pragma unroll
                for (int i = 0; i < R; i += 4) {
                    const int at = c * GP + warp * R + i;
                    *reinterpret_cast<float4*>(k + at) = make_float4(x[j][i], x[j][i + 1], x[j][i + 2], x[j][i + 3]);
                    if (!STATES)
                        *reinterpret_cast<float4*>(q + at) = make_float4(y[j][i], y[j][i + 1], y[j][i + 2], y[j][i + 3]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < GV / 32; ++j)
#pragma unroll
            for (int i = 0; i < R; ++i) {
                bad |= !(fabsf(z[j][i]) <= 3.4028235e38f);
                v[(warp * R + i) * GP + lane + 32 * j] = z[j][i];
            }
        bad = __syncthreads_or(bad);
        if (!STATES) {
            float s[4][4] = {}, o[4][4] = {};
#pragma unroll 4
            for (int x = 0; x < (i0 < m ? dkp : 0); ++x) {
                const float4 qx = *reinterpret_cast<const float4*>(q + x * GP + i0);
                fma44(s, qx, *reinterpret_cast<const float4*>(k + x * GP + j0));
                fma44(o, qx, *reinterpret_cast<const float4*>(S + x * GP + j0));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][j] *= pw[i0 + i + 1];
            __syncthreads();
#pragma unroll
            for (int j = 0; j < 4; ++j) {          // later tokens count nothing, whatever their scores
                float y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = j0 + j <= i0 + i ? s[i][j] * pw[i0 + i - j0 - j] : 0.0f;
                *reinterpret_cast<float4*>(pt + (j0 + j) * GP + i0) = make_float4(y[0], y[1], y[2], y[3]);
            }
            __syncthreads();
            if (!bad) {
#pragma unroll 4
                for (int x = 0; x < (i0 < m ? i0 + 4 : 0); ++x)
                    fma44(o, *reinterpret_cast<const float4*>(pt + x * GP + i0),
                          *reinterpret_cast<const float4*>(v + x * GP + j0));
            } else {                               // 0 * inf would reach rows before the infinity
                for (int x = 0; x < i0 + 4; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (x <= i0 + i)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                o[i][j] = fmaf(pt[x * GP + i0 + i], v[x * GP + j0 + j], o[i][j]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                T y[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) mx::round_to(i0 + i < m ? o[i][j] : 0.0f, y + j);
                T* to = og + (n0 + i0 + i) * ld + j0;
                if (n0 + i0 + i >= a.N || j0 >= nv) continue;
                if (wide) {
                    struct alignas(4 * sizeof(T)) Four { T x[4]; };
                    *reinterpret_cast<Four*>(to) = {{y[0], y[1], y[2], y[3]}};
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (j0 + j < nv) to[j] = y[j];
                }
            }
            __syncthreads();
        }
        // the rows of v by what is left of them at the chunk's end
        for (int i = t; i < m * GV; i += G_THREADS) v[i / GV * GP + i % GV] *= pw[m - 1 - i / GV];
        __syncthreads();
        const float fh = m == GC ? ch : lh, fl = m == GC ? cl : ll;
        for (int r = i0; r < dkp; r += 64) {
            float s[4][4] = {};
#pragma unroll 4
            for (int x = 0; x < mp; x += 4) {
                float4 kk[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) kk[i] = *reinterpret_cast<const float4*>(k + (r + i) * GP + x);
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const float4 vv = *reinterpret_cast<const float4*>(v + (x + y) * GP + j0);
                    const float* k0 = reinterpret_cast<const float*>(&kk[0]);
                    fma44(s, make_float4(k0[y], k0[4 + y], k0[8 + y], k0[12 + y]), vv);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float& x = S[(r + i) * GP + j0 + j];
                    x = fmaf(x, fh, fmaf(x, fl, s[i][j]));
                }
        }
    }
    if (!STATES && end) {                          // rows behind the last chunk
        for (int64_t n = chunks * GC + warp; n < a.N; n += G_THREADS / 32)
            for (int c = lane; c < nv; c += 32) mx::round_to(0.0f, og + n * ld + c);
    }
    __syncthreads();
    if (STATES || (end && a.state_out)) {
        for (int i = t; i < dk * GV; i += G_THREADS) {
            const int r = i / GV, c = i % GV;
            if (c >= nv) continue;
            if (STATES) work[seg * slot + r * GV + c] = S[r * GP + c];
            else a.state_out[state + (int64_t)r * a.dv + c] = S[r * GP + c];
        }
    }
}

// As for the tensor cores' form; a chunk of 64 tokens at 64 columns of k takes 19 us for the two blocks of
// an SM (5 for one in the pass before), both in proportion to dk.
int any_segments(int64_t items, int64_t chunks, int64_t dk) {
    const int64_t slots = dk <= 64 ? 296 : 148;
    int best = 1;
    int64_t least = 0;
    for (int n = 1; n <= 16 && (n == 1 || (chunks >= 2 * n && items <= slots)); ++n) {
        const int64_t cps = (chunks + n - 1) / n;
        if ((n - 1) * cps >= chunks) continue;
        const int64_t rounds = (items * n + slots - 1) / slots, before = (items * (n - 1) + slots - 1) / slots;
        const int64_t t = rounds * (cps * dk + 40) + before * (cps * dk / 4 + 40) + (n > 1 ? 60 : 0);
        if (n == 1 || t < least) {
            best = n;
            least = t;
        }
    }
    return best;
}
int64_t any_workspace(int64_t B, int64_t N, int64_t H, int64_t dk, int64_t dv) {
    const int64_t items = B * H * ((dv + GV - 1) / GV);
    const int segs = any_segments(items, (N + GC - 1) / GC, dk);
    return segs > 1 ? segs * items * dk * GV * 4 : 0;
}

constexpr int any_smem(int dk, bool states) {
    const int dkp = (dk + 3) / 4 * 4;
    return ((2 * dkp + (states ? 0 : dkp > GC ? dkp : GC) + GC) * GP + GC + 4) * 4;
}
static_assert(any_smem(MAX_DIM, false) <= 227 * 1024, "shared memory");
template <typename T, bool STATES>
int launch_any(AnyArgs p, cudaStream_t s) {
    // once per device, at the most that any call asks for
    if (const int st = allow_smem<decay_any_kernel<T, STATES>>(any_smem(MAX_DIM, STATES))) return st;
    p.items = (uint32_t)(p.a.B * p.a.H * p.tiles * (STATES ? p.segs - 1 : p.segs));
    return launch_k(decay_any_kernel<T, STATES>, dim3(p.items), dim3(G_THREADS), any_smem(p.a.dk, STATES), s, p);
}
template <typename T>
int run_any(const Args& a, void* work, int64_t bytes, cudaStream_t s) {
    const uint32_t tiles = (a.dv + GV - 1) / GV;
    const int64_t chunks = (a.N + GC - 1) / GC;
    const int segs = any_segments(a.B * a.H * tiles, chunks, a.dk);
    if (segs > 1 && (!work || !aligned16(work) || bytes < any_workspace(a.B, a.N, a.H, a.dk, a.dv)))
        return SNNB_ERR_ARG;
    const AnyArgs p = {a, tiles, 0, segs, (int)((chunks + segs - 1) / segs), static_cast<float*>(work)};
    if (segs > 1)
        if (const int st = launch_any<T, true>(p, s)) return st;
    return launch_any<T, false>(p, s);
}

// One token of each sequence: a thread block per sequence, head and ST_V columns of its state,
// which it reads and writes once.
constexpr int ST_THREADS = 256;
constexpr int ST_V = 32;

template <typename T>
__global__ void __launch_bounds__(ST_THREADS) decay_step_kernel(Args a, uint32_t tiles) {
    __shared__ float q[MAX_DIM], k[MAX_DIM], part[ST_THREADS / ST_V][ST_V];
    pdl_wait();
    pdl_trigger();
    const uint32_t tile = blockIdx.x % tiles, bh = blockIdx.x / tiles;
    const int64_t b = bh / a.H, h = bh - b * a.H, hk = h / (a.H / a.Hk);
    const int t = threadIdx.x, c = tile * ST_V + t % ST_V, r0 = t / ST_V;
    const T* qg = static_cast<const T*>(a.q) + b * a.qs[0] + h * a.qs[2];
    const T* kg = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
    for (int i = t; i < a.dk; i += ST_THREADS) {
        q[i] = to_f32(qg[i]) * a.scale;
        k[i] = to_f32(kg[i]);
    }
    __syncthreads();
    float s = 0.0f;
    if (c < a.dv) {
        const float v = to_f32(static_cast<const T*>(a.v)[b * a.vs[0] + hk * a.vs[2] + c]);
        const float l = a.decay[h];
        const int64_t base = (b * a.H + h) * a.dk * a.dv + c;
        for (int r = r0; r < a.dk; r += ST_THREADS / ST_V) {
            const float old = a.state_in ? a.state_in[base + (int64_t)r * a.dv] : 0.0f;
            const float x = l * old + k[r] * v;
            if (a.state_out) a.state_out[base + (int64_t)r * a.dv] = x;
            s += q[r] * x;
        }
    }
    part[r0][t % ST_V] = s;
    __syncthreads();
    if (t < ST_V && c < a.dv) {
        for (int i = 1; i < ST_THREADS / ST_V; ++i) s += part[i][t];
        mx::round_to(s, static_cast<T*>(a.out) + (b * a.H + h) * a.dv + c);
    }
}

// The same in float4s: LANES of them along a row of the state, as many rows at a time as the block
// has threads for, eight of a thread's in flight before q and k are there.  Bound: HBM, which the state
// crosses twice.  64 sequences x 32 heads of 128 x 128: 42.6 us, 6.3 TB/s (single floats: 86 us).
template <typename T, int LANES>
__global__ void __launch_bounds__(ST_THREADS) decay_step_vec_kernel(Args a, uint32_t tiles) {
    constexpr int ROWS = ST_THREADS / LANES, AHEAD = 8;
    __shared__ float q[MAX_DIM], k[MAX_DIM];
    __shared__ float4 part[ROWS][LANES];
    pdl_wait();
    pdl_trigger();
    const uint32_t bh = blockIdx.x / tiles, tile = blockIdx.x - bh * tiles;
    const uint32_t b = bh / (uint32_t)a.H, h = bh - b * (uint32_t)a.H, hk = h / (uint32_t)(a.H / a.Hk);
    const int t = threadIdx.x, c = (tile * LANES + t % LANES) * 4, r0 = t / LANES;
    const bool in = c < a.dv;
    const int64_t base = (int64_t)bh * a.dk * a.dv + c;
    const float* from = a.state_in + base;
    float* to = a.state_out + base;
    float4 x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
        x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (in && a.state_in && r0 + i * ROWS < a.dk)
            x[i] = *reinterpret_cast<const float4*>(from + (int64_t)(r0 + i * ROWS) * a.dv);
    }
    const T* qg = static_cast<const T*>(a.q) + b * a.qs[0] + h * a.qs[2];
    const T* kg = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
    if (t < a.dk) {
        q[t] = to_f32(qg[t]) * a.scale;
        k[t] = to_f32(kg[t]);
    }
    float v[4] = {};
    if (in) {
        const T* vg = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2] + c;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = to_f32(vg[j]);
    }
    const float l = a.decay[h];
    __syncthreads();
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int r = r0; r < a.dk; r += AHEAD * ROWS) {
        if (r != r0) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                if (in && a.state_in && r + i * ROWS < a.dk)
                    x[i] = *reinterpret_cast<const float4*>(from + (int64_t)(r + i * ROWS) * a.dv);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int n = r + i * ROWS;
            if (!in || n >= a.dk) continue;
            const float kn = k[n], qn = q[n];
            x[i] = make_float4(l * x[i].x + kn * v[0], l * x[i].y + kn * v[1], l * x[i].z + kn * v[2],
                               l * x[i].w + kn * v[3]);
            if (a.state_out) *reinterpret_cast<float4*>(to + (int64_t)n * a.dv) = x[i];
            s.x += qn * x[i].x; s.y += qn * x[i].y; s.z += qn * x[i].z; s.w += qn * x[i].w;
        }
    }
    part[r0][t % LANES] = s;
    __syncthreads();
    if (t < 4 * LANES) {                             // a column a thread
        const int col = tile * LANES * 4 + t;
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) y += reinterpret_cast<const float*>(part[i])[t];
        if (col < a.dv) mx::round_to(y, static_cast<T*>(a.out) + (int64_t)bh * a.dv + col);
    }
}

template <typename T>
int run_step(const Args& a, cudaStream_t s) {
    if (a.dv % 4 == 0 && aligned16(a.state_in) && aligned16(a.state_out)) {
        // rows as wide as the state's, up to 128 columns; narrower where that leaves SMs idle
        int lanes = 32;
        while (lanes > 8 && lanes * 2 >= a.dv) lanes /= 2;
        auto blocks = [&](int n) { return a.B * a.H * ((a.dv + 4 * n - 1) / (4 * n)); };
        while (lanes > 8 && blocks(lanes) < 148) lanes /= 2;
        const uint32_t tiles = (a.dv + 4 * lanes - 1) / (4 * lanes);
        auto k = lanes == 32   ? decay_step_vec_kernel<T, 32>
                 : lanes == 16 ? decay_step_vec_kernel<T, 16>
                               : decay_step_vec_kernel<T, 8>;
        return launch_k(k, dim3((unsigned)blocks(lanes)), dim3(ST_THREADS), 0, s, a, tiles);
    }
    const uint32_t tiles = (a.dv + ST_V - 1) / ST_V;
    return launch_k(decay_step_kernel<T>, dim3((unsigned)(a.B * a.H * tiles)), dim3(ST_THREADS), 0,
                    s, a, tiles);
}

bool heads_ok(int dtype, int64_t B, int64_t H, int64_t Hk, int64_t dk, int64_t dv) {
    return (dtype == SNNB_F32 || dtype == SNNB_F16 || dtype == SNNB_BF16) && B >= 0 && H >= 1 &&
           Hk >= 1 && H % Hk == 0 && dk >= 1 && dk <= MAX_DIM && dv >= 1 && dv <= MAX_DIM &&
           H <= 0x7fffff && B <= 0x7fffffff / (H * 8);
}
bool element_aligned(const void* p, int dtype) {
    return reinterpret_cast<uintptr_t>(p) % (dtype == SNNB_F32 ? 4 : 2) == 0;
}

}  // namespace
}  // namespace snnb

using namespace snnb;

extern "C" int64_t snnb_decay_attention_workspace_bytes(int dtype, int64_t B, int64_t N, int64_t H,
                                                        int64_t dk, int64_t dv) {
    if (!heads_ok(dtype, B, H, H, dk, dv) || N < 0 || N > MOST_TOKENS) return -1;
    if (B == 0 || N == 0) return 0;
    // strides and alignment decide between the forms
    const int64_t tc = decay::tc_workspace(dtype, B, N, H, dk, dv), any = any_workspace(B, N, H, dk, dv);
    return tc > any ? tc : any;
}

extern "C" int snnb_decay_attention(const void* q, const int64_t* q_strides, const void* k,
                                    const int64_t* k_strides, const void* v,
                                    const int64_t* v_strides, int dtype, int64_t B, int64_t N,
                                    int64_t H, int64_t Hkv, int64_t dk, int64_t dv,
                                    const float* decay, float scale, const float* state_in,
                                    const void* lengths, int lengths_dtype, void* out,
                                    float* state_out, void* workspace, int64_t workspace_bytes,
                                    snnb_stream_t stream) {
    if (const int inj = take_injected_status()) return inj;
    if (!heads_ok(dtype, B, H, Hkv, dk, dv) || N < 0 || N > MOST_TOKENS) return SNNB_ERR_ARG;
    if (N > (int64_t(1) << 40) / (H * dv) / (B ? B : 1)) return SNNB_ERR_ARG;
    if (lengths && lengths_dtype != 0 && lengths_dtype != 1) return SNNB_ERR_ARG;
    if (B == 0) return SNNB_OK;
    if (!decay || (N && (!q || !k || !v || !out || !q_strides || !k_strides || !v_strides)))
        return SNNB_ERR_ARG;
    for (const void* p : {q, k, v, (const void*)out})
        if (!element_aligned(p, dtype)) return SNNB_ERR_ARG;
    for (const void* p : {(const void*)decay, (const void*)state_in, (const void*)state_out})
        if (reinterpret_cast<uintptr_t>(p) % 4) return SNNB_ERR_ARG;
    if (reinterpret_cast<uintptr_t>(lengths) % (lengths_dtype ? 8 : 4)) return SNNB_ERR_ARG;
    Args a = {q, k, v, out, {0, 0, 0}, {0, 0, 0}, {0, 0, 0}, B, N, H, Hkv, (int)dk, (int)dv, decay,
              scale, state_in, state_out, lengths, lengths_dtype};
    for (int i = 0; i < 3 && N; ++i) {
        a.qs[i] = q_strides[i];
        a.ks[i] = k_strides[i];
        a.vs[i] = v_strides[i];
    }
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (N == 1 && !lengths) {                      // one token: no chunk
        if (dtype == SNNB_F32) return run_step<float>(a, s);
        if (dtype == SNNB_F16) return run_step<__half>(a, s);
        return run_step<__nv_bfloat16>(a, s);
    }
    // The tensor cores, where they take the arguments, whatever the length: bf16, 8 heads of 64, 2 tokens 6.0 us (on
    // the CUDA cores 8.7), 64 6.1 (14.2), 128 6.2 (25.5); 256 heads of 64, 2 tokens 12.0 (10.8), 9 12.1 (13.0).
    if (tc_takes(a, dtype)) return tc_run(a, dtype, workspace, workspace_bytes, s);
    if (dtype == SNNB_F32) return run_any<float>(a, workspace, workspace_bytes, s);
    if (dtype == SNNB_F16) return run_any<__half>(a, workspace, workspace_bytes, s);
    return run_any<__nv_bfloat16>(a, workspace, workspace_bytes, s);
}

extern "C" int snnb_decay_attention_step(const void* q, const int64_t* q_strides, const void* k,
                                         const int64_t* k_strides, const void* v,
                                         const int64_t* v_strides, int dtype, int64_t B, int64_t H,
                                         int64_t Hkv, int64_t dk, int64_t dv, const float* decay,
                                         float scale, const float* state_in, void* out,
                                         float* state_out, snnb_stream_t stream) {
    if (const int inj = take_injected_status()) return inj;
    if (!heads_ok(dtype, B, H, Hkv, dk, dv)) return SNNB_ERR_ARG;
    if (B == 0) return SNNB_OK;
    if (!q || !k || !v || !out || !q_strides || !k_strides || !v_strides || !decay || !state_in ||
        !state_out)
        return SNNB_ERR_ARG;
    for (const void* p : {q, k, v, (const void*)out})
        if (!element_aligned(p, dtype)) return SNNB_ERR_ARG;
    for (const void* p : {(const void*)decay, (const void*)state_in, (const void*)state_out})
        if (reinterpret_cast<uintptr_t>(p) % 4) return SNNB_ERR_ARG;
    const Args a = {q, k, v, out, {q_strides[0], 0, q_strides[1]}, {k_strides[0], 0, k_strides[1]},
                    {v_strides[0], 0, v_strides[1]}, B, 1, H, Hkv, (int)dk, (int)dv, decay, scale,
                    state_in, state_out, nullptr, 0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == SNNB_F32) return run_step<float>(a, s);
    if (dtype == SNNB_F16) return run_step<__half>(a, s);
    return run_step<__nv_bfloat16>(a, s);
}
