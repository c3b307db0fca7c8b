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
// Powers come from a table that float64 fills: they compound over the chunks.
#include "decay.cuh"

namespace snnb {
namespace {

using namespace decay;

constexpr int GC = 32;             // tokens of a chunk
constexpr int GV = 32;             // columns of the state that a thread block holds
constexpr int G_THREADS = 256;

// Every type, size and stride: products in float32 on the CUDA cores, a thread block per
// sequence, head and GV columns of its state.
template <typename T>
__global__ void __launch_bounds__(G_THREADS) decay_any_kernel(Args a, uint32_t tiles) {
    extern __shared__ float sm[];
    const int dk = a.dk;
    float* S = sm;                                 // [dk][GV]
    float* q = S + dk * GV;                        // [GC][dk + 1]
    float* k = q + GC * (dk + 1);
    float* v = k + GC * (dk + 1);                  // [GC][GV]
    float* p = v + GC * GV;                        // [GC][GC + 1]
    float* pw = p + GC * (GC + 1);                 // [GC + 1]
    pdl_wait();
    pdl_trigger();
    const uint32_t tile = blockIdx.x % tiles, bh = blockIdx.x / tiles;
    const int64_t b = bh / a.H, h = bh - b * a.H, hk = h / (a.H / a.Hk);
    const int c0 = tile * GV, nv = min(GV, a.dv - c0), t = threadIdx.x;
    const int64_t len = a.length(b);
    if (t <= GC) pw[t] = (float)power(a.decay[h], t);
    const float* s_in = a.state_in ? a.state_in + (b * a.H + h) * dk * a.dv + c0 : nullptr;
    for (int i = t; i < dk * GV; i += G_THREADS)
        S[i] = s_in && i % GV < nv ? s_in[(int64_t)(i / GV) * a.dv + i % GV] : 0.0f;
    const T* qg = static_cast<const T*>(a.q) + b * a.qs[0] + h * a.qs[2];
    const T* kg = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
    const T* vg = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2] + c0;
    T* og = static_cast<T*>(a.out) + (b * a.N * a.H + h) * a.dv + c0;
    for (int64_t n0 = 0; n0 < a.N; n0 += GC) {
        const int m = (int)max((int64_t)0, min((int64_t)GC, len - n0));
        if (m == 0) {                              // rows behind the sequence
            const int left = (int)min((int64_t)GC, a.N - n0);
            for (int i = t; i < left * GV; i += G_THREADS)
                if (i % GV < nv) mx::round_to(0.0f, og + (n0 + i / GV) * a.H * a.dv + i % GV);
            continue;
        }
        __syncthreads();
        for (int i = t; i < GC * dk; i += G_THREADS) {
            const int r = i / dk, c = i - r * dk;
            q[r * (dk + 1) + c] = r < m ? to_f32(qg[(n0 + r) * a.qs[1] + c]) * a.scale : 0.0f;
            k[r * (dk + 1) + c] = r < m ? to_f32(kg[(n0 + r) * a.ks[1] + c]) : 0.0f;
        }
        for (int i = t; i < GC * GV; i += G_THREADS) {
            const int r = i / GV, c = i % GV;
            v[i] = r < m && c < nv ? to_f32(vg[(n0 + r) * a.vs[1] + c]) : 0.0f;
        }
        __syncthreads();
        for (int i = t; i < GC * GC; i += G_THREADS) {
            const int r = i / GC, c = i % GC;
            float s = 0.0f;
            if (c <= r) {
                for (int x = 0; x < dk; ++x) s += q[r * (dk + 1) + x] * k[c * (dk + 1) + x];
                s *= pw[r - c];
            }
            p[r * (GC + 1) + c] = s;
        }
        __syncthreads();
        for (int i = t; i < GC * GV; i += G_THREADS) {
            const int r = i / GV, c = i % GV;
            float s = 0.0f;
            for (int x = 0; x < dk; ++x) s += q[r * (dk + 1) + x] * S[x * GV + c];
            s *= pw[r + 1];
            for (int x = 0; x <= r; ++x) s += p[r * (GC + 1) + x] * v[x * GV + c];
            if (n0 + r < a.N && c < nv)
                mx::round_to(r < m ? s : 0.0f, og + (n0 + r) * a.H * a.dv + c);
        }
        __syncthreads();
        for (int i = t; i < dk * GV; i += G_THREADS) {
            const int r = i / GV, c = i % GV;
            float s = pw[m] * S[i];
            for (int x = 0; x < m; ++x) s += pw[m - 1 - x] * k[x * (dk + 1) + r] * v[x * GV + c];
            S[i] = s;
        }
    }
    if (a.state_out) {
        float* s_out = a.state_out + (b * a.H + h) * dk * a.dv + c0;
        __syncthreads();
        for (int i = t; i < dk * GV; i += G_THREADS)
            if (i % GV < nv) s_out[(int64_t)(i / GV) * a.dv + i % GV] = S[i];
    }
}

template <typename T>
int run_any(const Args& a, cudaStream_t s) {
    const uint32_t tiles = (a.dv + GV - 1) / GV;
    const size_t smem = (size_t)(a.dk * GV + 2 * GC * (a.dk + 1) + GC * GV + GC * (GC + 1) + GC + 1) * 4;
    auto k = decay_any_kernel<T>;
    // once per device, at the most that any call asks for
    if (const int st = allow_smem<decay_any_kernel<T>>(
            (MAX_DIM * GV + 2 * GC * (MAX_DIM + 1) + GC * GV + GC * (GC + 1) + GC + 1) * 4))
        return st;
    return launch_k(k, dim3((unsigned)(a.B * a.H * tiles)), dim3(G_THREADS), smem, s, a, tiles);
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
            const float x = l * a.state_in[base + (int64_t)r * a.dv] + k[r] * v;
            a.state_out[base + (int64_t)r * a.dv] = x;
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
// has threads for, eight of a thread's in flight before q and k are there.
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
    for (int i = 0; i < AHEAD; ++i)
        if (in && r0 + i * ROWS < a.dk)
            x[i] = *reinterpret_cast<const float4*>(from + (int64_t)(r0 + i * ROWS) * a.dv);
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
                if (in && r + i * ROWS < a.dk)
                    x[i] = *reinterpret_cast<const float4*>(from + (int64_t)(r + i * ROWS) * a.dv);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int n = r + i * ROWS;
            if (!in || n >= a.dk) continue;
            const float kn = k[n], qn = q[n];
            x[i] = make_float4(l * x[i].x + kn * v[0], l * x[i].y + kn * v[1], l * x[i].z + kn * v[2],
                               l * x[i].w + kn * v[3]);
            *reinterpret_cast<float4*>(to + (int64_t)n * a.dv) = x[i];
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
    if (!heads_ok(dtype, B, H, H, dk, dv) || N < 0) return -1;
    return decay::tc_workspace(dtype, B, N, H, dk, dv);
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
    if (!heads_ok(dtype, B, H, Hkv, dk, dv) || N < 0) return SNNB_ERR_ARG;
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
    if (tc_takes(a, dtype)) return tc_run(a, dtype, workspace, workspace_bytes, s);
    if (dtype == SNNB_F32) return run_any<float>(a, s);
    if (dtype == SNNB_F16) return run_any<__half>(a, s);
    return run_any<__nv_bfloat16>(a, s);
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
