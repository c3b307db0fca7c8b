// Microscaled formats (blocks of 32 values along the last axis share a power-of-two scale):
// element conversions and the layout of the codes and scales of a tensor [rows, K].
//
//   element   E2M1 (4 bits, largest 6) or E4M3 (8 bits, largest 448); scale: the E8M0 byte b of
//             2^(b - 127), 255 = NaN
//   codes     rows of nb = ceil(K / 32) blocks: 16 bytes a block (E2M1, the even element in the
//             low four bits) or 32 bytes (E4M3); elements past K are zero
//   scales    groups of 512 bytes, one per 128 rows x 4 blocks, the groups of a row tile
//             consecutive: row r, block j is byte (r % 32) * 16 + (r % 128 / 32) * 4 + j % 4 of
//             group (r / 128) * ceil(nb / 4) + j / 4.  This is the order in which the tensor
//             core's block-scaled products want a tile's scales in tensor memory (lane r % 32,
//             32-bit column r % 128 / 32, byte j % 4), so a group goes there as it lies.
#pragma once

#include "common.cuh"

namespace snnb {
namespace mx {

constexpr int BLOCK = 32;
constexpr int GROUP_BYTES = 512;

template <int FMT> struct Fmt;
template <> struct Fmt<SNNB_MXFP4> {
    static constexpr int EMAX = 2;              // 6 = 1.5 * 2^2
    static constexpr int BLOCK_BYTES = 16;
    typedef uint32_t Codes8;                    // the codes of 8 elements
};
template <> struct Fmt<SNNB_MXFP8> {
    static constexpr int EMAX = 8;              // 448 = 1.75 * 2^8
    static constexpr int BLOCK_BYTES = 32;
    typedef uint2 Codes8;
};

__host__ __device__ __forceinline__ int64_t blocks_of(int64_t K) { return (K + BLOCK - 1) / BLOCK; }
__host__ __device__ __forceinline__ int64_t groups_of(int64_t K) { return (blocks_of(K) + 3) / 4; }

// Largest extents: indexes of blocks (rows padded to groups of 4) and of scale words stay below
// 2^31, byte offsets are 64-bit; row strides up to 2^40 elements in all.
inline bool sizes_ok(int64_t rows, int64_t K) {
    return rows >= 0 && K >= 1 && K <= 0x7fffffff - 255 && rows <= 0x7fffffff - 127 &&
           (rows + 127) * (groups_of(K) * 4) <= 0x7fffffff;
}
inline bool stride_ok(int64_t rows, int64_t ld) {
    return ld >= 0 && (rows <= 1 || ld <= (int64_t(1) << 40) / rows);
}

// 8 floats, already multiplied by the inverse scale, to codes: round to nearest, ties to even,
// magnitudes above the largest element become the largest.
__device__ __forceinline__ void encode8(const float (&v)[8], uint32_t& c) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(c)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
}
__device__ __forceinline__ void encode8(const float (&v)[8], uint2& c) {
    asm("{\n\t.reg .b16 h0, h1, h2, h3;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h0, %3, %2;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h1, %5, %4;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h2, %7, %6;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h3, %9, %8;\n\t"
        "mov.b32 %0, {h0, h1};\n\t"
        "mov.b32 %1, {h2, h3};\n\t}"
        : "=r"(c.x), "=r"(c.y)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
}

// Two float operations an instruction (each rounded as the scalar one is).
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// v = a * s.
__device__ __forceinline__ void scale8(const float (&a)[8], float s, float (&v)[8]) {
    const uint64_t ss = pack2(s, s);
#pragma unroll
    for (int i = 0; i < 8; i += 2) unpack2(mul2(pack2(a[i], a[i + 1]), ss), v[i], v[i + 1]);
}

// The values of 8 codes (exact: both element formats are subsets of f16).
__device__ __forceinline__ void halves_to_f32(uint32_t h, float& a, float& b) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    a = f.x;
    b = f.y;
}
__device__ __forceinline__ void decode8(uint32_t c, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(c));
#pragma unroll
    for (int i = 0; i < 4; ++i) halves_to_f32(h[i], v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ void decode8(uint2 c, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n\t.reg .b16 h0, h1, h2, h3;\n\t"
        "mov.b32 {h0, h1}, %4;\n\t"
        "mov.b32 {h2, h3}, %5;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, h0;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h1;\n\t"
        "cvt.rn.f16x2.e4m3x2 %2, h2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %3, h3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(c.x), "r"(c.y));
#pragma unroll
    for (int i = 0; i < 4; ++i) halves_to_f32(h[i], v[2 * i], v[2 * i + 1]);
}

// 2^(byte - 127); the value of byte 0 is subnormal, 255 is NaN.
__device__ __forceinline__ float scale_value(uint32_t byte) {
    const uint32_t bits = byte << 23;
    return __int_as_float((int)(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : bits));
}

// ---- quantising a block of 32 values held by 4 neighbouring lanes, 8 each ----------------
// Every lane of the warp calls.  The scale byte is floor(log2(largest magnitude)) - EMAX as an
// exponent: the exponent field of the largest magnitude's float minus EMAX, 0 for a block of
// zeros or float subnormals.  A block that holds an infinity or a NaN gets the byte 255 (NaN)
// and zero codes.

// The largest magnitude's exponent field among 8 values (255 where one is an infinity or NaN).
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint32_t top_exponent(const float (&x)[8]) {
    const float m = max_abs3(max_abs3(x[0], x[1], x[2]), max_abs3(x[3], x[4], x[5]),
                             max_abs3(x[6], x[7], x[7]));
    return ((uint32_t)__float_as_int(m) >> 23) & 255u;
}

// The same from the raw values.  bfloat16 has float's exponent field: compare pairs.
template <typename T> struct Raw8;
template <typename T>
__device__ __forceinline__ uint32_t top_exponent(const Raw8<T>&, const float (&x)[8]) {
    return top_exponent(x);
}
__device__ __forceinline__ uint32_t top_exponent(const Raw8<__nv_bfloat16>& r, const float (&x)[8]);

template <int FMT>
__device__ __forceinline__ uint32_t quantise_block(const float (&x)[8], uint32_t exponent,
                                                   typename Fmt<FMT>::Codes8& codes) {
    uint32_t e = max(exponent, __shfl_xor_sync(0xffffffffu, exponent, 1));
    e = max(e, __shfl_xor_sync(0xffffffffu, e, 2));
    const bool bad = e == 255;
    const uint32_t byte = bad ? 255u : (e > (uint32_t)Fmt<FMT>::EMAX ? e - Fmt<FMT>::EMAX : 0u);
    // 1 / scale = 2^(127 - byte), exact and normal (byte <= 252); a product that leaves the
    // normal range is far below the smallest element and rounds to zero either way
    const float inv = __int_as_float((int)((254u - byte) << 23));
    float v[8];
    scale8(x, inv, v);
    encode8(v, codes);
    if constexpr (FMT == SNNB_MXFP4) {
        codes = bad ? 0u : codes;
    } else {
        codes.x = bad ? 0u : codes.x;
        codes.y = bad ? 0u : codes.y;
    }
    return byte;
}

// The four scale bytes of 4 neighbouring blocks (16 lanes, one byte per 4 lanes) as one word,
// in every one of the 16 lanes; of a row of two blocks that 8 lanes hold, in those.
template <int LANES = 32>
__device__ __forceinline__ uint32_t join_scales(uint32_t byte, int lane) {
    uint32_t w = byte << (8 * ((lane >> 2) & (LANES >= 16 ? 3 : 1)));
    w |= __shfl_xor_sync(0xffffffffu, w, 4);
    if (LANES >= 16) w |= __shfl_xor_sync(0xffffffffu, w, 8);
    return w;
}

// Index of the 4-byte word of row `row`, group `g` along K (blocks 4 g .. 4 g + 3).
__device__ __forceinline__ uint32_t scale_word(uint32_t row, uint32_t g, uint32_t groups) {
    return ((row >> 7) * groups + g) * (GROUP_BYTES / 4) + (row & 31) * 4 + ((row >> 5) & 3);
}

// The scale bytes of rows past the tensor's last one, in its last row tile: zero.  All threads
// of the grid share the work.
__device__ __forceinline__ void zero_row_padding(uint32_t* scales, uint32_t rows, uint32_t groups,
                                                 uint64_t thread, uint64_t threads) {
    const uint32_t pad = (0u - rows) & 127u;
    for (uint64_t i = thread; i < (uint64_t)pad * groups; i += threads)
        scales[scale_word(rows + (uint32_t)(i % pad), (uint32_t)(i / pad), groups)] = 0;
}

// ---- 8 values of a row -------------------------------------------------------------------
template <typename T> struct Raw8 { uint4 v[sizeof(T) / 2]; };      // 16 bytes, 32 for float
__device__ __forceinline__ uint32_t top_exponent(const Raw8<__nv_bfloat16>& r, const float (&)[8]) {
    const uint32_t m = 0x7FFF7FFFu;
    const uint32_t t = __vmaxu2(__vmaxu2(r.v[0].x & m, r.v[0].y & m),
                                __vmaxu2(r.v[0].z & m, r.v[0].w & m));
    return max(t >> 16, t & 0xFFFFu) >> 7;
}

// Streaming 16-byte load: read once, not kept in L1.
__device__ __forceinline__ uint4 load16(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ float2 pair_f32(uint32_t u, const __half*) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
__device__ __forceinline__ float2 pair_f32(uint32_t u, const __nv_bfloat16*) {
    return make_float2(__int_as_float((int)(u << 16)), __int_as_float((int)(u & 0xFFFF0000u)));
}
template <typename T>
__device__ __forceinline__ void to_floats(const Raw8<T>& r, float (&v)[8]) {
    const uint32_t u[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = pair_f32(u[i], (const T*)nullptr);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
template <>
__device__ __forceinline__ void to_floats(const Raw8<float>& r, float (&v)[8]) {
    const uint32_t u[8] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w,
                           r.v[1].x, r.v[1].y, r.v[1].z, r.v[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __int_as_float((int)u[i]);
}

__device__ __forceinline__ uint32_t round_pair(float a, float b, const __half*) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t round_pair(float a, float b, const __nv_bfloat16*) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void from_floats(const float (&v)[8], Raw8<T>& r) {
    const T* t = nullptr;
    r.v[0] = make_uint4(round_pair(v[0], v[1], t), round_pair(v[2], v[3], t),
                        round_pair(v[4], v[5], t), round_pair(v[6], v[7], t));
}
template <>
__device__ __forceinline__ void from_floats(const float (&v)[8], Raw8<float>& r) {
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = (uint32_t)__float_as_int(v[i]);
    r.v[0] = make_uint4(u[0], u[1], u[2], u[3]);
    r.v[1] = make_uint4(u[4], u[5], u[6], u[7]);
}

// 16-byte aligned p.
template <typename T>
__device__ __forceinline__ Raw8<T> load_aligned8(const T* p) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = load16(reinterpret_cast<const uint4*>(p) + i);
    return r;
}
template <typename T>
__device__ __forceinline__ void store_aligned8(T* p, const Raw8<T>& r) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = r.v[i];
}
template <typename T>
__device__ __forceinline__ Raw8<T> zero8() {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = make_uint4(0, 0, 0, 0);
    return r;
}

// w[0 ..] shifted right by `bytes` (0 .. 15, a multiple of sizeof(T)) over its first N words.
template <typename T, int N>
__device__ __forceinline__ void shift_right(uint32_t (&w)[N + 4], uint32_t bytes) {
#pragma unroll
    for (int i = 0; i < N + 2; ++i) w[i] = bytes & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < N + 1; ++i) w[i] = bytes & 4 ? w[i + 1] : w[i];
    if (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (bytes & 2) * 8);
    }
}

// Whether aligned loads around a row's values may reach past its two ends: the bytes there belong
// to the tensor's span, from its first value to its last (gaps between its rows included).
struct RowEnds {
    bool before = false, after = false;
    __device__ __forceinline__ RowEnds() {}
    template <typename T>
    __device__ __forceinline__ RowEnds(const T* x, uint32_t rows, int64_t ld, uint32_t K, uint32_t row) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(x + (int64_t)row * ld);
        before = (at & ~uintptr_t(15)) >= reinterpret_cast<uintptr_t>(x);
        after = at + K * (uint64_t)sizeof(T) + 16 * (sizeof(T) / 2 + 1) <=
                reinterpret_cast<uintptr_t>(x + (int64_t)(rows - 1) * ld + K);
    }
};

// The values k .. k + 7 of a row of K at `row`, aligned to an element only; values past K are
// zero.  Two (float: three) aligned 16-byte loads around them, shifted into place, where those
// stay inside the row or the tensor's span; elsewhere one load per element.
template <typename T>
__device__ __forceinline__ Raw8<T> load_any8(const T* row, uint32_t k, uint32_t K, RowEnds ends = RowEnds()) {
    constexpr int W = (int)sizeof(T) * 2;                        // words of 8 values
    uint32_t w[W + 4];
    const T* p = row + k;
    if ((k >= 8 || ends.before) && (k + 16 <= K || ends.after)) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(p);
        const uint4* down = reinterpret_cast<const uint4*>(at & ~uintptr_t(15));
#pragma unroll
        for (int i = 0; i < W / 4 + 1; ++i) {
            const uint4 v = __ldg(down + i);
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
        shift_right<T, W>(w, (uint32_t)(at & 15));
        if (k + 8 > K) {                                         // the row's end
            const int n = (int)(K - k);
#pragma unroll
            for (int i = 0; i < W; ++i) {
                if (sizeof(T) == 4) w[i] = i < n ? w[i] : 0;
                else w[i] = 2 * i + 1 < n ? w[i] : 2 * i < n ? w[i] & 0xFFFFu : 0;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (k + i >= K) continue;
            if (sizeof(T) == 2)
                w[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(p) + i) << (16 * (i & 1));
            else
                w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
        }
    }
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < W / 4; ++i)
        r.v[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    return r;
}

// The counterpart store, of a whole warp in teams of TEAM lanes, one row each: a team's lane l
// holds 8 values for p (its own address, 8 l elements after lane 0's), the first n inside the row;
// lanes past a partial one have n <= 0.
// Aligned 16-byte pieces are put together from two neighbouring lanes, the one that holds a
// piece's first value stores it; what no whole piece covers goes out by elements.
template <typename T, int TEAM = 32>
__device__ __forceinline__ void store_any8(T* p, int n, const Raw8<T>& r, int lane) {
    constexpr int W = (int)sizeof(T) * 2;
    constexpr int PER = 16 / (int)sizeof(T);                     // elements of a piece
    uint32_t w[W], t[W + 4];                 // own words; with the next lane's first 4
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
        w[4 * i] = r.v[i].x; w[4 * i + 1] = r.v[i].y; w[4 * i + 2] = r.v[i].z; w[4 * i + 3] = r.v[i].w;
    }
#pragma unroll
    for (int i = 0; i < W; ++i) t[i] = w[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[W + i] = __shfl_down_sync(0xffffffffu, w[i], 1);
    const int next = max(0, __shfl_down_sync(0xffffffffu, n, 1));
    if (n <= 0) return;
    // elements before the first aligned address; the own and the next lane's values from there
    const int head = (int)((0u - (uint32_t)reinterpret_cast<uintptr_t>(p)) & 15u) / (int)sizeof(T);
    const int have = n < 8 ? n : 8 + ((lane & (TEAM - 1)) < TEAM - 1 ? next : 0);
    const int bytes = head * (int)sizeof(T);
    shift_right<T, W>(t, (uint32_t)bytes);
    int taken = head;
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
        if (head + (i + 1) * PER > have) continue;
        *reinterpret_cast<uint4*>(p + head + i * PER) =
            make_uint4(t[4 * i], t[4 * i + 1], t[4 * i + 2], t[4 * i + 3]);
        taken = head + (i + 1) * PER;
    }
    // the lane before stored [0, head) with its last piece, unless there is none or the values
    // here do not fill it
    const bool start = (lane & (TEAM - 1)) == 0 || n < head;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i >= n || !((i < head && start) || i >= taken)) continue;
        if (sizeof(T) == 2)
            reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        else
            reinterpret_cast<uint32_t*>(p)[i] = w[i];
    }
}

__device__ __forceinline__ void round_to(float v, float* p) { *p = v; }
__device__ __forceinline__ void round_to(float v, __half* p) { *p = __float2half_rn(v); }
__device__ __forceinline__ void round_to(float v, __nv_bfloat16* p) { *p = __float2bfloat16_rn(v); }

// n / d for n < 2^31 by a multiplication.
struct FastDiv {
    uint32_t d, mul, shift;
    FastDiv() = default;
    explicit FastDiv(uint32_t d_) : d(d_) {
        shift = 0;
        while (shift < 31 && (uint64_t(1) << shift) < d) ++shift;
        mul = (uint32_t)(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const {
        return (__umulhi(n, mul) + n) >> shift;
    }
};

}  // namespace mx
}  // namespace snnb
