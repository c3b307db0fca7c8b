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
    if (byte == 255) return __int_as_float(0x7FC00000);
    return byte == 0 ? __int_as_float(0x00400000) : __int_as_float((int)(byte << 23));
}

// One block of 32 values held by 4 neighbouring lanes, 8 each: the scale byte is
// floor(log2(largest magnitude)) - EMAX as an exponent, i.e. the exponent field of the largest
// magnitude's float minus EMAX (0 for a block of zeros or float subnormals).  A block that holds
// an infinity or a NaN gets the byte 255 (NaN) and zero codes.  Every lane of the warp calls.
template <int FMT>
__device__ __forceinline__ uint32_t quantise_block(const float (&x)[8],
                                                   typename Fmt<FMT>::Codes8& codes) {
    // magnitudes compare as integers, and an infinity or NaN is above every finite value
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, (uint32_t)__float_as_int(x[i]) & 0x7FFFFFFFu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t e = top >> 23;
    const uint32_t byte = e == 255 ? 255u : (e > (uint32_t)Fmt<FMT>::EMAX ? e - Fmt<FMT>::EMAX : 0u);
    // 1 / scale = 2^(127 - byte), exact and normal for byte <= 253; a product that leaves the
    // normal range is far below the smallest element and rounds to zero either way
    const float inv = __int_as_float((int)((254u - byte) << 23));
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = byte == 255 ? 0.0f : x[i] * inv;
    encode8(v, codes);
    return byte;
}

// The four scale bytes of 4 neighbouring blocks (16 lanes, one byte per 4 lanes) as one word,
// in every one of the 16 lanes.
__device__ __forceinline__ uint32_t join_scales(uint32_t byte, int lane) {
    uint32_t w = byte << (8 * ((lane >> 2) & 3));
    w |= __shfl_xor_sync(0xffffffffu, w, 4);
    w |= __shfl_xor_sync(0xffffffffu, w, 8);
    return w;
}

// Index of the 4-byte word of row `row`, group `g` along K (blocks 4 g .. 4 g + 3).
__device__ __forceinline__ int64_t scale_word(int64_t row, int64_t g, int64_t groups) {
    return ((row >> 7) * groups + g) * (GROUP_BYTES / 4) + (row & 31) * 4 + ((row >> 5) & 3);
}

// Walks the blocks of a tensor: block index q = row * per_row + j, advanced by a fixed step
// with one division at the start.
struct BlockWalk {
    int64_t row, j, drow, dj, per_row;
    __device__ BlockWalk(int64_t q, int64_t step, int64_t per_row_) : per_row(per_row_) {
        row = q / per_row;
        j = q - row * per_row;
        drow = step / per_row;
        dj = step - drow * per_row;
    }
    __device__ void next() {
        row += drow;
        j += dj;
        if (j >= per_row) {
            j -= per_row;
            ++row;
        }
    }
};

// The scale bytes of rows past the tensor's last one, in its last row tile: zero.
__device__ __forceinline__ void zero_row_padding(uint32_t* scales, int64_t rows, int64_t groups,
                                                 int64_t thread, int64_t threads) {
    const int64_t pad = ((rows + 127) & ~int64_t(127)) - rows;
    const int64_t words = pad * groups;
    if (thread >= words) return;
    for (BlockWalk w(thread, threads, groups); w.row < pad; w.next())
        scales[scale_word(rows + w.row, w.j, groups)] = 0;
}

// 8 consecutive elements at p as floats; `n` of them lie inside the row (0..8; the others read
// as zero).  VEC: p is 16-byte aligned and n is 0 or 8.
template <bool VEC>
__device__ __forceinline__ void load8(const float* p, int n, float (&v)[8]) {
    if (VEC) {
        float4 a = make_float4(0, 0, 0, 0), b = a;
        if (n > 0) {
            a = __ldg(reinterpret_cast<const float4*>(p));
            b = __ldg(reinterpret_cast<const float4*>(p) + 1);
        }
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? __ldg(p + i) : 0.0f;
    }
}
__device__ __forceinline__ float2 pair_f32(uint32_t u, const __half*) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
__device__ __forceinline__ float2 pair_f32(uint32_t u, const __nv_bfloat16*) {
    return make_float2(__int_as_float((int)(u << 16)), __int_as_float((int)(u & 0xFFFF0000u)));
}
template <bool VEC, typename T>
__device__ __forceinline__ void load8(const T* p, int n, float (&v)[8]) {
    if (VEC) {
        uint4 a = make_uint4(0, 0, 0, 0);
        if (n > 0) a = __ldg(reinterpret_cast<const uint4*>(p));
        const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = pair_f32(u[i], p);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.0f;
    }
}

__device__ __forceinline__ uint32_t round_pair(float a, float b, const __half*) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t round_pair(float a, float b, const __nv_bfloat16*) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void round_to(float v, float* p) { *p = v; }
__device__ __forceinline__ void round_to(float v, __half* p) { *p = __float2half_rn(v); }
__device__ __forceinline__ void round_to(float v, __nv_bfloat16* p) { *p = __float2bfloat16_rn(v); }

template <bool VEC>
__device__ __forceinline__ void store8(float* p, int n, const float (&v)[8]) {
    if (VEC) {
        if (n > 0) {
            reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = v[i];
    }
}
template <bool VEC, typename T>
__device__ __forceinline__ void store8(T* p, int n, const float (&v)[8]) {
    if (VEC) {
        if (n > 0)
            *reinterpret_cast<uint4*>(p) =
                make_uint4(round_pair(v[0], v[1], p), round_pair(v[2], v[3], p),
                           round_pair(v[4], v[5], p), round_pair(v[6], v[7], p));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) round_to(v[i], p + i);
    }
}

}  // namespace mx
}  // namespace snnb
