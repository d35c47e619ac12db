// What the layers of the network operators share: 16-bit conversions, activations, row stores.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace p2b {

int sm_count();

enum Activation { kGelu = 0, kSilu = 1, kNoActivation = 2 };

inline int64_t blocks_of(int64_t n, int64_t size) { return (n + size - 1) / size; }
// 16-bit rows `stride` elements apart that all start on 16-byte boundaries
inline bool aligned16(const void* p, int64_t stride) { return ((uintptr_t)p % 16) == 0 && stride % 8 == 0; }

template <bool kBf16> __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    if (kBf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool kBf16> __device__ __forceinline__ float2 unpack(uint32_t v) {
    if (kBf16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <bool kBf16> __device__ __forceinline__ float widen(uint16_t v) {
    if (kBf16) return __uint_as_float((uint32_t)v << 16);
    return __half2float(__ushort_as_half(v));
}
template <bool kBf16> __device__ __forceinline__ uint16_t narrow(float v) { return (uint16_t)pack<kBf16>(v, 0.0f); }

__device__ __forceinline__ float power_of_two(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 numbers in one register pair: an instruction works on both.
struct Two {
    uint64_t v;
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ Two(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
    __device__ __forceinline__ explicit Two(float both) : Two(both, both) {}
    __device__ __forceinline__ float2 apart() const {
        float2 r;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
        return r;
    }
};
__device__ __forceinline__ Two operator+(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
template <bool kBf16> __device__ __forceinline__ Two two_of(uint32_t word) {
    const float2 f = unpack<kBf16>(word);
    return Two(f.x, f.y);
}

// act(z), and act'(z) where asked for.  The normal distribution of the gelu is Abramowitz and Stegun 7.1.26 (off by 1.5e-7 at
// most), about half the instructions of erff, whose exponential is the density that the slope needs.  The epilogues of the
// layers last as long as their instructions: with erff a 128 x 128 tile took 14,000 clocks beside 12,300 of products.
template <int kActivation, bool kSlope> __device__ __forceinline__ Two activate(Two z, Two& slope) {
    if (kActivation == kNoActivation) {
        slope = Two(1.0f);
        return z;
    }
    const float2 zs = z.apart();
    if (kActivation == kGelu) {
        const float2 power = (z * z * Two(-0.72134752044448170f)).apart();
        const Two density(power_of_two(power.x), power_of_two(power.y));  // exp(-z^2 / 2)
        const float2 below_t = fma2(Two(fabsf(zs.x), fabsf(zs.y)), Two(0.3275911f * 0.70710678118654752f), Two(1.0f)).apart();
        const Two t(reciprocal(below_t.x), reciprocal(below_t.y));
        Two tail = fma2(t, Two(0.5f * 1.061405429f), Two(-0.5f * 1.453152027f));
        tail = fma2(tail, t, Two(0.5f * 1.421413741f));
        tail = fma2(tail, t, Two(-0.5f * 0.284496736f));
        tail = fma2(tail, t, Two(0.5f * 0.254829592f));
        // half less the tail beyond |z|, with z's sign, on half
        const float2 middle = fma2(tail * t, density * Two(-1.0f), Two(0.5f)).apart();
        const Two below = Two(copysignf(middle.x, zs.x), copysignf(middle.y, zs.y)) + Two(0.5f);
        if (kSlope) slope = fma2(z * Two(0.39894228040143268f), density, below);
        return z * below;
    }
    const float2 power = (z * Two(-1.4426950408889634f)).apart();
    const float2 over = (Two(power_of_two(power.x), power_of_two(power.y)) + Two(1.0f)).apart();
    const Two s(reciprocal(over.x), reciprocal(over.y));
    if (kSlope) slope = s * fma2(z, fma2(s, Two(-1.0f), Two(1.0f)), Two(1.0f));
    return z * s;
}

// bytes (16, 8, 4 or 2) on whose boundaries rows `stride` 16-bit elements apart all start
inline int row_alignment(const void* p, int64_t stride) {
    const uint64_t bits = (uint64_t)(uintptr_t)p | (uint64_t)(2 * stride) | 16;
    return (int)(bits & (~bits + 1));
}

// kWords * 2 neighbouring 16-bit values, the first `count` of which exist; the others read as zeros.
template <int kWords> __device__ __forceinline__ void load_words(const uint16_t* p, int count, bool vector, uint32_t (&q)[kWords]) {
    if (vector && count >= 2 * kWords) {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            q[4 * i] = v.x, q[4 * i + 1] = v.y, q[4 * i + 2] = v.z, q[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            q[i] = 2 * i < count ? p[2 * i] : 0;
            q[i] |= 2 * i + 1 < count ? (uint32_t)p[2 * i + 1] << 16 : 0;
        }
    }
}

// kCount neighbouring values of a row, the first `count` of which lie inside the tensor, in stores as wide as the rows' alignment
// allows.
template <bool kBf16, int kCount> __device__ __forceinline__ void store_row(void* out, int64_t at, const float (&v)[kCount], int count, int alignment) {
    uint16_t* p = reinterpret_cast<uint16_t*>(out) + at;
    if (count >= kCount && alignment > 2) {
        uint32_t q[kCount / 2];
#pragma unroll
        for (int i = 0; i < kCount / 2; ++i) q[i] = pack<kBf16>(v[2 * i], v[2 * i + 1]);
        if (alignment == 16) {
#pragma unroll
            for (int i = 0; i < kCount / 8; ++i) reinterpret_cast<uint4*>(p)[i] = make_uint4(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
        } else if (alignment == 8) {
#pragma unroll
            for (int i = 0; i < kCount / 4; ++i) reinterpret_cast<uint2*>(p)[i] = make_uint2(q[2 * i], q[2 * i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < kCount / 2; ++i) reinterpret_cast<uint32_t*>(p)[i] = q[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < kCount; ++i)
            if (i < count) p[i] = narrow<kBf16>(v[i]);
    }
}

// Outputs leave through panels of shared memory, 128 rows x 64 columns of 16 bits in the 128-byte swizzle, filled by the lanes that
// hold a row each.  (Stored from there, 16 bytes of 32 different rows an instruction, they were 2,048 requests a 128 x 128 tile at 3
// clocks each: a tile without any activation took 6,300 clocks.)
constexpr int kPanelBytes = 128 * 128;

// kCount (16 or 32) neighbouring values of row r from column `col` of the panel on.
template <bool kBf16, int kCount> __device__ __forceinline__ void put_panel(uint8_t* panel, int r, int col, const float (&v)[kCount]) {
#pragma unroll
    for (int i = 0; i < kCount / 8; ++i) {
        const int chunk = (col / 8 + i) ^ (r & 7);
        *reinterpret_cast<uint4*>(panel + r * 128 + chunk * 16) =
            make_uint4(pack<kBf16>(v[8 * i], v[8 * i + 1]), pack<kBf16>(v[8 * i + 2], v[8 * i + 3]), pack<kBf16>(v[8 * i + 4], v[8 * i + 5]),
                       pack<kBf16>(v[8 * i + 6], v[8 * i + 7]));
    }
}
// 32 rows of a panel, from r0 on, by `warps` warps to a matrix whose rows start on no 16-byte boundaries: two rows an instruction where
// they start on 8-byte ones, else one.
__device__ __forceinline__ void copy_panel(const uint8_t* panel, int r0, int warp, int warps, void* out, int64_t stride, int64_t row, int64_t rows, int col,
                                           int columns, int alignment, int lane) {
    if (alignment >= 8 && col + 64 <= columns) {
        const int c = lane % 16;
        uint16_t* p = reinterpret_cast<uint16_t*>(out) + (row + lane / 16 + 2 * warp) * stride + col + 4 * c;
#pragma unroll 4
        for (int i = 2 * warp + lane / 16; i < 32; i += 2 * warps, p += 2 * warps * stride) {
            const int r = r0 + i;
            if (row + i < rows) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(panel + r * 128 + ((c / 2) ^ (r & 7)) * 16 + c % 2 * 8);
        }
        return;
    }
    for (int i = warp; i < 32 && row + i < rows; i += warps) {
        const int r = r0 + i;
        const uint32_t two = *reinterpret_cast<const uint32_t*>(panel + r * 128 + ((lane / 4) ^ (r & 7)) * 16 + lane % 4 * 4);
        uint16_t* p = reinterpret_cast<uint16_t*>(out) + (row + i) * stride + col + 2 * lane;
        const int left = columns - col - 2 * lane;
        if (alignment >= 4 && left >= 2) {
            *reinterpret_cast<uint32_t*>(p) = two;
        } else {
            if (left >= 1) p[0] = (uint16_t)two;
            if (left >= 2) p[1] = (uint16_t)(two >> 16);
        }
    }
}

}  // namespace p2b
