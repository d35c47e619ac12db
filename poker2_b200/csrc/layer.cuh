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

// act(z), and act'(z) where asked for
template <int kActivation, bool kSlope> __device__ __forceinline__ float activate(float z, float& slope) {
    if (kActivation == kNoActivation) {
        slope = 1.0f;
        return z;
    }
    if (kActivation == kGelu) {
        const float below = 0.5f * (1.0f + erff(z * 0.70710678118654752f));
        if (kSlope) slope = fmaf(z, 0.39894228040143268f * __expf(-0.5f * z * z), below);
        return z * below;
    }
    const float s = __fdividef(1.0f, 1.0f + __expf(-z));
    if (kSlope) slope = s * fmaf(z, 1.0f - s, 1.0f);
    return z * s;
}

// 32 values of a row from column `first` on; `count` of them lie inside the tensor.
template <bool kBf16> __device__ __forceinline__ void store_row(void* out, int64_t at, const float (&v)[32], int count, bool vector) {
    uint16_t* p = reinterpret_cast<uint16_t*>(out) + at;
    if (vector && count >= 32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint4 q;
            q.x = pack<kBf16>(v[8 * i], v[8 * i + 1]);
            q.y = pack<kBf16>(v[8 * i + 2], v[8 * i + 3]);
            q.z = pack<kBf16>(v[8 * i + 4], v[8 * i + 5]);
            q.w = pack<kBf16>(v[8 * i + 6], v[8 * i + 7]);
            reinterpret_cast<uint4*>(p)[i] = q;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (i < count) p[i] = narrow<kBf16>(v[i]);
    }
}

}  // namespace p2b
