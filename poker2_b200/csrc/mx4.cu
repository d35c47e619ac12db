// Microscaled 4-bit values: rows in blocks of 32 that share a power-of-two scale; quantising, reading back, and the product
// of two such matrices on the block-scaled matrix instructions.
//
// A block's scale is the smallest power of two that brings its largest magnitude to 6 or below (no value is cut off); a
// value then goes to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6, ties to the even code.  Both steps are exact in fp32.
//
// Layout: values two a byte, the first in the low half, a row of ceil(width/32) * 16 bytes.  Scales (exponent + 127 in a byte,
// 255: the block holds an infinity or a NaN) as the matrix instructions read them: 512 bytes hold 128 rows x 4 blocks, at
// (row % 32) * 16 + (row % 128) / 32 * 4 + block % 4; an even number of these along the row, so that a step of 256 columns
// always finds two.  The entries behind the last row and the last block are zero.
#include "layer.cuh"
#include "tensor.cuh"

#include <type_traits>

namespace p2b {

using namespace tc;

// pieces of 512 scale bytes along a row of `width` values
__host__ __device__ __forceinline__ int64_t scale_pieces(int64_t width) { return (width + 255) / 256 * 2; }

// Eight neighbouring values as they lie in memory, and what is asked of them.
template <typename T> struct Eight {  // 16-bit types
    static constexpr bool kBf16 = sizeof(T) == 2 && !std::is_same<T, __half>::value;
    uint32_t w[4];
    __device__ __forceinline__ void load(const T* p) {
        const uint4 q = __ldg(reinterpret_cast<const uint4*>(p));
        w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
    }
    __device__ __forceinline__ void load_some(const T* p, int64_t count) {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (2 * i < count ? h[2 * i] : 0) | (2 * i + 1 < count ? (uint32_t)h[2 * i + 1] << 16 : 0);
    }
    // the largest magnitude as an ordered number (a NaN counts as the largest), to be taken over lanes, and the float it stands for
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = w[0] & 0x7FFF7FFFu;
#pragma unroll
        for (int i = 1; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
        return max(m & 0xFFFFu, m >> 16);
    }
    static __device__ __forceinline__ float magnitude(uint32_t top) { return widen<kBf16>((uint16_t)top); }
    __device__ __forceinline__ float2 pair(int i) const { return unpack<kBf16>(w[i]); }
    static __device__ __forceinline__ void store(T* p, const float2 (&v)[4]) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack<kBf16>(v[0].x, v[0].y), pack<kBf16>(v[1].x, v[1].y), pack<kBf16>(v[2].x, v[2].y), pack<kBf16>(v[3].x, v[3].y));
    }
    static __device__ __forceinline__ void put(T* p, float v) { *reinterpret_cast<uint16_t*>(p) = narrow<kBf16>(v); }
};
template <> struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = __ldg(reinterpret_cast<const float4*>(p));
        b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    }
    __device__ __forceinline__ void load_some(const float* p, int64_t count) {
        a = make_float4(count > 0 ? p[0] : 0.0f, count > 1 ? p[1] : 0.0f, count > 2 ? p[2] : 0.0f, count > 3 ? p[3] : 0.0f);
        b = make_float4(count > 4 ? p[4] : 0.0f, count > 5 ? p[5] : 0.0f, count > 6 ? p[6] : 0.0f, count > 7 ? p[7] : 0.0f);
    }
    __device__ __forceinline__ uint32_t top() const {
        const uint32_t m = max(max(__float_as_uint(a.x) & 0x7FFFFFFFu, __float_as_uint(a.y) & 0x7FFFFFFFu), max(__float_as_uint(a.z) & 0x7FFFFFFFu, __float_as_uint(a.w) & 0x7FFFFFFFu));
        const uint32_t n = max(max(__float_as_uint(b.x) & 0x7FFFFFFFu, __float_as_uint(b.y) & 0x7FFFFFFFu), max(__float_as_uint(b.z) & 0x7FFFFFFFu, __float_as_uint(b.w) & 0x7FFFFFFFu));
        return max(m, n);
    }
    static __device__ __forceinline__ float magnitude(uint32_t top) { return __uint_as_float(top); }
    __device__ __forceinline__ float2 pair(int i) const { return i == 0 ? make_float2(a.x, a.y) : i == 1 ? make_float2(a.z, a.w) : i == 2 ? make_float2(b.x, b.y) : make_float2(b.z, b.w); }
    static __device__ __forceinline__ void store(float* p, const float2 (&v)[4]) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    }
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};

// Scale byte of a block whose largest magnitude is `top`: top = 2^E m, 1 <= m < 2, is at most 6 * 2^(E-2) where m <= 1.5.
__device__ __forceinline__ uint32_t scale_byte(float top) {
    const uint32_t bits = __float_as_uint(top);
    if (bits >= 0x7F800000u) return 255u;
    const int e = (int)(bits >> 23) - ((bits & 0x7FFFFFu) > 0x400000u ? 1 : 2);
    return (uint32_t)(e > 0 ? e : 0);
}
// 2^(127 - byte) for the bytes that a finite block gets, 0 to 253
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float scale_of(uint32_t byte) {
    return byte == 255u ? __int_as_float(0x7FC00000) : byte ? __uint_as_float(byte << 23) : 5.8774717541114375e-39f;
}
// Eight values of magnitude 6 at most, two a byte, and back.
__device__ __forceinline__ uint32_t four_bit_codes(const float2 (&v)[4]) {
    uint32_t word;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(word)
        : "f"(v[0].x), "f"(v[0].y), "f"(v[1].x), "f"(v[1].y), "f"(v[2].x), "f"(v[2].y), "f"(v[3].x), "f"(v[3].y));
    return word;
}
__device__ __forceinline__ void four_bit_values(uint32_t word, float scale, float2 (&v)[4]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(word));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[i] = (Two(f.x, f.y) * Two(scale)).apart();
    }
}

template <typename T> __device__ __forceinline__ uint32_t codes_of(const Eight<T>& x, Two inverse) {
    float2 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 two = x.pair(i);
        v[i] = (Two(two.x, two.y) * inverse).apart();
    }
    return four_bit_codes(v);
}
// What eight values of a block become that four lanes have, and its scale byte.
template <typename T> __device__ __forceinline__ uint32_t quantise_eight(const Eight<T>& x, uint32_t& byte) {
    uint32_t top = x.top();
    top = max(top, __shfl_xor_sync(~0u, top, 1));
    top = max(top, __shfl_xor_sync(~0u, top, 2));
    byte = scale_byte(Eight<T>::magnitude(top));
    return codes_of(x, Two(byte == 255u ? 0.0f : inverse_scale(byte)));
}

// Two lanes take a block, a warp kWide times 512 neighbouring columns of a row: four 16-byte loads (16-bit types) on their way at once,
// 256 bytes of values and four scale words out a time.  Bound by memory and its instructions alike: 24576 x 2720 bf16 take 34 us (169 MB, 5
// TB/s); with four lanes a block, which spend as much on every scale for half as many values, 37.
constexpr int kWide = 2;
constexpr int kSpans = 4;

template <typename T>
__global__ void __launch_bounds__(256) mx4_quantise_kernel(const T* x, int64_t stride, int64_t rows, int width, uint8_t* values, uint8_t* scales,
                                                           int vector) {
    const int lane = threadIdx.x % 32;
    const int blocks = (width + 31) / 32, pieces = (width + 255) / 256 * 2, row_jobs = (width + 512 * kWide - 1) / (512 * kWide);
    const int64_t row_bytes = (int64_t)blocks * 16, all = (rows + 127) / 128 * 128 * row_jobs;
    for (int64_t job = (int64_t)blockIdx.x * 8 + threadIdx.x / 32; job < all; job += (int64_t)gridDim.x * 8) {
        const int64_t row = all < (1ll << 31) ? (uint32_t)job / (uint32_t)row_jobs : job / row_jobs;
        const int first = (int)(job - row * row_jobs) * 512 * kWide, col0 = first + lane * 16, inside = width - col0;
        const T* const p = x + row * stride + col0;
        const bool there = row < rows;
        Eight<T> v[2 * kWide];
        if (there && vector && first + 512 * kWide <= width) {
#pragma unroll
            for (int i = 0; i < 2 * kWide; ++i) v[i].load(p + i / 2 * 512 + i % 2 * 8);
        } else {
#pragma unroll
            for (int i = 0; i < 2 * kWide; ++i) {
                const int at = i / 2 * 512 + i % 2 * 8;
                if (there && vector && inside >= at + 8)
                    v[i].load(p + at);
                else
                    v[i].load_some(p + at, there ? inside - at : 0);
            }
        }
        uint2* const out = reinterpret_cast<uint2*>(values + row * row_bytes + col0 / 2);
        const int piece = first / 128 + lane / 8;
        uint32_t* const row_scales = reinterpret_cast<uint32_t*>(scales + (row / 128 * pieces + piece) * 512 + row % 32 * 16 + row % 128 / 32 * 4);
        const int left = there ? blocks * 32 - col0 : 0;
#pragma unroll
        for (int i = 0; i < kWide; ++i) {
            if (first + 512 * i >= width) break;
            uint32_t top = max(v[2 * i].top(), v[2 * i + 1].top());
            top = max(top, __shfl_xor_sync(~0u, top, 1));
            const uint32_t byte = scale_byte(Eight<T>::magnitude(top));
            const Two inverse(byte == 255u ? 0.0f : inverse_scale(byte));
            const uint2 codes = make_uint2(codes_of(v[2 * i], inverse), codes_of(v[2 * i + 1], inverse));
            if (left > i * 512) out[i * 32] = codes;
            uint32_t four = byte << (8 * (lane / 2 % 4));
            four |= __shfl_xor_sync(~0u, four, 2);
            four |= __shfl_xor_sync(~0u, four, 4);
            if (lane % 8 == 0 && piece + 4 * i < pieces) row_scales[i * 512] = four;
        }
    }
}

// Back: four lanes a block, a warp kSpans times 256 columns, so that the stores of a warp are 512 bytes in a row (24576 x 2720 bf16: 31
// us; with two lanes a block and half a sector a store, 44).
template <typename T>
__global__ void __launch_bounds__(256) mx4_dequantise_kernel(const uint8_t* values, const uint8_t* scales, int64_t rows, int width, T* out,
                                                             int64_t stride, int vector) {
    const int lane = threadIdx.x % 32;
    const int spans = (width + 255) / 256, row_jobs = (spans + kSpans - 1) / kSpans;
    const int64_t row_bytes = (int64_t)((width + 31) / 32) * 16, all = rows * row_jobs;
    for (int64_t job = (int64_t)blockIdx.x * 8 + threadIdx.x / 32; job < all; job += (int64_t)gridDim.x * 8) {
        const int64_t row = all < (1ll << 31) ? (uint32_t)job / (uint32_t)row_jobs : job / row_jobs;
        const int first = (int)(job - row * row_jobs) * kSpans;
        const uint8_t* const row_scales = scales + (row / 128 * spans * 2 + lane / 16) * 512 + row % 32 * 16 + row % 128 / 32 * 4 + lane / 4 % 4;
        uint32_t word[kSpans], byte[kSpans];
#pragma unroll
        for (int i = 0; i < kSpans; ++i) {
            const int col = (first + i) * 256 + lane * 8;
            word[i] = col < width ? __ldg(reinterpret_cast<const uint32_t*>(values + row * row_bytes + col / 2)) : 0;
            byte[i] = col < width ? __ldg(row_scales + (int64_t)(first + i) * 1024) : 0;
        }
#pragma unroll
        for (int i = 0; i < kSpans; ++i) {
            if (first + i >= spans) break;
            const int col = (first + i) * 256 + lane * 8;
            float2 v[4];
            four_bit_values(word[i], scale_of(byte[i]), v);
            T* p = out + row * stride + col;
            if (vector && col + 8 <= width) {
                Eight<T>::store(p, v);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (col + 2 * j < width) Eight<T>::put(p + 2 * j, v[j].x);
                    if (col + 2 * j + 1 < width) Eight<T>::put(p + 2 * j + 1, v[j].y);
                }
            }
        }
    }
}

// y = act(A W^T + bias): tiles of 128 rows x 128 columns, steps of 256 columns of A and W (128 bytes a row), the scales of a step
// copied from shared to tensor memory by the thread that issues the matrix instructions, in their order.
struct Mx4Args {
    CUtensorMap a, w, to, sa, sw;  // (the maps of the scales: pairs alone)
    const uint8_t *a_scales, *w_scales;
    const void* bias;
    void* out;
    uint8_t *out_values, *out_scales;  // the result quantised, instead of out
    int64_t out_stride, rows;
    int columns, steps, tiles_m, tiles_n;
    int vector_bias, align_out, pairs;
};

constexpr int kTile = 128;
constexpr int kMxStages = 4;
constexpr int kScaleBytes = 1024;  // two pieces
constexpr int kMxStage = 2 * (kTile * 128 + kScaleBytes);
constexpr int kMxShared = kMxStages * kMxStage + 4 * kPanelBytes + 1024;
constexpr int kMxEpilogueWarps = 16;
constexpr int kMxThreads = 32 * (kMxEpilogueWarps + 2);
constexpr int kScaleSets = 4;      // sets of scale columns in tensor memory, used in turn
constexpr uint32_t kMxTmem = 512;  // two accumulators, scales behind them
constexpr uint32_t kScaleColumn = 2 * kTile;

// 32 accumulators of a row from column `col` on to act(. + bias), rounded to 16 bits: two to a word of y.
template <bool kBf16, int kActivation>
__device__ __forceinline__ void finish_block(const Mx4Args& args, const uint32_t (&g)[32], int col, bool ok, uint32_t (&y)[16]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        uint32_t bias[8];
        load_words(reinterpret_cast<const uint16_t*>(args.bias) + col + 16 * j, args.bias ? args.columns - col - 16 * j : 0, args.vector_bias, bias);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            Two slope;
            const uint32_t* two = g + 16 * j + 2 * i;
            const float2 v = activate<kActivation, false>(Two(__uint_as_float(two[0]), __uint_as_float(two[1])) + two_of<kBf16>(bias[i]), slope).apart();
            y[8 * j + i] = ok ? pack<kBf16>(v.x, v.y) : 0x7FFF7FFFu;  // (a NaN in either type)
        }
    }
}
// A row's 64 neighbouring results from column `col` on, quantised as mx4_quantise_kernel would: 32 bytes of values, two scales.  Rows behind
// the last have scales of zero; columns behind the last count as zeros (no weight, no bias: they are, but where the row holds a block that
// is not finite).
template <bool kBf16> __device__ __forceinline__ void store_quantised(const Mx4Args& args, int64_t row, int col, const uint32_t (&y)[2][16]) {
    using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
    if (col >= (args.columns + 255) / 256 * 256 || row >= (args.rows + 127) / 128 * 128) return;
    const int64_t row_bytes = (int64_t)((args.columns + 31) / 32) * 16, pieces = scale_pieces(args.columns);
    uint32_t bytes = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        Eight<T> v[4];
        uint32_t top = 0, codes[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[i].w[k] = y[j][4 * i + k];
        }
        const int left = args.columns - col - 32 * j;
        if (left < 32) {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i / 4].w[i % 4] &= (2 * i < left ? 0xFFFFu : 0u) | (2 * i + 1 < left ? 0xFFFF0000u : 0u);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, v[i].top());
        const uint32_t byte = row < args.rows ? scale_byte(Eight<T>::magnitude(top)) : 0;
        const Two inverse(byte == 255u ? 0.0f : inverse_scale(byte));
#pragma unroll
        for (int i = 0; i < 4; ++i) codes[i] = codes_of(v[i], inverse);
        bytes |= byte << (8 * j);
        if (row < args.rows && col + 32 * j < args.columns)
            *reinterpret_cast<uint4*>(args.out_values + row * row_bytes + (col + 32 * j) / 2) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
    }
    uint8_t* at = args.out_scales + (row / 128 * pieces + col / 128) * 512 + row % 32 * 16 + row % 128 / 32 * 4 + col / 32 % 4;
    *reinterpret_cast<uint16_t*>(at) = (uint16_t)bytes;
}
template <bool kBf16> __device__ __forceinline__ void put_block(uint8_t* panel, int r, int col, const uint32_t (&y)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint4*>(panel + r * 128 + ((col / 8 + i) ^ (r & 7)) * 16) = make_uint4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
}

template <int kOut, int kActivation, bool kQuantised>  // kOut 0 bf16, 1 fp16
__global__ void __launch_bounds__(kMxThreads, 1) mx4_linear_kernel(const __grid_constant__ Mx4Args args) {
    constexpr bool kBf16 = kOut == 0;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t bars[2 * kMxStages + 4];
    __shared__ uint32_t tmem_at;
    __shared__ volatile int given_up;
    const uint32_t ring = (smem_addr(raw) + 1023) & ~1023u, bar0 = smem_addr(bars);
    auto full = [&](int s) { return bar0 + 8 * s; };
    auto empty = [&](int s) { return bar0 + 8 * (kMxStages + s); };
    auto acc_full = [&](int s) { return bar0 + 8 * (2 * kMxStages + s); };
    auto acc_empty = [&](int s) { return bar0 + 8 * (2 * kMxStages + 2 + s); };
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        given_up = 0;
        for (int s = 0; s < kMxStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(acc_full(s), 1);
            mbar_init(acc_empty(s), kMxEpilogueWarps / 2);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMxEpilogueWarps + 1) tmem_alloc(smem_addr(&tmem_at), kMxTmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    const int tiles = args.tiles_m * args.tiles_n, steps = args.steps;

    if (warp == kMxEpilogueWarps) {
        if (lane == 0) {
            tma_prefetch_map(&args.a);
            tma_prefetch_map(&args.w);
            int s = 0;
            uint32_t phase = 1;  // (the stages begin empty)
            bool ok = true;
            for (int64_t tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
                const int m = (int)(tile / args.tiles_n), n = (int)(tile % args.tiles_n);
                for (int k = 0; k < steps; ++k) {
                    if (!mbar_wait(empty(s), phase, &given_up)) {
                        ok = false;
                        break;
                    }
                    const uint32_t a = ring + s * kMxStage;
                    mbar_expect(full(s), kMxStage);
                    tma_load_2d(a, &args.a, k * 128, m * kTile, full(s));
                    tma_load_2d(a + kTile * 128, &args.w, k * 128, n * kTile, full(s));
                    bulk_load(a + 2 * kTile * 128, args.a_scales + ((int64_t)m * steps + k) * kScaleBytes, kScaleBytes, full(s));
                    bulk_load(a + 2 * kTile * 128 + kScaleBytes, args.w_scales + ((int64_t)n * steps + k) * kScaleBytes, kScaleBytes, full(s));
                    if (++s == kMxStages) s = 0, phase ^= 1;
                }
            }
            if (!ok) let_settle();  // the copies in flight land before the block's memory goes
        }
        __syncwarp();
    } else if (warp == kMxEpilogueWarps + 1) {
        if (lane == 0) {
            uint32_t used = 0, phase = 0;
            int s = 0, turn = 0;
            bool ok = true;
            for (int64_t tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, ++turn) {
                const int acc = turn & 1;
                if (turn >= 2 && !mbar_wait(acc_empty(acc), (uint32_t)(turn / 2 - 1) & 1, &given_up)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                for (int k = 0; k < steps; ++k, ++used) {
                    if (!mbar_wait(full(s), phase, &given_up)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = ring + s * kMxStage, w = a + kTile * 128, sa = w + kTile * 128, sw = sa + kScaleBytes;
                    const uint32_t ta = tmem + kScaleColumn + (uint32_t)(used % kScaleSets) * 16, tw = ta + 8;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        tmem_copy_scales(ta + 4 * i, scale_desc(sa + 512 * i));
                        tmem_copy_scales(tw + 4 * i, scale_desc(sw + 512 * i));
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        mma_mx4(tmem + acc * kTile, operand_desc(a + 32 * i, 1024, 16), operand_desc(w + 32 * i, 1024, 16), mx4_idesc(kTile, kTile, i & 1),
                                ta + 4 * (i >> 1), tw + 4 * (i >> 1), k > 0 || i > 0);
                    tc_commit(empty(s));
                    if (++s == kMxStages) s = 0, phase ^= 1;
                }
                if (ok) tc_commit(acc_full(acc));
            }
            if (!ok) let_settle();  // the matrix instructions in flight end before their tensor memory is freed
        }
        __syncwarp();
    } else {
        // Two groups of eight warps take the tiles in turn, each its own accumulator: a tile's epilogue is a chain of waits (with one
        // group of sixteen it took 3.1 us whatever the products took).  A warp has 32 rows and 64 columns, a panel's quarter of its own.
        const int quadrant = warp % 4, half = warp / 4 % 2, acc = warp / 8, r = quadrant * 32 + lane;
        uint8_t* const panel = raw + (ring - smem_addr(raw)) + kMxStages * kMxStage + (2 * acc + half) * kPanelBytes;
        int turn = acc;
        for (int64_t tile = blockIdx.x + (int64_t)acc * gridDim.x; tile < tiles; tile += 2 * (int64_t)gridDim.x, turn += 2) {
            const int64_t row0 = tile / args.tiles_n * kTile + quadrant * 32;
            const int n = (int)(tile % args.tiles_n), col = n * kTile + 64 * half;
            const bool ok = mbar_wait(acc_full(acc), (uint32_t)(turn / 2) & 1, &given_up);
            tc_fence_after();
            if (!kQuantised && lane == 0) store_wait_read<0>();
            __syncwarp();
            uint32_t y[2][16];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t g[32];
                tmem_load_32(tmem + ((uint32_t)(quadrant * 32) << 16) + acc * kTile + 64 * half + 32 * j, g);
                tmem_load_wait();
                if (j == 1) {  // the accumulator is read
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(acc_empty(acc));
                }
                finish_block<kBf16, kActivation>(args, g, col + 32 * j, ok, y[j]);
                if (!kQuantised) put_block<kBf16>(panel, r, 32 * j, y[j]);
            }
            if (kQuantised) {
                store_quantised<kBf16>(args, row0 + lane, col, y);
                // (the odd piece behind a last tile of 128 columns has no tile of its own)
                if (n + 1 == args.tiles_n && n % 2 == 0) {
                    const uint32_t none[2][16] = {};
                    store_quantised<kBf16>(args, row0 + lane, col + 128, none);
                }
                continue;
            }
            if (args.align_out == 16) {
                async_fence();
                __syncwarp();
                if (lane == 0) {
                    if (row0 < args.rows && col < args.columns) tma_store_2d(&args.to, col, (int)row0, smem_addr(panel) + quadrant * 4096);
                    store_commit();
                }
            } else {
                __syncwarp();
                copy_panel(panel, quadrant * 32, 0, 1, args.out, args.out_stride, row0, args.rows, col, args.columns, args.align_out, lane);
            }
        }
        if (lane == 0) store_wait();
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMxEpilogueWarps + 1) {
        tc_fence_after();
        tmem_free(tmem, kMxTmem);
    }
}

// Pairs of blocks, 256 x 256 outputs: each block brings its 128 rows of A, 128 of the 256 rows of W, and the scales of the former
// and of all of the latter: 35 KB a step for 512 clocks of matrix instructions, where the blocks by themselves need 35 KB for
// 256 and wait for them (436 ns a step; 24576 rows of 1536 x 1536 with a gelu: 64 against 49 us).  The accumulators fill half of tensor memory and the scales a fifth, so there is one set: the
// epilogue takes them into registers at once, and the products of the next tile begin while it works on those.
constexpr int kPairStages = 4;
constexpr int kPairStage = 2 * kTile * 128 + 3 * kScaleBytes + 1024;  // (a stage starts on a 1024-byte boundary)
constexpr int kPairBytes = 2 * kTile * 128 + 3 * kScaleBytes;
constexpr int kPairShared = kPairStages * kPairStage + 4 * kPanelBytes + 1024;
constexpr uint32_t kPairScales = 256;  // column of the scales

template <int kOut, int kActivation, bool kQuantised>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kMxThreads, 1) mx4_pair_kernel(const __grid_constant__ Mx4Args args) {
    constexpr bool kBf16 = kOut == 0;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t bars[2 * kPairStages + 2];
    __shared__ uint32_t tmem_at;
    __shared__ volatile int given_up;
    const uint32_t ring = (smem_addr(raw) + 1023) & ~1023u, bar0 = smem_addr(bars);
    auto full = [&](int s) { return bar0 + 8 * s; };
    auto empty = [&](int s) { return bar0 + 8 * (kPairStages + s); };
    const uint32_t acc_full = bar0 + 16 * kPairStages, acc_empty = acc_full + 8;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = (int)pair_rank(), pair = blockIdx.x / 2, pairs = gridDim.x / 2;
    if (threadIdx.x == 0) {
        given_up = 0;
        for (int s = 0; s < kPairStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        mbar_init(acc_full, 1);
        mbar_init(acc_empty, 2 * kMxEpilogueWarps);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMxEpilogueWarps + 1) pair_tmem_alloc(smem_addr(&tmem_at), kMxTmem);
    tc_fence_before();
    __syncthreads();
    pair_sync();
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    const int tiles = args.tiles_m * args.tiles_n, steps = args.steps;

    if (warp == kMxEpilogueWarps) {
        if (lane == 0) {
            tma_prefetch_map(&args.a);
            tma_prefetch_map(&args.w);
            tma_prefetch_map(&args.sa);
            tma_prefetch_map(&args.sw);
            const uint32_t leader_full = in_leader(full(0));
            int s = 0;
            uint32_t phase = 1;  // (the stages begin empty)
            bool ok = true;
            for (int64_t tile = pair; ok && tile < tiles; tile += pairs) {
                const int m = (int)(tile / args.tiles_n) * 2 + rank, n = (int)(tile % args.tiles_n) * 2;  // in 128 rows
                for (int k = 0; k < steps; ++k) {
                    if (!pair_wait(empty(s), phase, &given_up)) {
                        ok = false;
                        break;
                    }
                    const uint32_t a = ring + s * kPairStage, sa = a + 2 * kTile * 128, bar = leader_full + 8 * s;
                    if (rank == 0) mbar_expect(full(s), 2 * kPairBytes);
                    pair_load_2d(a, &args.a, k * 128, m * kTile, bar);
                    pair_load_2d(a + kTile * 128, &args.w, k * 128, (n + rank) * kTile, bar);
                    // (groups of 128 rows behind the last read as zeros)
                    pair_load_2d(sa, &args.sa, 0, (m * steps + k) * 8, bar);
                    for (int i = 0; i < 2; ++i) pair_load_2d(sa + (1 + i) * kScaleBytes, &args.sw, 0, ((n + i) * steps + k) * 8, bar);
                    if (++s == kPairStages) s = 0, phase ^= 1;
                }
            }
            if (!ok) let_settle();
        }
        __syncwarp();
    } else if (warp == kMxEpilogueWarps + 1) {
        if (lane == 0 && rank == 0) {
            uint32_t used = 0, phase = 0;
            int s = 0, turn = 0;
            bool ok = true;
            for (int64_t tile = pair; ok && tile < tiles; tile += pairs, ++turn) {
                if (turn >= 1 && !pair_wait(acc_empty, (uint32_t)(turn - 1) & 1, &given_up)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                for (int k = 0; k < steps; ++k, ++used) {
                    if (!pair_wait(full(s), phase, &given_up)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = ring + s * kPairStage, w = a + kTile * 128, sa = w + kTile * 128, sw = sa + kScaleBytes;
                    const uint32_t ta = tmem + kPairScales + (used % kScaleSets) * 24, tw = ta + 8;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {  // a piece of 128 columns of K: four columns for A, eight for the two groups of W
                        pair_copy_scales(ta + 4 * i, scale_desc(sa + 512 * i));
                        pair_copy_scales(tw + 8 * i, scale_desc(sw + 512 * i));
                        pair_copy_scales(tw + 8 * i + 4, scale_desc(sw + kScaleBytes + 512 * i));
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        pair_mma_mx4(tmem, operand_desc(a + 32 * i, 1024, 16), operand_desc(w + 32 * i, 1024, 16), pair_mx4_idesc(256, i & 1), ta + 4 * (i >> 1),
                                     tw + 8 * (i >> 1), k > 0 || i > 0);
                    pair_commit(empty(s));
                    if (++s == kPairStages) s = 0, phase ^= 1;
                }
                if (ok) pair_commit(acc_full);
            }
            if (!ok) let_settle();
        }
        __syncwarp();
    } else {
        // A warp has 32 rows and 64 columns: a panel's quarter of its own.
        const int quadrant = warp % 4, part = warp / 4, r = quadrant * 32 + lane;
        uint8_t* const panel = raw + (ring - smem_addr(raw)) + kPairStages * kPairStage + part * kPanelBytes;
        int turn = 0;
        for (int64_t tile = pair; tile < tiles; tile += pairs, ++turn) {
            const int64_t row0 = tile / args.tiles_n * 256 + rank * 128 + quadrant * 32;
            const int col = (int)(tile % args.tiles_n) * 256 + 64 * part;
            const bool ok = pair_wait(acc_full, (uint32_t)turn & 1, &given_up);
            tc_fence_after();
            uint32_t g[2][32];
            const uint32_t from = tmem + ((uint32_t)(quadrant * 32) << 16) + 64 * part;
            tmem_load_32(from, g[0]);
            tmem_load_32(from + 32, g[1]);
            tmem_load_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                pair_arrive(in_leader(acc_empty));
                if (!kQuantised) store_wait_read<0>();
            }
            __syncwarp();
            uint32_t y[2][16];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                finish_block<kBf16, kActivation>(args, g[j], col + 32 * j, ok, y[j]);
                if (!kQuantised) put_block<kBf16>(panel, r, 32 * j, y[j]);
            }
            if (kQuantised) {
                store_quantised<kBf16>(args, row0 + lane, col, y);
                continue;
            }
            if (args.align_out == 16) {
                async_fence();
                __syncwarp();
                if (lane == 0) {
                    if (row0 < args.rows && col < args.columns) tma_store_2d(&args.to, col, (int)row0, smem_addr(panel) + quadrant * 4096);
                    store_commit();
                }
            } else {
                __syncwarp();
                copy_panel(panel, quadrant * 32, 0, 1, args.out, args.out_stride, row0, args.rows, col, args.columns, args.align_out, lane);
                __syncwarp();
            }
        }
        if (lane == 0) store_wait();
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    pair_sync();
    if (warp == kMxEpilogueWarps + 1) {
        tc_fence_after();
        pair_tmem_free(tmem, kMxTmem);
    }
}

// Few rows of x as they are: every block quantises them for itself (a chunk of kChunk columns at a time, in shared memory as the
// values they stand for), a warp takes a column of the product.  One launch, and no 128 rows of which most are empty: 1 row of 1536 x
// 1536 takes 3.6 us, in the two launches of the general way 9.6; 4 rows 7.1 and 9.6; at 8 rows it would be 12.3 and 9.4.
constexpr int kFewRows = 4;
constexpr int kChunk = 1024;

template <typename T, int kMost, bool kBf16, int kActivation>
__global__ void __launch_bounds__(256) mx4_few_kernel(const T* x, int64_t x_stride, int rows, int width, const uint8_t* w_values, const uint8_t* w_scales,
                                                      const uint16_t* bias, int columns, uint16_t* out, int64_t out_stride, int vector) {
    __shared__ __align__(16) float values[kMost][kChunk];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, column = blockIdx.x * 8 + warp;
    const int blocks = (width + 31) / 32, spans = (width + 255) / 256;
    const int64_t row_bytes = (int64_t)blocks * 16;
    const uint8_t* const w = w_values + column * row_bytes;
    const uint8_t* const scale_at = w_scales + ((int64_t)(column / 128) * spans * 2 + lane / 16) * 512 + column % 32 * 16 + column % 128 / 32 * 4 + lane / 4 % 4;
    float sum[kMost];
#pragma unroll
    for (int r = 0; r < kMost; ++r) sum[r] = 0.0f;
    for (int first = 0; first < spans; first += kChunk / 256) {
        uint32_t word[kChunk / 256], byte[kChunk / 256];
#pragma unroll
        for (int i = 0; i < kChunk / 256; ++i) {
            const int col = (first + i) * 256 + lane * 8;
            const bool there = column < columns && col < blocks * 32;
            word[i] = there ? __ldg(reinterpret_cast<const uint32_t*>(w + col / 2)) : 0;
            byte[i] = there ? __ldg(scale_at + (int64_t)(first + i) * 1024) : 0;
        }
        if (first > 0) __syncthreads();
        for (int job = warp; job < rows * (kChunk / 256); job += 8) {
            const int r = job / (kChunk / 256), i = job % (kChunk / 256), col = (first + i) * 256 + lane * 8;
            Eight<T> v;
            if (vector && col + 8 <= width)
                v.load(x + r * x_stride + col);
            else
                v.load_some(x + r * x_stride + col, width - col);
            uint32_t b;
            // (by way of a shuffle: codes handed straight from their packing to their unpacking came out as zeros, nvcc 12.9)
            const uint32_t word_x = __shfl_sync(~0u, quantise_eight<T>(v, b), lane);
            float2 q[4];
            four_bit_values(word_x, scale_of(b), q);
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<float2*>(&values[r][i * 256 + lane * 8 + 2 * j]) = q[j];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kChunk / 256; ++i) {
            if (first + i >= spans) break;
            float2 f[4];
            four_bit_values(word[i], scale_of(byte[i]), f);
#pragma unroll
            for (int r = 0; r < kMost; ++r)
                if (r < rows) {
                    const float4 a = *reinterpret_cast<const float4*>(&values[r][i * 256 + lane * 8]), b = *reinterpret_cast<const float4*>(&values[r][i * 256 + lane * 8 + 4]);
                    float part = fmaf(a.x, f[0].x, sum[r]);
                    part = fmaf(a.y, f[0].y, part);
                    part = fmaf(a.z, f[1].x, part);
                    part = fmaf(a.w, f[1].y, part);
                    part = fmaf(b.x, f[2].x, part);
                    part = fmaf(b.y, f[2].y, part);
                    part = fmaf(b.z, f[3].x, part);
                    sum[r] = fmaf(b.w, f[3].y, part);
                }
        }
    }
#pragma unroll
    for (int r = 0; r < kMost; ++r)
#pragma unroll
        for (int o = 16; o > 0; o /= 2) sum[r] += __shfl_xor_sync(~0u, sum[r], o);
    if (column >= columns) return;
#pragma unroll
    for (int r = 0; r < kMost; ++r)
        if (lane == r && r < rows) {
            Two slope;
            out[r * out_stride + column] = narrow<kBf16>(activate<kActivation, false>(Two(sum[r] + (bias ? widen<kBf16>(bias[column]) : 0.0f)), slope).apart().x);
        }
}

template <typename T, bool kBf16, int kActivation>
static int launch_few(const void* x, int64_t x_stride, int rows, int width, const void* w_values, const void* w_scales, const void* bias, int columns, void* out,
                      int64_t out_stride, cudaStream_t stream) {
    const int vector = (uintptr_t)x % 16 == 0 && (rows == 1 || x_stride % (16 / (int)sizeof(T)) == 0);
    auto* kernel = rows == 1 ? mx4_few_kernel<T, 1, kBf16, kActivation> : rows == 2 ? mx4_few_kernel<T, 2, kBf16, kActivation> : mx4_few_kernel<T, kFewRows, kBf16, kActivation>;
    kernel<<<(unsigned)blocks_of(columns, 8), 256, 0, stream>>>((const T*)x, x_stride, rows, width, (const uint8_t*)w_values, (const uint8_t*)w_scales,
                                                               (const uint16_t*)bias, columns, (uint16_t*)out, out_stride, vector);
    return check_cuda(cudaGetLastError(), "mx4_few_kernel");
}

static SharedLimit g_limit[2][3][2], g_pair_limit[2][3][2];

// Blocks by themselves while each gets at most one tile: a pair walks as long as a block and ends with twice the epilogue (1024 rows of
// 1536 x 2720 with a gelu: 13.4 against 16.7 us); pairs beyond (2048 rows: 16.7 against 19.0; 24576: 71 against 101).
static bool paired(int64_t rows, int64_t columns) { return blocks_of(rows, kTile) * blocks_of(columns, kTile) > sm_count(); }

template <int kOut, int kActivation, bool kQuantised> static int launch_linear(const Mx4Args& args, cudaStream_t stream) {
    if (args.pairs) {
        auto* kernel = mx4_pair_kernel<kOut, kActivation, kQuantised>;
        int rc = allow_shared(g_pair_limit[kOut][kActivation][kQuantised], (const void*)kernel, kPairShared);
        if (rc) return rc;
        const int tiles = args.tiles_m * args.tiles_n, most = sm_count() / 2;
        kernel<<<2 * (tiles < most ? tiles : most), kMxThreads, kPairShared, stream>>>(args);
        return check_cuda(cudaGetLastError(), "mx4_pair_kernel");
    }
    auto* kernel = mx4_linear_kernel<kOut, kActivation, kQuantised>;
    int rc = allow_shared(g_limit[kOut][kActivation][kQuantised], (const void*)kernel, kMxShared);
    if (rc) return rc;
    const int tiles = args.tiles_m * args.tiles_n;
    kernel<<<tiles < sm_count() ? tiles : sm_count(), kMxThreads, kMxShared, stream>>>(args);
    return check_cuda(cudaGetLastError(), "mx4_linear_kernel");
}

constexpr int64_t kMostRows = 1ll << 30;
constexpr int32_t kMostWidth = 1 << 20;

static int check_matrix(const char* name, int64_t rows, int32_t width) {
    if (rows < 0 || rows > kMostRows || width < 1 || width > kMostWidth)
        return set_error(P2B_ERR_ARG, "%s: %lld rows of %d are out of range", name, (long long)rows, width);
    return P2B_OK;
}
static unsigned warp_grid(int64_t jobs) {
    const int64_t blocks = blocks_of(jobs, 8), most = (int64_t)sm_count() * 8;
    return (unsigned)(blocks < most ? blocks : most);
}

}  // namespace p2b

using namespace p2b;

extern "C" int64_t p2b_mx4_value_bytes(int64_t rows, int32_t width) { return rows < 0 || width < 1 ? -1 : rows * blocks_of(width, 32) * 16; }
extern "C" int64_t p2b_mx4_scale_bytes(int64_t rows, int32_t width) {
    return rows < 0 || width < 1 ? -1 : blocks_of(rows, 128) * scale_pieces(width) * 512;
}

static int check_source(const char* name, const void* x, int64_t x_stride, int64_t rows, int32_t width, int32_t dtype) {
    int rc = check_matrix(name, rows, width);
    if (rc) return rc;
    if (dtype < 0 || dtype > 2) return set_error(P2B_ERR_ARG, "%s: unknown type %d (0 bf16, 1 fp16, 2 fp32)", name, dtype);
    if (rows > 0 && (!x || x_stride < 0 || (uintptr_t)x % (dtype == 2 ? 4 : 2)))
        return set_error(P2B_ERR_ARG, "%s: x must lie on its elements' boundaries, its rows no negative number apart", name);
    return P2B_OK;
}

extern "C" int p2b_mx4_quantise(const void* x, int64_t x_stride, int64_t rows, int32_t width, int32_t dtype, void* values, void* scales, void* stream) {
    int rc = check_source("p2b_mx4_quantise", x, x_stride, rows, width, dtype);
    if (rc || rows == 0) return rc;
    if (!values || !scales || ((uintptr_t)values % 16) || ((uintptr_t)scales % 16))
        return set_error(P2B_ERR_ARG, "p2b_mx4_quantise: values and scales must lie on 16-byte boundaries");
    const int vector = (uintptr_t)x % 16 == 0 && x_stride % (dtype == 2 ? 4 : 8) == 0;
    const unsigned grid = warp_grid(blocks_of(rows, 128) * 128 * blocks_of(width, 512 * kWide));
    cudaStream_t st = (cudaStream_t)stream;
    uint8_t *v = (uint8_t*)values, *s = (uint8_t*)scales;
    if (dtype == 0) mx4_quantise_kernel<<<grid, 256, 0, st>>>((const __nv_bfloat16*)x, x_stride, rows, width, v, s, vector);
    if (dtype == 1) mx4_quantise_kernel<<<grid, 256, 0, st>>>((const __half*)x, x_stride, rows, width, v, s, vector);
    if (dtype == 2) mx4_quantise_kernel<<<grid, 256, 0, st>>>((const float*)x, x_stride, rows, width, v, s, vector);
    return check_cuda(cudaGetLastError(), "mx4_quantise_kernel");
}

extern "C" int p2b_mx4_dequantise(const void* values, const void* scales, int64_t rows, int32_t width, int32_t dtype, void* out, int64_t out_stride,
                                  void* stream) {
    int rc = check_matrix("p2b_mx4_dequantise", rows, width);
    if (rc) return rc;
    if (dtype < 0 || dtype > 2) return set_error(P2B_ERR_ARG, "p2b_mx4_dequantise: unknown type %d (0 bf16, 1 fp16, 2 fp32)", dtype);
    if (rows == 0) return P2B_OK;
    if (!out || !values || !scales || (rows > 1 && out_stride < width))
        return set_error(P2B_ERR_ARG, "p2b_mx4_dequantise: null array or rows that overlap");
    if (((uintptr_t)values % 16) || ((uintptr_t)scales % 16) || (uintptr_t)out % (dtype == 2 ? 4 : 2))
        return set_error(P2B_ERR_ARG, "p2b_mx4_dequantise: values and scales must lie on 16-byte boundaries, out on its element's");
    const int vector = (uintptr_t)out % 16 == 0 && out_stride % (dtype == 2 ? 4 : 8) == 0;
    const unsigned grid = warp_grid(rows * blocks_of(width, 256 * kSpans));
    cudaStream_t st = (cudaStream_t)stream;
    const uint8_t *v = (const uint8_t*)values, *s = (const uint8_t*)scales;
    if (dtype == 0) mx4_dequantise_kernel<<<grid, 256, 0, st>>>(v, s, rows, width, (__nv_bfloat16*)out, out_stride, vector);
    if (dtype == 1) mx4_dequantise_kernel<<<grid, 256, 0, st>>>(v, s, rows, width, (__half*)out, out_stride, vector);
    if (dtype == 2) mx4_dequantise_kernel<<<grid, 256, 0, st>>>(v, s, rows, width, (float*)out, out_stride, vector);
    return check_cuda(cudaGetLastError(), "mx4_dequantise_kernel");
}

extern "C" int p2b_mx4_few_rows(void) { return kFewRows; }

extern "C" int p2b_mx4_linear_few(const void* x, int64_t x_stride, int32_t x_dtype, int64_t rows, const void* w_values, const void* w_scales, int32_t columns,
                                  int32_t width, const void* bias, int32_t dtype, int32_t activation, void* out, int64_t out_stride, void* stream) {
    const char* name = "p2b_mx4_linear_few";
    int rc = check_matrix(name, columns, width);
    if (rc) return rc;
    if (rows < 0 || rows > kFewRows || columns < 1) return set_error(P2B_ERR_ARG, "%s: %lld rows and %d columns (0 to %d rows)", name, (long long)rows, columns, kFewRows);
    if (dtype < 0 || dtype > 1 || x_dtype < 0 || x_dtype > 2) return set_error(P2B_ERR_ARG, "%s: unknown type (x %d, result %d)", name, x_dtype, dtype);
    if (activation < 0 || activation > 2) return set_error(P2B_ERR_ARG, "%s: unknown activation %d (0 gelu, 1 silu, 2 none)", name, activation);
    if (rows == 0) return P2B_OK;
    if (!x || !w_values || !w_scales || !out || x_stride < 0 || (rows > 1 && out_stride < columns))
        return set_error(P2B_ERR_ARG, "%s: null array or rows that overlap", name);
    if ((uintptr_t)w_values % 16 || (uintptr_t)w_scales % 16) return set_error(P2B_ERR_ARG, "%s: values and scales must lie on 16-byte boundaries", name);
    if ((uintptr_t)out % 2 || (uintptr_t)bias % 2 || (uintptr_t)x % (x_dtype == 2 ? 4 : 2)) return set_error(P2B_ERR_ARG, "%s: x, out and bias must lie on their elements' boundaries", name);
    auto few = [&](auto element) {
        using T = decltype(element);
        auto* f = dtype == 0 ? (activation == 0 ? launch_few<T, true, 0> : activation == 1 ? launch_few<T, true, 1> : launch_few<T, true, 2>)
                             : (activation == 0 ? launch_few<T, false, 0> : activation == 1 ? launch_few<T, false, 1> : launch_few<T, false, 2>);
        return f(x, x_stride, (int)rows, width, w_values, w_scales, bias, columns, out, out_stride, (cudaStream_t)stream);
    };
    return x_dtype == 0 ? few(__nv_bfloat16()) : x_dtype == 1 ? few(__half()) : few(0.0f);
}

static int prepare_linear(const char* name, Mx4Args& args, const void* a_values, const void* a_scales, int64_t rows, const void* w_values, const void* w_scales,
                          int32_t columns, int32_t width, const void* bias, int32_t dtype, int32_t activation, void* out, int64_t out_stride, void* out_values,
                          void* out_scales) {
    const bool quantised = out_values || out_scales;
    int rc = check_matrix(name, rows, width);
    if (!rc) rc = check_matrix(name, columns, width);
    if (rc) return rc;
    // (tiles and rows of 128 scale bytes are counted in 32 bits)
    if (columns < 1 || blocks_of(rows, kTile) * blocks_of(columns, kTile) > 0x7FFF0000ll || (blocks_of(rows, kTile) + 1) * blocks_of(width, 256) > 0x0FFF0000ll ||
        (blocks_of(columns, kTile) + 1) * blocks_of(width, 256) > 0x0FFF0000ll)
        return set_error(P2B_ERR_ARG, "%s: %lld x %d outputs are out of range", name, (long long)rows, columns);
    if (dtype < 0 || dtype > 1) return set_error(P2B_ERR_ARG, "%s: unknown type %d (0 bf16, 1 fp16)", name, dtype);
    if (activation < 0 || activation > 2) return set_error(P2B_ERR_ARG, "%s: unknown activation %d (0 gelu, 1 silu, 2 none)", name, activation);
    if (rows == 0) return P2B_OK;
    if (!a_values || !a_scales || !w_values || !w_scales || (quantised ? !out_values || !out_scales : !out || (rows > 1 && out_stride < columns)))
        return set_error(P2B_ERR_ARG, "%s: null array or rows that overlap", name);
    for (const void* p : {a_values, a_scales, w_values, w_scales, (const void*)out_values, (const void*)out_scales})
        if ((uintptr_t)p % 16) return set_error(P2B_ERR_ARG, "%s: values and scales must lie on 16-byte boundaries", name);
    if ((uintptr_t)out % 2 || (uintptr_t)bias % 2) return set_error(P2B_ERR_ARG, "%s: out and bias must lie on 2-byte boundaries", name);
    const int64_t row_bytes = blocks_of(width, 32) * 16;
    rc = encode_rows(&args.a, a_values, 1, row_bytes, rows, row_bytes, kTile);
    if (!rc) rc = encode_rows(&args.w, w_values, 1, row_bytes, columns, row_bytes, kTile);
    if (rc) return rc;
    args.out_values = (uint8_t*)out_values, args.out_scales = (uint8_t*)out_scales;
    args.align_out = row_alignment(out, rows > 1 ? out_stride : 0);
    if (!quantised && args.align_out == 16) rc = encode_rows(&args.to, out, 2, columns, rows, 2 * (rows > 1 ? out_stride : blocks_of(columns, 8) * 8), 32);
    if (rc) return rc;
    args.a_scales = (const uint8_t*)a_scales, args.w_scales = (const uint8_t*)w_scales, args.bias = bias, args.out = out;
    args.out_stride = out_stride, args.rows = rows, args.columns = columns;
    args.steps = (int)blocks_of(width, 256);
    args.pairs = paired(rows, columns);
    if (args.pairs) {
        rc = encode_pieces(&args.sa, a_scales, blocks_of(rows, 128) * args.steps);
        if (!rc) rc = encode_pieces(&args.sw, w_scales, blocks_of(columns, 128) * args.steps);
        if (rc) return rc;
    }
    const int edge = args.pairs ? 256 : kTile;
    args.tiles_m = (int)blocks_of(rows, edge), args.tiles_n = (int)blocks_of(columns, edge);
    args.vector_bias = aligned16(bias, 0);
    return P2B_OK;
}

static int run_linear(const Mx4Args& args, int32_t dtype, int32_t activation, cudaStream_t stream) {
    auto launch = [&](auto type) {
        constexpr int kOut = decltype(type)::value;
        auto* f = args.out_values ? (activation == 0 ? launch_linear<kOut, 0, true> : activation == 1 ? launch_linear<kOut, 1, true> : launch_linear<kOut, 2, true>)
                                  : (activation == 0 ? launch_linear<kOut, 0, false> : activation == 1 ? launch_linear<kOut, 1, false> : launch_linear<kOut, 2, false>);
        return f(args, stream);
    };
    return dtype == 0 ? launch(std::integral_constant<int, 0>()) : launch(std::integral_constant<int, 1>());
}

extern "C" int p2b_mx4_linear(const void* a_values, const void* a_scales, int64_t rows, const void* w_values, const void* w_scales, int32_t columns,
                              int32_t width, const void* bias, int32_t dtype, int32_t activation, void* out, int64_t out_stride, void* stream) {
    if (rows > 0 && !out) return set_error(P2B_ERR_ARG, "p2b_mx4_linear: null array");
    Mx4Args args{};
    const int rc = prepare_linear("p2b_mx4_linear", args, a_values, a_scales, rows, w_values, w_scales, columns, width, bias, dtype, activation, out, out_stride, nullptr,
                                  nullptr);
    return rc || rows == 0 ? rc : run_linear(args, dtype, activation, (cudaStream_t)stream);
}

extern "C" int p2b_mx4_linear_mx4(const void* a_values, const void* a_scales, int64_t rows, const void* w_values, const void* w_scales, int32_t columns,
                                  int32_t width, const void* bias, int32_t dtype, int32_t activation, void* out_values, void* out_scales, void* stream) {
    if (rows > 0 && (!out_values || !out_scales)) return set_error(P2B_ERR_ARG, "p2b_mx4_linear_mx4: null array");
    Mx4Args args{};
    const int rc = prepare_linear("p2b_mx4_linear_mx4", args, a_values, a_scales, rows, w_values, w_scales, columns, width, bias, dtype, activation, nullptr, 0, out_values,
                                  out_scales);
    return rc || rows == 0 ? rc : run_linear(args, dtype, activation, (cudaStream_t)stream);
}

extern "C" int64_t p2b_mx4_linear_rows_scratch_bytes(int64_t rows, int32_t width) {
    if (rows < 0 || width < 1) return -1;
    return rows <= kFewRows ? 0 : p2b_mx4_scale_bytes(rows, width) + p2b_mx4_value_bytes(rows, width);
}

extern "C" int p2b_mx4_linear_rows(const void* x, int64_t x_stride, int32_t x_dtype, int64_t rows, const void* w_values, const void* w_scales, int32_t columns,
                                   int32_t width, const void* bias, int32_t dtype, int32_t activation, void* out, int64_t out_stride, void* scratch,
                                   int64_t scratch_bytes, void* stream) {
    if (rows <= kFewRows)
        return p2b_mx4_linear_few(x, x_stride, x_dtype, rows, w_values, w_scales, columns, width, bias, dtype, activation, out, out_stride, stream);
    int rc = check_source("p2b_mx4_linear_rows", x, x_stride, rows, width, x_dtype);
    if (rc) return rc;
    if (!scratch || (uintptr_t)scratch % 16 || scratch_bytes < p2b_mx4_linear_rows_scratch_bytes(rows, width))
        return set_error(P2B_ERR_ARG, "p2b_mx4_linear_rows: scratch of %lld bytes on a 16-byte boundary is needed",
                         (long long)p2b_mx4_linear_rows_scratch_bytes(rows, width));
    uint8_t *scales = (uint8_t*)scratch, *values = scales + p2b_mx4_scale_bytes(rows, width);
    // (the product's arguments are looked at before anything is launched)
    Mx4Args args{};
    rc = prepare_linear("p2b_mx4_linear_rows", args, values, scales, rows, w_values, w_scales, columns, width, bias, dtype, activation, out, out_stride, nullptr, nullptr);
    if (!rc) rc = p2b_mx4_quantise(x, x_stride, rows, width, x_dtype, values, scales, stream);
    return rc ? rc : run_linear(args, dtype, activation, (cudaStream_t)stream);
}
