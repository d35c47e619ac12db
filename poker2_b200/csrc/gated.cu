// Gated hidden layer, h = act(x Wg^T + bg) * (x Wu^T + bu), and its gradients, on the tensor cores.
//
// One tile of 128 rows holds 128 gate and 128 up columns next to each other in tensor memory (one matrix instruction of
// 256 columns, its operand half from Wg, half from Wu), so the activation and the product happen on the accumulators and
// neither projection goes through memory.  The backward pass takes the same products again instead of keeping them: its first
// kernel ends in dgate = dh * up * act'(gate), dup = dh * act(gate) (16-bit, side by side in work space), from which
// dx = dgate Wg + dup Wu, dWg = dgate^T x, dWu = dup^T x and the column sums follow.
#include "layer.cuh"
#include "tensor.cuh"

namespace p2b {

using namespace tc;

enum GatedMode { kForward = 0, kGradHidden = 1, kGradInput = 2, kGradWeight = 3 };

struct GatedArgs {
    CUtensorMap a, b0, b1;
    const void *bias_gate, *bias_up, *grad_h;
    void *out0, *out1;
    int64_t grad_stride, out_stride;
    int64_t rows;         // rows of x
    int width, hidden;    // columns of x, rows of either weight
    int hidden_padded;    // columns of dgate (and dup) in work space: a multiple of 128
    int k_blocks;         // steps of 64 along the reduction (kGradInput: of each half)
    int tiles_m, tiles_n;
    int activation;
    int vector_in, vector_out;  // 16-byte loads of grad_h, stores of the outputs
};

constexpr int kRows = 128;     // rows of a tile
constexpr int kStep = 64;      // reduction columns of a stage: 128 bytes
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 32 * (kEpilogueWarps + 2);

template <int kCols> __host__ __device__ constexpr int stages() { return kCols == 256 ? 4 : 6; }
template <int kCols> __host__ __device__ constexpr int stage_bytes() { return kRows * 128 + kCols * 128; }
template <int kCols> __host__ __device__ constexpr int shared_bytes() { return stages<kCols>() * stage_bytes<kCols>() + 1024; }

template <int kMode, int kCols, bool kBf16, int kActivation>
__global__ void __launch_bounds__(kThreads, 1) gated_kernel(const __grid_constant__ GatedArgs args) {
    constexpr int kStages = stages<kCols>();
    constexpr bool kPaired = kMode == kForward || kMode == kGradHidden;  // gate and up columns in one tile
    constexpr int kTileCols = kPaired ? kCols / 2 : kCols;               // output columns of a tile
    constexpr uint32_t kTmem = 2 * kCols < 32 ? 32 : 2 * kCols;
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t bars[2 * kStages + 5];
    __shared__ uint32_t tmem_at;
    __shared__ volatile int given_up;

    const uint32_t ring = (smem_addr(raw) + 1023) & ~1023u;
    const uint32_t bar0 = smem_addr(bars);
    auto full = [&](int s) { return bar0 + 8 * s; };
    auto empty = [&](int s) { return bar0 + 8 * (kStages + s); };
    auto acc_full = [&](int s) { return bar0 + 8 * (2 * kStages + s); };
    auto acc_empty = [&](int s) { return bar0 + 8 * (2 * kStages + 2 + s); };
    const uint32_t last = bar0 + 8 * (2 * kStages + 4);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        given_up = 0;
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(acc_full(s), 1);
            mbar_init(acc_empty(s), 32 * kEpilogueWarps);
        }
        mbar_init(last, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kEpilogueWarps + 1) tmem_alloc(smem_addr(&tmem_at), kTmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    const int tiles = args.tiles_m * args.tiles_n;
    const int steps = kMode == kGradInput ? 2 * args.k_blocks : args.k_blocks;

    if (warp == kEpilogueWarps) {
        if (lane == 0) {
            tma_prefetch_map(&args.a);
            tma_prefetch_map(&args.b0);
            if (kMode != kGradWeight) tma_prefetch_map(&args.b1);
            int64_t issued = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
                const int m0 = tile / args.tiles_n * kRows, n0 = tile % args.tiles_n * kTileCols;
                for (int k = 0; k < steps; ++k, ++issued) {
                    const int s = (int)(issued % kStages);
                    if (issued >= kStages && !mbar_wait(empty(s), (uint32_t)(issued / kStages - 1) & 1, &given_up)) {
                        ok = false;
                        break;
                    }
                    const uint32_t a = ring + s * stage_bytes<kCols>(), b = a + kRows * 128;
                    mbar_expect(full(s), stage_bytes<kCols>());
                    if (kPaired) {
                        tma_load_2d(a, &args.a, k * kStep, m0, full(s));
                        tma_load_2d(b, &args.b0, k * kStep, n0, full(s));
                        tma_load_2d(b + kTileCols * 128, &args.b1, k * kStep, n0, full(s));
                    } else if (kMode == kGradInput) {
                        const bool second = k >= args.k_blocks;
                        const int f0 = (second ? k - args.k_blocks : k) * kStep;
                        tma_load_2d(a, &args.a, f0 + (second ? args.hidden_padded : 0), m0, full(s));
                        for (int c = 0; c < kCols / 64; ++c)
                            tma_load_2d(b + c * 8192, second ? &args.b1 : &args.b0, n0 + 64 * c, f0, full(s));
                    } else {
                        for (int c = 0; c < kRows / 64; ++c) tma_load_2d(a + c * 8192, &args.a, m0 + 64 * c, k * kStep, full(s));
                        for (int c = 0; c < kCols / 64; ++c) tma_load_2d(b + c * 8192, &args.b0, n0 + 64 * c, k * kStep, full(s));
                    }
                }
            }
            if (!ok)  // the copies in flight land before the block's memory goes
                for (int64_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i) {
                    volatile int still = 0;
                    mbar_wait(full((int)(i % kStages)), (uint32_t)(i / kStages) & 1, &still);
                }
        }
        __syncwarp();
    } else if (warp == kEpilogueWarps + 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = f16_idesc(kBf16, kMode == kGradWeight, !kPaired, kRows, kCols);
            int64_t used = 0;
            int turn = 0;
            bool ok = true;
            for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, ++turn) {
                const int acc = turn & 1;
                if (turn >= 2 && !mbar_wait(acc_empty(acc), (uint32_t)(turn / 2 - 1) & 1, &given_up)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                for (int k = 0; k < steps; ++k, ++used) {
                    const int s = (int)(used % kStages);
                    if (!mbar_wait(full(s), (uint32_t)(used / kStages) & 1, &given_up)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = ring + s * stage_bytes<kCols>(), b = a + kRows * 128;
#pragma unroll
                    for (int i = 0; i < kStep / 16; ++i) {
                        // rows along the reduction: 32 bytes on within the swizzled row, else 16 rows of 128 bytes
                        const uint64_t da = kMode == kGradWeight ? operand_desc(a + 2048 * i, 1024, 8192) : operand_desc(a + 32 * i, 1024, 16);
                        const uint64_t db = kPaired ? operand_desc(b + 32 * i, 1024, 16) : operand_desc(b + 2048 * i, 1024, 8192);
                        mma_f16(tmem + acc * kCols, da, db, idesc, k > 0 || i > 0);
                    }
                    tc_commit(empty(s));
                }
                if (ok) tc_commit(acc_full(acc));
            }
            if (!ok) {  // the matrix instructions in flight end before their tensor memory is freed
                volatile int still = 0;
                tc_commit(last);
                mbar_wait(last, 0, &still);
            }
        }
        __syncwarp();
    } else {
        const int quadrant = warp % 4, half = warp / 4;
        const uint32_t lanes = (uint32_t)(quadrant * 32) << 16;
        int turn = 0;
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++turn) {
            const int64_t row = (int64_t)(tile / args.tiles_n) * kRows + quadrant * 32 + lane;
            const int n0 = tile % args.tiles_n * kTileCols, acc = turn & 1;
            const bool ok = mbar_wait(acc_full(acc), (uint32_t)(turn / 2) & 1, &given_up);
            tc_fence_after();
            for (int c = 32 * half; c < kTileCols; c += 64) {
                const uint32_t from = tmem + lanes + acc * kCols + c;
                const int col = n0 + c;
                float v[32];
                if (kPaired) {
                    uint32_t g[32], u[32];
                    tmem_load_32(from, g);
                    tmem_load_32(from + kTileCols, u);
                    float bias_g = 0.0f, bias_u = 0.0f;
                    if (col + lane < args.hidden) {
                        if (args.bias_gate) bias_g = widen<kBf16>(reinterpret_cast<const uint16_t*>(args.bias_gate)[col + lane]);
                        if (args.bias_up) bias_u = widen<kBf16>(reinterpret_cast<const uint16_t*>(args.bias_up)[col + lane]);
                    }
                    if (kMode == kForward) {
                        tmem_load_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            float slope;
                            const float gate = __uint_as_float(g[i]) + __shfl_sync(~0u, bias_g, i);
                            const float up = __uint_as_float(u[i]) + __shfl_sync(~0u, bias_u, i);
                            v[i] = activate<kActivation, false>(gate, slope) * up;
                        }
                    } else {
                        const uint16_t* dh = reinterpret_cast<const uint16_t*>(args.grad_h) + row * args.grad_stride + col;
                        const bool inside = row < args.rows;
                        uint32_t d[16];
                        if (inside && args.vector_in && col + 32 <= args.hidden) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint4 q = __ldg(reinterpret_cast<const uint4*>(dh) + i);
                                d[4 * i] = q.x, d[4 * i + 1] = q.y, d[4 * i + 2] = q.z, d[4 * i + 3] = q.w;
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                d[i] = inside && col + 2 * i < args.hidden ? dh[2 * i] : 0;
                                d[i] |= inside && col + 2 * i + 1 < args.hidden ? (uint32_t)dh[2 * i + 1] << 16 : 0;
                            }
                        }
                        tmem_load_wait();
                        float w[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            float slope;
                            const float gate = __uint_as_float(g[i]) + __shfl_sync(~0u, bias_g, i);
                            const float up = __uint_as_float(u[i]) + __shfl_sync(~0u, bias_u, i);
                            const float a = activate<kActivation, true>(gate, slope);
                            const float2 pair = unpack<kBf16>(d[i / 2]);
                            const float grad = i % 2 ? pair.y : pair.x;
                            // (zero behind the last column, also where a row of x is not finite)
                            v[i] = !ok ? __int_as_float(0x7FC00000) : col + i < args.hidden ? grad * up * slope : 0.0f;
                            w[i] = !ok ? __int_as_float(0x7FC00000) : col + i < args.hidden ? grad * a : 0.0f;
                        }
                        if (inside) store_row<kBf16>(args.out0, row * args.out_stride + args.hidden_padded + col, w, 32, true);
                    }
                } else {
                    uint32_t g[32];
                    tmem_load_32(from, g);
                    tmem_load_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(g[i]);
                }
                if (kMode != kGradHidden && !ok)
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __int_as_float(0x7FC00000);
                if (kMode == kForward) {
                    if (row < args.rows) store_row<kBf16>(args.out0, row * args.out_stride + col, v, args.hidden - col, args.vector_out);
                } else if (kMode == kGradHidden) {
                    if (row < args.rows) store_row<kBf16>(args.out0, row * args.out_stride + col, v, 32, true);
                } else if (kMode == kGradInput) {
                    if (row < args.rows) store_row<kBf16>(args.out0, row * args.out_stride + col, v, args.width - col, args.vector_out);
                } else {
                    const bool up = row >= args.hidden_padded;
                    const int64_t f = up ? row - args.hidden_padded : row;
                    if (f < args.hidden && (up ? args.out1 : args.out0))
                        store_row<kBf16>(up ? args.out1 : args.out0, f * args.out_stride + col, v, args.width - col, args.vector_out);
                }
            }
            tc_fence_before();
            mbar_arrive(acc_empty(acc));
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kEpilogueWarps + 1) {
        tc_fence_after();
        tmem_free(tmem, kTmem);
    }
}

// Few rows: a warp takes one gate and one up row of the weights, which pass through the chip once, against all rows of x.
// Bound by the way from L2 and the launch: at 1 row, width 1536, hidden 1024 the weights are 6.3 MB.
template <int kMost, bool kBf16, int kActivation>
__global__ void __launch_bounds__(128) gated_few_kernel(const uint16_t* x, int64_t x_stride, const uint16_t* wg, int64_t wg_stride,
                                                        const uint16_t* wu, int64_t wu_stride, const uint16_t* bg, const uint16_t* bu,
                                                        int rows, int width, int hidden, uint16_t* h, int64_t h_stride, int vector) {
    const int f = blockIdx.x * 4 + threadIdx.x / 32, lane = threadIdx.x % 32;
    if (f >= hidden) return;
    float g[kMost], u[kMost];
#pragma unroll
    for (int r = 0; r < kMost; ++r) g[r] = u[r] = 0.0f;
    const uint16_t *pg = wg + f * wg_stride, *pu = wu + f * wu_stride;
    if (vector) {
#pragma unroll 2
        for (int k = lane * 8; k + 8 <= width; k += 256) {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(pg + k)), b = __ldg(reinterpret_cast<const uint4*>(pu + k));
            const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int r = 0; r < kMost; ++r)
                if (r < rows) {
                    const uint4 c = __ldg(reinterpret_cast<const uint4*>(x + r * x_stride + k));
                    const uint32_t wc[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 p = unpack<kBf16>(wa[i]), q = unpack<kBf16>(wb[i]), v = unpack<kBf16>(wc[i]);
                        g[r] = fmaf(p.y, v.y, fmaf(p.x, v.x, g[r]));
                        u[r] = fmaf(q.y, v.y, fmaf(q.x, v.x, u[r]));
                    }
                }
        }
    }
    for (int k = (vector ? width / 8 * 8 : 0) + lane; k < width; k += 32) {
        const float a = widen<kBf16>(pg[k]), b = widen<kBf16>(pu[k]);
#pragma unroll
        for (int r = 0; r < kMost; ++r)
            if (r < rows) {
                const float v = widen<kBf16>(x[r * x_stride + k]);
                g[r] = fmaf(a, v, g[r]);
                u[r] = fmaf(b, v, u[r]);
            }
    }
#pragma unroll
    for (int r = 0; r < kMost; ++r)
#pragma unroll
        for (int o = 16; o > 0; o /= 2) {
            g[r] += __shfl_xor_sync(~0u, g[r], o);
            u[r] += __shfl_xor_sync(~0u, u[r], o);
        }
#pragma unroll
    for (int r = 0; r < kMost; ++r)
        if (lane == r && r < rows) {
            float slope;
            const float gate = g[r] + (bg ? widen<kBf16>(bg[f]) : 0.0f), up = u[r] + (bu ? widen<kBf16>(bu[f]) : 0.0f);
            h[r * h_stride + f] = narrow<kBf16>(activate<kActivation, false>(gate, slope) * up);
        }
}

// Column sums of dgate | dup: a block adds `chunk` rows of 64 columns, and a second launch the blocks' sums in their order.
template <bool kBf16>
__global__ void __launch_bounds__(256) column_sums_kernel(const uint16_t* d, int64_t stride, int64_t rows, int64_t chunk, float* partial, int columns) {
    __shared__ float2 part[8][32];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int col = blockIdx.x * 64 + 2 * lane;
    const int64_t first = blockIdx.y * chunk, end = first + chunk < rows ? first + chunk : rows;
    float2 sum = {0.0f, 0.0f};
    for (int64_t r = first + warp; r < end; r += 8) {
        const float2 v = unpack<kBf16>(*reinterpret_cast<const uint32_t*>(d + r * stride + col));
        sum.x += v.x;
        sum.y += v.y;
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0) {
#pragma unroll
        for (int w = 1; w < 8; ++w) {
            sum.x += part[w][lane].x;
            sum.y += part[w][lane].y;
        }
        float* p = partial + (int64_t)blockIdx.y * columns + col;
        p[0] = sum.x;
        p[1] = sum.y;
    }
}
template <bool kBf16>
__global__ void __launch_bounds__(128) column_totals_kernel(const float* partial, int parts, int hidden, int hidden_padded, uint16_t* gate, uint16_t* up) {
    const int c = blockIdx.x * 128 + threadIdx.x;
    if (c >= 2 * hidden_padded) return;
    float sum = 0.0f;
    for (int p = 0; p < parts; ++p) sum += partial[(int64_t)p * 2 * hidden_padded + c];
    const bool second = c >= hidden_padded;
    const int f = second ? c - hidden_padded : c;
    uint16_t* out = second ? up : gate;
    if (f < hidden && out) out[f] = narrow<kBf16>(sum);
}

static SharedLimit g_limit[4][2][2][2];

template <int kMode, int kCols, bool kBf16, int kActivation> static int launch(const GatedArgs& args, cudaStream_t stream) {
    auto* kernel = gated_kernel<kMode, kCols, kBf16, kActivation>;
    int rc = allow_shared(g_limit[kMode][kCols == 256][kBf16][kActivation], (const void*)kernel, shared_bytes<kCols>());
    if (rc) return rc;
    const int tiles = args.tiles_m * args.tiles_n;
    kernel<<<tiles < sm_count() ? tiles : sm_count(), kThreads, shared_bytes<kCols>(), stream>>>(args);
    return check_cuda(cudaGetLastError(), "gated_kernel");
}
template <int kMode, int kCols> static int launch(const GatedArgs& args, bool bf16, cudaStream_t stream) {
    if (kMode == kGradInput || kMode == kGradWeight)
        return bf16 ? launch<kMode, kCols, true, 0>(args, stream) : launch<kMode, kCols, false, 0>(args, stream);
    if (args.activation == kGelu)
        return bf16 ? launch<kMode, kCols, true, kGelu>(args, stream) : launch<kMode, kCols, false, kGelu>(args, stream);
    return bf16 ? launch<kMode, kCols, true, kSilu>(args, stream) : launch<kMode, kCols, false, kSilu>(args, stream);
}


constexpr int kFewRows = 8;
constexpr int64_t kMostRows = 1ll << 30;
constexpr int kMostColumns = 1 << 20;

static int check_layer(const char* name, const void* x, int64_t x_stride, const void* wg, int64_t wg_stride, const void* wu, int64_t wu_stride,
                       int64_t rows, int32_t width, int32_t hidden, int32_t dtype, int32_t activation) {
    if (rows < 0 || rows > kMostRows || width < 1 || width > kMostColumns || hidden < 1 || hidden > kMostColumns)
        return set_error(P2B_ERR_ARG, "%s: %lld rows, width %d, hidden %d are out of range", name, (long long)rows, width, hidden);
    // (tiles are counted in 32 bits)
    if ((rows + 127) / 128 * ((hidden + 31) / 32) > 0x7FFF0000ll || (rows + 127) / 128 * ((width + 31) / 32) > 0x7FFF0000ll)
        return set_error(P2B_ERR_ARG, "%s: %lld rows of %d to %d are too many for one call", name, (long long)rows, width, hidden);
    if (dtype < 0 || dtype > 1) return set_error(P2B_ERR_ARG, "%s: unknown type %d (0 bf16, 1 fp16)", name, dtype);
    if (activation < 0 || activation > 1) return set_error(P2B_ERR_ARG, "%s: unknown activation %d (0 gelu, 1 silu)", name, activation);
    if ((rows > 0 && !x) || !wg || !wu) return set_error(P2B_ERR_ARG, "%s: null operand", name);
    if ((rows > 1 && x_stride < width) || (hidden > 1 && (wg_stride < width || wu_stride < width)))
        return set_error(P2B_ERR_ARG, "%s: rows overlap", name);
    return P2B_OK;
}

// Maps of x (rows x 64 boxes) and of the weights for the paired products.
static int paired_maps(GatedArgs& args, const void* x, int64_t x_stride, const void* wg, int64_t wg_stride, const void* wu, int64_t wu_stride, int cols) {
    int rc = encode_rows(&args.a, x, 2, args.width, args.rows, 2 * x_stride, kRows);
    if (!rc) rc = encode_rows(&args.b0, wg, 2, args.width, args.hidden, 2 * wg_stride, cols / 2);
    if (!rc) rc = encode_rows(&args.b1, wu, 2, args.width, args.hidden, 2 * wu_stride, cols / 2);
    args.k_blocks = (int)blocks_of(args.width, kStep);
    args.tiles_m = (int)blocks_of(args.rows, kRows);
    args.tiles_n = (int)blocks_of(args.hidden, cols / 2);
    return rc;
}

// A tile of 32 hidden columns where the wide ones would leave more than half of the multiprocessors without one.
static bool narrow_tiles(int64_t rows, int32_t hidden) { return 2 * blocks_of(rows, kRows) * blocks_of(hidden, 128) <= sm_count(); }

template <bool kBf16, int kActivation>
static int launch_few(const void* x, int64_t x_stride, const void* wg, int64_t wg_stride, const void* wu, int64_t wu_stride, const void* bg,
                      const void* bu, int rows, int width, int hidden, void* h, int64_t h_stride, cudaStream_t stream) {
    const int vector = aligned16(x, rows > 1 ? x_stride : 0) && aligned16(wg, wg_stride) && aligned16(wu, wu_stride);
    auto* kernel = rows == 1 ? gated_few_kernel<1, kBf16, kActivation> : rows <= 4 ? gated_few_kernel<4, kBf16, kActivation> : gated_few_kernel<kFewRows, kBf16, kActivation>;
    kernel<<<(unsigned)blocks_of(hidden, 4), 128, 0, stream>>>((const uint16_t*)x, x_stride, (const uint16_t*)wg, wg_stride, (const uint16_t*)wu, wu_stride,
                                                              (const uint16_t*)bg, (const uint16_t*)bu, rows, width, hidden, (uint16_t*)h, h_stride, vector);
    return check_cuda(cudaGetLastError(), "gated_few_kernel");
}

}  // namespace p2b

using namespace p2b;

extern "C" int p2b_gated_few_rows(void) { return kFewRows; }

extern "C" int p2b_gated_forward(const void* x, int64_t x_stride, const void* wg, int64_t wg_stride, const void* wu, int64_t wu_stride,
                                 const void* bg, const void* bu, int64_t rows, int32_t width, int32_t hidden, int32_t dtype,
                                 int32_t activation, void* h, int64_t h_stride, void* stream) {
    int rc = check_layer("p2b_gated_forward", x, x_stride, wg, wg_stride, wu, wu_stride, rows, width, hidden, dtype, activation);
    if (rc) return rc;
    if (rows == 0) return P2B_OK;
    if (!h || (rows > 1 && h_stride < hidden)) return set_error(P2B_ERR_ARG, "p2b_gated_forward: null output or rows that overlap");
    const bool bf16 = dtype == 0;
    cudaStream_t st = (cudaStream_t)stream;
    if (rows <= kFewRows) {
        auto* few = activation == kGelu ? (bf16 ? launch_few<true, kGelu> : launch_few<false, kGelu>) : (bf16 ? launch_few<true, kSilu> : launch_few<false, kSilu>);
        return few(x, x_stride, wg, wg_stride, wu, wu_stride, bg, bu, (int)rows, width, hidden, h, h_stride, st);
    }
    if (!aligned16(x, x_stride) || !aligned16(wg, hidden > 1 ? wg_stride : 0) || !aligned16(wu, hidden > 1 ? wu_stride : 0))
        return set_error(P2B_ERR_ARG, "p2b_gated_forward: rows of x and of the weights must start on 16-byte boundaries");
    GatedArgs args{};
    args.rows = rows, args.width = width, args.hidden = hidden, args.activation = activation;
    args.bias_gate = bg, args.bias_up = bu, args.out0 = h, args.out_stride = h_stride, args.vector_out = aligned16(h, h_stride);
    const bool slim = narrow_tiles(rows, hidden);
    rc = paired_maps(args, x, x_stride, wg, hidden > 1 ? wg_stride : blocks_of(width, 8) * 8, wu, hidden > 1 ? wu_stride : blocks_of(width, 8) * 8, slim ? 64 : 256);
    if (rc) return rc;
    return slim ? launch<kForward, 64>(args, bf16, st) : launch<kForward, 256>(args, bf16, st);
}

static int sum_parts(int64_t rows) { return (int)(rows < 64 * 64 ? blocks_of(rows, 64) : 64); }

extern "C" int64_t p2b_gated_backward_scratch_bytes(int64_t rows, int32_t hidden) {
    if (rows < 0 || rows > kMostRows || hidden < 1 || hidden > kMostColumns) return -1;
    const int64_t columns = 2 * blocks_of(hidden, 128) * 128;
    return 2 * rows * columns + 4 * columns * sum_parts(rows);
}

extern "C" int p2b_gated_backward(const void* grad_h, int64_t grad_stride, const void* x, int64_t x_stride, const void* wg, int64_t wg_stride,
                                  const void* wu, int64_t wu_stride, const void* bg, const void* bu, int64_t rows, int32_t width,
                                  int32_t hidden, int32_t dtype, int32_t activation, void* dx, int64_t dx_stride, void* dwg, void* dwu,
                                  void* dbg, void* dbu, void* scratch, int64_t scratch_bytes, void* stream) {
    int rc = check_layer("p2b_gated_backward", x, x_stride, wg, wg_stride, wu, wu_stride, rows, width, hidden, dtype, activation);
    if (rc) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if (rows == 0) {  // no row: gradients of the weights are zero
        for (void* w : {dwg, dwu})
            if (w && (rc = check_cuda(cudaMemsetAsync(w, 0, (size_t)2 * width * hidden, st), "p2b_gated_backward"))) return rc;
        for (void* b : {dbg, dbu})
            if (b && (rc = check_cuda(cudaMemsetAsync(b, 0, (size_t)2 * hidden, st), "p2b_gated_backward"))) return rc;
        return P2B_OK;
    }
    if (!grad_h || (rows > 1 && grad_stride < hidden)) return set_error(P2B_ERR_ARG, "p2b_gated_backward: null gradient or rows that overlap");
    if (dx && rows > 1 && dx_stride < width) return set_error(P2B_ERR_ARG, "p2b_gated_backward: rows of dx overlap");
    if (!aligned16(x, rows > 1 ? x_stride : 0) || !aligned16(wg, hidden > 1 ? wg_stride : 0) || !aligned16(wu, hidden > 1 ? wu_stride : 0))
        return set_error(P2B_ERR_ARG, "p2b_gated_backward: rows of x and of the weights must start on 16-byte boundaries");
    if (!scratch || ((uintptr_t)scratch % 16) != 0 || scratch_bytes < p2b_gated_backward_scratch_bytes(rows, hidden))
        return set_error(P2B_ERR_ARG, "p2b_gated_backward: scratch of %lld bytes on a 16-byte boundary is needed",
                         (long long)p2b_gated_backward_scratch_bytes(rows, hidden));
    const bool bf16 = dtype == 0;
    const int64_t whole = blocks_of(width, 8) * 8;
    if (rows == 1) x_stride = whole;
    if (hidden == 1) wg_stride = wu_stride = whole;
    GatedArgs args{};
    args.rows = rows, args.width = width, args.hidden = hidden, args.activation = activation;
    args.hidden_padded = (int)blocks_of(hidden, 128) * 128;
    args.bias_gate = bg, args.bias_up = bu, args.grad_h = grad_h, args.grad_stride = grad_stride;
    args.vector_in = aligned16(grad_h, rows > 1 ? grad_stride : 0);
    const int64_t columns = 2 * (int64_t)args.hidden_padded;
    args.out0 = scratch, args.out_stride = columns;
    rc = paired_maps(args, x, x_stride, wg, wg_stride, wu, wu_stride, 256);
    if (!rc) rc = launch<kGradHidden, 256>(args, bf16, st);
    if (rc) return rc;
    if (dx) {
        GatedArgs in = args;
        rc = encode_rows(&in.a, scratch, 2, columns, rows, 2 * columns, kRows);
        if (!rc) rc = encode_rows(&in.b0, wg, 2, width, hidden, 2 * wg_stride, kStep);
        if (!rc) rc = encode_rows(&in.b1, wu, 2, width, hidden, 2 * wu_stride, kStep);
        if (rc) return rc;
        in.k_blocks = (int)blocks_of(hidden, kStep);
        in.tiles_n = (int)blocks_of(width, 256);
        in.out0 = dx, in.out_stride = dx_stride, in.vector_out = aligned16(dx, rows > 1 ? dx_stride : 0);
        rc = launch<kGradInput, 256>(in, bf16, st);
        if (rc) return rc;
    }
    if (dwg || dwu) {
        GatedArgs in = args;
        rc = encode_rows(&in.a, scratch, 2, columns, rows, 2 * columns, kStep);
        if (!rc) rc = encode_rows(&in.b0, x, 2, width, rows, 2 * x_stride, kStep);
        if (rc) return rc;
        in.k_blocks = (int)blocks_of(rows, kStep);
        in.tiles_m = (int)(columns / kRows);
        in.tiles_n = (int)blocks_of(width, 256);
        in.out0 = dwg, in.out1 = dwu, in.out_stride = width;
        in.vector_out = (!dwg || aligned16(dwg, width)) && (!dwu || aligned16(dwu, width));
        rc = launch<kGradWeight, 256>(in, bf16, st);
        if (rc) return rc;
    }
    if (dbg || dbu) {
        float* partial = (float*)((char*)scratch + 2 * rows * columns);
        const int parts = sum_parts(rows);
        const dim3 grid((unsigned)(columns / 64), parts);
        const int64_t chunk = blocks_of(rows, parts);
        auto* sums = bf16 ? column_sums_kernel<true> : column_sums_kernel<false>;
        auto* totals = bf16 ? column_totals_kernel<true> : column_totals_kernel<false>;
        sums<<<grid, 256, 0, st>>>((const uint16_t*)scratch, columns, rows, chunk, partial, (int)columns);
        totals<<<(unsigned)(columns / 128), 128, 0, st>>>(partial, parts, hidden, args.hidden_padded, (uint16_t*)dbg, (uint16_t*)dbu);
        rc = check_cuda(cudaGetLastError(), "column sums");
    }
    return rc;
}
