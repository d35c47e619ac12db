// Gated hidden layer, h = act(x Wg^T + bg) * (x Wu^T + bu), and its gradients, on the tensor cores.
//
// One tile of 128 rows holds 128 gate and 128 up columns next to each other in tensor memory (one matrix instruction of
// 256 columns, its operand half from Wg, half from Wu), so the activation and the product happen on the accumulators and
// neither projection goes through memory.  Bound by the matrix instructions and what feeds them: 24576 rows of 1536 -> 1024 (155
// GFLOP, 2 x 1024 x 1536 weights in L2) take 110 to 125 us, 1.24 to 1.41 PFLOP/s; 1.21 GB of operand tiles come
// out of L2 meanwhile, 9.7 to 11 TB/s.  The backward pass takes the
// same products again or, in large layers, finds gate and up in fp32 as the forward pass of the step kept them (`keeps` below).  From
// them come dgate = dh * up * act'(gate) and dup = dh * act(gate) (16-bit, side by side in work space), and from these
// dx = dgate Wg + dup Wu, dWg = dgate^T x, dWu = dup^T x and the column sums.
#include "layer.cuh"
#include "tensor.cuh"

namespace p2b {

using namespace tc;

enum GatedMode { kForward = 0, kGradHidden = 1, kGradients = 2, kForwardKept = 3 };

struct GatedArgs {
    CUtensorMap a, b0, b1;   // kForward, kGradHidden: x, Wg, Wu; kGradients: dgate | dup by rows, Wg, Wu
    CUtensorMap at, bt;      // kGradients: dgate | dup and x with the reduction along their rows
    CUtensorMap to, to_wg, to_wu;  // the outputs out, dwg, dwu, where their rows start on 16-byte boundaries
    CUtensorMap kept;              // kForwardKept: gate and up in fp32, upper halves and then lower halves side by side
    const void *bias_gate, *bias_up, *grad_h;
    void *out, *dwg, *dwu;   // h, dgate | dup or dx; the gradients of the weights
    float* sums;             // column sums of dgate | dup over 32 rows each, left by kGradHidden for kGradients (NULL: not wanted)
    void *dbg, *dbu;         // kGradients: the gradients of the biases, from the sums
    int parts;               // 16-bit numbers that dgate and dup are kept in: 1, or 2 whose sum they are
    int64_t grad_stride, out_stride;
    int64_t rows;            // rows of x
    int width, hidden;       // columns of x, rows of either weight
    int hidden_padded;       // columns of dgate (and dup) in work space: a multiple of 128
    int steps, steps_w;      // steps of 64 along the reduction of a tile; kGradients: of dx, of the weights
    int tiles_n, tiles;      // tiles of out
    int tiles_w_n, tiles_w;  // kGradients: tiles of the weights' gradients, and how many of the
    int ahead;               //   other tiles a pair without a last one of those takes in its place
    int vector_in, vector_bias;      // 16-byte loads of grad_h and of the biases
    int align_out, align_w;          // row_alignment of the outputs
};

constexpr int kRows = 128;   // rows of a block's tile
constexpr int kStep = 64;    // reduction columns of a stage: 128 bytes
constexpr int kEpilogueWarps = 16;
constexpr int kThreads = 32 * (kEpilogueWarps + 2);

// Sum over the warp's lanes of each of 32 values: lane l ends with the sum of value l.  Half of the values change places in
// every round, 31 exchanges in all.
__device__ __forceinline__ float lane_sums(float (&v)[32], int lane) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2) {
        const bool upper = lane & o;
#pragma unroll
        for (int i = 0; i < o; ++i) {
            const float give = upper ? v[i] : v[i + o], keep = upper ? v[i + o] : v[i];
            v[i] = keep + __shfl_xor_sync(~0u, give, o);
        }
    }
    return v[0];
}

// The biases as the epilogues read them: of up to kBiasColumns hidden units from shared memory, zeros behind the last, else from
// where they are.
constexpr int kBiasColumns = 2048;
struct Biases {
    const uint16_t *gate, *up;
    int count_gate, count_up;  // entries that may be read
    bool vector;
};
__device__ __forceinline__ Biases stage_biases(const GatedArgs& args, uint16_t* area, int threads) {
    const uint16_t *gate = reinterpret_cast<const uint16_t*>(args.bias_gate), *up = reinterpret_cast<const uint16_t*>(args.bias_up);
    if (args.hidden_padded > kBiasColumns) return {gate, up, gate ? args.hidden : 0, up ? args.hidden : 0, (bool)args.vector_bias};
    for (int f = threadIdx.x; f < args.hidden_padded; f += threads) {
        area[f] = gate && f < args.hidden ? gate[f] : 0;
        area[args.hidden_padded + f] = up && f < args.hidden ? up[f] : 0;
    }
    return {area, area + args.hidden_padded, args.hidden_padded, args.hidden_padded, true};
}

// Two fp32 numbers as their upper and their lower halves, and back.
__device__ __forceinline__ void keep(float2 v, uint32_t& upper, uint32_t& lower) {
    upper = __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x7632);
    lower = __byte_perm(__float_as_uint(v.x), __float_as_uint(v.y), 0x5410);
}
__device__ __forceinline__ Two kept_pair(uint32_t upper, uint32_t lower) {
    return Two(__uint_as_float(__byte_perm(lower, upper, 0x5410)), __uint_as_float(__byte_perm(lower, upper, 0x7632)));
}
__device__ __forceinline__ void put_words(uint8_t* panel, int r, int col, const uint32_t (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
        *reinterpret_cast<uint4*>(panel + r * 128 + ((col / 8 + i) ^ (r & 7)) * 16) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
}

// 16 hidden columns of a warp's 32 rows, from the accumulators of gate and up to h (v[0..15]) or to dgate and dup (v[0..15], v[16..31]).
// (grad: 16 columns of grad_h, loaded before the accumulators were waited for; kept: kForwardKept, the halves of gate and up.)
template <int kMode, bool kBf16, int kActivation>
__device__ __forceinline__ void finish_hidden(const GatedArgs& args, const Biases& bias, const uint32_t (&grad)[8], uint32_t gate_at, uint32_t up_at,
                                              int64_t row, int col, bool ok, float (&v)[32], uint32_t (&kept)[4][8]) {
    uint32_t g[16], u[16], bg[8], bu[8];
    tmem_load_16(gate_at, g);
    tmem_load_16(up_at, u);
    load_words(bias.gate + col, bias.count_gate - col, bias.vector, bg);
    load_words(bias.up + col, bias.count_up - col, bias.vector, bu);
    const bool inside = row < args.rows;
    tmem_load_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        Two slope;
        const Two gate = Two(__uint_as_float(g[2 * i]), __uint_as_float(g[2 * i + 1])) + two_of<kBf16>(bg[i]);
        const Two up = Two(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1])) + two_of<kBf16>(bu[i]);
        const Two a = activate<kActivation, kMode == kGradHidden>(gate, slope);
        if (kMode == kForward || kMode == kForwardKept) {
            const float2 h = (a * up).apart();
            v[2 * i] = ok ? h.x : __int_as_float(0x7FC00000);
            v[2 * i + 1] = ok ? h.y : __int_as_float(0x7FC00000);
            if (kMode == kForwardKept) {
                const float2 gates = gate.apart(), ups = up.apart();
                keep(ok ? gates : make_float2(__int_as_float(0x7FC00000), __int_as_float(0x7FC00000)), kept[0][i], kept[2][i]);
                keep(ups, kept[1][i], kept[3][i]);
            }
        } else {
            const Two dh = two_of<kBf16>(grad[i]);
            const float2 dgate = (dh * up * slope).apart(), dup = (dh * a).apart();
            // (zero behind the last row and column, also where x is not finite)
            const bool first = inside && col + 2 * i < args.hidden, second = inside && col + 2 * i + 1 < args.hidden;
            v[2 * i] = !ok ? __int_as_float(0x7FC00000) : first ? dgate.x : 0.0f;
            v[2 * i + 1] = !ok ? __int_as_float(0x7FC00000) : second ? dgate.y : 0.0f;
            v[16 + 2 * i] = !ok ? __int_as_float(0x7FC00000) : first ? dup.x : 0.0f;
            v[17 + 2 * i] = !ok ? __int_as_float(0x7FC00000) : second ? dup.y : 0.0f;
        }
    }
}
__device__ __forceinline__ void split(const float (&v)[32], float (&lower)[16], float (&upper)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) lower[i] = v[i], upper[i] = v[16 + i];
}
// v minus its value in 16 bits
template <bool kBf16> __device__ __forceinline__ void take_rounded(float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float rest = v[i] - widen<kBf16>(narrow<kBf16>(v[i]));
        v[i] = isfinite(rest) ? rest : 0.0f;  // (the first part says it already)
    }
}
// Column sums of dgate and dup (16 columns each) over the warp's 32 rows.
__device__ __forceinline__ void sum_hidden(const GatedArgs& args, float (&v)[32], int64_t row, int col, int lane) {
    if (!args.sums || row - lane >= args.rows) return;
    const float sum = lane_sums(v, lane);
    args.sums[(row / 32) * 2 * args.hidden_padded + (lane < 16 ? 0 : args.hidden_padded - 16) + col + lane] = sum;
}

// Gradients of the biases: the column sums of 32 rows each, added up.  512 threads (16 warps, barrier 5) take 32 columns at a time, a
// warp every sixteenth of the sums.  kGradients does it while its first tile is on its way.
template <bool kBf16> __device__ __forceinline__ void add_bias_gradients(const GatedArgs& args, float* area, int block, int blocks) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t sums = (args.rows + 31) / 32;
    for (int c0 = block * 32; c0 < 2 * args.hidden_padded; c0 += blocks * 32) {
        float sum = 0.0f;
#pragma unroll 4
        for (int64_t p = warp; p < sums; p += 16) sum += args.sums[p * 2 * args.hidden_padded + c0 + lane];
        area[threadIdx.x] = sum;
        group_sync(5, 512);
        if (warp == 0) {
#pragma unroll
            for (int w = 1; w < 16; ++w) sum += area[w * 32 + lane];
            const bool second = c0 >= args.hidden_padded;
            const int f = c0 + lane - (second ? args.hidden_padded : 0);
            uint16_t* out = reinterpret_cast<uint16_t*>(second ? args.dbu : args.dbg);
            if (f < args.hidden && out) out[f] = narrow<kBf16>(sum);
        }
        group_sync(5, 512);
    }
}

// Which tiles a pair takes, the same for its producers, its matrix instructions and its epilogues.  kGradients: first the tiles
// of the weights' gradients, pair after pair; the pairs that get one less of them go ahead on the tiles of dx.
template <int kMode> struct Walk {
    int pair, pairs, next, free_pairs, ahead_left, behind;
    bool on_weights;
    __device__ __forceinline__ Walk(const GatedArgs& args, int pair_, int pairs_) : pair(pair_), pairs(pairs_), next(pair_) {
        on_weights = kMode == kGradients && args.tiles_w > 0;
        const int extra = kMode == kGradients ? args.tiles_w % pairs : 0;
        free_pairs = extra > 0 ? pairs - extra : 0;
        ahead_left = extra > 0 && pair >= extra ? args.ahead : 0;
        behind = extra > 0 ? min(args.ahead * free_pairs, args.tiles) : 0;
        if (!on_weights) enter(args);
    }
    __device__ __forceinline__ void enter(const GatedArgs& args) {
        on_weights = false;
        next = ahead_left > 0 ? pair - (pairs - free_pairs) : behind + pair;
    }
    // the next tile; false when there is none left
    __device__ __forceinline__ bool take(const GatedArgs& args, int& tile, bool& weights) {
        if (on_weights) {
            if (next < args.tiles_w) {
                tile = next, weights = true;
                next += pairs;
                return true;
            }
            enter(args);
        }
        weights = false;
        if (ahead_left > 0) {
            if (next < behind) {
                tile = next;
                next += free_pairs;
                if (--ahead_left == 0) next = behind + pair;
                return true;
            }
            ahead_left = 0;
            next = behind + pair;
        }
        if (next >= args.tiles) return false;
        tile = next;
        next += pairs;
        return true;
    }
};

// Pairs of blocks: 256 rows x 256 accumulator columns a tile, of which a block holds 128 rows of one operand and 128 of the other, so
// that a step of 64 brings 32 KB to each multiprocessor for 512 clocks of matrix instructions (a block by itself: 48 KB).
// Accumulators in turn: the epilogue of a tile runs beside the products of the next.
constexpr int kPairStages = 5;
constexpr int kPairStage = 2 * kRows * 128;
constexpr int kBiasBytes = 4 * kBiasColumns;
constexpr int kPairShared = kPairStages * kPairStage + 2 * kPanelBytes + kBiasBytes + 1024;

template <int kMode, bool kBf16, int kActivation>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) gated_pair_kernel(const __grid_constant__ GatedArgs args) {
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t bars[2 * kPairStages + 5];
    __shared__ uint32_t tmem_at;
    __shared__ volatile int given_up;
    const uint32_t ring = (smem_addr(raw) + 1023) & ~1023u, bar0 = smem_addr(bars);
    auto full = [&](int s) { return bar0 + 8 * s; };
    auto empty = [&](int s) { return bar0 + 8 * (kPairStages + s); };
    auto acc_full = [&](int s) { return bar0 + 8 * (2 * kPairStages + s); };
    auto acc_empty = [&](int s) { return bar0 + 8 * (2 * kPairStages + 2 + s); };
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = (int)pair_rank(), pair = blockIdx.x / 2, pairs = gridDim.x / 2;
    if (threadIdx.x == 0) {
        given_up = 0;
        for (int s = 0; s < kPairStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(acc_full(s), 1);
            mbar_init(acc_empty(s), 2 * kEpilogueWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kEpilogueWarps + 1) pair_tmem_alloc(smem_addr(&tmem_at), 512);
    Biases bias{};
    uint8_t* const panels = raw + (ring - smem_addr(raw)) + kPairStages * kPairStage;
    if (kMode != kGradients) bias = stage_biases(args, reinterpret_cast<uint16_t*>(panels + 2 * kPanelBytes), kThreads);
    tc_fence_before();
    __syncthreads();
    pair_sync();
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    Walk<kMode> walk(args, pair, pairs);
    int tile;
    bool weights;

    if (warp == kEpilogueWarps) {
        if (lane == 0) {
            tma_prefetch_map(&args.a);
            tma_prefetch_map(&args.b0);
            tma_prefetch_map(&args.b1);
            // (the thread that issues the copies sets the pace of the products: stages and coordinates are counted, not divided)
            const uint32_t leader_full = in_leader(full(0));
            int s = 0;
            uint32_t phase = 1;  // (the stages begin empty)
            bool ok = true;
            while (ok && walk.take(args, tile, weights)) {
                const int across = weights ? args.tiles_w_n : args.tiles_n, steps = weights ? args.steps_w : args.steps;
                const int m0 = tile / across * 256 + rank * 128, n = tile % across;
                // kGradients: the reduction goes over dgate (with Wg), dup (with Wu), then the rests of both; or twice over the rows of x
                const int run = kMode != kGradients ? 0 : (weights ? steps / args.parts : steps / (2 * args.parts)) * kStep;
                int side = 0, at = 0;
                for (int k = 0; k < steps; ++k) {
                    if (!pair_wait(empty(s), phase, &given_up)) {
                        ok = false;
                        break;
                    }
                    const uint32_t a = ring + s * kPairStage, b = a + kRows * 128, bar = leader_full + 8 * s;
                    if (rank == 0) mbar_expect(full(s), 2 * kPairStage);
                    if (kMode != kGradients) {
                        pair_load_2d(a, &args.a, at, m0, bar);
                        pair_load_2d(b, rank == 0 ? &args.b0 : &args.b1, at, n * 128, bar);
                    } else if (weights) {
                        for (int c = 0; c < 2; ++c) {
                            pair_load_2d(a + c * 8192, &args.at, m0 + 64 * c + 2 * side * args.hidden_padded, at, bar);
                            pair_load_2d(b + c * 8192, &args.bt, n * 256 + rank * 128 + 64 * c, at, bar);
                        }
                    } else {
                        pair_load_2d(a, &args.a, at + side * args.hidden_padded, m0, bar);
                        for (int c = 0; c < 2; ++c)
                            pair_load_2d(b + c * 8192, side & 1 ? &args.b1 : &args.b0, n * 256 + rank * 128 + 64 * c, at, bar);
                    }
                    at += kStep;
                    if (kMode == kGradients && at == run) at = 0, ++side;
                    if (++s == kPairStages) s = 0, phase ^= 1;
                }
            }
            if (!ok) let_settle();
        }
        __syncwarp();
    } else if (warp == kEpilogueWarps + 1) {
        if (lane == 0 && rank == 0) {
            int s = 0, turn = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (; ok && walk.take(args, tile, weights); ++turn) {
                const int acc = turn & 1, steps = weights ? args.steps_w : args.steps;
                if (turn >= 2 && !pair_wait(acc_empty(acc), (uint32_t)(turn / 2 - 1) & 1, &given_up)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t idesc = f16_idesc(kBf16, weights, kMode == kGradients, 256, 256);
                // rows along the reduction: 32 bytes on within the swizzled row, else 16 rows of 128 bytes
                const uint64_t a0 = weights ? operand_desc(ring, 1024, 8192) : operand_desc(ring, 1024, 16);
                const uint64_t b0 = kMode == kGradients ? operand_desc(ring + kRows * 128, 1024, 8192) : operand_desc(ring + kRows * 128, 1024, 16);
                const uint32_t a_on = weights ? 2048 >> 4 : 32 >> 4, b_on = kMode == kGradients ? 2048 >> 4 : 32 >> 4;
                uint32_t add = 0;
                for (int k = 0; k < steps; ++k) {
                    if (!pair_wait(full(s), phase, &given_up)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t da = a0 + s * (kPairStage >> 4), db = b0 + s * (kPairStage >> 4);
#pragma unroll
                    for (int i = 0; i < kStep / 16; ++i) {
                        pair_mma_f16(tmem + acc * 256, da + i * a_on, db + i * b_on, idesc, add);
                        add = 1;
                    }
                    pair_commit(empty(s));
                    if (++s == kPairStages) s = 0, phase ^= 1;
                }
                if (ok) pair_commit(acc_full(acc));
            }
            if (!ok) let_settle();
        }
        __syncwarp();
    } else {
        // The four warps of a quadrant (32 rows) fill its part of the panels; their first thread stores it.
        const int quadrant = warp % 4, part = warp / 4, r = quadrant * 32 + lane;
        const bool storer = part == 0 && lane == 0;
        const uint32_t lanes = (uint32_t)(quadrant * 32) << 16;
        if (kMode == kGradients && args.sums) add_bias_gradients<kBf16>(args, reinterpret_cast<float*>(panels), blockIdx.x, gridDim.x);
        for (int turn = 0; walk.take(args, tile, weights); ++turn) {
            const int across = weights ? args.tiles_w_n : args.tiles_n, n = tile % across, acc = turn & 1;
            const int64_t row = (int64_t)(tile / across) * 256 + rank * 128 + r, row0 = row - lane;
            const uint32_t from = tmem + lanes + acc * 256;
            const bool up = weights && row0 >= args.hidden_padded;  // (a block's 128 rows lie on one side)
            const int64_t first = up ? row0 - args.hidden_padded : row0, rows = weights ? args.hidden : args.rows;
            void* const out = weights ? (up ? args.dwu : args.dwg) : args.out;
            const CUtensorMap* const map = weights ? (up ? &args.to_wu : &args.to_wg) : &args.to;
            const int64_t stride = weights ? args.width : args.out_stride;
            const int alignment = weights ? args.align_w : args.align_out;
            uint32_t grad[2][8];
            if (kMode == kGradHidden)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int col = n * 128 + 64 * j + 16 * part;
                    load_words(reinterpret_cast<const uint16_t*>(args.grad_h) + row * args.grad_stride + col, row < args.rows ? args.hidden - col : 0,
                               args.vector_in, grad[j]);
                }
            const bool ok = pair_wait(acc_full(acc), (uint32_t)(turn / 2) & 1, &given_up);
            tc_fence_after();
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                // forward: 64 columns, one panel after the other; dgate and dup: 64 columns each; other gradients: 128 columns
                if (storer) {
                    if (kMode == kForward)
                        store_wait_read<1>();
                    else
                        store_wait_read<0>();
                }
                group_sync(1 + quadrant, 128);
                const int col = kMode == kGradients ? n * 256 + 128 * j : n * 128 + 64 * j;
                float v[32];
                uint32_t kept[4][8];
                if (kMode == kGradients) {
                    uint32_t g[32];
                    tmem_load_32(from + 128 * j + 32 * part, g);
                    tmem_load_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = ok ? __uint_as_float(g[i]) : __int_as_float(0x7FC00000);
                    put_panel<kBf16>(panels + part / 2 * kPanelBytes, r, part % 2 * 32, v);
                } else {
                    float lower[16], upper[16];
                    const int c = 64 * j + 16 * part;
                    finish_hidden<kMode, kBf16, kActivation>(args, bias, grad[j], from + c, from + 128 + c, row, n * 128 + c, ok, v, kept);
                    split(v, lower, upper);
                    put_panel<kBf16>(panels + (kMode == kForward ? j : 0) * kPanelBytes, r, 16 * part, lower);
                    if (kMode == kGradHidden) put_panel<kBf16>(panels + kPanelBytes, r, 16 * part, upper);
                }
                if (j == 1) {  // the accumulators are read
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) pair_arrive(in_leader(acc_empty(acc)));
                }
                if (alignment == 16) {
                    async_fence();
                    group_sync(1 + quadrant, 128);
                    if (storer) {
                        if (first < rows && out) {
                            const uint32_t src = smem_addr(panels) + quadrant * 4096;
                            const int columns = kMode == kForward || kMode == kForwardKept ? args.hidden : kMode == kGradHidden ? args.hidden_padded : args.width;
                            if (col < columns) tma_store_2d(map, col, (int)first, src + (kMode == kForward ? j : 0) * kPanelBytes);
                            if (kMode == kGradHidden) tma_store_2d(map, args.hidden_padded + col, (int)first, src + kPanelBytes);
                            if (kMode == kGradients && col + 64 < columns) tma_store_2d(map, col + 64, (int)first, src + kPanelBytes);
                        }
                        store_commit();
                    }
                } else {
                    group_sync(1 + quadrant, 128);
                    const int columns = kMode == kForward || kMode == kForwardKept ? args.hidden : args.width;
                    if (out)
                        for (int p = 0; p < (kMode == kGradients ? 2 : 1); ++p)
                            copy_panel(panels + (kMode == kForward ? j : p) * kPanelBytes, quadrant * 32, part, 4, out, stride, first, rows, col + 64 * p, columns,
                                       alignment, lane);
                }
                if (kMode == kForwardKept)
#pragma unroll
                    for (int p = 0; p < 2; ++p) {  // the upper halves of gate and up, then the lower ones
                        if (storer) store_wait_read<0>();
                        group_sync(1 + quadrant, 128);
                        put_words(panels, r, 16 * part, kept[2 * p]);
                        put_words(panels + kPanelBytes, r, 16 * part, kept[2 * p + 1]);
                        async_fence();
                        group_sync(1 + quadrant, 128);
                        if (storer) {
                            const uint32_t src = smem_addr(panels) + quadrant * 4096;
                            if (first < rows) {
                                tma_store_2d(&args.kept, 2 * p * args.hidden_padded + col, (int)first, src);
                                tma_store_2d(&args.kept, (2 * p + 1) * args.hidden_padded + col, (int)first, src + kPanelBytes);
                            }
                            store_commit();
                        }
                    }
                if (kMode == kGradHidden && args.parts == 2) {  // what the rounding left, behind dgate | dup
                    float lower[16], upper[16];
                    split(v, lower, upper);
                    take_rounded<kBf16>(lower);
                    take_rounded<kBf16>(upper);
                    if (storer) store_wait_read<0>();
                    group_sync(1 + quadrant, 128);
                    put_panel<kBf16>(panels, r, 16 * part, lower);
                    put_panel<kBf16>(panels + kPanelBytes, r, 16 * part, upper);
                    async_fence();
                    group_sync(1 + quadrant, 128);
                    if (storer) {
                        const uint32_t src = smem_addr(panels) + quadrant * 4096;
                        if (first < rows) {
                            tma_store_2d(map, 2 * args.hidden_padded + col, (int)first, src);
                            tma_store_2d(map, 3 * args.hidden_padded + col, (int)first, src + kPanelBytes);
                        }
                        store_commit();
                    }
                }
                if (kMode == kGradHidden) sum_hidden(args, v, row, n * 128 + 64 * j + 16 * part, lane);
            }
        }
        if (storer) store_wait();
    }
    tc_fence_before();
    __syncthreads();
    pair_sync();
    if (warp == kEpilogueWarps + 1) {
        tc_fence_after();
        pair_tmem_free(tmem, 512);
    }
}

// Blocks by themselves, 128 rows x 32 hidden columns: for few rows, where tiles of the pairs would leave most multiprocessors
// without work and what counts is the length of a block's walk along the reduction.
constexpr int kSlimStages = 8;
constexpr int kSlimStage = (kRows + 64) * 128;
constexpr int kSlimShared = kSlimStages * kSlimStage + kBiasBytes + 1024;

template <int kMode, bool kBf16, int kActivation>
__global__ void __launch_bounds__(192, 1) gated_slim_kernel(const __grid_constant__ GatedArgs args) {
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t bars[2 * kSlimStages + 1];
    __shared__ uint32_t tmem_at;
    __shared__ volatile int given_up;
    const uint32_t ring = (smem_addr(raw) + 1023) & ~1023u, bar0 = smem_addr(bars), done = bar0 + 16 * kSlimStages;
    auto full = [&](int s) { return bar0 + 8 * s; };
    auto empty = [&](int s) { return bar0 + 8 * (kSlimStages + s); };
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t m0 = (int64_t)(blockIdx.x / args.tiles_n) * kRows;
    const int n0 = blockIdx.x % args.tiles_n * 32;
    if (threadIdx.x == 0) {
        given_up = 0;
        for (int s = 0; s < kSlimStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 5) tmem_alloc(smem_addr(&tmem_at), 64);
    const Biases bias = stage_biases(args, reinterpret_cast<uint16_t*>(raw + (ring - smem_addr(raw)) + kSlimStages * kSlimStage), 192);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_at;
    const int steps = args.steps;
    if (warp == 4) {
        if (lane == 0) {
            bool ok = true;
            int issued = 0;
            for (; issued < steps; ++issued) {
                const int s = issued % kSlimStages, round = issued / kSlimStages;
                if (round > 0 && !mbar_wait(empty(s), (round - 1) & 1, &given_up)) {
                    ok = false;
                    break;
                }
                const uint32_t a = ring + s * kSlimStage, b = a + kRows * 128;
                mbar_expect(full(s), kSlimStage);
                tma_load_2d(a, &args.a, issued * kStep, (int)m0, full(s));
                tma_load_2d(b, &args.b0, issued * kStep, n0, full(s));
                tma_load_2d(b + 32 * 128, &args.b1, issued * kStep, n0, full(s));
            }
            if (!ok) let_settle();
        }
        __syncwarp();
    } else if (warp == 5) {
        if (lane == 0) {
            bool ok = true;
            for (int k = 0; k < steps; ++k) {
                const int s = k % kSlimStages;
                if (!mbar_wait(full(s), (k / kSlimStages) & 1, &given_up)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t a = ring + s * kSlimStage, b = a + kRows * 128;
#pragma unroll
                for (int i = 0; i < kStep / 16; ++i)
                    mma_f16(tmem, operand_desc(a + 32 * i, 1024, 16), operand_desc(b + 32 * i, 1024, 16), f16_idesc(kBf16, false, false, kRows, 64), k > 0 || i > 0);
                tc_commit(empty(s));
            }
            if (ok)
                tc_commit(done);
            else
                let_settle();
        }
        __syncwarp();
    } else {
        const int64_t row = m0 + warp * 32 + lane;
        uint32_t grad[2][8];
        if (kMode == kGradHidden)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                load_words(reinterpret_cast<const uint16_t*>(args.grad_h) + row * args.grad_stride + n0 + 16 * j,
                           row < args.rows ? args.hidden - n0 - 16 * j : 0, args.vector_in, grad[j]);
        const bool ok = mbar_wait(done, 0, &given_up);
        tc_fence_after();
        const uint32_t from = tmem + ((uint32_t)(warp * 32) << 16);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float v[32], lower[16], upper[16];
            const int col = n0 + 16 * j;
            uint32_t none[4][8];
            finish_hidden<kMode, kBf16, kActivation>(args, bias, grad[j], from + 16 * j, from + 32 + 16 * j, row, col, ok, v, none);
            split(v, lower, upper);
            if (row < args.rows) {
                if (kMode == kForward) {
                    store_row<kBf16>(args.out, row * args.out_stride + col, lower, args.hidden - col, args.align_out);
                } else {
                    store_row<kBf16>(args.out, row * args.out_stride + col, lower, 16, 16);
                    store_row<kBf16>(args.out, row * args.out_stride + args.hidden_padded + col, upper, 16, 16);
                    if (args.parts == 2) {
                        take_rounded<kBf16>(lower);
                        take_rounded<kBf16>(upper);
                        store_row<kBf16>(args.out, row * args.out_stride + 2 * args.hidden_padded + col, lower, 16, 16);
                        store_row<kBf16>(args.out, row * args.out_stride + 3 * args.hidden_padded + col, upper, 16, 16);
                    }
                }
            }
            if (kMode == kGradHidden) sum_hidden(args, v, row, col, lane);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 5) {
        tc_fence_after();
        tmem_free(tmem, 64);
    }
}

// Few rows: a warp takes one gate and one up row of the weights, which pass through the chip once, against all rows of x.
// Bound by the way from L2 and by the launch: 1 row, width 1536, hidden 1024 (6.3 MB of weights) take 3.1 us, 2 TB/s.
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
#pragma unroll(kMost == 1 ? 6 : 3)
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
            Two slope;
            const float gate = g[r] + (bg ? widen<kBf16>(bg[f]) : 0.0f), up = u[r] + (bu ? widen<kBf16>(bu[f]) : 0.0f);
            h[r * h_stride + f] = narrow<kBf16>(activate<kActivation, false>(Two(gate), slope).apart().x * up);
        }
}

// dgate and dup (and their sums over 32 rows) from gate and up as the forward pass kept them, with the bits that kGradHidden would give:
// the same numbers, the sums in the order of lane_sums.  A block takes 32 rows x 128 hidden columns, a thread 8 columns of rows ty
// and ty + 16.  Bound by memory, 14 bytes a hidden value: 8192 x 1024 take 22 us, 5.3 TB/s.
template <bool kBf16, int kActivation>
__global__ void __launch_bounds__(256) gated_kept_kernel(const __grid_constant__ GatedArgs args, const uint16_t* kept) {
    __shared__ float sums[8][16][17];  // half of the sixteen rows at a time, 8 columns of dgate and dup for each of 16 threads
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16, col = blockIdx.x * 128 + 8 * tx;
    const int64_t row0 = (int64_t)blockIdx.y * 32, wide = 4 * (int64_t)args.hidden_padded;
    float total[16];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int64_t row = row0 + ty + 16 * k;
        const bool inside = row < args.rows;
        uint32_t dh[4], half[4][4];
        load_words(reinterpret_cast<const uint16_t*>(args.grad_h) + row * args.grad_stride + col, inside ? args.hidden - col : 0, args.vector_in, dh);
#pragma unroll
        for (int p = 0; p < 4; ++p) load_words(kept + row * wide + p * args.hidden_padded + col, inside ? 8 : 0, true, half[p]);
        float d[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            Two slope;
            const Two gate = kept_pair(half[0][i], half[2][i]), up = kept_pair(half[1][i], half[3][i]), grad = two_of<kBf16>(dh[i]);
            const Two a = activate<kActivation, true>(gate, slope);
            const float2 dgate = (grad * up * slope).apart(), dup = (grad * a).apart();
            const bool first = inside && col + 2 * i < args.hidden, second = inside && col + 2 * i + 1 < args.hidden;
            d[2 * i] = first ? dgate.x : 0.0f, d[2 * i + 1] = second ? dgate.y : 0.0f;
            d[8 + 2 * i] = first ? dup.x : 0.0f, d[9 + 2 * i] = second ? dup.y : 0.0f;
        }
        if (inside) {
            uint16_t* out = reinterpret_cast<uint16_t*>(args.out) + row * args.out_stride + col;
            *reinterpret_cast<uint4*>(out) = make_uint4(pack<kBf16>(d[0], d[1]), pack<kBf16>(d[2], d[3]), pack<kBf16>(d[4], d[5]), pack<kBf16>(d[6], d[7]));
            *reinterpret_cast<uint4*>(out + args.hidden_padded) =
                make_uint4(pack<kBf16>(d[8], d[9]), pack<kBf16>(d[10], d[11]), pack<kBf16>(d[12], d[13]), pack<kBf16>(d[14], d[15]));
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) total[i] = k == 0 ? d[i] : total[i] + d[i];
    }
    if (!args.sums) return;
#pragma unroll
    for (int o = 8; o > 0; o /= 2) {
        if (ty >= o && ty < 2 * o)
#pragma unroll
            for (int i = 0; i < 16; ++i) sums[ty - o][tx][i] = total[i];
        __syncthreads();
        if (ty < o)
#pragma unroll
            for (int i = 0; i < 16; ++i) total[i] += sums[ty][tx][i];
        __syncthreads();
    }
    if (ty == 0) {
        float* to = args.sums + (int64_t)blockIdx.y * 2 * args.hidden_padded + col;
#pragma unroll
        for (int i = 0; i < 8; ++i) to[i] = total[i], to[args.hidden_padded + i] = total[8 + i];
    }
}

// (by itself where no other gradient is wanted)
template <bool kBf16> __global__ void __launch_bounds__(512) bias_gradient_kernel(const __grid_constant__ GatedArgs args) {
    __shared__ float area[512];
    add_bias_gradients<kBf16>(args, area, blockIdx.x, gridDim.x);
}

static SharedLimit g_pair_limit[4][2][2], g_slim_limit[2][2][2];

template <int kMode, bool kBf16, int kActivation> static int launch_pairs(const GatedArgs& args, cudaStream_t stream) {
    auto* kernel = gated_pair_kernel<kMode, kBf16, kActivation>;
    int rc = allow_shared(g_pair_limit[kMode][kBf16][kActivation], (const void*)kernel, kPairShared);
    if (rc) return rc;
    const int tiles = args.tiles + args.tiles_w, pairs = sm_count() / 2;
    kernel<<<2 * (tiles < pairs ? tiles : pairs), kThreads, kPairShared, stream>>>(args);
    return check_cuda(cudaGetLastError(), "gated_pair_kernel");
}
template <int kMode, bool kBf16, int kActivation> static int launch_slim(const GatedArgs& args, cudaStream_t stream) {
    auto* kernel = gated_slim_kernel<kMode, kBf16, kActivation>;
    int rc = allow_shared(g_slim_limit[kMode][kBf16][kActivation], (const void*)kernel, kSlimShared);
    if (rc) return rc;
    kernel<<<args.tiles, 192, kSlimShared, stream>>>(args);
    return check_cuda(cudaGetLastError(), "gated_slim_kernel");
}
template <int kMode> static int launch_hidden(const GatedArgs& args, bool slim, bool bf16, int activation, cudaStream_t st) {
    if (slim)
        return activation == kGelu ? (bf16 ? launch_slim<kMode, true, kGelu>(args, st) : launch_slim<kMode, false, kGelu>(args, st))
                                   : (bf16 ? launch_slim<kMode, true, kSilu>(args, st) : launch_slim<kMode, false, kSilu>(args, st));
    return activation == kGelu ? (bf16 ? launch_pairs<kMode, true, kGelu>(args, st) : launch_pairs<kMode, false, kGelu>(args, st))
                               : (bf16 ? launch_pairs<kMode, true, kSilu>(args, st) : launch_pairs<kMode, false, kSilu>(args, st));
}

// From five rows on the slim tiles are as fast (1536 x 1024: 3.1 us at 1 row, 7.4 at 4, 10.8 at 6, 13.3 at 8; slim 10.7 at any).
constexpr int kFewRows = 4;
constexpr int64_t kMostRows = 1ll << 30;
constexpr int kMostColumns = 1 << 20;

static int check_layer(const char* name, const void* x, int64_t x_stride, const void* wg, int64_t wg_stride, const void* wu, int64_t wu_stride,
                       const void* bg, const void* bu, int64_t rows, int32_t width, int32_t hidden, int32_t dtype, int32_t activation) {
    if (rows < 0 || rows > kMostRows || width < 1 || width > kMostColumns || hidden < 1 || hidden > kMostColumns)
        return set_error(P2B_ERR_ARG, "%s: %lld rows, width %d, hidden %d are out of range", name, (long long)rows, width, hidden);
    // (tiles are counted in 32 bits)
    if ((rows + 127) / 128 * ((hidden + 31) / 32) > 0x7FFF0000ll || (rows + 127) / 128 * ((width + 31) / 32) > 0x7FFF0000ll)
        return set_error(P2B_ERR_ARG, "%s: %lld rows of %d to %d are too many for one call", name, (long long)rows, width, hidden);
    if (dtype < 0 || dtype > 1) return set_error(P2B_ERR_ARG, "%s: unknown type %d (0 bf16, 1 fp16)", name, dtype);
    if (activation < 0 || activation > 1) return set_error(P2B_ERR_ARG, "%s: unknown activation %d (0 gelu, 1 silu)", name, activation);
    if ((rows > 0 && !x) || !wg || !wu) return set_error(P2B_ERR_ARG, "%s: null operand", name);
    if ((uintptr_t)x % 2 || (uintptr_t)wg % 2 || (uintptr_t)wu % 2 || (uintptr_t)bg % 2 || (uintptr_t)bu % 2)
        return set_error(P2B_ERR_ARG, "%s: an operand lies on no 2-byte boundary", name);
    if ((rows > 1 && x_stride < width) || (hidden > 1 && (wg_stride < width || wu_stride < width)))
        return set_error(P2B_ERR_ARG, "%s: rows overlap", name);
    return P2B_OK;
}

// Operands whose rows do not start on 16-byte boundaries, as the copies into shared memory want them, are copied to rows that do: all that
// need it in one launch, 16 bytes a thread.
struct AlignJob {
    const uint16_t* from;
    int64_t stride, rows;
    uint16_t* to;
};
struct AlignArgs {
    AlignJob job[3];
    int width, whole;  // columns, and rounded up to a multiple of 8
};
__global__ void __launch_bounds__(256) align_rows_kernel(const __grid_constant__ AlignArgs args) {
    const AlignJob job = args.job[blockIdx.y];
    const int groups = args.whole / 8;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < job.rows * groups; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / groups;
        const int col = (int)(i - row * groups) * 8;
        const uint16_t* p = job.from + row * job.stride + col;
        uint32_t q[4];
        load_words(p, args.width - col, false, q);
        *reinterpret_cast<uint4*>(job.to + row * args.whole + col) = make_uint4(q[0], q[1], q[2], q[3]);
    }
}
static int64_t align_bytes(int64_t rows, int64_t width, int64_t hidden) { return 2 * (rows + 2 * hidden) * (blocks_of(width, 8) * 8); }
// x, gate and up weights with rows and strides; those that need it become copies in `area`.
static int align_operands(const char* name, const void** at, int64_t* stride, const int64_t* rows, int width, void* area, int64_t bytes, cudaStream_t st) {
    AlignArgs args{};
    args.width = width, args.whole = (int)blocks_of(width, 8) * 8;
    uint16_t* to = (uint16_t*)area;
    int jobs = 0;
    int64_t most = 0;
    for (int i = 0; i < 3; ++i) {
        if (aligned16(at[i], rows[i] > 1 ? stride[i] : 0)) {
            if (rows[i] <= 1) stride[i] = args.whole;
            continue;
        }
        args.job[jobs++] = {(const uint16_t*)at[i], stride[i], rows[i], to};
        at[i] = to, stride[i] = args.whole;
        to += rows[i] * args.whole;
        most = rows[i] > most ? rows[i] : most;
    }
    if (!jobs) return P2B_OK;
    if (!area || (uintptr_t)area % 16 || (char*)to - (char*)area > bytes)
        return set_error(P2B_ERR_ARG, "%s: rows of x or of a weight start on no 16-byte boundaries, and there is no scratch for copies that do", name);
    const int64_t blocks = blocks_of(most * (args.whole / 8), 256), fit = 8 * sm_count();
    align_rows_kernel<<<dim3((unsigned)(blocks < fit ? blocks : fit), jobs), 256, 0, st>>>(args);
    return check_cuda(cudaGetLastError(), "align_rows_kernel");
}

// Slim tiles where they fit the chip at once: 512 rows of 1536 x 1024 take 11.8 us in slim tiles, 14.3 in pairs; 600 rows, a wave and
// some, 20.8 and 14.4.
static bool slim_tiles(int64_t rows, int32_t hidden) { return blocks_of(rows, kRows) * blocks_of(hidden, 32) <= sm_count(); }

// Tiles and maps of x and the weights for the products that end in hidden columns.
static int hidden_maps(GatedArgs& args, bool slim, const void* x, int64_t x_stride, const void* wg, int64_t wg_stride, const void* wu, int64_t wu_stride) {
    int rc = encode_rows(&args.a, x, 2, args.width, args.rows, 2 * x_stride, kRows);
    if (!rc) rc = encode_rows(&args.b0, wg, 2, args.width, args.hidden, 2 * wg_stride, slim ? 32 : 128);
    if (!rc) rc = encode_rows(&args.b1, wu, 2, args.width, args.hidden, 2 * wu_stride, slim ? 32 : 128);
    args.steps = (int)blocks_of(args.width, kStep);
    args.tiles_n = (int)blocks_of(args.hidden, slim ? 32 : 128);
    args.tiles = (int)blocks_of(args.rows, slim ? kRows : 256) * args.tiles_n;
    return rc;
}

template <bool kBf16, int kActivation>
static int launch_few(const void* x, int64_t x_stride, const void* wg, int64_t wg_stride, const void* wu, int64_t wu_stride, const void* bg,
                      const void* bu, int rows, int width, int hidden, void* h, int64_t h_stride, cudaStream_t stream) {
    const int vector = aligned16(x, rows > 1 ? x_stride : 0) && aligned16(wg, wg_stride) && aligned16(wu, wu_stride);
    auto* kernel = rows == 1 ? gated_few_kernel<1, kBf16, kActivation> : rows == 2 ? gated_few_kernel<2, kBf16, kActivation> : gated_few_kernel<kFewRows, kBf16, kActivation>;
    kernel<<<(unsigned)blocks_of(hidden, 4), 128, 0, stream>>>((const uint16_t*)x, x_stride, (const uint16_t*)wg, wg_stride, (const uint16_t*)wu, wu_stride,
                                                              (const uint16_t*)bg, (const uint16_t*)bu, rows, width, hidden, (uint16_t*)h, h_stride, vector);
    return check_cuda(cudaGetLastError(), "gated_few_kernel");
}

// Whether the forward pass of a training step keeps gate and up for the backward pass, or that takes the projections again.  Kept
// they are 8 bytes a hidden value (of hidden rounded up to 128) to write and to read, taken again 4 * width operations.  Both passes of 8192 rows to 1024, taken
// again and kept: width 512 115 and 110 us, 1024 133 and 121, 1536 180 and 156, 2720 306 and 248.  Below a width of 1024 that is not
// worth the memory, and below 2^33 products autograd takes longer on the host than the kernels (1000 rows of 1536 to 1024: 57 and 47 us
// of kernels, 125 and 132 for the call).  The kernels that keep them are the pairs'.
constexpr int kKeptWidth = 1024;
constexpr int64_t kKeptProducts = 1ll << 33;
static bool keeps(int64_t rows, int64_t width, int64_t hidden) {
    return width >= kKeptWidth && rows * hidden >= blocks_of(kKeptProducts, width) && rows > kFewRows && !slim_tiles(rows, (int32_t)hidden);
}

}  // namespace p2b

using namespace p2b;

extern "C" int p2b_gated_few_rows(void) { return kFewRows; }

extern "C" int64_t p2b_gated_kept_bytes(int64_t rows, int32_t width, int32_t hidden) {
    if (rows < 0 || rows > kMostRows || width < 1 || width > kMostColumns || hidden < 1 || hidden > kMostColumns) return -1;
    return keeps(rows, width, hidden) ? 8 * rows * blocks_of(hidden, 128) * 128 : 0;
}

extern "C" int64_t p2b_gated_align_bytes(int64_t rows, int32_t width, int32_t hidden) {
    return rows < 0 || rows > kMostRows || width < 1 || width > kMostColumns || hidden < 1 || hidden > kMostColumns ? -1 : align_bytes(rows, width, hidden);
}

extern "C" int p2b_gated_forward(const void* x, int64_t x_stride, const void* wg, int64_t wg_stride, const void* wu, int64_t wu_stride,
                                 const void* bg, const void* bu, int64_t rows, int32_t width, int32_t hidden, int32_t dtype,
                                 int32_t activation, void* h, int64_t h_stride, void* kept, void* scratch, int64_t scratch_bytes, void* stream) {
    int rc = check_layer("p2b_gated_forward", x, x_stride, wg, wg_stride, wu, wu_stride, bg, bu, rows, width, hidden, dtype, activation);
    if (rc) return rc;
    if (rows == 0) return P2B_OK;
    if (!h || (rows > 1 && h_stride < hidden)) return set_error(P2B_ERR_ARG, "p2b_gated_forward: null output or rows that overlap");
    if ((uintptr_t)h % 2) return set_error(P2B_ERR_ARG, "p2b_gated_forward: the output lies on no 2-byte boundary");
    if (kept && ((uintptr_t)kept % 16 || !p2b_gated_kept_bytes(rows, width, hidden)))
        return set_error(P2B_ERR_ARG, "p2b_gated_forward: kept lies on a 16-byte boundary and is NULL where p2b_gated_kept_bytes is 0");
    const bool bf16 = dtype == 0;
    cudaStream_t st = (cudaStream_t)stream;
    if (rows <= kFewRows) {
        auto* few = activation == kGelu ? (bf16 ? launch_few<true, kGelu> : launch_few<false, kGelu>) : (bf16 ? launch_few<true, kSilu> : launch_few<false, kSilu>);
        return few(x, x_stride, wg, wg_stride, wu, wu_stride, bg, bu, (int)rows, width, hidden, h, h_stride, st);
    }
    const void* at[3] = {x, wg, wu};
    int64_t stride[3] = {x_stride, wg_stride, wu_stride};
    const int64_t count[3] = {rows, hidden, hidden};
    rc = align_operands("p2b_gated_forward", at, stride, count, width, scratch, scratch_bytes, st);
    if (rc) return rc;
    GatedArgs args{};
    args.rows = rows, args.width = width, args.hidden = hidden;
    args.hidden_padded = (int)blocks_of(hidden, 128) * 128;
    args.bias_gate = bg, args.bias_up = bu, args.out = h, args.out_stride = h_stride, args.align_out = row_alignment(h, rows > 1 ? h_stride : 0);
    args.vector_bias = aligned16(bg, 0) && aligned16(bu, 0);
    const bool slim = slim_tiles(rows, hidden);
    rc = hidden_maps(args, slim, at[0], stride[0], at[1], stride[1], at[2], stride[2]);
    if (!rc && !slim && args.align_out == 16) rc = encode_rows(&args.to, h, 2, hidden, rows, 2 * (rows > 1 ? h_stride : blocks_of(hidden, 8) * 8), 32);
    if (!rc && kept) {
        const int64_t wide = 4 * (int64_t)args.hidden_padded;
        rc = encode_rows(&args.kept, kept, 2, wide, rows, 2 * wide, 32);
        if (rc) return rc;
        return activation == kGelu ? (bf16 ? launch_pairs<kForwardKept, true, kGelu>(args, st) : launch_pairs<kForwardKept, false, kGelu>(args, st))
                                   : (bf16 ? launch_pairs<kForwardKept, true, kSilu>(args, st) : launch_pairs<kForwardKept, false, kSilu>(args, st));
    }
    return rc ? rc : launch_hidden<kForward>(args, slim, bf16, activation, st);
}

// dgate and dup are rounded to 16 bits on their way into the products, which makes the gradients' error 1.4 times that of their
// last rounding alone.  Two 16-bit numbers for each would take it away and make the products twice as long (1000 rows of 1536 x 1024: 35
// -> 48 us for the whole pass).  Small layers have them all the same, for 1 us (16 rows of 72 x 64: 11.1 -> 11.9
// us): a layer's gradients are therefore more exact on few rows than on many.
constexpr int64_t kSmallProducts = 1ll << 24;
static int parts_of(int64_t rows, int64_t width, int64_t hidden) { return rows * hidden <= kSmallProducts / width ? 2 : 1; }

extern "C" int64_t p2b_gated_backward_scratch_bytes(int64_t rows, int32_t width, int32_t hidden) {
    if (rows < 0 || rows > kMostRows || width < 1 || width > kMostColumns || hidden < 1 || hidden > kMostColumns) return -1;
    const int64_t columns = 2 * blocks_of(hidden, 128) * 128;
    return 2 * rows * columns * parts_of(rows, width, hidden) + 4 * columns * blocks_of(rows, 32);  // dgate | dup, their column sums
}

extern "C" int p2b_gated_backward(const void* grad_h, int64_t grad_stride, const void* x, int64_t x_stride, const void* wg, int64_t wg_stride,
                                  const void* wu, int64_t wu_stride, const void* bg, const void* bu, int64_t rows, int32_t width,
                                  int32_t hidden, int32_t dtype, int32_t activation, void* dx, int64_t dx_stride, void* dwg, void* dwu,
                                  void* dbg, void* dbu, const void* kept, void* scratch, int64_t scratch_bytes, void* stream) {
    int rc = check_layer("p2b_gated_backward", x, x_stride, wg, wg_stride, wu, wu_stride, bg, bu, rows, width, hidden, dtype, activation);
    if (rc) return rc;
    for (const void* p : {grad_h, (const void*)dx, (const void*)dwg, (const void*)dwu, (const void*)dbg, (const void*)dbu})
        if ((uintptr_t)p % 2) return set_error(P2B_ERR_ARG, "p2b_gated_backward: a gradient lies on no 2-byte boundary");
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
    if (!scratch || ((uintptr_t)scratch % 16) != 0 || scratch_bytes < p2b_gated_backward_scratch_bytes(rows, width, hidden))
        return set_error(P2B_ERR_ARG, "p2b_gated_backward: scratch of %lld bytes on a 16-byte boundary is needed",
                         (long long)p2b_gated_backward_scratch_bytes(rows, width, hidden));
    if (kept && ((uintptr_t)kept % 16 || !p2b_gated_kept_bytes(rows, width, hidden)))
        return set_error(P2B_ERR_ARG, "p2b_gated_backward: kept lies on a 16-byte boundary and is NULL where p2b_gated_kept_bytes is 0");
    const bool bf16 = dtype == 0;
    const int64_t whole = blocks_of(width, 8) * 8, own = p2b_gated_backward_scratch_bytes(rows, width, hidden);
    const void* at[3] = {x, wg, wu};
    int64_t stride[3] = {x_stride, wg_stride, wu_stride};
    const int64_t count[3] = {rows, hidden, hidden};
    rc = align_operands("p2b_gated_backward", at, stride, count, width, (char*)scratch + own, scratch_bytes - own, st);
    if (rc) return rc;
    x = at[0], wg = at[1], wu = at[2];
    x_stride = stride[0], wg_stride = stride[1], wu_stride = stride[2];
    GatedArgs args{};
    args.rows = rows, args.width = width, args.hidden = hidden;
    args.hidden_padded = (int)blocks_of(hidden, 128) * 128;
    args.parts = parts_of(rows, width, hidden);
    const int64_t columns = 2 * (int64_t)args.hidden_padded, wide = columns * args.parts;
    if (dbg || dbu) args.sums = (float*)((char*)scratch + 2 * rows * wide);
    GatedArgs next = args;
    args.bias_gate = bg, args.bias_up = bu, args.grad_h = grad_h, args.grad_stride = grad_stride;
    args.vector_in = aligned16(grad_h, rows > 1 ? grad_stride : 0), args.vector_bias = aligned16(bg, 0) && aligned16(bu, 0);
    args.out = scratch, args.out_stride = wide;
    if (kept) {
        auto* kernel = activation == kGelu ? (bf16 ? gated_kept_kernel<true, kGelu> : gated_kept_kernel<false, kGelu>)
                                           : (bf16 ? gated_kept_kernel<true, kSilu> : gated_kept_kernel<false, kSilu>);
        for (int64_t done = 0; done < rows; done += 32ll * 65535) {  // (blocks of 32 rows, 65,535 to a launch)
            GatedArgs part = args;
            part.rows = rows - done < 32ll * 65535 ? rows - done : 32ll * 65535;
            part.grad_h = (const uint16_t*)grad_h + done * grad_stride;
            part.out = (uint16_t*)scratch + done * wide;
            if (args.sums) part.sums = args.sums + done / 32 * columns;
            const dim3 grid((unsigned)(args.hidden_padded / 128), (unsigned)blocks_of(part.rows, 32));
            kernel<<<grid, 256, 0, st>>>(part, (const uint16_t*)kept + done * 4 * args.hidden_padded);
            if ((rc = check_cuda(cudaGetLastError(), "gated_kept_kernel"))) return rc;
        }
    } else {
        const bool slim = slim_tiles(rows, args.hidden_padded);
        rc = hidden_maps(args, slim, x, x_stride, wg, wg_stride, wu, wu_stride);
        // every column of the work space is written, those behind the last hidden unit as zeros
        args.tiles_n = args.hidden_padded / (slim ? 32 : 128);
        args.tiles = (int)blocks_of(rows, slim ? kRows : 256) * args.tiles_n;
        args.align_out = 16;
        if (!rc && !slim) rc = encode_rows(&args.to, scratch, 2, wide, rows, 2 * wide, 32);
        if (!rc) rc = launch_hidden<kGradHidden>(args, slim, bf16, activation, st);
        if (rc) return rc;
    }
    if (dx || dwg || dwu) {
        next.out = dx, next.out_stride = dx_stride, next.align_out = row_alignment(dx, rows > 1 ? dx_stride : 0);
        next.dwg = dwg, next.dwu = dwu, next.align_w = row_alignment((const void*)((uintptr_t)dwg | (uintptr_t)dwu), hidden > 1 ? width : 0);
        next.dbg = dbg, next.dbu = dbu;
        rc = encode_rows(&next.a, scratch, 2, wide, rows, 2 * wide, kRows);
        if (!rc) rc = encode_rows(&next.b0, wg, 2, width, hidden, 2 * wg_stride, kStep);
        if (!rc) rc = encode_rows(&next.b1, wu, 2, width, hidden, 2 * wu_stride, kStep);
        if (!rc) rc = encode_rows(&next.at, scratch, 2, wide, rows, 2 * wide, kStep);
        if (!rc) rc = encode_rows(&next.bt, x, 2, width, rows, 2 * x_stride, kStep);
        if (!rc && dx && next.align_out == 16) rc = encode_rows(&next.to, dx, 2, width, rows, 2 * (rows > 1 ? dx_stride : whole), 32);
        for (int i = 0; i < 2; ++i)
            if (!rc && (i ? dwu : dwg) && next.align_w == 16)
                rc = encode_rows(i ? &next.to_wu : &next.to_wg, i ? dwu : dwg, 2, width, hidden, 2 * (hidden > 1 ? (int64_t)width : whole), 32);
        if (rc) return rc;
        next.steps = 2 * args.parts * (int)blocks_of(hidden, kStep);
        next.steps_w = args.parts * (int)blocks_of(rows, kStep);
        next.tiles_n = next.tiles_w_n = (int)blocks_of(width, 256);
        next.tiles = dx ? (int)blocks_of(rows, 256) * next.tiles_n : 0;
        next.tiles_w = dwg || dwu ? (int)(columns / 256) * next.tiles_w_n : 0;
        next.ahead = (next.steps_w + next.steps / 2) / next.steps;
        rc = bf16 ? launch_pairs<kGradients, true, 0>(next, st) : launch_pairs<kGradients, false, 0>(next, st);
    } else if (args.sums) {
        next.dbg = dbg, next.dbu = dbu;
        const unsigned blocks = (unsigned)(columns / 32);
        if (bf16)
            bias_gradient_kernel<true><<<blocks, 512, 0, st>>>(next);
        else
            bias_gradient_kernel<false><<<blocks, 512, 0, st>>>(next);
        rc = check_cuda(cudaGetLastError(), "bias_gradient_kernel");
    }
    return rc;
}
