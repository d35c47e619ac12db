// Clipped policy loss with a KL term over the hands of a batch of states, and its gradient, in one pass over the data.
//
// Per state and hand, over the legal actions a with p = softmax(logits), q the old policy, A the advantages, t the target:
//   l = -sum_a min(p_a A_a, clip(p_a, (1-e) q_a, (1+e) q_a) A_a) + k sum_a t_a (log t_a - log p_a)
//   dl/dz_a = -p_a (g_a - sum_b g_b p_b) + k (p_a sum_b t_b - t_a),   g_a = A_a where the first side of the min is taken, else 0
// and the loss is sum(w l) / sum(w) over the hands of states with a legal action.  (q min(r A, clip(r, 1-e, 1+e) A) with the ratio
// r = p/q, summed over the actions instead of sampled; written without the division, so q = 0 is no special case.)
//
// Bound by memory: an action's logit, three fp32 policies and the gradient; 4096 states of 1326 hands and 8 actions, bf16 logits (708
// MB) take 140 us, 5.1 TB/s.  A block takes 256 hands, whose arrays come as one
// bulk copy each (hands of 5 actions are 20 bytes: read by thread they would be five sectors an instruction).  Which side
// of the min is taken is decided in 64 bits where 32 might get it wrong: the gradient jumps there.
#include "layer.cuh"
#include "tensor.cuh"

#include <type_traits>

namespace p2b {

using namespace tc;

constexpr int kHands = 256;       // hands of a block
constexpr int kMostActions = 16;
constexpr int kMassBlocks = 592;  // four a multiprocessor
constexpr int kMassChunk = 2048;
constexpr int kLossStages = 3;
constexpr int kLossBlocks = 1024;  // at most
// Tiles that one block takes by itself, in one launch and without work space: as long on the device as two launches for the hands of one
// state (1326 of 5 actions: 9.8 and 9.4 us), and a launch less for the host; 8 tiles would take 11.7 and 7.2.
constexpr int kAlone = 6;

struct LossArgs {
    const void* logits;
    const float *old_policy, *advantages, *target, *weights;
    const uint8_t* legal;
    int64_t states, total;  // total = states * hands
    int hands;
    double clip;
    float kl;
    int bulk;
    // scratch: [0] blocks done, then the mass sums, then the loss sums
    unsigned long long* done;
    double *mass, *sums;
    uint32_t* masks;  // legal actions of every state, a bit each (with mass_parts > 0)
    int mass_parts;
    uint64_t magic;   // ceil(2^64 / hands)
    float* loss;
    void* grad;
    int wide;                // fp16 logits: grad is fp32
    float factor;            // of the gradient, times *factor_at (NULL: 1), before its only rounding
    const float* factor_at;
};

__device__ __forceinline__ double block_sum(double v, double* area) {
#pragma unroll
    for (int o = 16; o > 0; o /= 2) v += __shfl_xor_sync(~0u, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) area[threadIdx.x / 32] = v;
    __syncthreads();
    double sum = 0.0;
    for (int i = 0; i < kHands / 32; ++i) sum += area[i];
    return sum;
}

// Sum of the weights of the hands whose state has a legal action: a warp takes a state's hands, kMassChunk at most; a part for
// every block, in a fixed order.
__global__ void __launch_bounds__(kHands) loss_mass_kernel(const float* weights, const uint8_t* legal, int64_t states, int hands, int actions,
                                                           unsigned long long* done, double* mass, uint32_t* masks) {
    __shared__ double area[kHands / 32];
    const int lane = threadIdx.x % 32, chunks = (hands + kMassChunk - 1) / kMassChunk;
    double sum = 0.0;
    for (int64_t job = (int64_t)blockIdx.x * 8 + threadIdx.x / 32; job < states * chunks; job += (int64_t)gridDim.x * 8) {
        const int64_t state = chunks == 1 ? job : job / chunks;
        const int first = (int)(job - state * chunks) * kMassChunk, count = min(hands - first, kMassChunk);
        const uint32_t open = __ballot_sync(~0u, lane < actions && legal[state * actions + min(lane, actions - 1)] != 0);
        if (lane == 0 && first == 0) masks[state] = open;
        if (open == 0) continue;
        if (!weights) {
            if (lane == 0) sum += (double)count;
            continue;
        }
        const float* w = weights + state * hands + first;
        double part[4] = {0.0, 0.0, 0.0, 0.0};
        int h = lane;
        for (; h + 7 * 32 < count; h += 8 * 32) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __ldg(w + h + 32 * i);
#pragma unroll
            for (int i = 0; i < 8; ++i) part[i % 4] += (double)v[i];
        }
        for (; h < count; h += 32) part[0] += (double)w[h];
        sum += (part[0] + part[1]) + (part[2] + part[3]);
    }
    sum = block_sum(sum, area);
    if (threadIdx.x == 0) {
        mass[blockIdx.x] = sum;
        if (blockIdx.x == 0) *done = 0;
    }
}

template <typename T> __device__ __forceinline__ float as_float(T v);
template <> __device__ __forceinline__ float as_float(float v) { return v; }
template <> __device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half(v); }

__device__ __forceinline__ float small_power_of_two(float x) {  // (subnormal results are kept)
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A hand's kActions values from shared memory, in reads as wide as the hands' distance allows (8 fp32 values apart, single reads would
// meet in four banks).
template <int kActions, typename T> __device__ __forceinline__ void read_hand(const T* p, float (&v)[kActions]) {
    constexpr int kBytes = kActions * (int)sizeof(T), kWide = kBytes % 16 == 0 ? 16 : kBytes % 8 == 0 ? 8 : kBytes % 4 == 0 ? 4 : 2;
    constexpr int kEach = kWide / (int)sizeof(T) > 0 ? kWide / (int)sizeof(T) : 1;
#pragma unroll
    for (int i = 0; i < kActions / kEach; ++i) {
        T part[kEach];
        if (kWide == 16) *reinterpret_cast<uint4*>(part) = reinterpret_cast<const uint4*>(p)[i];
        if (kWide == 8) *reinterpret_cast<uint2*>(part) = reinterpret_cast<const uint2*>(p)[i];
        if (kWide == 4) *reinterpret_cast<uint32_t*>(part) = reinterpret_cast<const uint32_t*>(p)[i];
        if (kWide == 2) *reinterpret_cast<uint16_t*>(part) = reinterpret_cast<const uint16_t*>(p)[i];
#pragma unroll
        for (int j = 0; j < kEach; ++j) v[i * kEach + j] = as_float(part[j]);
    }
}
template <int kActions, typename T> __device__ __forceinline__ void write_hand(T* p, const float (&v)[kActions]) {
    constexpr int kBytes = kActions * (int)sizeof(T), kWide = kBytes % 16 == 0 ? 16 : kBytes % 8 == 0 ? 8 : kBytes % 4 == 0 ? 4 : 2;
    constexpr int kEach = kWide / (int)sizeof(T) > 0 ? kWide / (int)sizeof(T) : 1;
#pragma unroll
    for (int i = 0; i < kActions / kEach; ++i) {
        T part[kEach];
#pragma unroll
        for (int j = 0; j < kEach; ++j) part[j] = from_float<T>(v[i * kEach + j]);
        if (kWide == 16) reinterpret_cast<uint4*>(p)[i] = *reinterpret_cast<const uint4*>(part);
        if (kWide == 8) reinterpret_cast<uint2*>(p)[i] = *reinterpret_cast<const uint2*>(part);
        if (kWide == 4) reinterpret_cast<uint32_t*>(p)[i] = *reinterpret_cast<const uint32_t*>(part);
        if (kWide == 2) reinterpret_cast<uint16_t*>(p)[i] = *reinterpret_cast<const uint16_t*>(part);
    }
}

__device__ __forceinline__ float log_two(float x) {  // of a normal number; a NaN stays one
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float log_two_of_target(float x) { return log_two(fmaxf(x, 1.17549435e-38f)); }  // (a subnormal number counts as the smallest normal)

// Which of the doubtful actions of a hand are free: probabilities so near an end of their interval that 32 bits may put them on the
// wrong side are compared in 64.  (Masks go in and out: an address taken of the caller's arrays would put them into memory.)
template <int kActions, typename T>
__device__ __noinline__ uint32_t settle_hand(const T* z, const float* old, const float* adv, uint32_t open, uint32_t doubtful, double clip) {
    double top = -INFINITY, total = 0.0;
    for (int a = 0; a < kActions; ++a)
        if (open >> a & 1) top = fmax(top, (double)as_float(z[a]));
    for (int a = 0; a < kActions; ++a)
        if (open >> a & 1) total += exp((double)as_float(z[a]) - top);
    uint32_t free = 0;
    for (int a = 0; a < kActions; ++a)
        if (doubtful >> a & 1) {
            const double exact = exp((double)as_float(z[a]) - top) / total, end = (adv[a] > 0.0f ? 1.0 + clip : 1.0 - clip) * (double)old[a];
            free |= (adv[a] > 0.0f ? exact <= end : exact >= end) ? 1u << a : 0u;
        }
    return free;
}

// Blocks a multiprocessor that registers are to leave room for, as many as shared memory does (8 actions, one block instead of two: 217 us
// instead of 150 for 4096 states).
constexpr int blocks_held(int actions) { return actions <= 4 ? 4 : actions == 5 ? 3 : actions <= 10 ? 2 : 1; }

// Blocks stay: each takes every gridDim.x-th tile of 256 hands, with the tiles after the present one on their way into the other
// two of three stages (two stages in all: half as long again for the states above).  The gradient overwrites the logits (in fp32: the
// targets) of its stage and leaves from there.
template <int kActions, typename T>
__global__ void __launch_bounds__(kHands, blocks_held(kActions)) policy_loss_kernel(const __grid_constant__ LossArgs args) {
    extern __shared__ __align__(16) uint8_t area[];
    __shared__ double sums[kHands / 32];
    __shared__ uint64_t bar_words[kLossStages];
    __shared__ volatile int given_up;
    __shared__ bool last_block;
    constexpr int kStage = kHands * (kActions * ((int)sizeof(T) + 12) + 4), kWords = kHands * kActions * 4, kLogits = kHands * kActions * (int)sizeof(T);
    const int tid = threadIdx.x;
    const bool wide = std::is_same<T, __half>::value && args.wide;
    const int64_t tiles = (args.total + kHands - 1) / kHands;
    auto bar = [&](int s) { return smem_addr(bar_words + s); };
    auto whole = [&](int64_t tile) { return args.bulk && tile < tiles && (tile + 1) * kHands <= args.total; };
    auto fetch = [&](int64_t tile, int s) {
        const int64_t first = tile * kHands;
        const uint32_t at = smem_addr(area) + s * kStage, b = bar(s);
        mbar_expect(b, kLogits + kWords + (args.old_policy ? 2 * kWords : 0) + (args.weights ? kHands * 4 : 0));
        bulk_load(at, reinterpret_cast<const T*>(args.logits) + first * kActions, kLogits, b);
        bulk_load(at + kLogits + 2 * kWords, args.target + first * kActions, kWords, b);
        if (args.old_policy) {
            bulk_load(at + kLogits, args.old_policy + first * kActions, kWords, b);
            bulk_load(at + kLogits + kWords, args.advantages + first * kActions, kWords, b);
        }
        if (args.weights) bulk_load(at + kLogits + 3 * kWords, args.weights + first, kHands * 4, b);
    };
    if (tid == 0) {
        given_up = 0;
        for (int s = 0; s < kLossStages; ++s) mbar_init(bar(s), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int s = 0; s < kLossStages - 1; ++s)
            if (whole(blockIdx.x + (int64_t)s * gridDim.x)) fetch(blockIdx.x + (int64_t)s * gridDim.x, s);
    }
    // meanwhile the sum of the weights
    double mass = 0.0;
    if (args.mass_parts > 0) {
        for (int i = tid; i < args.mass_parts; i += kHands) mass += __ldcg(args.mass + i);
    } else {  // a single block, few hands
        for (int i = tid; i < (int)args.total; i += kHands) {
            bool open = false;
            for (int a = 0; a < kActions; ++a) open |= args.legal[i / args.hands * kActions + a] != 0;
            if (open) mass += args.weights ? (double)args.weights[i] : 1.0;
        }
    }
    mass = block_sum(mass, sums);
    const bool nothing = mass <= 0.0;  // (an undefined mass is not nothing)
    // (masses whose reciprocal fp32 has no room for: weights and mass are lifted alike, a power of two)
    const float lift = mass < 0x1p-100 ? 0x1p100f : mass > 0x1p100 ? 0x1p-100f : 1.0f;
    const float inverse = nothing ? 0.0f : (float)(1.0 / (mass * lift)), share = inverse * (args.factor_at ? args.factor * *args.factor_at : args.factor);
    const float undefined_mass = mass < INFINITY ? 0.0f : __int_as_float(0x7FC00000);  // (goes the way of undefined logits)
    const float low_end = (float)(1.0 - args.clip), high_end = (float)(1.0 + args.clip);

    double loss_sum = 0.0;
    int turn = 0;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++turn) {
        const int s = turn % kLossStages;
        const int64_t first = tile * kHands;
        const int count = (int)(args.total - first < kHands ? args.total - first : kHands);
        const bool bulk = whole(tile);
        uint8_t* const stage = area + s * kStage;
        T* const z_s = reinterpret_cast<T*>(stage);
        float* const old_s = reinterpret_cast<float*>(stage + kLogits);
        float *const adv_s = old_s + kHands * kActions, *const target_s = adv_s + kHands * kActions, *const weight_s = target_s + kHands * kActions;
        if (!bulk) {
            for (int i = tid; i < count * kActions; i += kHands) {
                z_s[i] = reinterpret_cast<const T*>(args.logits)[first * kActions + i];
                target_s[i] = args.target[first * kActions + i];
                if (args.old_policy) {
                    old_s[i] = args.old_policy[first * kActions + i];
                    adv_s[i] = args.advantages[first * kActions + i];
                }
            }
            if (args.weights && tid < count) weight_s[tid] = args.weights[first + tid];
            __syncthreads();
        }
        uint32_t open = 0;
        if (tid < count) {
            // the hand's state, a multiplication instead of a division: one too large where the product carries the reciprocal's excess
            const int64_t at = first + tid;
            int64_t state = args.magic ? (int64_t)__umul64hi((uint64_t)at, args.magic) : at;
            state -= state * args.hands > at;
            if (args.mass_parts > 0) {
                open = __ldcg(args.masks + state);
            } else {
#pragma unroll
                for (int a = 0; a < kActions; ++a) open |= (args.legal[state * kActions + a] != 0 ? 1u : 0u) << a;
            }
        }
        // (a stage that no bulk copy filled has not moved its barrier: only the last tile of all is one)
        const bool ok = !bulk || mbar_wait(bar(s), (uint32_t)(turn / kLossStages) & 1, &given_up);
        if (!ok && tid == 0) let_settle();  // the copies in flight land before the block's memory goes

        if (tid < count) {
            const float weight = args.weights ? weight_s[tid] : 1.0f;
            T* const z_own = z_s + tid * kActions;
            float p[kActions], t[kActions], q[kActions], g[kActions];
            read_hand<kActions, T>(z_own, p);
            read_hand<kActions, float>(target_s + tid * kActions, t);
            if (args.old_policy) {
                read_hand<kActions, float>(old_s + tid * kActions, q);
                read_hand<kActions, float>(adv_s + tid * kActions, g);
            }
            float top = -INFINITY;
#pragma unroll
            for (int a = 0; a < kActions; ++a) {
                const bool legal = open & 1u << a;
                p[a] = legal ? p[a] : -INFINITY;
                t[a] = legal ? t[a] : 0.0f;
                q[a] = legal ? q[a] : 1.0f;
                g[a] = legal ? g[a] : 0.0f;
                top = fmaxf(top, p[a]);
            }
            // no legal action, or a hand that does not count: nothing, whatever else is there
            if (weight != 0.0f && open != 0) {
                float d[kActions], total = undefined_mass, targets = 0.0f, divergence = 0.0f;
                // (in powers of two; logarithms are lg2.approx, off by 2^-22, of which the loss averages a whole batch)
#pragma unroll
                for (int a = 0; a < kActions; ++a) {
                    d[a] = (p[a] - top) * 1.4426950408889634f;
                    p[a] = small_power_of_two(d[a]);
                    total += p[a];
                    targets += t[a];
                    const float more = fmaf(t[a], log_two_of_target(t[a]) - d[a], divergence);
                    divergence = t[a] > 0.0f ? more : divergence;
                }
                divergence = 0.69314718055994531f * fmaf(targets, log_two(total), divergence);
                const float rcp = reciprocal(total);
                float scale = weight * lift * share, pulled = scale * args.kl;
                float surrogate = 0.0f, pull = 0.0f;
                // A sum that is NaN: no action that the logits leave is nothing, something undefined stays so at the legal actions.  (Of the
                // logits again: a maximum passes over NaN, which is no -inf.)
                auto undefined = [&] {
                    uint32_t left = 0;
#pragma unroll 1
                    for (int a = 0; a < kActions; ++a) left = open >> a & 1 && as_float(z_own[a]) != -INFINITY ? open : left;
#pragma unroll
                    for (int a = 0; a < kActions; ++a) {
                        p[a] = left & 1u << a ? p[a] : 0.0f;
                        t[a] = left ? t[a] : 0.0f;
                    }
                    scale = pulled = 1.0f;
                    if (left == 0) divergence = surrogate = targets = 0.0f;
                };
                if (args.old_policy) {
                    uint32_t doubtful = 0;
#pragma unroll
                    for (int a = 0; a < kActions; ++a) {
                        p[a] *= rcp;
                        q[a] *= g[a] > 0.0f ? high_end : low_end;
                        // p is off by 1.5e-6 of itself and 1e-7 for every halving below the top, and by its last bits where those are few
                        // (undefined counts as doubtful)
                        doubtful |= fabsf(p[a] - q[a]) > fmaf(q[a], fmaf(fminf(-d[a], 200.0f), 1e-7f, 2e-6f), 1e-43f) ? 0u : 1u << a;
                        const float moving = p[a] * g[a], fixed = q[a] * g[a];
                        const bool free = moving <= fixed;
                        surrogate += free ? moving : fixed;
                        d[a] = free ? g[a] : 0.0f;
                        pull += free ? moving : 0.0f;
                    }
                    if (doubtful && total != total) {
                        undefined();
                    } else if (doubtful) {
                        const uint32_t free = settle_hand<kActions, T>(z_own, old_s + tid * kActions, adv_s + tid * kActions, open, doubtful, args.clip);
                        surrogate = pull = 0.0f;
#pragma unroll
                        for (int a = 0; a < kActions; ++a) {
                            const bool moves = doubtful >> a & 1 ? free >> a & 1 : p[a] * g[a] <= q[a] * g[a];
                            surrogate = fmaf(moves ? p[a] : q[a], g[a], surrogate);
                            d[a] = moves ? g[a] : 0.0f;
                            pull = fmaf(d[a], p[a], pull);
                        }
                    }
                    const float base = fmaf(pulled, targets, scale * pull);
#pragma unroll
                    for (int a = 0; a < kActions; ++a) p[a] = fmaf(p[a], fmaf(-scale, d[a], base), -pulled * t[a]);
                } else {
#pragma unroll
                    for (int a = 0; a < kActions; ++a) p[a] *= rcp;
                    if (total != total) undefined();
#pragma unroll
                    for (int a = 0; a < kActions; ++a) p[a] = pulled * fmaf(p[a], targets, -t[a]);
                }
                loss_sum += (double)weight * (double)(args.kl * divergence - surrogate);
            } else {
#pragma unroll
                for (int a = 0; a < kActions; ++a) p[a] = 0.0f;
            }
            if (!ok) loss_sum = __longlong_as_double(0x7FF8000000000000ll);
            if (args.grad) {
                if (!ok)
#pragma unroll
                    for (int a = 0; a < kActions; ++a) p[a] = __int_as_float(0x7FC00000);
                if (wide)  // (in the place of the targets, which are read)
                    write_hand<kActions, float>(target_s + tid * kActions, p);
                else
                    write_hand<kActions, T>(z_own, p);
            }
        }
        if (bulk) async_fence();
        __syncthreads();
        if (bulk && tid == 0) {
            if (args.grad)
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(
                                 reinterpret_cast<uint8_t*>(args.grad) + first * kActions * (wide ? 4 : (int)sizeof(T))),
                             "r"(wide ? smem_addr(target_s) : smem_addr(z_s)), "r"((uint32_t)(wide ? kWords : kLogits))
                             : "memory");
            store_commit();
            store_wait_read<1>();  // the gradient of the tile before has left its stage, which takes the tile after the next
            const int64_t next = tile + (int64_t)(kLossStages - 1) * gridDim.x;
            if (whole(next)) fetch(next, (turn + kLossStages - 1) % kLossStages);
        }
        if (!bulk && args.grad)
            for (int i = tid; i < count * kActions; i += kHands) {
                if (wide)
                    reinterpret_cast<float*>(args.grad)[first * kActions + i] = target_s[i];
                else
                    reinterpret_cast<T*>(args.grad)[first * kActions + i] = z_s[i];
            }
        if (!args.bulk) __syncthreads();
    }
    loss_sum = block_sum(loss_sum, sums);
    // the block that comes last adds the parts up, in their order
    if (gridDim.x == 1) {
        if (tid == 0) *args.loss = nothing ? 0.0f : (float)(loss_sum / mass);
    } else {
        if (tid == 0) {
            args.sums[blockIdx.x] = loss_sum;
            __threadfence();
            last_block = atomicAdd(args.done, 1ull) == gridDim.x - 1;
        }
        __syncthreads();
        if (last_block) {
            __threadfence();
            double sum = 0.0;
            for (int i = tid; i < (int)gridDim.x; i += kHands) sum += __ldcg(args.sums + i);
            sum = block_sum(sum, sums);
            if (tid == 0) *args.loss = nothing ? 0.0f : (float)(sum / mass);
        }
    }
    if (tid == 0) store_wait();
}

// grad * factor, the factor on the device; 16 bytes a thread, the first `whole` values in whole sixteens.
template <typename T> __global__ void __launch_bounds__(256) scale_kernel(const T* in, const float* factor, T* out, int64_t n, int64_t whole) {
    constexpr int kEach = 16 / (int)sizeof(T);
    const float f = *factor;
    const int64_t step = (int64_t)gridDim.x * 256, begin = (int64_t)blockIdx.x * 256 + threadIdx.x;
    for (int64_t i = begin; i < whole / kEach; i += step) {
        __align__(16) T v[kEach];
        *reinterpret_cast<uint4*>(v) = __ldg(reinterpret_cast<const uint4*>(in) + i);
#pragma unroll
        for (int j = 0; j < kEach; ++j) v[j] = from_float<T>(as_float(v[j]) * f);
        reinterpret_cast<uint4*>(out)[i] = *reinterpret_cast<const uint4*>(v);
    }
    for (int64_t i = whole + begin; i < n; i += step) out[i] = from_float<T>(as_float(in[i]) * f);
}

// The same of a gradient in fp32, for fp16 logits: an entry is of the size of 1 / (states * hands), 2e-7 for 4096 states, and fp16 ends at
// 6e-8, so it takes the factor before it is rounded.  Up to a factor of 2, where that can bring nothing back, it is rounded before as well,
// as the gradient by itself is: the same bits times the factor, two half steps of fp16 more at most.
__global__ void __launch_bounds__(256) scale_wide_kernel(const float* in, const float* factor, __half* out, int64_t n, int64_t whole) {
    const float f = *factor;
    const bool before = fabsf(f) <= 2.0f;
    auto scaled = [&](float g) { return __float2half((before ? __half2float(__float2half(g)) : g) * f); };
    const int64_t step = (int64_t)gridDim.x * 256, begin = (int64_t)blockIdx.x * 256 + threadIdx.x;
    for (int64_t i = begin; i < whole / 8; i += step) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(in) + 2 * i), b = __ldg(reinterpret_cast<const float4*>(in) + 2 * i + 1);
        __align__(16) const __half v[8] = {scaled(a.x), scaled(a.y), scaled(a.z), scaled(a.w), scaled(b.x), scaled(b.y), scaled(b.z), scaled(b.w)};
        reinterpret_cast<uint4*>(out)[i] = *reinterpret_cast<const uint4*>(v);
    }
    for (int64_t i = whole + begin; i < n; i += step) out[i] = scaled(in[i]);
}

static SharedLimit g_limit[kMostActions + 1][3];

template <int kActions, typename T> static int launch_loss(const LossArgs& args, int type, cudaStream_t stream) {
    auto* kernel = policy_loss_kernel<kActions, T>;
    constexpr int shared = kLossStages * kHands * (kActions * (int)(sizeof(T) + 12) + 4);
    int rc = allow_shared(g_limit[kActions][type], (const void*)kernel, shared);
    if (rc) return rc;
    const int64_t tiles = blocks_of(args.total, kHands), fit = (int64_t)sm_count() * (shared <= 56 * 1024 ? 4 : shared <= 75 * 1024 ? 3 : shared <= 113 * 1024 ? 2 : 1);
    const int64_t blocks = args.mass_parts == 0 ? 1 : tiles < fit ? tiles : fit;
    kernel<<<(unsigned)(blocks < kLossBlocks ? blocks : kLossBlocks), kHands, shared, stream>>>(args);
    return check_cuda(cudaGetLastError(), "policy_loss_kernel");
}
template <typename T, int kActions = kMostActions> static int launch_actions(const LossArgs& args, int actions, int type, cudaStream_t stream) {
    if (actions == kActions) return launch_loss<kActions, T>(args, type, stream);
    if constexpr (kActions > 1) return launch_actions<T, kActions - 1>(args, actions, type, stream);
    return P2B_ERR_ARG;
}

}  // namespace p2b

using namespace p2b;

static bool loss_sizes(int64_t states, int32_t hands, int32_t actions) {
    return states >= 0 && hands >= 1 && actions >= 1 && actions <= kMostActions && states <= (1ll << 38) / hands;
}

extern "C" int64_t p2b_policy_loss_scratch_bytes(int64_t states, int32_t hands) {
    if (loss_sizes(states, hands, 1) && states * hands <= kAlone * kHands) return 0;
    return loss_sizes(states, hands, 1) ? 8 * (1 + kMassBlocks + kLossBlocks) + blocks_of(states, 2) * 8 : -1;
}

extern "C" int p2b_policy_loss_scaled(const void* logits, const float* old_policy, const float* advantages, const float* target, const uint8_t* legal,
                                      const float* weights, int64_t states, int32_t hands, int32_t actions, int32_t dtype, double clip, float kl,
                                      float* loss, void* grad, int32_t grad_dtype, float factor, const float* factor_at, void* scratch,
                                      int64_t scratch_bytes, void* stream) {
    const char* name = "p2b_policy_loss";
    if (!loss_sizes(states, hands, actions))
        return set_error(P2B_ERR_ARG, "%s: %lld states of %d hands and %d actions are out of range (1 to %d actions)", name, (long long)states, hands, actions, kMostActions);
    if (dtype < 0 || dtype > 2) return set_error(P2B_ERR_ARG, "%s: unknown type %d (0 bf16, 1 fp16, 2 fp32)", name, dtype);
    if (!(clip >= 0.0 && clip < 1.0) || !(kl >= 0.0f && kl <= 3.4028234e38f)) return set_error(P2B_ERR_ARG, "%s: clip lies in [0, 1), kl is not negative", name);
    const int64_t bytes = p2b_policy_loss_scratch_bytes(states, hands);
    if (!loss || (bytes > 0 && !scratch) || scratch_bytes < bytes || (uintptr_t)scratch % 8)
        return set_error(P2B_ERR_ARG, "%s: loss and scratch of %lld bytes on an 8-byte boundary are needed", name,
                         (long long)bytes);
    if ((old_policy == nullptr) != (advantages == nullptr)) return set_error(P2B_ERR_ARG, "%s: the old policy and the advantages come together", name);
    if (states > 0 && (!logits || !target || !legal)) return set_error(P2B_ERR_ARG, "%s: null array", name);
    if (grad_dtype != dtype && (grad_dtype != 2 || dtype != 1)) return set_error(P2B_ERR_ARG, "%s: the gradient has the logits' type, or is fp32 where they are fp16", name);
    if (!(factor >= -3.4028234e38f && factor <= 3.4028234e38f)) return set_error(P2B_ERR_ARG, "%s: the gradient's factor is not finite", name);
    const uintptr_t four = (uintptr_t)old_policy | (uintptr_t)advantages | (uintptr_t)target | (uintptr_t)weights | (uintptr_t)loss | (uintptr_t)factor_at;
    if (four % 4 || (uintptr_t)logits % (dtype == 2 ? 4 : 2) || (uintptr_t)grad % (grad_dtype == 2 ? 4 : 2)) return set_error(P2B_ERR_ARG, "%s: an array lies off its elements' boundaries", name);
    cudaStream_t st = (cudaStream_t)stream;
    if (states == 0) return check_cuda(cudaMemsetAsync(loss, 0, 4, st), name);
    LossArgs args{};
    args.logits = logits, args.old_policy = old_policy, args.advantages = advantages, args.target = target, args.weights = weights, args.legal = legal;
    args.states = states, args.total = states * hands, args.hands = hands, args.clip = clip, args.kl = kl, args.loss = loss, args.grad = grad;
    args.wide = grad_dtype != dtype, args.factor = factor, args.factor_at = factor_at;
    args.bulk = (((uintptr_t)old_policy | (uintptr_t)advantages | (uintptr_t)target | (uintptr_t)weights | (uintptr_t)logits | (uintptr_t)grad) % 16) == 0;
    args.done = (unsigned long long*)scratch;
    args.mass = (double*)scratch + 1;
    args.sums = args.mass + kMassBlocks;
    args.masks = (uint32_t*)(args.sums + kLossBlocks);
    args.magic = hands == 1 ? 0 : ~0ull / (uint64_t)hands + 1;
    if (args.total > kAlone * kHands) {
        const int64_t jobs = states * blocks_of(hands, kMassChunk);
        args.mass_parts = (int)(jobs < 8 * kMassBlocks ? blocks_of(jobs, 8) : kMassBlocks);
        loss_mass_kernel<<<args.mass_parts, kHands, 0, st>>>(weights, legal, states, hands, actions, args.done, args.mass, args.masks);
        int rc = check_cuda(cudaGetLastError(), "loss_mass_kernel");
        if (rc) return rc;
    }
    if (dtype == 0) return launch_actions<__nv_bfloat16>(args, actions, 0, st);
    if (dtype == 1) return launch_actions<__half>(args, actions, 1, st);
    return launch_actions<float>(args, actions, 2, st);
}

extern "C" int p2b_policy_loss(const void* logits, const float* old_policy, const float* advantages, const float* target, const uint8_t* legal,
                               const float* weights, int64_t states, int32_t hands, int32_t actions, int32_t dtype, double clip, float kl,
                               float* loss, void* grad, void* scratch, int64_t scratch_bytes, void* stream) {
    return p2b_policy_loss_scaled(logits, old_policy, advantages, target, legal, weights, states, hands, actions, dtype, clip, kl, loss, grad, dtype, 1.0f, nullptr,
                                  scratch, scratch_bytes, stream);
}

extern "C" int p2b_policy_loss_scale(const void* grad, const float* factor, int64_t n, int32_t dtype, void* out, void* stream) {
    if (n < 0 || dtype < 0 || dtype > 2) return set_error(P2B_ERR_ARG, "p2b_policy_loss_scale: %lld values of type %d", (long long)n, dtype);
    if (n == 0) return P2B_OK;
    if (!grad || !factor || !out) return set_error(P2B_ERR_ARG, "p2b_policy_loss_scale: null array");
    if ((uintptr_t)factor % 4 || ((uintptr_t)grad | (uintptr_t)out) % (dtype == 2 ? 4 : 2))
        return set_error(P2B_ERR_ARG, "p2b_policy_loss_scale: an array lies off its elements' boundaries");
    const int64_t each = dtype == 2 ? 4 : 8, whole = ((uintptr_t)grad | (uintptr_t)out) % 16 ? 0 : n / each * each;
    const int64_t blocks = blocks_of(n, 256 * each), most = 8 * sm_count();
    const unsigned grid = (unsigned)(blocks < most ? blocks : most);
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == 0) scale_kernel<<<grid, 256, 0, st>>>((const __nv_bfloat16*)grad, factor, (__nv_bfloat16*)out, n, whole);
    if (dtype == 1) scale_kernel<<<grid, 256, 0, st>>>((const __half*)grad, factor, (__half*)out, n, whole);
    if (dtype == 2) scale_kernel<<<grid, 256, 0, st>>>((const float*)grad, factor, (float*)out, n, whole);
    return check_cuda(cudaGetLastError(), "scale_kernel");
}

extern "C" int p2b_policy_loss_scale_fp32(const float* grad, const float* factor, int64_t n, void* out, void* stream) {
    const char* name = "p2b_policy_loss_scale_fp32";
    if (n < 0) return set_error(P2B_ERR_ARG, "%s: %lld values", name, (long long)n);
    if (n == 0) return P2B_OK;
    if (!grad || !factor || !out) return set_error(P2B_ERR_ARG, "%s: null array", name);
    if (((uintptr_t)factor | (uintptr_t)grad) % 4 || (uintptr_t)out % 2) return set_error(P2B_ERR_ARG, "%s: an array lies off its elements' boundaries", name);
    const int64_t whole = ((uintptr_t)grad | (uintptr_t)out) % 16 ? 0 : n / 8 * 8, blocks = blocks_of(n, 256 * 8), most = 8 * sm_count();
    scale_wide_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, (cudaStream_t)stream>>>(grad, factor, (__half*)out, n, whole);
    return check_cuda(cudaGetLastError(), "scale_wide_kernel");
}
