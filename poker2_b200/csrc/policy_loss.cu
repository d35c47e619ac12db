// Clipped policy loss with a KL term over the hands of a batch of states, and its gradient, in one pass over the data.
//
// Per state and hand, over the legal actions a with p = softmax(logits), q the old policy, A the advantages, t the target:
//   l = -sum_a min(p_a A_a, clip(p_a, (1-e) q_a, (1+e) q_a) A_a) + k sum_a t_a (log t_a - log p_a)
//   dl/dz_a = -p_a (g_a - sum_b g_b p_b) + k (p_a sum_b t_b - t_a),   g_a = A_a where the first side of the min is taken, else 0
// and the loss is sum(w l) / sum(w) over the hands of states with a legal action.  (q min(r A, clip(r, 1-e, 1+e) A) with the ratio
// r = p/q, summed over the actions instead of sampled; written without the division, so q = 0 is no special case.)
//
// Bound by memory: an action's logit, three fp32 policies and the gradient.  A block takes 256 hands, whose arrays come as one
// bulk copy each (hands of 5 actions are 20 bytes: read by thread they would be five sectors an instruction).  Which side
// of the min is taken is decided in 64 bits where 32 might get it wrong: the gradient jumps there.
#include "layer.cuh"
#include "tensor.cuh"

namespace p2b {

using namespace tc;

constexpr int kHands = 256;       // hands of a block
constexpr int kMostActions = 16;
constexpr int kMassBlocks = 296;  // two a multiprocessor
constexpr int kMassChunk = 2048;

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
    int mass_parts;
    float* loss;
    void* grad;
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

// Sum of the weights of the hands whose state has a legal action: a part for every block, in a fixed order.
__global__ void __launch_bounds__(kHands) loss_mass_kernel(const float* weights, const uint8_t* legal, int64_t states, int hands, int actions,
                                                           unsigned long long* done, double* mass) {
    __shared__ double area[kHands / 32];
    const int64_t chunks = (hands + kMassChunk - 1) / kMassChunk;
    double sum = 0.0;
    for (int64_t job = blockIdx.x; job < states * chunks; job += gridDim.x) {
        const int64_t state = job / chunks;
        const int first = (int)(job - state * chunks) * kMassChunk, end = min(hands, first + kMassChunk);
        bool any = false;
        for (int a = 0; a < actions; ++a) any |= legal[state * actions + a] != 0;
        if (!any) continue;
        for (int h = first + threadIdx.x; h < end; h += kHands) sum += weights ? (double)weights[state * hands + h] : 1.0;
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

// The probability of action `which` in 64 bits.
template <int kActions, typename T> __device__ __noinline__ double exact_probability(const T* z, uint32_t open, int which) {
    double top = -INFINITY, sum = 0.0;
    for (int a = 0; a < kActions; ++a)
        if (open >> a & 1) top = fmax(top, (double)as_float(z[a]));
    for (int a = 0; a < kActions; ++a)
        if (open >> a & 1) sum += exp((double)as_float(z[a]) - top);
    return exp((double)as_float(z[which]) - top) / sum;
}

template <int kActions, typename T>
__global__ void __launch_bounds__(kHands) policy_loss_kernel(const __grid_constant__ LossArgs args) {
    extern __shared__ __align__(16) uint8_t area[];
    __shared__ double sums[kHands / 32];
    __shared__ uint64_t bar_word;
    __shared__ volatile int given_up;
    __shared__ bool last_block;
    T* z_s = reinterpret_cast<T*>(area);
    float* old_s = reinterpret_cast<float*>(area + kHands * kActions * sizeof(T));
    float* adv_s = old_s + kHands * kActions;
    float* target_s = adv_s + kHands * kActions;
    float* weight_s = target_s + kHands * kActions;
    const int64_t first = (int64_t)blockIdx.x * kHands;
    const int count = (int)(args.total - first < kHands ? args.total - first : kHands);
    const bool bulk = args.bulk && count == kHands;
    const uint32_t bar = smem_addr(&bar_word);
    const int tid = threadIdx.x;
    if (tid == 0) {
        given_up = 0;
        mbar_init(bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (bulk) {
            constexpr uint32_t words = kHands * kActions * 4, z_bytes = kHands * kActions * sizeof(T);
            mbar_expect(bar, z_bytes + words + (args.old_policy ? 2 * words : 0) + (args.weights ? kHands * 4 : 0));
            bulk_load(smem_addr(z_s), reinterpret_cast<const T*>(args.logits) + first * kActions, z_bytes, bar);
            bulk_load(smem_addr(target_s), args.target + first * kActions, words, bar);
            if (args.old_policy) {
                bulk_load(smem_addr(old_s), args.old_policy + first * kActions, words, bar);
                bulk_load(smem_addr(adv_s), args.advantages + first * kActions, words, bar);
            }
            if (args.weights) bulk_load(smem_addr(weight_s), args.weights + first, kHands * 4, bar);
        }
    }
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
    }
    // meanwhile the sum of the weights, and the hand's legal actions
    double mass = 0.0;
    for (int i = tid; i < args.mass_parts; i += kHands) mass += args.mass[i];
    mass = block_sum(mass, sums);  // (a barrier of the block: what the threads copied is there)
    const float inverse = mass > 0.0 ? (float)(1.0 / mass) : 0.0f;
    uint32_t open = 0;
    if (tid < count) {
        const int64_t state0 = first / args.hands;
        const int64_t state = state0 + ((int)(first - state0 * args.hands) + tid) / args.hands;
#pragma unroll
        for (int a = 0; a < kActions; ++a) open |= (args.legal[state * kActions + a] != 0 ? 1u : 0u) << a;
    }
    const bool ok = !bulk || mbar_wait(bar, 0, &given_up);
    if (!ok && tid == 0) {  // the copies in flight land before the block's memory goes
        volatile int still = 0;
        mbar_wait(bar, 0, &still);
    }

    double loss = 0.0;
    if (tid < count) {
        const float weight = args.weights ? weight_s[tid] : 1.0f;
        T* z_own = z_s + tid * kActions;
        float p[kActions], d[kActions];
        float top = -INFINITY;
#pragma unroll
        for (int a = 0; a < kActions; ++a) {
            p[a] = as_float(z_own[a]);
            if (open >> a & 1) top = fmaxf(top, p[a]);
        }
        // no legal action, or none that the logits leave, or a hand that does not count: nothing, whatever else is there
        if (weight != 0.0f && open != 0 && top != -INFINITY) {
            float total = 0.0f;
#pragma unroll
            for (int a = 0; a < kActions; ++a) {
                d[a] = p[a] - top;
                p[a] = open >> a & 1 ? expf(d[a]) : 0.0f;
                total += p[a];
            }
            const float log_total = logf(total), rcp = 1.0f / total;
            float surrogate = 0.0f, divergence = 0.0f, targets = 0.0f, pull = 0.0f;
            float g[kActions];
#pragma unroll
            for (int a = 0; a < kActions; ++a) {
                p[a] *= rcp;
                g[a] = 0.0f;
                if (open >> a & 1) {
                    const float t = target_s[tid * kActions + a];
                    targets += t;
                    if (t > 0.0f) divergence = fmaf(t, logf(t) - (d[a] - log_total), divergence);
                    if (args.old_policy) {
                        const float q = old_s[tid * kActions + a], adv = adv_s[tid * kActions + a];
                        const float low = (float)(1.0 - args.clip) * q, high = (float)(1.0 + args.clip) * q;
                        bool free = adv > 0.0f ? p[a] <= high : p[a] >= low;
                        const float border = adv > 0.0f ? high : low;
                        if (fabsf(p[a] - border) <= border * fmaf(fabsf(d[a]), 1e-7f, 1e-5f)) {
                            const double exact = exact_probability<kActions>(z_own, open, a);
                            free = adv > 0.0f ? exact <= (1.0 + args.clip) * (double)q : exact >= (1.0 - args.clip) * (double)q;
                        }
                        g[a] = free ? adv : 0.0f;
                        surrogate = fmaf(free ? p[a] : border, adv, surrogate);
                        pull = fmaf(g[a], p[a], pull);
                    }
                }
            }
            loss = (double)weight * (double)(args.kl * divergence - surrogate);
            const float scale = weight * inverse;
#pragma unroll
            for (int a = 0; a < kActions; ++a) {
                const float t = open >> a & 1 ? target_s[tid * kActions + a] : 0.0f;
                d[a] = scale * (args.kl * (p[a] * targets - t) - p[a] * (g[a] - pull));
            }
        } else {
#pragma unroll
            for (int a = 0; a < kActions; ++a) d[a] = 0.0f;
        }
        if (args.grad)
#pragma unroll
            for (int a = 0; a < kActions; ++a) z_own[a] = from_float<T>(ok ? d[a] : __int_as_float(0x7FC00000));
    }
    if (!ok) loss = __longlong_as_double(0x7FF8000000000000ll);
    loss = block_sum(loss, sums);
    if (args.grad) {
        if (bulk) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncthreads();
            if (tid == 0) {
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(reinterpret_cast<T*>(args.grad) + first * kActions),
                             "r"(smem_addr(z_s)), "r"((uint32_t)(kHands * kActions * sizeof(T)))
                             : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
        } else {
            for (int i = tid; i < count * kActions; i += kHands) reinterpret_cast<T*>(args.grad)[first * kActions + i] = z_s[i];
        }
    }
    // the block that comes last adds the parts up, in their order
    if (tid == 0) {
        args.sums[blockIdx.x] = loss;
        __threadfence();
        last_block = atomicAdd(args.done, 1ull) == gridDim.x - 1;
    }
    __syncthreads();
    if (last_block) {
        __threadfence();
        double sum = 0.0;
        for (int64_t i = tid; i < gridDim.x; i += kHands) sum += __ldcg(args.sums + i);
        sum = block_sum(sum, sums);
        if (tid == 0) *args.loss = mass > 0.0 ? (float)(sum / mass) : 0.0f;
    }
    if (bulk && args.grad && tid == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// grad * factor, the factor on the device
template <typename T> __global__ void __launch_bounds__(256) scale_kernel(const T* in, const float* factor, T* out, int64_t n) {
    const float f = *factor;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[i] = from_float<T>(as_float(in[i]) * f);
}

static SharedLimit g_limit[kMostActions + 1][3];

template <int kActions, typename T> static int launch_loss(const LossArgs& args, int type, cudaStream_t stream) {
    auto* kernel = policy_loss_kernel<kActions, T>;
    constexpr int shared = kHands * (kActions * (int)(sizeof(T) + 12) + 4);
    int rc = allow_shared(g_limit[kActions][type], (const void*)kernel, shared);
    if (rc) return rc;
    kernel<<<(unsigned)blocks_of(args.total, kHands), kHands, shared, stream>>>(args);
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
    return loss_sizes(states, hands, 1) ? 8 * (1 + kMassBlocks + blocks_of(states * hands, kHands)) : -1;
}

extern "C" int p2b_policy_loss(const void* logits, const float* old_policy, const float* advantages, const float* target, const uint8_t* legal,
                               const float* weights, int64_t states, int32_t hands, int32_t actions, int32_t dtype, double clip, float kl,
                               float* loss, void* grad, void* scratch, int64_t scratch_bytes, void* stream) {
    const char* name = "p2b_policy_loss";
    if (!loss_sizes(states, hands, actions))
        return set_error(P2B_ERR_ARG, "%s: %lld states of %d hands and %d actions are out of range (1 to %d actions)", name, (long long)states, hands, actions, kMostActions);
    if (dtype < 0 || dtype > 2) return set_error(P2B_ERR_ARG, "%s: unknown type %d (0 bf16, 1 fp16, 2 fp32)", name, dtype);
    if (!(clip >= 0.0 && clip < 1.0) || !(kl >= 0.0f && kl <= 3.4028234e38f)) return set_error(P2B_ERR_ARG, "%s: clip lies in [0, 1), kl is not negative", name);
    if (!loss || !scratch || scratch_bytes < p2b_policy_loss_scratch_bytes(states, hands) || (uintptr_t)scratch % 8)
        return set_error(P2B_ERR_ARG, "%s: loss and scratch of %lld bytes on an 8-byte boundary are needed", name,
                         (long long)p2b_policy_loss_scratch_bytes(states, hands));
    if ((old_policy == nullptr) != (advantages == nullptr)) return set_error(P2B_ERR_ARG, "%s: the old policy and the advantages come together", name);
    if (states > 0 && (!logits || !target || !legal)) return set_error(P2B_ERR_ARG, "%s: null array", name);
    const int size = dtype == 2 ? 4 : 2;
    const uintptr_t four = (uintptr_t)old_policy | (uintptr_t)advantages | (uintptr_t)target | (uintptr_t)weights | (uintptr_t)loss;
    if (four % 4 || ((uintptr_t)logits | (uintptr_t)grad) % size) return set_error(P2B_ERR_ARG, "%s: an array lies off its elements' boundaries", name);
    cudaStream_t st = (cudaStream_t)stream;
    if (states == 0) return check_cuda(cudaMemsetAsync(loss, 0, 4, st), name);
    LossArgs args{};
    args.logits = logits, args.old_policy = old_policy, args.advantages = advantages, args.target = target, args.weights = weights, args.legal = legal;
    args.states = states, args.total = states * hands, args.hands = hands, args.clip = clip, args.kl = kl, args.loss = loss, args.grad = grad;
    args.bulk = (((uintptr_t)old_policy | (uintptr_t)advantages | (uintptr_t)target | (uintptr_t)weights | (uintptr_t)logits | (uintptr_t)grad) % 16) == 0;
    args.done = (unsigned long long*)scratch;
    args.mass = (double*)scratch + 1;
    args.sums = args.mass + kMassBlocks;
    const int64_t jobs = states * blocks_of(hands, kMassChunk);
    args.mass_parts = (int)(jobs < kMassBlocks ? jobs : kMassBlocks);
    loss_mass_kernel<<<args.mass_parts, kHands, 0, st>>>(weights, legal, states, hands, actions, args.done, args.mass);
    int rc = check_cuda(cudaGetLastError(), "loss_mass_kernel");
    if (rc) return rc;
    if (dtype == 0) return launch_actions<__nv_bfloat16>(args, actions, 0, st);
    if (dtype == 1) return launch_actions<__half>(args, actions, 1, st);
    return launch_actions<float>(args, actions, 2, st);
}

extern "C" int p2b_policy_loss_scale(const void* grad, const float* factor, int64_t n, int32_t dtype, void* out, void* stream) {
    if (n < 0 || dtype < 0 || dtype > 2) return set_error(P2B_ERR_ARG, "p2b_policy_loss_scale: %lld values of type %d", (long long)n, dtype);
    if (n == 0) return P2B_OK;
    if (!grad || !factor || !out) return set_error(P2B_ERR_ARG, "p2b_policy_loss_scale: null array");
    const int64_t blocks = blocks_of(n, 1024);
    const unsigned grid = (unsigned)(blocks < 8 * sm_count() ? blocks : 8 * sm_count());
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == 0) scale_kernel<<<grid, 256, 0, st>>>((const __nv_bfloat16*)grad, factor, (__nv_bfloat16*)out, n);
    if (dtype == 1) scale_kernel<<<grid, 256, 0, st>>>((const __half*)grad, factor, (__half*)out, n);
    if (dtype == 2) scale_kernel<<<grid, 256, 0, st>>>((const float*)grad, factor, (float*)out, n);
    return check_cuda(cudaGetLastError(), "scale_kernel");
}
