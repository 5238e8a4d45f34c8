// Routing to experts with a choice of scores, a balance bias and groups of experts (jq_moe_route_topk).
//
//   s = softmax(l) or 1 / (1 + exp(-l));  c = s + bias
//   group score = sum of the group_top largest c of a group; the groups_kept best groups stay
//   idx = the k largest c of the groups that stay, descending;  w = s[idx] (/ (sum + 1e-20)) * scale
//
// Bound: T * E logits read once; at the sizes of a serving step it is latency, the k dependent selections of a warp.
// One warp per token, a lane holds PER >= E / 32 of the row's keys in registers.  Which expert is taken hangs on
// neighbouring scores, so c is compared in float64 (float32 scores put close neighbours on the wrong side about once in
// 4096 tokens x 256 experts); where c grows with the logit alone -- no bias, and at most the best expert of a group
// counts -- the order of the logits is the order of the scores and 32-bit keys do.  A key is the value's bits made
// monotonic as an unsigned integer, so an arg-max over the warp is two redux steps per 32 bits instead of ten
// shuffles; equal keys go to the lower expert.  A NaN logit counts as -inf, a score of zero; +inf takes the limit.
#include "jq_common.cuh"

namespace jq {

constexpr int ROUTE2_MAX_E = 1024;
constexpr int ROUTE2_MAX_GROUPS = 32;
constexpr int ROUTE2_WARPS = 4;

__device__ __forceinline__ uint32_t redux_max(uint32_t v) { return __reduce_max_sync(0xFFFFFFFFu, v); }
__device__ __forceinline__ uint32_t redux_min(uint32_t v) { return __reduce_min_sync(0xFFFFFFFFu, v); }

// monotonic keys; 0 is below every number's key and stands for "not to be chosen".  -0 and 0 are one score.
__device__ __forceinline__ uint32_t order_key(float v) {
    v = v != v ? -INFINITY : v + 0.f;
    const uint32_t b = __float_as_uint(v);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(double v) {
    v = v != v ? -(double)INFINITY : v + 0.0;
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
}
// largest key of the warp, known to every lane
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return redux_max(k); }
__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
    const uint32_t hi = redux_max((uint32_t)(k >> 32));
    const uint32_t lo = redux_max((uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return (uint64_t)hi << 32 | lo;
}

template <bool F64> struct RouteKey { using V = float; using K = uint32_t; };
template <> struct RouteKey<true> { using V = double; using K = uint64_t; };

struct RouteArgs {
    const void* logits;
    int64_t ld;
    const float* bias;
    int32_t* idx;
    float* w;
    int T, E, k, sigmoid, groups, kept, top, renorm;
    float scale;
};

template <typename LT> __device__ __forceinline__ float load_logit(const RouteArgs& a, int64_t t, int e) {
    const float v = Elt<LT>::to_f32(reinterpret_cast<const LT*>(a.logits)[t * a.ld + e]);
    return v != v ? -INFINITY : v;
}
// exp(l - mx) without inf - inf
__device__ __forceinline__ double exp_below(float l, float mx) { return l == mx ? (mx == -INFINITY ? 0.0 : 1.0) : exp((double)l - (double)mx); }

template <typename LT, int PER, bool F64>
__global__ void __launch_bounds__(32 * ROUTE2_WARPS)
route_groups_kernel(const RouteArgs a) {
    using V = typename RouteKey<F64>::V;
    using K = typename RouteKey<F64>::K;
    extern __shared__ __align__(16) uint8_t route_smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t t = (int64_t)blockIdx.x * ROUTE2_WARPS + warp;
    if (t >= a.T) return;                                  // no block-wide barrier below
    const int E = a.E;

    float l[PER];
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane + 32 * i;
        l[i] = e < E ? load_logit<LT>(a, t, e) : -INFINITY;
        mx = fmaxf(mx, l[i]);
    }
    double sum = 0.0;                                      // of the softmax; unused with sigmoid scores
    V c[PER];
    if (!a.sigmoid) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, d));
        if constexpr (F64) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                c[i] = lane + 32 * i < E ? exp_below(l[i], mx) : 0.0;
                sum += c[i];
            }
        } else {                                           // only the weights see the sum: float32 terms
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (l[i] != -INFINITY) part += l[i] == mx ? 1.f : expf(l[i] - mx);
            sum = part;
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
        if (sum == 0.0) sum = 1.0;                         // a row of -inf: every score is zero
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane + 32 * i;
        if constexpr (F64) {
            c[i] = a.sigmoid ? 1.0 / (1.0 + exp(-(double)l[i])) : c[i] / sum;
            if (a.bias && e < E) c[i] += (double)a.bias[e];
        } else {
            c[i] = l[i];
        }
    }

    uint32_t keep = 0xFFFFFFFFu;                           // bit per group
    const int per = E / a.groups;
    if (a.groups > 1) {
        V* row = reinterpret_cast<V*>(route_smem) + (size_t)warp * E;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (lane + 32 * i < E) row[lane + 32 * i] = c[i] != c[i] ? -(V)INFINITY : c[i];
        __syncwarp();
        // L lanes per group (a power of two): two largest of the lane's share, then a butterfly over the L lanes
        int L = 1;
        while (2 * L * a.groups <= 32) L *= 2;
        const int g = lane / L;
        V best = -(V)INFINITY, second = -(V)INFINITY;
        if (g < a.groups)
            for (int j = lane % L; j < per; j += L) {
                const V v = row[g * per + j];
                second = v > best ? best : (v > second ? v : second);
                best = v > best ? v : best;
            }
        for (int d = L / 2; d > 0; d >>= 1) {
            const V b2 = __shfl_xor_sync(0xFFFFFFFFu, best, d), s2 = __shfl_xor_sync(0xFFFFFFFFu, second, d);
            const V low = best < b2 ? best : b2, high = best < b2 ? b2 : best;
            const V s = second > s2 ? second : s2;
            best = high;
            second = low > s ? low : s;
        }
        const K mine = order_key(a.top == 2 ? best + second : best);
        int rank = 0;
        for (int o = 0; o < a.groups; ++o) {
            const K other = __shfl_sync(0xFFFFFFFFu, mine, o * L);
            rank += (other > mine || (other == mine && o < g)) ? 1 : 0;
        }
        const uint32_t in = __ballot_sync(0xFFFFFFFFu, g < a.groups && rank < a.kept);      // L equal bits per group
        keep = 0;
        for (int o = 0; o < a.groups; ++o) keep |= ((in >> (o * L)) & 1u) << o;
    }

    K key[PER];
    K best = 0;
    int bi = 0;                                            // register index of the lane's best; the lower expert on ties
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane + 32 * i;
        key[i] = e < E && (a.groups == 1 || (keep >> (e / per) & 1u)) ? order_key(c[i]) : (K)0;
        if (key[i] > best) { best = key[i]; bi = i; }
    }
    double chosen = 0.0;                                   // sum of the chosen scores
    for (int j0 = 0; j0 < a.k; j0 += 32) {
        const int n = min(32, a.k - j0);
        int mine = 0;
        for (int j = 0; j < n; ++j) {
            const K top = warp_max(best);
            const int e = (int)redux_min(best == top ? (uint32_t)(lane + 32 * bi) : 0xFFFFFFFFu);
            if (lane == j) mine = e;
            if (lane == (e & 31)) {                        // the owner looks for its next one
                best = 0;
                const int gone = e >> 5;
                bi = 0;
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    if (i == gone) key[i] = 0;
                    if (key[i] > best) { best = key[i]; bi = i; }
                }
            }
            __syncwarp();
        }
        double s = 0.0;
        if (lane < n) {
            const float lv = load_logit<LT>(a, t, mine);
            s = a.sigmoid ? 1.0 / (1.0 + exp(-(double)lv)) : exp_below(lv, mx) / sum;
            a.idx[t * a.k + j0 + lane] = mine;
        }
        chosen += s;
        if (a.k > 32 && lane < n) a.w[t * a.k + j0 + lane] = (float)s;        // scaled below, once the sum is known
        if (a.k <= 32) {
            double norm = a.scale;
            if (a.renorm) {
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) chosen += __shfl_xor_sync(0xFFFFFFFFu, chosen, d);
                norm = (double)a.scale / (chosen + 1e-20);
            }
            if (lane < n) a.w[t * a.k + lane] = (float)(s * norm);
            return;
        }
    }
    double norm = a.scale;
    if (a.renorm) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) chosen += __shfl_xor_sync(0xFFFFFFFFu, chosen, d);
        norm = (double)a.scale / (chosen + 1e-20);
    }
    for (int j = lane; j < a.k; j += 32) {                 // the lane's own stores of above
        float* p = a.w + t * a.k + j;
        *p = (float)((double)*p * norm);
    }
}

template <typename LT, int PER, bool F64>
static int launch_route(const RouteArgs& a, cudaStream_t st) {
    const unsigned blocks = (unsigned)((a.T + ROUTE2_WARPS - 1) / ROUTE2_WARPS);
    const size_t smem = a.groups > 1 ? (size_t)ROUTE2_WARPS * a.E * sizeof(typename RouteKey<F64>::V) : 0;
    static_assert(ROUTE2_WARPS * ROUTE2_MAX_E * sizeof(double) <= 48 * 1024, "no opt-in shared memory");
    route_groups_kernel<LT, PER, F64><<<blocks, 32 * ROUTE2_WARPS, smem, st>>>(a);
    return check_launch("moe_route_topk");
}

template <typename LT>
static int launch_route_e(const RouteArgs& a, bool f64, cudaStream_t st) {
#define JQ_ROUTE_PER(P) return f64 ? launch_route<LT, P, true>(a, st) : launch_route<LT, P, false>(a, st)
    if (a.E <= 64) JQ_ROUTE_PER(2);
    if (a.E <= 128) JQ_ROUTE_PER(4);
    if (a.E <= 256) JQ_ROUTE_PER(8);
    if (a.E <= 512) JQ_ROUTE_PER(16);
    JQ_ROUTE_PER(32);
#undef JQ_ROUTE_PER
}

}  // namespace jq

extern "C" int jq_moe_route_topk(const void* logits, int logits_dtype, int64_t ld, int64_t T, int num_experts, int k, int score,
                                 const float* bias, int groups, int groups_kept, int group_top, int renorm, float scale,
                                 int32_t* idx_out, float* w_out, jq_stream_t stream) {
    using namespace jq;
    JQ_REQUIRE(num_experts > 0 && num_experts <= ROUTE2_MAX_E, JQ_EUNSUPPORTED, "jq_moe_route_topk takes 1 to %d experts, got %d",
               ROUTE2_MAX_E, num_experts);
    JQ_REQUIRE(score == JQ_SCORE_SOFTMAX || score == JQ_SCORE_SIGMOID, JQ_EINVAL, "unknown score kind %d", score);
    JQ_REQUIRE(groups >= 1 && groups <= ROUTE2_MAX_GROUPS && num_experts % groups == 0, JQ_EINVAL,
               "groups must be 1 to %d and divide the number of experts (%d), got %d", ROUTE2_MAX_GROUPS, num_experts, groups);
    JQ_REQUIRE(groups_kept >= 1 && groups_kept <= groups, JQ_EINVAL, "groups_kept must be 1 to %d, got %d", groups, groups_kept);
    JQ_REQUIRE(groups == 1 || ((group_top == 1 || group_top == 2) && group_top <= num_experts / groups), JQ_EINVAL,
               "group_top must be 1 or 2 and at most the experts of a group (%d), got %d", num_experts / groups, group_top);
    JQ_REQUIRE(k >= 1 && k <= groups_kept * (num_experts / groups), JQ_EINVAL,
               "k must be 1 to the experts of the groups that are kept (%d), got %d", groups_kept * (num_experts / groups), k);
    JQ_REQUIRE(valid_dtype(logits_dtype), JQ_EINVAL, "logits must be f32, f16 or bf16");
    JQ_REQUIRE(T >= 0 && ld >= num_experts, JQ_EINVAL, "T must not be negative, ld at least the number of experts");
    JQ_REQUIRE(T < (1ll << 30), JQ_EUNSUPPORTED, "too many rows");
    if (T == 0) return JQ_OK;
    JQ_REQUIRE(logits && idx_out && w_out, JQ_EINVAL, "null pointer");
    RouteArgs a;
    a.logits = logits; a.ld = ld; a.bias = bias; a.idx = idx_out; a.w = w_out;
    a.T = (int)T; a.E = num_experts; a.k = k; a.sigmoid = score == JQ_SCORE_SIGMOID;
    // all groups kept is no grouping
    a.groups = groups_kept == groups ? 1 : groups;
    a.kept = groups_kept; a.top = group_top; a.renorm = renorm; a.scale = scale;
    const bool f64 = bias != nullptr || (a.groups > 1 && group_top == 2);
    JQ_DISPATCH_DTYPE(logits_dtype, LT, return launch_route_e<LT>(a, f64, (cudaStream_t)stream));
    return JQ_OK;
}
