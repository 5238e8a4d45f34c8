// Routing to experts with a choice of scores, a balance bias and groups of experts (jq_moe_route_topk).
//
//   s = softmax(l) or 1 / (1 + exp(-l));  c = s + bias
//   group score = sum of the group_top largest c of a group; the groups_kept best groups stay
//   idx = the k largest c of the groups that stay, descending;  w = s[idx] (/ (sum + 1e-20)) * scale
//
// Bound: T * E logits read once; at the sizes of a serving step it is latency, the k dependent selections of a warp.
// One warp per token, a lane holds PER >= E / 32 of the row's keys in registers: values made monotonic as unsigned
// integers, so the arg-max of the warp is two redux steps; equal keys go to the lower expert.
// Which expert is taken hangs on neighbouring scores: float32 scores put close neighbours on the wrong side about once in
// 4096 tokens x 256 experts, and float64 ones for every expert cost 12 us for 61 tokens x 512.  So a token is selected on
// float32 scores together with a bound of their error, and what the bound leaves open is settled in float64: the groups, if
// two at the cut are closer than the bound, and the order of the chosen experts and of those within the bound of the last,
// if there are neighbours among them that close.  The slowest token of a call is its time, so this path is kept short too
// (the whole token again in float64: 22 us for 4096 x 256).  Where c grows with the logit alone (no bias, and at most the
// best expert of a group counts) the order of the logits is the order of the scores, exactly.  A NaN logit counts as -inf, a
// score of zero; +inf takes the limit.
// Weights that are not renormalised hold the softmax's sum: it is taken in float64 then (61 tokens, 512 experts 7.7 us, 5.9 with a
// float32 sum, whose ten roundings left weights up to three half steps off; 4096 tokens, 256 experts 10.0 and 8.1).
// Measured: one token, 128 experts, softmax 2.5 us (an empty launch is 2); 61 tokens, 512 experts, bias, 10 of them 6.8; sigmoid,
// bias, the best 4 of 8 groups of 32, 8 experts: 592 tokens 5.6, 4096 tokens 12 to 14 by how close their scores lie (latency up to one
// token per scheduler, then issue of the selections, the groups and the scores in like parts).
#include "jq_launch.cuh"

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
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }
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

// How the choice scores are held: the logits themselves (their order is the scores'), or float32 with a bound of the error.
enum RouteMode { ROUTE_LOGIT, ROUTE_SCREEN };
// How far the difference of two float32 choice scores may be off, in units u = 2^-23.  The fast exponential of -d is off by
// 2 + 1.16 d units of its value.  A softmax score is at most top = 1 / sum: exponential 2 top (where d = 0), its argument and the
// quotient 1.5 top; the sum, common to both scores, by the mean of 2 + 1.16 d over the terms, at most 11 for 1024 experts, and
// ten additions by halves: 16 top for the difference.  23 top for two scores.  A sigmoid score is off by 1 from its
// exponential (s (1 - s) (2 + 1.16 d) < 1), 2 from the quotient and 1 from the sum in it: 8 for two.  The sum of a group's
// two largest is off by twice as much.  Adding the bias rounds each by half a unit of |c|, the group's sum once more: 4 of the
// largest |c|.  46 top, 16 and 4, each taken about twice as large.
__device__ __forceinline__ float choice_error(bool sigmoid, float top, float largest) {
    return (sigmoid ? 0x1p-18f : 0x1p-16f * top) + 0x1p-20f * largest;
}

// sum by halves (E of 1024: ten additions deep), and the largest key with its place, the lower place on ties
template <int PER> __device__ __forceinline__ float lane_sum(const float (&c)[PER]) {
    float p[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) p[i] = c[i];
#pragma unroll
    for (int w = PER / 2; w > 0; w /= 2)
#pragma unroll
        for (int i = 0; i < w; ++i) p[i] += p[i + w];
    return p[0];
}
template <int PER> __device__ __forceinline__ void lane_best(const uint32_t (&key)[PER], uint32_t& best, int& at) {
    uint32_t k[PER];
    int ix[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) { k[i] = key[i]; ix[i] = i; }
#pragma unroll
    for (int w = PER / 2; w > 0; w /= 2)
#pragma unroll
        for (int i = 0; i < w; ++i) {
            const bool left = k[2 * i] >= k[2 * i + 1];
            k[i] = left ? k[2 * i] : k[2 * i + 1];
            ix[i] = left ? ix[2 * i] : ix[2 * i + 1];
        }
    best = k[0];
    at = ix[0];
}

struct RouteArgs {
    const void* logits;
    int64_t ld;
    const float* bias;
    int32_t* idx;
    float* w;
    int T, E, k, sigmoid, groups, kept, top, renorm;
    int per;                         // experts of a group
    int lanes_log2;                  // lanes of the warp per group: as many as fit
    float scale;
};

template <typename LT> __device__ __forceinline__ float load_logit(const RouteArgs& a, int64_t t, int e) {
    const float v = Elt<LT>::to_f32(reinterpret_cast<const LT*>(a.logits)[t * a.ld + e]);
    return v != v ? -INFINITY : v;
}
// exp(l - mx) without inf - inf
__device__ __forceinline__ double exp_below(float l, float mx) { return l == mx ? (mx == -INFINITY ? 0.0 : 1.0) : exp((double)l - (double)mx); }

// Which groups stay, as a bit for each of a group's 1 << lanes_log2 lanes, from the choice scores of the token in shared memory.  near: set (in every lane)
// when a group at the cut is within `close` of another.
template <typename V>
__device__ __forceinline__ uint32_t kept_groups(const RouteArgs& a, const V* row, int lane, float close, bool& near) {
    // L lanes per group: two largest of the lane's share, then a butterfly over the L lanes
    const int L = 1 << a.lanes_log2, g = lane >> a.lanes_log2;
    V best = -(V)INFINITY, second = -(V)INFINITY;
    if (g < a.groups)
#pragma unroll 8
        for (int j = lane & (L - 1); j < a.per; j += L) {
            const V v = row[g * a.per + j];
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
    const V score = a.top == 2 ? best + second : best;
    const auto mine = order_key(score);
    int rank = 0;
    bool touch = false;
    for (int o = 0; o < a.groups; ++o) {
        const auto other = __shfl_sync(0xFFFFFFFFu, mine, o << a.lanes_log2);
        const V value = __shfl_sync(0xFFFFFFFFu, score, o << a.lanes_log2);
        rank += (other > mine || (other == mine && o < g)) ? 1 : 0;
        touch |= o != g && !(fabs(value - score) > (V)close);            // two infinities differ by NaN, which is near
    }
    near = __any_sync(0xFFFFFFFFu, g < a.groups && touch && (rank == a.kept - 1 || rank == a.kept));
    return __ballot_sync(0xFFFFFFFFu, g < a.groups && rank < a.kept);
}

template <typename LT> __device__ __forceinline__ double exact_score(const RouteArgs& a, int64_t t, int e, float mx, double sum) {
    const float lv = load_logit<LT>(a, t, e);
    return a.sigmoid ? 1.0 / (1.0 + exp(-(double)lv)) : exp_below(lv, mx) / sum;
}
// Results of up to 32 selections from j0 on: lane j holds expert `mine`.  Returns the sum of their scores.  MANY: k may be above 32.
template <typename LT, bool MANY>
__device__ __forceinline__ double store_chosen(const RouteArgs& a, int64_t t, int lane, int j0, int n, int mine, float mx, double sum) {
    double s = 0.0, chosen;
    if (lane < n) {
        s = exact_score<LT>(a, t, mine, mx, sum);
        a.idx[t * a.k + j0 + lane] = mine;
    }
    chosen = s;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) chosen += __shfl_xor_sync(0xFFFFFFFFu, chosen, d);
    if (!MANY || a.k <= 32) {                              // of more: when the sum of all is known
        s *= a.renorm ? (double)a.scale / (chosen + 1e-20) : (double)a.scale;
        if (lane < n) a.w[t * a.k + j0 + lane] = (float)s;
    }
    return chosen;
}
template <typename LT>
__device__ __forceinline__ void store_weights(const RouteArgs& a, int64_t t, int lane, float mx, double sum, double chosen) {
    if (a.k <= 32) return;
    const double norm = a.renorm ? (double)a.scale / (chosen + 1e-20) : (double)a.scale;
#pragma unroll 1
    for (int j = lane; j < a.k; j += 32)                   // the lane's own choices
        a.w[t * a.k + j] = (float)(exact_score<LT>(a, t, a.idx[t * a.k + j], mx, sum) * norm);
}

// Sum of the softmax, and the choice scores of a whole token, in float64; four exponentials at a time (a row of them unrolled is
// so much code that fetching it takes longer than running it).
template <typename LT>
__device__ __forceinline__ double exact_sum_here(const RouteArgs& a, int64_t t, int lane, float mx) {
    double sum = 0.0;
#pragma unroll 4
    for (int e = lane; e < a.E; e += 32) sum += exp_below(load_logit<LT>(a, t, e), mx);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    return sum == 0.0 ? 1.0 : sum;                         // a row of -inf: every score is zero
}
template <typename LT> __device__ __noinline__ double exact_sum(const RouteArgs& a, int64_t t, int lane, float mx) {
    return exact_sum_here<LT>(a, t, lane, mx);
}
template <typename LT>
__device__ __forceinline__ double exact_choice(const RouteArgs& a, int64_t t, int e, float mx, double sum) {
    double c = exact_score<LT>(a, t, e, mx, sum);
    if (a.bias) c += (double)a.bias[e];
    return c != c ? -(double)INFINITY : c;
}
template <typename LT>
__device__ __noinline__ void exact_row(const RouteArgs& a, int64_t t, int lane, double* row, float mx, double sum) {
#pragma unroll 4
    for (int e = lane; e < a.E; e += 32) row[e] = exact_choice<LT>(a, t, e, mx, sum);
    __syncwarp();
}

// The n candidates, one per lane, in the order of their exact scores (place: n ints).
template <typename LT>
__device__ __noinline__ int exact_order(const RouteArgs& a, int64_t t, int lane, int n, int mine, int* place, float mx, double sum) {
    const uint64_t key = lane < n ? order_key(exact_choice<LT>(a, t, mine, mx, sum)) : 0ull;
    int rank = 0;
    for (int o = 0; o < n; ++o) {
        const uint64_t other = __shfl_sync(0xFFFFFFFFu, key, o);
        const int oe = __shfl_sync(0xFFFFFFFFu, mine, o);
        rank += other > key || (other == key && oe < mine) ? 1 : 0;
    }
    if (lane < n) place[rank] = mine;
    __syncwarp();
    return lane < n ? place[lane] : 0;
}

// One token on 32-bit keys (row: E doubles of shared memory, or floats where the logits decide).  Returns false (the same in
// every lane) where the token is to be done in float64: more than 32 experts too close to tell, or weights that hold the screen's sum.
template <typename LT, int PER, RouteMode MODE>
__device__ __forceinline__ bool route_token(const RouteArgs& a, int64_t t, int lane, void* row, const float (&l)[PER], float mx) {
    const int E = a.E;
    float sum = 1.f;                                       // of the softmax, for the screen
    float c[PER];
    if (MODE == ROUTE_SCREEN && !a.sigmoid) {
        const float m = mx == -INFINITY ? 0.f : mx;        // exp(-inf) = 0 of masked experts, places past E and empty rows
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const float d = mx == INFINITY ? (l[i] == INFINITY ? 0.f : -INFINITY) : l[i] - m;
            c[i] = __expf(d);
        }
        sum = lane_sum<PER>(c);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
        if (sum == 0.f) sum = 1.f;                         // a row of -inf: every score is zero
    }
    float close = 0.f;
    double sum64 = 0.0;                                    // computed when it is needed
    if constexpr (MODE == ROUTE_LOGIT) {
#pragma unroll
        for (int i = 0; i < PER; ++i) c[i] = l[i];
    } else {
        float largest = 0.f;                               // |c| of the token; a NaN is passed over, it counts as -inf
        const float inv = 1.f / sum;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = lane + 32 * i;
            c[i] = a.sigmoid ? __fdividef(1.f, 1.f + __expf(-l[i])) : c[i] * inv;
            if (a.bias && e < E) c[i] += a.bias[e];
            largest = fmaxf(largest, fabsf(c[i]));
        }
        close = choice_error(a.sigmoid, inv, __uint_as_float(redux_max(__float_as_uint(largest))));
        if (!(close < INFINITY)) return false;             // an infinite bias
    }
    uint32_t keep = 0xFFFFFFFFu;
    if (a.groups > 1) {
        float* row32 = reinterpret_cast<float*>(row);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (lane + 32 * i < E) row32[lane + 32 * i] = c[i] != c[i] ? -INFINITY : c[i];
        __syncwarp();
        bool near;
        keep = kept_groups<float>(a, row32, lane, close, near);
        __syncwarp();                                      // the row is written again
        if (MODE == ROUTE_SCREEN && near) {
            if (!a.sigmoid) sum64 = exact_sum<LT>(a, t, lane, mx);
            exact_row<LT>(a, t, lane, reinterpret_cast<double*>(row), mx, sum64);
            keep = kept_groups<double>(a, reinterpret_cast<double*>(row), lane, 0.f, near);
            __syncwarp();
        }
    }
    uint32_t key[PER];
    const float per_group = 1.f / (float)a.per;            // (e + 1/2) / per is never within 2^-12 of a whole number
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane + 32 * i;
        key[i] = e < E && (keep >> ((int)(((float)e + 0.5f) * per_group) << a.lanes_log2) & 1u) ? order_key(c[i]) : 0u;
    }
    uint32_t best, before = 0;
    int bi;                                                // register index of the lane's best
    lane_best<PER>(key, best, bi);
    double chosen = 0.0;
    for (int j0 = 0; j0 < a.k; j0 += 32) {
        int n = min(32, a.k - j0), mine = 0;
        bool open = false;
        for (int j = 0;; ++j) {
            const uint32_t top = redux_max(best);
            if (MODE == ROUTE_LOGIT && j == n) break;
            if constexpr (MODE == ROUTE_SCREEN) {          // two infinities differ by NaN, which is close
                const bool touch = j > 0 && top != 0 && !(key_value(before) - key_value(top) > close);
                if (j >= n && !touch) break;               // the chosen ones and those within the bound of the last of them
                if (j == 32) return false;
                open |= touch;
                before = top;
            }
            const int e = (int)redux_min(best == top ? (uint32_t)(lane + 32 * bi) : 0xFFFFFFFFu);
            if (lane == j) mine = e;
            if (lane == (e & 31)) {                        // the owner looks for its next one
                const int gone = e >> 5;
#pragma unroll
                for (int i = 0; i < PER; ++i)
                    if (i == gone) key[i] = 0;
                lane_best<PER>(key, best, bi);
            }
            __syncwarp();
            if constexpr (MODE == ROUTE_SCREEN)
                if (j >= n) n = j + 1;
        }
        if constexpr (MODE == ROUTE_SCREEN) {
            if (open) {                                    // k <= 32 here
                if (!a.sigmoid && sum64 == 0.0) sum64 = exact_sum<LT>(a, t, lane, mx);
                mine = exact_order<LT>(a, t, lane, n, mine, reinterpret_cast<int*>(row), mx, sum64);
            }
            n = min(32, a.k - j0);
        }
        // A renormalised weight does not hold the sum, so the screen's (or none, where the logits decide) does for it, unless the
        // chosen scores are so small, against the largest, that the 1e-20 beside their own sum counts.
        // (A call costs a copy of the arguments at the kernel's start, which the form without others is spared.)
        if (!a.sigmoid && !a.renorm && sum64 == 0.0)
            sum64 = MODE == ROUTE_LOGIT ? exact_sum_here<LT>(a, t, lane, mx) : exact_sum<LT>(a, t, lane, mx);
        const double got = store_chosen<LT, MODE == ROUTE_LOGIT>(a, t, lane, j0, n, mine, mx, sum64 != 0.0 ? sum64 : (double)sum);
        if constexpr (MODE == ROUTE_LOGIT) chosen += got;
        else if (!a.sigmoid && sum64 == 0.0 && got < 1e-12) return false;
    }
    if constexpr (MODE == ROUTE_LOGIT) store_weights<LT>(a, t, lane, mx, sum64 != 0.0 ? sum64 : 1.0, chosen);
    return true;
}

// A whole token in float64, in shared memory: more than 32 experts to choose, or too many too close to each other.
template <typename LT>
__device__ __noinline__ void route_token_exact(const RouteArgs& a, int64_t t, int lane, double* row, float mx) {
    const double sum = a.sigmoid ? 1.0 : exact_sum<LT>(a, t, lane, mx);
    exact_row<LT>(a, t, lane, row, mx, sum);
    uint32_t keep = 0xFFFFFFFFu;
    if (a.groups > 1) {
        bool near;
        keep = kept_groups<double>(a, row, lane, 0.f, near);
        __syncwarp();
    }
    // keys take the scores' places; the lane's best is found by walking its share
    uint64_t* key = reinterpret_cast<uint64_t*>(row);
    uint64_t best = 0;
    int at = 0;
    for (int e = lane; e < a.E; e += 32) {
        const uint64_t k = a.groups == 1 || (keep >> (e / a.per << a.lanes_log2) & 1u) ? order_key(row[e]) : 0ull;
        key[e] = k;
        if (k > best) { best = k; at = e; }
    }
    double chosen = 0.0;
    for (int j0 = 0; j0 < a.k; j0 += 32) {
        const int n = min(32, a.k - j0);
        int mine = 0;
        for (int j = 0; j < n; ++j) {
            const uint64_t top = warp_max(best);
            const int e = (int)redux_min(best == top ? (uint32_t)at : 0xFFFFFFFFu);
            if (lane == j) mine = e;
            if (lane == (e & 31)) {
                key[e] = 0;
                best = 0;
                for (int i = lane; i < a.E; i += 32)
                    if (key[i] > best) { best = key[i]; at = i; }
            }
            __syncwarp();
        }
        chosen += store_chosen<LT, true>(a, t, lane, j0, n, mine, mx, sum);
    }
    store_weights<LT>(a, t, lane, mx, sum, chosen);
}

// SCREEN: the order of the logits does not decide
template <typename LT, int PER, bool SCREEN>
__global__ void __launch_bounds__(32 * ROUTE2_WARPS)
route_groups_kernel(const RouteArgs a) {
    extern __shared__ __align__(16) uint8_t route_smem[];
    overlap_enter();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t t = (int64_t)blockIdx.x * ROUTE2_WARPS + warp;
    if (t >= a.T) return;                                  // no block-wide barrier below
    float l[PER];
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane + 32 * i;
        l[i] = e < a.E ? load_logit<LT>(a, t, e) : -INFINITY;
        mx = fmaxf(mx, l[i]);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, d));
    if constexpr (SCREEN) {
        double* row = reinterpret_cast<double*>(route_smem) + (size_t)warp * a.E;
        if (a.k > 32 || !route_token<LT, PER, ROUTE_SCREEN>(a, t, lane, row, l, mx))
            route_token_exact<LT>(a, t, lane, row, mx);
    } else {
        route_token<LT, PER, ROUTE_LOGIT>(a, t, lane, reinterpret_cast<float*>(route_smem) + (size_t)warp * a.E, l, mx);
    }
}

template <typename LT, int PER, bool SCREEN>
static int launch_route(const RouteArgs& a, cudaStream_t st) {
    const unsigned blocks = (unsigned)((a.T + ROUTE2_WARPS - 1) / ROUTE2_WARPS);
    const size_t smem = SCREEN || a.groups > 1 ? (size_t)ROUTE2_WARPS * a.E * (SCREEN ? sizeof(double) : sizeof(float)) : 0;
    static_assert(ROUTE2_WARPS * ROUTE2_MAX_E * sizeof(double) <= 48 * 1024, "no opt-in shared memory");
    JQ_CUDA_OK(launch_overlapped(route_groups_kernel<LT, PER, SCREEN>, dim3(blocks), 32 * ROUTE2_WARPS, smem, st, a));
    return JQ_OK;
}

template <typename LT>
static int launch_route_e(const RouteArgs& a, bool screen, cudaStream_t st) {
#define JQ_ROUTE_PER(P) return screen ? launch_route<LT, P, true>(a, st) : launch_route<LT, P, false>(a, st)
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
    a.per = num_experts / a.groups;
    a.lanes_log2 = 0;
    while (a.groups > 1 && a.groups << (a.lanes_log2 + 1) <= 32) ++a.lanes_log2;
    a.kept = groups_kept; a.top = group_top; a.renorm = renorm; a.scale = scale;
    const bool screen = bias != nullptr || (a.groups > 1 && group_top == 2);
    JQ_DISPATCH_DTYPE(logits_dtype, LT, return launch_route_e<LT>(a, screen, (cudaStream_t)stream));
    return JQ_OK;
}
