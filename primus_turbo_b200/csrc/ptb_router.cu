// Top-k routing of a mixture-of-experts layer, and its gradient.
//
//   s = softmax(l) or 1 / (1 + exp(-l));  c = s + bias;  the k largest c of the kept groups (ties: the lowest index);
//   p = scaling * s, or normalised over the chosen: the softmax of the chosen logits, s / (sum of the chosen s + 1e-20) for sigmoid
//
// One warp per token.  Lane i holds the V neighbouring experts [i * V, i * V + V) in registers, so a row is read once, in
// 16-byte pieces, a lane's order is the experts' order, and a group of experts is a run of lanes.  A round of the selection is
// a warp maximum of order-preserving integer keys and a ballot for the first lane that has it.  Where a key has low bits to spare (16-bit
// logits; scores that are only nearly right, see below) an expert's place in its lane goes there, each lane sorts its keys once,
// two instructions an exchange, and the lane that lost its best moves the others up.
//
// What is compared: without bias and groups the logits themselves (both score functions are increasing), which is
// exact.  With them the choice hangs on sums of scores, and two experts a rounding apart would be taken in an order that depends on how
// exp was rounded: what counts are 64-bit scores.  They took 40 of 69 us for every row (16384 tokens, 256 experts in 8 groups), so a token's
// choice is first made from 32-bit scores, and made again in 64 bits only where two values that it hangs on are nearer to each
// other than their error.  Probabilities are 32-bit arithmetic.
#include "ptb_common.cuh"

namespace ptb {
namespace {

constexpr int kMaxTopk    = 32;   // chosen expert r lives in lane r
constexpr int kMaxExperts = 1024; // 32 lanes of 32
constexpr float kTiny     = 1e-20f;
constexpr int kRows       = 4;    // of a CTA

struct RouterArgs {
    const void *logits;
    int64_t T, row_stride;
    int E, k, groups, topk_groups;
    int softmax, normalize;
    float scaling;
    const float *bias;
    float *probs;   // [T, k], or
    float *table;   // [T, E] with
    uint8_t *map;   // [T, E]
    int64_t *ids;   // [T, k]
};

// Order-preserving keys.  0: not available (a logit of -inf).  NaN is the largest.  -0 and +0 are one value.
__device__ __forceinline__ uint32_t key_of(float v) {
    if (v != v) return 0xffffffffu;
    if (v == -INFINITY) return 0u;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(double v) {
    if (v != v) return ~0ull;
    const uint64_t u = (uint64_t) __double_as_longlong(v + 0.0);
    return u ^ ((u >> 63) ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ double value_of(uint64_t k) {
    return __longlong_as_double((long long) (k ^ ((k >> 63) ? 1ull << 63 : ~0ull)));
}

__device__ __forceinline__ uint32_t warp_max_key(uint32_t k) { return __reduce_max_sync(0xffffffffu, k); }
__device__ __forceinline__ uint64_t warp_max_key(uint64_t k) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t) (k >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t) (k >> 32) == hi ? (uint32_t) k : 0u);
    return (uint64_t) hi << 32 | lo;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The lane's V logits, -inf past the last expert.
template <typename T, int V> __device__ __forceinline__ void load_row(const T *row, int E, int first, bool vec, float (&l)[V]) {
    constexpr int kBytes = V * (int) sizeof(T);
    if (vec && first + V <= E) {
        if constexpr (kBytes >= 16) {
            uint4 u[kBytes / 16];
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) u[i] = reinterpret_cast<const uint4 *>(row + first)[i];
#pragma unroll
            for (int j = 0; j < V; ++j) l[j] = to_f32(reinterpret_cast<const T *>(u)[j]);
            return;
        } else if constexpr (kBytes == 8) {
            const uint2 u = *reinterpret_cast<const uint2 *>(row + first);
#pragma unroll
            for (int j = 0; j < V; ++j) l[j] = to_f32(reinterpret_cast<const T *>(&u)[j]);
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) l[j] = first + j < E ? to_f32(row[first + j]) : -INFINITY;
}

// Two largest keys of a pair of pairs.
template <typename K> __device__ __forceinline__ void merge_two(K &a, K &b, K c, K d) {
    const K hi = a > c ? a : c, lo = a > c ? c : a;
    const K b2 = a > c ? b : d;
    a = hi;
    b = lo > b2 ? lo : b2;
}

// Takes the k best of `key` (V a lane): the r-th ends in lane r as expert my_e; -1 once nothing is left.
template <typename K, int V> __device__ __forceinline__ void choose(K (&key)[V], int k, int lane, int first, int &my_e) {
    my_e   = -1;
    K best = 0;
    int at = 0;
    auto look = [&] {
        best = key[0]; at = 0;
#pragma unroll
        for (int j = 1; j < V; ++j)
            if (key[j] > best) { best = key[j]; at = j; }
    };
    look();
    for (int r = 0; r < k; ++r) {
        const K top = warp_max_key(best);
        if (top == 0) break;
        const int win = __ffs((int) __ballot_sync(0xffffffffu, best == top)) - 1;
        const int e   = __shfl_sync(0xffffffffu, first + at, win);
        if (lane == r) my_e = e;
        if (lane == win) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j == at) key[j] = 0;
            look();
        }
    }
}

// The groups with the largest `mine` (lane g has group g's), as bits.  kGap: false if the last that is kept and the first that is not are not
// further apart than `tol`.
template <typename K, bool kGap> __device__ __forceinline__ uint32_t best_groups(K mine, const RouterArgs &a, int lane, float tol, bool &clear) {
    uint32_t keep = 0;
    K before = 0;
    if (lane >= a.groups) mine = 0;
    for (int r = 0; r < a.topk_groups + (kGap ? 1 : 0); ++r) {
        const K best = warp_max_key(mine);
        if (best == 0) break;
        if (kGap && r == a.topk_groups) {
            clear = clear && value_of(before) - value_of(best) > tol;
            break;
        }
        before = best;
        const int win = __ffs((int) __ballot_sync(0xffffffffu, mine == best)) - 1;
        keep |= 1u << win;
        if (lane == win) mine = 0;
    }
    return keep;
}
// The key of the sum of a group's two largest.
template <typename K, typename F> __device__ __forceinline__ K group_score(K one, K two) {
    return one == 0 ? (K) 0 : key_of(two == 0 ? value_of(one) : (one == ~(K) 0 ? (F) NAN : value_of(one)) + value_of(two));
}

// ---- sorted lanes ----------------------------------------------------------------------------------------------------------------
// Keys with the expert's place in the lane in their low bits (the first place highest: ties go to it).
template <int V> struct Places {
    static constexpr uint32_t kMask = V - 1;
    static __device__ __forceinline__ uint32_t with(uint32_t key, int j) { return key == 0 ? 0u : (key & ~kMask) | (uint32_t) (V - 1 - j); }
    static __device__ __forceinline__ int of(uint32_t key) { return V - 1 - (int) (key & kMask); }
};
template <int V> __device__ __forceinline__ void sort_down(uint32_t (&key)[V]) { // odd-even merge sort
#pragma unroll
    for (int p = 1; p < V; p <<= 1)
#pragma unroll
        for (int q = p; q > 0; q >>= 1)
#pragma unroll
            for (int i = q % p; i + q < V; i += 2 * q)
#pragma unroll
                for (int j = 0; j < q; ++j)
                    if (i + j + q < V && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const uint32_t x = key[i + j], y = key[i + j + q];
                        key[i + j]     = max(x, y);
                        key[i + j + q] = min(x, y);
                    }
}
template <int V, bool kGap>
__device__ __forceinline__ bool choose_sorted(uint32_t (&key)[V], int k, int lane, int first, int &my_e, float tol) {
    constexpr uint32_t kMask = Places<V>::kMask;
    my_e            = -1;
    bool clear      = true;
    uint32_t before = 0;
    for (int r = 0; r < k + (kGap ? 1 : 0); ++r) {
        const uint32_t best = key[0] & ~kMask, top = warp_max_key(best);
        if (top == 0) break;
        if (kGap && r > 0) clear = clear && value_of(before) - value_of(top) > tol;
        before = top;
        if (r == k) break;
        const int win = __ffs((int) __ballot_sync(0xffffffffu, best == top)) - 1;
        const int e   = __shfl_sync(0xffffffffu, first + Places<V>::of(key[0]), win);
        if (lane == r) my_e = e;
        if (lane == win) {
#pragma unroll
            for (int j = 0; j + 1 < V; ++j) key[j] = key[j + 1];
            key[V - 1] = 0;
        }
    }
    return clear;
}
template <int V> __device__ __forceinline__ bool keep_groups_sorted(uint32_t (&key)[V], const RouterArgs &a, int lane, int first, float tol) {
    constexpr uint32_t kMask = Places<V>::kMask;
    const int size = a.E / a.groups, span = size / V; // span: lanes of a group
    bool clear = true;
    if (size % V == 0 && (span & (span - 1)) == 0) {
        uint32_t one = key[0] & ~kMask, two = V > 1 ? key[V > 1 ? 1 : 0] & ~kMask : 0u;
        for (int o = 1; o < span; o <<= 1) {
            const uint32_t p = __shfl_xor_sync(0xffffffffu, one, o), q = __shfl_xor_sync(0xffffffffu, two, o);
            merge_two<uint32_t>(one, two, p, q);
        }
        const uint32_t mine = __shfl_sync(0xffffffffu, group_score<uint32_t, float>(one, two), (lane * span) & 31);
        const uint32_t keep = best_groups<uint32_t, true>(mine, a, lane, tol, clear);
        if (!(keep >> (first < a.E ? first / size : 0) & 1))
#pragma unroll
            for (int j = 0; j < V; ++j) key[j] = 0;
        return clear;
    }
    uint32_t mine = 0;
    for (int g = 0; g < a.groups; ++g) {
        uint32_t one = 0, two = 0;
#pragma unroll
        for (int j = 0; j < V; ++j)
            if ((first + Places<V>::of(key[j])) / size == g) merge_two<uint32_t>(one, two, key[j] & ~kMask, 0u);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t p = __shfl_xor_sync(0xffffffffu, one, o), q = __shfl_xor_sync(0xffffffffu, two, o);
            merge_two<uint32_t>(one, two, p, q);
        }
        if (lane == g) mine = group_score<uint32_t, float>(one, two);
    }
    const uint32_t keep = best_groups<uint32_t, true>(mine, a, lane, tol, clear);
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (key[j] != 0 && !(keep >> ((first + Places<V>::of(key[j])) / size) & 1)) key[j] = 0;
    sort_down<V>(key);
    return clear;
}

// The lane's experts' biases.
template <int V> __device__ __forceinline__ void load_bias(const RouterArgs &a, int first, float (&b)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) b[j] = a.bias != nullptr && first + j < a.E ? a.bias[first + j] : 0.0f;
}

// The choice from 64-bit scores.  Few rows need it, and the last of them end the kernel: what counts is how long one takes, so a lane's
// exps run side by side as far as registers reach.
template <typename T, int V> __device__ __noinline__ int choose_wide(const T *row, const RouterArgs &a, int lane, bool vec) {
    constexpr int kSide = V <= 8 ? V : 1;
    const int first     = lane * V;
    float l[V], b[V];
    load_row<T, V>(row, a.E, first, vec, l);
    load_bias<V>(a, first, b);
    double c[V], z = 0.0;
    float top = l[0];
#pragma unroll
    for (int j = 1; j < V; ++j) top = fmaxf(top, l[j]);
    top = a.softmax ? warp_max(top) : 0.0f;
#pragma unroll kSide
    for (int j = 0; j < V; ++j) {
        const double x = (double) l[j] - (double) top;
        c[j]           = l[j] == -INFINITY ? 0.0 : exp(a.softmax ? x : -x);
        z += c[j];
    }
    if (a.softmax) z = warp_sum(z);
    uint64_t key[V];
#pragma unroll kSide
    for (int j = 0; j < V; ++j) {
        const double s = a.softmax ? c[j] / z : 1.0 / (1.0 + c[j]);
        key[j]         = l[j] == -INFINITY ? 0ull : key_of(s + (double) b[j]);
    }
    if (a.groups > a.topk_groups) {
        const int size = a.E / a.groups, span = size / V;
        uint64_t mine  = 0;
        bool clear     = true;
        if (size % V == 0 && (span & (span - 1)) == 0) { // a group: span lanes
            uint64_t one = 0, two = 0;
#pragma unroll kSide
            for (int j = 0; j < V; ++j) merge_two<uint64_t>(one, two, key[j], 0ull);
            for (int o = 1; o < span; o <<= 1) {
                const uint64_t p = __shfl_xor_sync(0xffffffffu, one, o), q = __shfl_xor_sync(0xffffffffu, two, o);
                merge_two<uint64_t>(one, two, p, q);
            }
            mine = __shfl_sync(0xffffffffu, group_score<uint64_t, double>(one, two), (lane * span) & 31);
        } else {
            for (int g = 0; g < a.groups; ++g) {
                uint64_t one = 0, two = 0;
#pragma unroll kSide
                for (int j = 0; j < V; ++j)
                    if ((first + j) / size == g) merge_two<uint64_t>(one, two, key[j], 0ull);
                for (int o = 1; o < 32; o <<= 1) {
                    const uint64_t p = __shfl_xor_sync(0xffffffffu, one, o), q = __shfl_xor_sync(0xffffffffu, two, o);
                    merge_two<uint64_t>(one, two, p, q);
                }
                if (lane == g) mine = group_score<uint64_t, double>(one, two);
            }
        }
        const uint32_t keep = best_groups<uint64_t, false>(mine, a, lane, 0.0f, clear);
#pragma unroll kSide
        for (int j = 0; j < V; ++j)
            if (first + j < a.E && !(keep >> ((first + j) / size) & 1)) key[j] = 0;
    }
    int my_e;
    choose<uint64_t, V>(key, a.k, lane, first, my_e);
    return my_e;
}

// Bound by instructions (1300 a row, 76 % of issue slots) and by the latency of the selection's rounds, so by how many warps an SM holds: 16384 tokens, 256 experts, 4 of 8 groups, fp32,
// with the backward pass: 40.3, 39.1 and 40.8 us for 32, 40 and 48 warps (the last spill), 49.7 with no limit.
template <typename T, int V, bool kWide>
__global__ void __launch_bounds__(kRows * 32, V <= 8 ? 40 / kRows : 4) router_kernel(const __grid_constant__ RouterArgs a) {
    grid_dep_begin();
    const int lane  = threadIdx.x & 31;
    const int64_t t = (int64_t) blockIdx.x * kRows + (threadIdx.x >> 5);
    if (t >= a.T) return;
    const int E = a.E, first = lane * V;
    const T *row = (const T *) a.logits + t * a.row_stride;
    const bool vec = (reinterpret_cast<uintptr_t>(a.logits) | (uintptr_t) (a.row_stride * (int64_t) sizeof(T))) % (V * sizeof(T) >= 16 ? 16 : 8) == 0;
    float l[V];
    load_row<T, V>(row, E, first, vec, l);

    float top = l[0];
#pragma unroll
    for (int j = 1; j < V; ++j) top = fmaxf(top, l[j]);
    top = warp_max(top); // NaN is passed over here and comes back through the sums

    int my_e;
    if constexpr (!kWide) {
        uint32_t key[V];
        if constexpr (sizeof(T) == 2) { // the logits' own low bits are all alike
#pragma unroll
            for (int j = 0; j < V; ++j) key[j] = Places<V>::with(key_of(l[j]), j);
            sort_down<V>(key);
            choose_sorted<V, false>(key, a.k, lane, first, my_e, 0.0f);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) key[j] = key_of(l[j]);
            choose<uint32_t, V>(key, a.k, lane, first, my_e);
        }
    } else {
        // 32-bit scores, fast and nearly right.  Of w, the largest score and bias, in units u = 2^-23 w: the fast exp is within 2 + 1.2 |x| units of
        // its last place.  Softmax: exp(x) (2 + 1.7 |x|), x <= 0 (itself rounded), is largest at 0, so a score is off by 2 u, the sum that divides
        // all alike left aside, and 1 for the product.  Sigmoid, s = 1 / (1 + exp(-x)): s ((2 + 1.2 |x|) (1 - s) + 2.5) is below 5 u where the
        // largest logit is 0 or more (w is 1/2 at least), and below (5 + 1.2 |x|) u with x the largest logit where it is less, since s is about
        // exp(x) and w may be no more.  Adding the bias 1/2 u; the low bits that are given away V u.  So two scores further apart than
        // 11 u + 2 V u + 2.4 |x| u are in their right order: tol is more.  Below exp(-64) the quotient comes near its smallest numbers.
        float c[V], b[V], widest = 0.0f;
        load_bias<V>(a, first, b);
        float z = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            c[j] = l[j] == -INFINITY ? 0.0f : a.softmax ? __expf(l[j] - top) : __fdividef(1.0f, 1.0f + __expf(-l[j]));
            z += c[j];
        }
        if (a.softmax) z = __fdiv_rn(1.0f, warp_sum(z));
        uint32_t key[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float s = a.softmax ? c[j] * z : c[j];
            widest        = fmaxf(widest, s + fabsf(b[j]));
            key[j]        = l[j] == -INFINITY ? 0u : Places<V>::with(key_of(s + b[j]), j);
        }
        sort_down<V>(key);
        const float below = a.softmax || top >= 0.0f || top == -INFINITY ? 0.0f : -top; // (of a row of nothing no score is compared)
        const float tol   = warp_max(widest) * (0x1p-18f + V * 0x1p-22f + below * 0x1p-21f);
        bool clear = tol < INFINITY && below <= 64.0f;
        if (a.groups > a.topk_groups) clear = keep_groups_sorted<V>(key, a, lane, first, 2.0f * tol) && clear;
        clear = choose_sorted<V, true>(key, a.k, lane, first, my_e, tol) && clear;
        if (!clear) my_e = choose_wide<T, V>(row, a, lane, vec); // (one answer for the warp)
    }
    const float my_l = my_e < 0 ? -INFINITY : to_f32(row[my_e]);

    // probabilities, lane r the r-th chosen expert's
    float p = 0.0f;
    if (a.softmax) {
        // normalised over the chosen, a softmax is the softmax of their logits alone
        const float ref = a.normalize ? warp_max(my_l) : top;
        const float e   = my_e < 0 ? 0.0f : expf(my_l - ref);
        float z = e;
        if (!a.normalize) {
            z = 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) z += l[j] == -INFINITY ? 0.0f : expf(l[j] - ref);
        }
        z = warp_sum(z);
        p = my_e < 0 ? 0.0f : __fdiv_rn(e, z);
    } else {
        p = my_e < 0 ? 0.0f : __fdiv_rn(1.0f, 1.0f + expf(-my_l));
        if (a.normalize) {
            const float sum = warp_sum(p) + kTiny;
            p = __fdiv_rn(p, sum);
        }
    }
    p *= a.scaling;
    if (my_e < 0) p = 0.0f;
    if (lane < a.k) {
        a.ids[t * a.k + lane] = my_e;
        if (a.probs != nullptr) a.probs[t * a.k + lane] = p;
    }
    if (a.table != nullptr) {
        // zeros first, then the chosen experts over them
        float *out     = a.table + t * E;
        uint8_t *flags = a.map + t * E;
        if (E % V == 0 && V % 4 == 0) { // rows of the tables start on V elements, and so do the lanes
            if (first < E) {
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    *reinterpret_cast<float4 *>(out + first + j)     = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    *reinterpret_cast<uint32_t *>(flags + first + j) = 0;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (first + j < E) { out[first + j] = 0.0f; flags[first + j] = 0; }
        }
        __syncwarp();
        if (my_e >= 0) { out[my_e] = p; flags[my_e] = 1; }
    }
}

struct RouterBwdArgs {
    const void *logits;
    int64_t T, row_stride;
    int E, k, softmax, normalize, dense; // dense: grad is [T, E], otherwise [T, k]
    float scaling;
    const int64_t *ids;
    const float *grad;
    int64_t grad_stride;
    void *grad_logits; // [T, E]
};

// dl from dp, g = scaling * dp.  Softmax over all: dl_e = s_e (g_e - sum g s), g = 0 for the others; over the chosen: the same among
// them, and nothing for the others.  Sigmoid: dl_i = s_i (1 - s_i) ds_i with ds_i = g_i, or normalised, D = sum s + 1e-20:
// ds_i = (g_i - sum g s / D) / D.  Only the softmax over all reads the whole row again.
template <typename T, int V>
__global__ void __launch_bounds__(kRows * 32) router_bwd_kernel(const RouterBwdArgs a) {
    grid_dep_begin();
    const int lane  = threadIdx.x & 31;
    const int64_t t = (int64_t) blockIdx.x * kRows + (threadIdx.x >> 5);
    if (t >= a.T) return;
    const int E = a.E, first = lane * V;
    const T *row = (const T *) a.logits + t * a.row_stride;
    const int e  = lane < a.k ? (int) a.ids[t * a.k + lane] : -1;
    float g = 0.0f, x = -INFINITY;
    if (e >= 0) {
        g = a.grad[t * a.grad_stride + (a.dense ? e : lane)] * a.scaling;
        x = to_f32(row[e]);
    }
    float d[V];
    float v; // the chosen expert's gradient
    if (a.softmax && !a.normalize) {
        float l[V];
        const bool vec = (reinterpret_cast<uintptr_t>(a.logits) | (uintptr_t) (a.row_stride * (int64_t) sizeof(T))) % (V * sizeof(T) >= 16 ? 16 : 8) == 0;
        load_row<T, V>(row, E, first, vec, l);
        float top = l[0];
#pragma unroll
        for (int j = 1; j < V; ++j) top = fmaxf(top, l[j]);
        top = warp_max(top);
        float z = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            d[j] = l[j] == -INFINITY ? 0.0f : expf(l[j] - top);
            z += d[j];
        }
        z = warp_sum(z);
        const float s   = e < 0 ? 0.0f : __fdiv_rn(expf(x - top), z);
        const float dot = warp_sum(g * s);
        const float c   = z > 0.0f || z != z ? __fdiv_rn(-dot, z) : 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] *= c;
        v = s * (g - dot);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = 0.0f;
        if (a.softmax) {
            const float top = warp_max(x);
            const float w   = e < 0 ? 0.0f : expf(x - top);
            const float sum = warp_sum(w); // every lane takes part in a sum, chosen or not
            const float s   = e < 0 ? 0.0f : __fdiv_rn(w, sum);
            const float dot = warp_sum(g * s);
            v = s * (g - dot);
        } else {
            const float u = e < 0 ? 0.0f : expf(-fabsf(x)); // s and 1 - s without cancellation
            const float big = __fdiv_rn(1.0f, 1.0f + u), small = __fdiv_rn(u, 1.0f + u);
            const float s = e < 0 ? 0.0f : (x >= 0.0f ? big : x < 0.0f ? small : x), s1 = x >= 0.0f ? small : big;
            if (a.normalize) {
                const float D = warp_sum(s) + kTiny;
                g = __fdiv_rn(g - __fdiv_rn(warp_sum(g * s), D), D);
            }
            v = g * s * s1;
        }
        if (e < 0) v = 0.0f;
    }
    T *out = (T *) a.grad_logits + t * E;
    constexpr int kBytes = V * (int) sizeof(T);
    if (kBytes >= 8 && E % V == 0) {
        if (first < E) {
            T r[V];
#pragma unroll
            for (int j = 0; j < V; ++j) r[j] = from_f32<T>(d[j]);
            if constexpr (kBytes >= 16) {
#pragma unroll
                for (int i = 0; i < kBytes / 16; ++i) {
                    uint4 w;
                    memcpy(&w, r + i * (16 / (int) sizeof(T)), 16);
                    reinterpret_cast<uint4 *>(out + first)[i] = w;
                }
            } else if constexpr (kBytes == 8) {
                uint2 w;
                memcpy(&w, r, 8);
                *reinterpret_cast<uint2 *>(out + first) = w;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (first + j < E) out[first + j] = from_f32<T>(d[j]);
    }
    __syncwarp();
    if (e >= 0) out[e] = from_f32<T>(v); // over the row
}

#define PTB_SWITCH_LANE_EXPERTS(E, V, ...)                    \
    if ((E) <= 32) { constexpr int V = 1; __VA_ARGS__; }      \
    else if ((E) <= 64) { constexpr int V = 2; __VA_ARGS__; } \
    else if ((E) <= 128) { constexpr int V = 4; __VA_ARGS__; }\
    else if ((E) <= 256) { constexpr int V = 8; __VA_ARGS__; }\
    else if ((E) <= 512) { constexpr int V = 16; __VA_ARGS__; }\
    else { constexpr int V = 32; __VA_ARGS__; }

int check_shape(const char *who, int64_t T, int64_t E, int64_t row_stride, int64_t k, int score_function) {
    PTB_REQUIRE(T >= 0 && E >= 1 && k >= 1 && k <= E, PTB_ERR_ARG, "%s: bad sizes", who);
    PTB_REQUIRE(E <= kMaxExperts, PTB_ERR_TOO_LARGE, "%s: more than %d experts", who, kMaxExperts);
    PTB_REQUIRE(k <= kMaxTopk, PTB_ERR_TOO_LARGE, "%s: more than %d experts per token", who, kMaxTopk);
    PTB_REQUIRE(T <= kRows * 2147483647ll, PTB_ERR_TOO_LARGE, "%s: too many tokens", who);
    PTB_REQUIRE(T <= 1 || row_stride >= E, PTB_ERR_ARG, "%s: rows overlap", who);
    PTB_REQUIRE(score_function == PTB_SCORE_SOFTMAX || score_function == PTB_SCORE_SIGMOID, PTB_ERR_ARG, "%s: unknown score function %d", who, score_function);
    return 0;
}

} // namespace
} // namespace ptb

using namespace ptb;

extern "C" {
#pragma GCC visibility push(default)

int ptb_topk_router(const void *logits, int dtype, int64_t T, int64_t E, int64_t row_stride, int64_t k, int score_function,
                    const float *bias, int64_t groups, int64_t topk_groups, int normalize, float scaling, int64_t *ids,
                    float *probs, float *table, void *map, ptb_stream_t stream) {
    if (int rc = check_shape("topk_router", T, E, row_stride, k, score_function)) return rc;
    PTB_REQUIRE(is_hp(dtype), PTB_ERR_ARG, "topk_router: logits must be fp32, fp16 or bf16");
    PTB_REQUIRE(groups >= 1 && groups <= 32 && E % groups == 0, PTB_ERR_ARG, "topk_router: groups must divide the experts, 32 at most");
    PTB_REQUIRE(topk_groups >= 1 && topk_groups <= groups, PTB_ERR_ARG, "topk_router: bad number of kept groups");
    PTB_REQUIRE(k <= E / groups * topk_groups, PTB_ERR_ARG, "topk_router: the kept groups have fewer than k experts");
    if (T == 0) return 0;
    PTB_REQUIRE(logits && ids && (probs || table), PTB_ERR_ARG, "topk_router: null pointer");
    PTB_REQUIRE((table == nullptr) == (map == nullptr), PTB_ERR_ARG, "topk_router: the table and the map come together");
    PTB_REQUIRE(aligned16(table) && aligned16(map), PTB_ERR_ALIGN, "topk_router: the table and the map must be 16-byte aligned");
    const RouterArgs a{logits, T, row_stride, (int) E, (int) k, (int) groups, (int) topk_groups, score_function == PTB_SCORE_SOFTMAX,
                       normalize != 0, scaling, bias, probs, table, (uint8_t *) map, ids};
    const dim3 grid((unsigned) cdiv<int64_t>(T, kRows));
    const bool wide = bias != nullptr || (groups > 1 && topk_groups < groups);
    PTB_SWITCH_HP(dtype, X, PTB_SWITCH_LANE_EXPERTS(E, V, {
        if (wide)
            PTB_CUDA(launch_after(router_kernel<X, V, true>, grid, kRows * 32, 0, (cudaStream_t) stream, 1, a));
        else
            PTB_CUDA(launch_after(router_kernel<X, V, false>, grid, kRows * 32, 0, (cudaStream_t) stream, 1, a));
    }));
    PTB_LAUNCH_CHECK("router_kernel");
    return 0;
}

int ptb_topk_router_bwd(const void *logits, int dtype, int64_t T, int64_t E, int64_t row_stride, int64_t k, int score_function,
                        int normalize, float scaling, const int64_t *ids, const float *grad, int64_t grad_stride, int dense,
                        void *grad_logits, ptb_stream_t stream) {
    if (int rc = check_shape("topk_router_bwd", T, E, row_stride, k, score_function)) return rc;
    PTB_REQUIRE(is_hp(dtype), PTB_ERR_ARG, "topk_router_bwd: logits must be fp32, fp16 or bf16");
    if (T == 0) return 0;
    PTB_REQUIRE(logits && ids && grad && grad_logits, PTB_ERR_ARG, "topk_router_bwd: null pointer");
    PTB_REQUIRE(aligned16(grad_logits), PTB_ERR_ALIGN, "topk_router_bwd: the gradient must be 16-byte aligned");
    const RouterBwdArgs a{logits, T, row_stride, (int) E, (int) k, score_function == PTB_SCORE_SOFTMAX, normalize != 0, dense != 0,
                          scaling, ids, grad, grad_stride, grad_logits};
    const dim3 grid((unsigned) cdiv<int64_t>(T, kRows));
    PTB_SWITCH_HP(dtype, X, PTB_SWITCH_LANE_EXPERTS(E, V, {
        PTB_CUDA(launch_after(router_bwd_kernel<X, V>, grid, kRows * 32, 0, (cudaStream_t) stream, 1, a));
    }));
    PTB_LAUNCH_CHECK("router_bwd_kernel");
    return 0;
}

#pragma GCC visibility pop
} // extern "C"
