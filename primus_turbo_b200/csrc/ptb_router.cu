// Top-k routing of a mixture-of-experts layer, and its gradient.
//
//   s = softmax(l) or 1 / (1 + exp(-l));  c = s + bias;  the k largest c of the kept groups (ties: the lowest index);
//   p = scaling * s, or normalised over the chosen: the softmax of the chosen logits, s / (sum of the chosen s + 1e-20) for sigmoid
//
// One warp per token.  Lane i holds the V neighbouring experts [i * V, i * V + V) in registers, so a row is read once, in
// 16-byte pieces, a lane's order is the experts' order, and a group of experts is a run of lanes.  A round of the selection is
// a warp maximum of order-preserving integer keys and a ballot for the first lane that has it; only the lane that lost its best
// expert looks for its next one.
//
// What is compared: without bias and groups the logits themselves (both score functions are increasing), which is
// exact.  With them the choice hangs on sums of scores, and two experts a rounding apart would be taken in an order that
// depends on how exp was rounded: those scores are computed in 64 bits.  Probabilities are 32-bit arithmetic.
#include "ptb_common.cuh"

namespace ptb {
namespace {

constexpr int kMaxTopk    = 32;   // chosen expert r lives in lane r
constexpr int kMaxExperts = 1024; // 32 lanes of 32
constexpr float kTiny     = 1e-20f;

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
__device__ __forceinline__ void merge_two(uint64_t &a, uint64_t &b, uint64_t c, uint64_t d) {
    const uint64_t hi = a > c ? a : c, lo = a > c ? c : a;
    const uint64_t b2 = a > c ? b : d;
    a = hi;
    b = lo > b2 ? lo : b2;
}

// Takes the k best of `key` (V a lane): chosen[r] ends in lane r as (expert, its logit); -1 once nothing is left.
template <typename K, int V>
__device__ __forceinline__ void choose(K (&key)[V], const float (&l)[V], int k, int lane, int first, int &my_e, float &my_l) {
    my_e = -1;
    my_l = -INFINITY;
    K best  = 0;
    int at  = 0;
    float v = -INFINITY;
    auto look = [&] {
        best = key[0]; at = 0; v = l[0];
#pragma unroll
        for (int j = 1; j < V; ++j)
            if (key[j] > best) { best = key[j]; at = j; v = l[j]; }
    };
    look();
    for (int r = 0; r < k; ++r) {
        const K top = warp_max_key(best);
        if (top == 0) break;
        const int win = __ffs((int) __ballot_sync(0xffffffffu, best == top)) - 1;
        const int e   = __shfl_sync(0xffffffffu, first + at, win);
        const float x = __shfl_sync(0xffffffffu, v, win);
        if (lane == r) { my_e = e; my_l = x; }
        if (lane == win) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j == at) key[j] = 0;
            look();
        }
    }
}

template <typename T, int V, bool kWide>
__global__ void __launch_bounds__(256) router_kernel(const RouterArgs a) {
    grid_dep_begin();
    const int lane  = threadIdx.x & 31;
    const int64_t t = (int64_t) blockIdx.x * 8 + (threadIdx.x >> 5);
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
    float my_l;
    if constexpr (!kWide) {
        uint32_t key[V];
#pragma unroll
        for (int j = 0; j < V; ++j) key[j] = key_of(l[j]);
        choose<uint32_t, V>(key, l, a.k, lane, first, my_e, my_l);
    } else {
        double c[V];
        if (a.softmax) {
            double z = 0.0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                c[j] = l[j] == -INFINITY ? 0.0 : exp((double) l[j] - (double) top);
                z += c[j];
            }
            z = warp_sum(z);
#pragma unroll
            for (int j = 0; j < V; ++j) c[j] = c[j] / z;
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) c[j] = 1.0 / (1.0 + exp(-(double) l[j]));
        }
        uint64_t key[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (a.bias != nullptr && first + j < E) c[j] += (double) a.bias[first + j];
            key[j] = l[j] == -INFINITY ? 0ull : key_of(c[j]);
        }
        if (a.groups > 1) {
            const int size = E / a.groups;
            uint64_t mine = 0; // lane g: the sum of group g's two largest
            auto score = [](uint64_t one, uint64_t two) {
                return one == 0 ? 0ull : key_of(two == 0 ? value_of(one) : (one == ~0ull ? NAN : value_of(one)) + value_of(two));
            };
            const int span = size / V; // lanes of a group
            if (size % V == 0 && (span & (span - 1)) == 0) {
                uint64_t one = 0, two = 0;
#pragma unroll
                for (int j = 0; j < V; ++j) merge_two(one, two, key[j], 0ull);
                for (int o = 1; o < span; o <<= 1) {
                    const uint64_t p = __shfl_xor_sync(0xffffffffu, one, o), q = __shfl_xor_sync(0xffffffffu, two, o);
                    merge_two(one, two, p, q);
                }
                mine = __shfl_sync(0xffffffffu, score(one, two), (lane * span) & 31);
            } else {
                for (int g = 0; g < a.groups; ++g) {
                    uint64_t one = 0, two = 0;
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if ((first + j) / size == g) merge_two(one, two, key[j], 0ull);
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const uint64_t p = __shfl_xor_sync(0xffffffffu, one, o), q = __shfl_xor_sync(0xffffffffu, two, o);
                        merge_two(one, two, p, q);
                    }
                    if (lane == g) mine = score(one, two);
                }
            }
            if (lane >= a.groups) mine = 0;
            uint32_t keep = 0;
            for (int r = 0; r < a.topk_groups; ++r) {
                const uint64_t best = warp_max_key(mine);
                if (best == 0) break;
                const int win = __ffs((int) __ballot_sync(0xffffffffu, mine == best)) - 1;
                keep |= 1u << win;
                if (lane == win) mine = 0;
            }
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (first + j < E && !(keep >> ((first + j) / size) & 1)) key[j] = 0;
        }
        choose<uint64_t, V>(key, l, a.k, lane, first, my_e, my_l);
    }

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
        float d[V];
        uint32_t on = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = 0.0f;
        for (int r = 0; r < a.k; ++r) {
            const int e   = __shfl_sync(0xffffffffu, my_e, r) - first;
            const float v = __shfl_sync(0xffffffffu, p, r);
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (e == j) { d[j] = v; on |= 1u << j; }
        }
        float *out     = a.table + t * E;
        uint8_t *flags = a.map + t * E;
        if (E % V == 0 && V % 4 == 0) { // rows of the tables start on V elements, and so do the lanes
            if (first < E) {
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    *reinterpret_cast<float4 *>(out + first + j) = make_float4(d[j], d[(j + 1) % V], d[(j + 2) % V], d[(j + 3) % V]);
                    const uint32_t b = on >> j & 15;
                    *reinterpret_cast<uint32_t *>(flags + first + j) = (b & 1) | (b & 2) << 7 | (b & 4) << 14 | (b & 8) << 21;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (first + j < E) { out[first + j] = d[j]; flags[first + j] = on >> j & 1; }
        }
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
__global__ void __launch_bounds__(256) router_bwd_kernel(const RouterBwdArgs a) {
    grid_dep_begin();
    const int lane  = threadIdx.x & 31;
    const int64_t t = (int64_t) blockIdx.x * 8 + (threadIdx.x >> 5);
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
    float v; // the chosen expert's gradient (added to the row's)
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
        v = g * s;
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
    for (int r = 0; r < a.k; ++r) {
        const int at   = __shfl_sync(0xffffffffu, e, r) - first;
        const float dv = __shfl_sync(0xffffffffu, v, r);
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (at == j) d[j] += dv;
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
    PTB_REQUIRE(T <= 8ll * 2147483647ll, PTB_ERR_TOO_LARGE, "%s: too many tokens", who);
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
    const dim3 grid((unsigned) cdiv<int64_t>(T, 8));
    const bool wide = bias != nullptr || (groups > 1 && topk_groups < groups);
    PTB_SWITCH_HP(dtype, X, PTB_SWITCH_LANE_EXPERTS(E, V, {
        if (wide)
            PTB_CUDA(launch_after(router_kernel<X, V, true>, grid, 256, 0, (cudaStream_t) stream, 1, a));
        else
            PTB_CUDA(launch_after(router_kernel<X, V, false>, grid, 256, 0, (cudaStream_t) stream, 1, a));
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
    const dim3 grid((unsigned) cdiv<int64_t>(T, 8));
    PTB_SWITCH_HP(dtype, X, PTB_SWITCH_LANE_EXPERTS(E, V, {
        PTB_CUDA(launch_after(router_bwd_kernel<X, V>, grid, 256, 0, (cudaStream_t) stream, 1, a));
    }));
    PTB_LAUNCH_CHECK("router_bwd_kernel");
    return 0;
}

#pragma GCC visibility pop
} // extern "C"
