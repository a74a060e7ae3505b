// A mixture-of-experts feed-forward layer for a few tokens:
//   y[t] = sum_j p[t, j] * W2[e] (silu(W1[e] x_t, first half) * (W1[e] x_t, second half)),  e = ids[t, j]
// from weights as they are kept: 16-bit, FP8 with inverse scales, or 4-bit groups.
//
// Three kernels: a list of the experts that are hit and their tokens, gate + up projection with the activation, down projection
// with the weighted sum over a token's experts.  What bounds them is reading the weights of the experts that are hit, once.
//
//  * moe_gate_up_kernel: one CTA per eight channels of one hit expert: the 16 rows of its MMAs are eight gate rows and the eight up
//    rows that go with them, so both halves of a channel meet in one lane and the activation needs no exchange.  Its warps share k.
//  * moe_down_kernel: one CTA per 16 output columns, over all experts that are hit: its warps share the list of (expert, block of k)
//    and keep one 32-bit sum per token and column each, added up in a fixed order at the end.  Nothing is added in memory, so no
//    atomics, no second pass, and the same result every time.
//
// The activation h between the two is kept as a sum of two bf16 (16 bits of mantissa): its rounding is not felt in the result, and
// the second MMA costs nothing next to the weights.
#include "ptb_few_rows.cuh"

namespace ptb {
namespace {

constexpr int kMaxTokens  = PTB_MOE_FEW_MAX_TOKENS;
constexpr int kMaxPairs   = PTB_MOE_FEW_MAX_PAIRS;
constexpr int kMaxExperts = 1024;

// One expert-major weight [E, rows, K].
struct ExpertWeight {
    const uint8_t *data;
    int64_t row_bytes, expert_bytes;
    const void *scale; // fp32 (8-bit) or bf16 (4-bit)
    const uint8_t *zero;
    int64_t scale_expert; // elements from expert to expert
    int scale_row, scale_k, row_shift; // 8-bit: row r, block b at (r >> row_shift) * scale_row + b * scale_k
    int groups; // 4-bit: scales a row
};

template <int FMT> __device__ __forceinline__ RowScale<FMT> row_scale(const ExpertWeight &w, int64_t e, int row, int rows) {
    RowScale<FMT> r{};
    if constexpr (FMT == kWInt4) {
        const int64_t at = (e * rows + row) * w.groups;
        r.s4    = (const __nv_bfloat16 *) w.scale + at;
        r.z4    = w.zero != nullptr ? w.zero + at : nullptr;
        r.count = w.groups;
    } else if constexpr (FMT != kW16) {
        r.s8     = (const float *) w.scale + e * w.scale_expert + (int64_t) (row >> w.row_shift) * w.scale_row;
        r.stride = w.scale_k;
    }
    return r;
}

// What the list kernel leaves for the others (in the workspace).  A slot is one (expert, token) pair, expert-major, tokens in order.
struct Lists {
    int *active;     // [0]: how many experts are hit; [1 + a]: the a-th of them, in increasing order
    int *first;      // [a]: its first slot; [number hit]: slots in all
    int *token;      // of a slot
    float *prob;     // of a slot
};
__host__ __device__ inline int64_t list_words(int64_t pairs) { return 1 + pairs + (pairs + 1) + pairs + pairs; }
__host__ __device__ inline Lists lists_at(void *ws, int64_t pairs) {
    int *p = (int *) ws;
    return {p, p + 1 + pairs, p + 2 + 2 * pairs, (float *) (p + 2 + 3 * pairs)};
}

// A token that names an expert twice has one slot with the sum of the two probabilities.  Ids outside [0, E) have none.
__global__ void __launch_bounds__(1024) moe_list_kernel(const int64_t *ids, const float *probs, int T, int k, int E, Lists out) {
    grid_dep_begin();
    __shared__ int count[kMaxExperts];
    __shared__ short id[kMaxPairs];
    __shared__ int warp_hit[32], warp_slots[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = T * k;
    count[tid] = 0;
    int mine = -1;
    if (tid < n) {
        const int64_t e = ids[tid];
        mine = e >= 0 && e < E ? (int) e : -1;
        id[tid] = (short) mine;
    }
    __syncthreads();
    float p = 0.0f;
    if (mine >= 0) {
        const int row = tid / k * k;
        p = probs[tid];
        for (int j = row; j < row + k; ++j)
            if (j != tid && id[j] == mine) {
                if (j < tid) { mine = -1; break; } // counted with the earlier one
                p += probs[j];
            }
        if (mine >= 0) atomicAdd(&count[mine], 1);
    }
    __syncthreads();
    // thread e: where expert e's slots start, and its place among those that are hit
    const int c = count[tid];
    int hit = c > 0, slots = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int h = __shfl_up_sync(0xffffffffu, hit, o), s = __shfl_up_sync(0xffffffffu, slots, o);
        if (lane >= o) { hit += h; slots += s; }
    }
    if (lane == 31) { warp_hit[warp] = hit; warp_slots[warp] = slots; }
    __syncthreads();
    int hit0 = 0, slots0 = 0;
    for (int w = 0; w < warp; ++w) { hit0 += warp_hit[w]; slots0 += warp_slots[w]; }
    hit += hit0;
    slots += slots0;
    if (c > 0) {
        out.active[hit] = tid; // hit counts from one here
        out.first[hit - 1] = slots - c;
    }
    if (tid == 1023) {
        out.active[0] = hit;
        out.first[hit] = slots;
    }
    count[tid] = slots - c; // from now on the next free slot
    // pairs in order, 32 at a time: lanes with the same expert take neighbouring slots
    __shared__ short own[kMaxPairs];
    __shared__ float prob[kMaxPairs];
    if (tid < n) { own[tid] = (short) mine; prob[tid] = p; }
    __syncthreads();
    if (warp != 0) return;
    for (int base = 0; base < n; base += 32) {
        const int i = base + lane, e = i < n ? own[i] : -1;
        const unsigned same = __match_any_sync(0xffffffffu, e);
        if (e >= 0) {
            const int slot  = count[e] + __popc(same & ((1u << lane) - 1));
            out.token[slot] = i / k;
            out.prob[slot]  = prob[i];
        }
        __syncwarp();
        if (e >= 0 && (same >> lane) == 1u) count[e] += __popc(same); // the last lane of each expert
        __syncwarp();
    }
}

struct GateUpArgs {
    const void *x;
    int64_t ldx;
    int H, I;
    ExpertWeight w;
    Lists lists;
    __nv_bfloat16 *h_hi, *h_lo; // [slots, I]
};

constexpr int kGateUpWarps = 8;

template <typename T, int FMT, int G, int NT>
__global__ void __launch_bounds__(32 * kGateUpWarps) moe_gate_up_kernel(const GateUpArgs a) {
    grid_dep_begin();
    const int hit = blockIdx.y;
    if (hit >= a.lists.active[0]) return;
    __shared__ float part[kGateUpWarps][NT * 8][17];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int r0 = blockIdx.x * 8, row = min(r0 + g, a.I - 1);
    const int64_t e = a.lists.active[1 + hit];
    const int begin = a.lists.first[hit], end = a.lists.first[hit + 1];
    const uint8_t *wa = a.w.data + e * a.w.expert_bytes + row * a.w.row_bytes, *wb = wa + (int64_t) a.I * a.w.row_bytes;
    const RowScale<FMT> sa = row_scale<FMT>(a.w, e, row, 2 * a.I), sb = row_scale<FMT>(a.w, e, a.I + row, 2 * a.I);
    const int blocks = (a.H + kKB - 1) / kKB;
    constexpr int kAhead = FMT == kWInt4 ? 4 : FMT == kW16 ? 1 : 2;
    for (int s0 = begin; s0 < end; s0 += NT * 8) {
        const T *x[NT];
        bool live[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int s = s0 + i * 8 + g;
            live[i]     = s < end;
            x[i]        = (const T *) a.x + (live[i] ? a.lists.token[s] : 0) * a.ldx;
        }
        float acc[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
        for (int kb = warp; kb < blocks; kb += kGateUpWarps * kAhead) {
            RowPiece<FMT> pa[kAhead], pb[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (kb + u * kGateUpWarps < blocks) {
                    pa[u].load(wa, kb + u * kGateUpWarps, t, a.H);
                    pb[u].load(wb, kb + u * kGateUpWarps, t, a.H);
                }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int b = kb + u * kGateUpWarps;
                if (b < blocks)
                    few_rows_block<T, FMT, G, NT, 1>(acc, b, pa[u], pb[u], sa, sb, [&](int i, int q, int) {
                        const int k = b * kKB + octet_k<FMT>(q, t);
                        return live[i] && k < a.H ? *reinterpret_cast<const uint4 *>(x[i] + k) : make_uint4(0, 0, 0, 0);
                    });
            }
        }
        __syncthreads(); // the sums of the eights before are read
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            part[warp][i * 8 + 2 * t][g]         = acc[i][0];
            part[warp][i * 8 + 2 * t + 1][g]     = acc[i][1];
            part[warp][i * 8 + 2 * t][g + 8]     = acc[i][2];
            part[warp][i * 8 + 2 * t + 1][g + 8] = acc[i][3];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < NT * 64; i += 32 * kGateUpWarps) {
            const int m = i / 8, r = i % 8;
            if (s0 + m >= end || r0 + r >= a.I) continue;
            float gate = 0.0f, up = 0.0f;
#pragma unroll
            for (int w = 0; w < kGateUpWarps; ++w) {
                gate += part[w][m][r];
                up += part[w][m][r + 8];
            }
            const float h = swiglu_prob(gate, up, 1.0f);
            const __nv_bfloat16 hi = __float2bfloat16_rn(h);
            const float rest = h - __bfloat162float(hi);
            const int64_t at = (int64_t) (s0 + m) * a.I + r0 + r;
            a.h_hi[at] = hi;
            a.h_lo[at] = __float2bfloat16_rn(fabsf(h) < INFINITY ? rest : 0.0f);
        }
    }
}

struct DownArgs {
    int T, H, I;
    ExpertWeight w;
    Lists lists;
    const __nv_bfloat16 *h_hi, *h_lo;
    void *out; // [T, H]
};

constexpr int kDownWarps = 16;

template <typename T, int FMT, int G, int NT>
__global__ void __launch_bounds__(32 * kDownWarps) moe_down_kernel(const DownArgs a) {
    grid_dep_begin();
    extern __shared__ float sums[]; // [warp][token][17]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 16, ra = min(n0 + g, a.H - 1), rb = min(n0 + g + 8, a.H - 1);
    float *mine = sums + (int64_t) warp * a.T * 17;
    for (int i = lane; i < a.T * 17; i += 32) mine[i] = 0.0f;
    __syncwarp();
    const int hits = a.lists.active[0], blocks = (a.I + kKB - 1) / kKB, total = hits * blocks;
    const int last = (int) ((int64_t) (warp + 1) * total / kDownWarps);
    using M = __nv_bfloat16; // the MMA's type: h is bf16 here whatever x is
    // fp16 weights become the sum of two bf16, exactly
    constexpr bool kSplit = FMT == kW16 && std::is_same<T, __half>::value;
    for (int item = (int) ((int64_t) warp * total / kDownWarps); item < last;) {
        const int hit = item / blocks, from = item - hit * blocks, to = min(blocks, from + last - item);
        item += to - from;
        const int64_t e = a.lists.active[1 + hit];
        const int begin = a.lists.first[hit], end = a.lists.first[hit + 1];
        const uint8_t *wa = a.w.data + e * a.w.expert_bytes + ra * a.w.row_bytes, *wb = a.w.data + e * a.w.expert_bytes + rb * a.w.row_bytes;
        const RowScale<FMT> sa = row_scale<FMT>(a.w, e, ra, a.H), sb = row_scale<FMT>(a.w, e, rb, a.H);
        constexpr int kAhead = FMT == kWInt4 ? 4 : FMT == kW16 ? 1 : 2;
        for (int s0 = begin; s0 < end; s0 += NT * 8) {
            int64_t row[NT];
            bool live[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int s = s0 + i * 8 + g;
                live[i]     = s < end;
                row[i]      = (int64_t) (live[i] ? s : begin) * a.I;
            }
            float acc[NT][4];
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
            for (int kb = from; kb < to; kb += kAhead) {
                RowPiece<FMT> pa[kAhead], pb[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; ++u)
                    if (kb + u < to) {
                        pa[u].load(wa, kb + u, t, a.I);
                        pb[u].load(wb, kb + u, t, a.I);
                    }
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const int b = kb + u;
                    if (b >= to) break;
                    auto x = [&](int i, int q, int term) {
                        const int k = b * kKB + octet_k<FMT>(q, t);
                        const __nv_bfloat16 *h = (term == 0 ? a.h_hi : a.h_lo) + row[i] + k;
                        return live[i] && k < a.I ? *reinterpret_cast<const uint4 *>(h) : make_uint4(0, 0, 0, 0);
                    };
                    if constexpr (!kSplit) {
                        few_rows_block<M, FMT, G, NT, 2>(acc, b, pa[u], pb[u], sa, sb, x);
                    } else {
                        RowPiece<FMT> ha, hb, la, lb;
                        auto split = [](const RowPiece<FMT> &p, RowPiece<FMT> &hi, RowPiece<FMT> &lo) {
#pragma unroll
                            for (int v = 0; v < RowPiece<FMT>::kVecs; ++v) {
                                const __half2 *f = reinterpret_cast<const __half2 *>(&p.v[v]);
                                __nv_bfloat162 h2[4], l2[4];
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const float2 w = __half22float2(f[j]);
                                    h2[j] = __float22bfloat162_rn(w);
                                    const float2 r = __bfloat1622float2(h2[j]);
                                    l2[j] = __float22bfloat162_rn(make_float2(fabsf(w.x) < INFINITY ? w.x - r.x : 0.0f, fabsf(w.y) < INFINITY ? w.y - r.y : 0.0f));
                                }
                                memcpy(&hi.v[v], h2, 16);
                                memcpy(&lo.v[v], l2, 16);
                            }
                        };
                        split(pa[u], ha, la);
                        split(pb[u], hb, lb);
                        few_rows_block<M, FMT, G, NT, 2>(acc, b, ha, hb, sa, sb, x);
                        few_rows_block<M, FMT, G, NT, 1>(acc, b, la, lb, sa, sb, x);
                    }
                }
            }
            // a slot's token and probability; a token has one slot an expert, so no two lanes add to one place
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int s = s0 + i * 8 + 2 * t + c;
                    if (s < end) {
                        float *to_add = mine + a.lists.token[s] * 17;
                        const float p = a.lists.prob[s];
                        to_add[g] += p * acc[i][c];
                        to_add[g + 8] += p * acc[i][2 + c];
                    }
                }
            __syncwarp();
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.T * 16; i += 32 * kDownWarps) {
        const int m = i / 16, n = i % 16;
        if (n0 + n >= a.H) continue;
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kDownWarps; ++w) s += sums[((int64_t) w * a.T + m) * 17 + n];
        ((T *) a.out)[(int64_t) m * a.H + n0 + n] = from_f32<T>(s);
    }
}

template <typename T, int FMT, int G, int NT>
int launch_layer(const GateUpArgs &u, const DownArgs &d, int max_hits, cudaStream_t st) {
    PTB_CUDA(launch_after(moe_gate_up_kernel<T, FMT, G, NT>, dim3((unsigned) cdiv(u.I, 8), (unsigned) max_hits), 32 * kGateUpWarps, 0, st, 1, u));
    PTB_LAUNCH_CHECK("moe_gate_up_kernel");
    const size_t smem = sizeof(float) * kDownWarps * d.T * 17;
    auto down = moe_down_kernel<T, FMT, G, NT>;
    if (smem > 48 * 1024) PTB_CUDA(cudaFuncSetAttribute(down, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) smem));
    PTB_CUDA(launch_after(down, dim3((unsigned) cdiv(d.H, 16)), 32 * kDownWarps, smem, st, 1, d));
    PTB_LAUNCH_CHECK("moe_down_kernel");
    return 0;
}

template <typename T, int FMT, int G> int launch_tokens(const GateUpArgs &u, const DownArgs &d, int max_hits, cudaStream_t st) {
    if (d.T <= 8) return launch_layer<T, FMT, G, 1>(u, d, max_hits, st);
    return launch_layer<T, FMT, G, 2>(u, d, max_hits, st);
}

template <typename T> int launch_format(int format, int group, const GateUpArgs &u, const DownArgs &d, int max_hits, cudaStream_t st) {
    switch (format) {
    case PTB_E4M3: return launch_tokens<T, kWE4M3, 128>(u, d, max_hits, st);
    case PTB_E5M2: return launch_tokens<T, kWE5M2, 128>(u, d, max_hits, st);
    case PTB_INT4:
        if (group == 32) return launch_tokens<T, kWInt4, 32>(u, d, max_hits, st);
        if (group == 64) return launch_tokens<T, kWInt4, 64>(u, d, max_hits, st);
        return launch_tokens<T, kWInt4, 128>(u, d, max_hits, st);
    default: return launch_tokens<T, kW16, 128>(u, d, max_hits, st);
    }
}

// One weight's description from the arguments of the C call.
int describe(const char *who, const PtbExpertWeight &p, int format, int64_t rows, int64_t K, ExpertWeight &w) {
    PTB_REQUIRE(p.data != nullptr, PTB_ERR_ARG, "moe_few_tokens: %s has no data", who);
    PTB_REQUIRE(aligned16(p.data), PTB_ERR_ALIGN, "moe_few_tokens: %s must be 16-byte aligned", who);
    w      = ExpertWeight{};
    w.data = (const uint8_t *) p.data;
    w.row_bytes = format == PTB_INT4 ? cdiv<int64_t>(K, kKB) * kInt4BlockBytes : format == PTB_E4M3 || format == PTB_E5M2 ? K : 2 * K;
    w.expert_bytes = w.row_bytes * rows;
    if (format == PTB_INT4) {
        PTB_REQUIRE(p.group == 32 || p.group == 64 || p.group == 128, PTB_ERR_ARG, "moe_few_tokens: %s: the group size must be 32, 64 or 128", who);
        w.groups = (int) cdiv<int64_t>(K, p.group);
        w.zero   = (const uint8_t *) p.zero;
    }
    if (format == PTB_INT4 || format == PTB_E4M3 || format == PTB_E5M2) PTB_REQUIRE(p.scale != nullptr, PTB_ERR_ARG, "moe_few_tokens: %s has no scales", who);
    w.scale = p.scale;
    switch (p.granularity) { // of an 8-bit weight
    case PTB_BLOCKWISE:
        w.scale_k   = 1;
        w.scale_row = (int) cdiv<int64_t>(K, 128);
        w.row_shift = 7;
        w.scale_expert = w.scale_row * cdiv<int64_t>(rows, 128);
        break;
    case PTB_ROWWISE:
        w.scale_row = 1;
        w.scale_expert = rows;
        break;
    default: break; // one scale: all strides 0
    }
    return 0;
}

} // namespace
} // namespace ptb

using namespace ptb;

extern "C" {
#pragma GCC visibility push(default)

int64_t ptb_moe_few_tokens_workspace(int64_t T, int64_t k, int64_t I) {
    if (T < 0 || k < 0 || I < 0 || T > kMaxTokens || T * k > kMaxPairs) return -1;
    return T * k * I * 4 + (list_words(T * k) * 4 + 15) / 16 * 16;
}

int ptb_moe_few_tokens(const void *x, int dtype, int64_t ldx, int64_t T, int64_t H, int64_t I, int64_t E, const int64_t *ids, const float *probs,
                       int64_t k, int format, const PtbExpertWeight *gate_up, const PtbExpertWeight *down, void *workspace, void *out,
                       ptb_stream_t stream) {
    PTB_REQUIRE(T >= 0 && H >= 1 && I >= 1 && E >= 1 && k >= 1, PTB_ERR_ARG, "moe_few_tokens: bad sizes");
    PTB_REQUIRE(dtype == PTB_BF16 || dtype == PTB_F16, PTB_ERR_ARG, "moe_few_tokens: x must be bf16 or fp16");
    PTB_REQUIRE(format == dtype || format == PTB_E4M3 || format == PTB_E5M2 || format == PTB_INT4, PTB_ERR_ARG,
                "moe_few_tokens: the weights must be of x's type, FP8 or 4-bit");
    PTB_REQUIRE(T <= kMaxTokens && T * k <= kMaxPairs, PTB_ERR_TOO_LARGE, "moe_few_tokens: at most %d tokens and %d (token, expert) pairs", kMaxTokens, kMaxPairs);
    PTB_REQUIRE(E <= kMaxExperts, PTB_ERR_TOO_LARGE, "moe_few_tokens: more than %d experts", kMaxExperts);
    PTB_REQUIRE(H <= 1 << 20 && I <= 1 << 20, PTB_ERR_TOO_LARGE, "moe_few_tokens: layer too wide");
    const int64_t step = format == PTB_E4M3 || format == PTB_E5M2 ? 16 : 8;
    PTB_REQUIRE(H % step == 0 && I % step == 0, PTB_ERR_ALIGN, "moe_few_tokens: the widths must be multiples of %d", (int) step);
    PTB_REQUIRE(T <= 1 || (ldx % 8 == 0 && ldx >= H), PTB_ERR_ALIGN, "moe_few_tokens: the row pitch of x must be a multiple of 8, and no less than a row");
    if (T == 0) return 0;
    PTB_REQUIRE(x && ids && probs && gate_up && down && workspace && out, PTB_ERR_ARG, "moe_few_tokens: null pointer");
    PTB_REQUIRE(aligned16(x) && aligned16(workspace), PTB_ERR_ALIGN, "moe_few_tokens: x and the workspace must be 16-byte aligned");
    PTB_REQUIRE(format != PTB_INT4 || gate_up->group == down->group, PTB_ERR_ARG, "moe_few_tokens: both weights must have the same group size");
    GateUpArgs u{};
    DownArgs d{};
    if (int rc = describe("the gate and up weight", *gate_up, format, 2 * I, H, u.w)) return rc;
    if (int rc = describe("the down weight", *down, format, H, I, d.w)) return rc;
    const int64_t pairs = T * k;
    __nv_bfloat16 *h = (__nv_bfloat16 *) workspace;
    const Lists lists = lists_at(h + 2 * pairs * I, pairs);
    u.x = x; u.ldx = ldx; u.H = (int) H; u.I = (int) I; u.lists = lists; u.h_hi = h; u.h_lo = h + pairs * I;
    d.T = (int) T; d.H = (int) H; d.I = (int) I; d.lists = lists; d.h_hi = u.h_hi; d.h_lo = u.h_lo; d.out = out;
    cudaStream_t st = (cudaStream_t) stream;
    PTB_CUDA(launch_after(moe_list_kernel, dim3(1), 1024, 0, st, 1, ids, probs, (int) T, (int) k, (int) E, lists));
    PTB_LAUNCH_CHECK("moe_list_kernel");
    const int max_hits = (int) imin(E, pairs);
    if (dtype == PTB_BF16) return launch_format<__nv_bfloat16>(format, gate_up->group, u, d, max_hits, st);
    return launch_format<__half>(format, gate_up->group, u, d, max_hits, st);
}

#pragma GCC visibility pop
} // extern "C"
