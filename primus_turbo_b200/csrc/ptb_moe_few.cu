// A mixture-of-experts feed-forward layer for a few tokens:
//   y[t] = sum_j p[t, j] * W2[e] (silu(W1[e] x_t, first half) * (W1[e] x_t, second half)),  e = ids[t, j]
// from weights as they are kept: 16-bit, FP8 with inverse scales, or 4-bit groups.
//
// What bounds it is reading the weights of the experts that are hit, once.  For a token or a few (at most 8 tokens and 32 (token,
// expert) pairs, as far as x and h fit into shared memory) two kernels, whose CTAs find the pairs of the experts themselves:
//
//  * moe_gate_up_token_kernel: the 16 rows of a tile are eight gate rows and the eight up rows that go with them, so both halves of a
//    channel are put together at the end of a tile.  The activation h is weighted with p there.
//  * moe_down_token_kernel: a tile is 16 output columns of all experts, whose blocks of k are one long k; the eight columns of the
//    MMA are the tokens.  Nothing is added in memory: no atomics, no second pass, and the same bits every time.
//
// Measured: 8 of 128 experts of 2048 x 768 in 4 bits 15 us (the weights are 3), 8 experts of 7168 x 2048 in FP8 62 us, where the weights are 54.
//
// For more tokens four: moe_list_kernel sorts the pairs by expert, beside the scaling of x; moe_gate_up_kernel on an expert's own tokens;
// moe_down_kernel writes a 32-bit row per pair and moe_merge_kernel adds up a token's rows in the router's order.
//
// Measured: FP8, 24 tokens, 128 experts of 2048 x 768, 93 us where the weights that are hit are 73; 4-bit see ptb_few_rows.cuh; 16-bit, 64 tokens, 16
// experts of 2880 x 1440, 106 us where the weights are 61: its 368 CTAs have 296 places, and the second wave leaves three quarters of them empty.
//
// The activation h between the two products is kept in 32 bits and then scaled like x, or scaled at once, per 64 channels: to fp16
// (2^-12 of each value; with fp16 results what that leaves is a second term), for 4-bit weights and few tokens to integers (2^-22 of the
// block's largest).  With 16-bit weights it is two bf16 (2^-17).  One fp16 turns over the
// last bit of some bf16 results (8e-4 of their norm, where rounding them is 1.7e-3); the other forms are hardly felt.
#include "ptb_few_tokens.cuh"

namespace ptb {
namespace {

constexpr int kMaxTokens  = PTB_MOE_FEW_MAX_TOKENS;
constexpr int kMaxPairs   = PTB_MOE_FEW_MAX_PAIRS;
constexpr int kMaxExperts = 1024;

// One expert-major weight [E, rows, K].
struct ExpertWeight {
    CUtensorMap map;
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
        r.s4    = (const uint16_t *) w.scale + at;
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
    int *slot;       // of a pair; -1 where it has none
};
__host__ __device__ inline int64_t list_words(int64_t pairs) { return 1 + pairs + (pairs + 1) + pairs + pairs + pairs; }
__host__ __device__ inline Lists lists_at(void *ws, int64_t pairs) {
    int *p = (int *) ws;
    return {p, p + 1 + pairs, p + 2 + 2 * pairs, (float *) (p + 2 + 3 * pairs), p + 2 + 4 * pairs};
}

// A token that names an expert twice has one slot with the sum of the two probabilities.  Ids outside [0, E) have none.
// CTAs from 1 on split x, if there are any.
template <typename X, int FMT>
__global__ void __launch_bounds__(1024) moe_list_kernel(const int64_t *ids, const float *probs, int T, int k, int E, Lists out, const X *x, int64_t ldx, int H,
                                                        const ScaledRows terms) {
    grid_dep_wait();
    grid_dep_open();
    if (blockIdx.x > 0) {
        if constexpr (kScaledX<FMT>) {
            const int blocks = (H + kKB - 1) / kKB, i = (blockIdx.x - 1) * 32 + (threadIdx.x >> 5);
            if (i < T * blocks) scale_block<X, FMT>(x + i / blocks * ldx, H, i % blocks, i / blocks, terms);
        }
        return;
    }
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
            out.slot[i]     = slot;
        } else if (i < n) {
            out.slot[i] = -1;
        }
        __syncwarp();
        if (e >= 0 && (same >> lane) == 1u) count[e] += __popc(same); // the last lane of each expert
        __syncwarp();
    }
}

struct LayerArgs {
    const void *x;
    int64_t ldx;
    int T, k, E, H, I;
    const int64_t *ids;
    const float *probs;
    ExpertWeight w1, w2;
    float *h32;                 // two kernels: [pairs, I], at the first pair with this token and expert
    Lists lists;                // four kernels:
    ScaledRows xs, hs;          // x [T, H] and h [slots, I], or with 16-bit weights
    __nv_bfloat16 *h_hi, *h_lo; // h in two parts
    float *rows;                // [slots, H]
    void *out;
};

// ---- a token or a few -----------------------------------------------------------------------------------------------------------
constexpr int kTokenPairs = 32;

// Which experts are hit, and at which pair each has its h for each token (-1: none), with what weight.
struct Pairs {
    int hits;
    int expert[kTokenPairs];
    signed char slot[kTokenPairs * kTokenCols];
    float weight[kTokenPairs * kTokenCols];
};
// Called by one warp; lane i has pair i.
__device__ __forceinline__ void find_pairs(const LayerArgs &a, Pairs &out) {
    const int lane = threadIdx.x & 31, n = a.T * a.k;
    int e = -1;
    float p = 0.0f;
    if (lane < n) {
        const int64_t id = a.ids[lane];
        if (id >= 0 && id < a.E) {
            e = (int) id;
            p = a.probs[lane];
        }
    }
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const bool first = e >= 0 && __ffs((int) same) - 1 == lane;
    const unsigned firsts = __ballot_sync(0xffffffffu, first);
    const int hit = __popc(firsts & ((1u << (__ffs((int) same) - 1)) - 1)); // of the expert of this lane's pair
    if (first) out.expert[hit] = e;
    if (lane == 0) out.hits = __popc(firsts);
    // a token that names an expert twice has it once, with the sum of the two weights
    const unsigned own = (unsigned) ((1ull << a.k) - 1);
#pragma unroll 1
    for (int c = 0; c < a.T; ++c) {
        const unsigned mine = same >> (c * a.k) & own;
        float sum = 0.0f;
#pragma unroll 1
        for (unsigned left = __reduce_or_sync(0xffffffffu, first ? mine : 0u); left != 0; left &= left - 1) {
            const int j   = __ffs((int) left) - 1;
            const float v = __shfl_sync(0xffffffffu, p, c * a.k + j);
            if (mine >> j & 1) sum += v;
        }
        if (first) {
            out.slot[hit * kTokenCols + c]   = (signed char) (mine == 0 ? -1 : c * a.k + __ffs((int) mine) - 1);
            out.weight[hit * kTokenCols + c] = sum;
        }
    }
}

// The warp's rows of expert e: eight gate rows from r0 on and the up rows that go with them, or 16 rows of the down weight.
template <int FMT> __device__ __forceinline__ void aim_gate_up(LaneRows<FMT> &out, const ExpertWeight &w, int64_t e, int r0, int I) {
    const int r  = min(r0 + lane_row(), I - 1);
    out.row      = r0;
    out.slab     = (int) e * 2;
    out.scale[0] = row_scale<FMT>(w, e, r, 2 * I);
    out.scale[1] = row_scale<FMT>(w, e, I + r, 2 * I);
}
template <int FMT> __device__ __forceinline__ void aim_down(LaneRows<FMT> &out, const ExpertWeight &w, int64_t e, int r0, int H) {
    const int r  = r0 + lane_row();
    out.row      = r0;
    out.slab     = (int) e;
    out.scale[0] = row_scale<FMT>(w, e, min(r, H - 1), H);
    out.scale[1] = row_scale<FMT>(w, e, min(r + 8, H - 1), H);
}

template <int FMT> struct GateUpTokenRows : LaneRows<FMT> {
    const LayerArgs &a;
    const Pairs &pairs;
    int tiles; // of an expert
    __device__ __forceinline__ GateUpTokenRows(const LayerArgs &a, const Pairs &pairs, int tiles) : a(a), pairs(pairs), tiles(tiles) {}
    __device__ __forceinline__ void open(int tile, int) {
        const int hit = tile / tiles;
        aim_gate_up<FMT>(*this, a.w1, pairs.expert[hit], (tile - hit * tiles) * 8, a.I);
    }
};

template <typename T, int FMT, int G>
__global__ void __launch_bounds__(32 * kTokenWarps, 1) moe_gate_up_token_kernel(const __grid_constant__ LayerArgs a, int shares) {
    extern __shared__ __align__(16) uint8_t raw[];
    uint8_t *smem = aligned(raw);
    __shared__ Pairs pairs;
    grid_dep_wait(); // the kernel before this one is somebody else's
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tiles = (a.I + 7) / 8, blocks = (a.H + kKB - 1) / kKB;
    constexpr int kTerms = FMT == kWInt4 ? kIntTerms : 1;
    if (warp == 0) find_pairs(a, pairs);
    __syncthreads();
    few_tokens_walk<T, FMT, G, kTerms, false, false, false>(
        smem, &a.w1.map, a.T, pairs.hits * tiles, shares, 1, a.H, GateUpTokenRows<FMT>(a, pairs, tiles),
        [&](uint8_t *x, uint8_t *runs) {
            stage_blocks<T, T, FMT, G, kTerms>(x, runs, blocks, a.T, [&](int block, int col, int &left) {
                left = a.H - block * kKB;
                return (const T *) a.x + col * a.ldx + block * kKB;
            });
        },
        [&](int tile, auto &&sum) {
            const int hit = tile / tiles, r0 = (tile - hit * tiles) * 8;
            for (int i = lane; i < a.T * 8; i += 32) {
                const int c = i / 8, r = i % 8, slot = pairs.slot[hit * kTokenCols + c];
                if (slot >= 0 && r0 + r < a.I) a.h32[(int64_t) slot * a.I + r0 + r] = swiglu_prob(sum(c, r), sum(c, r + 8), pairs.weight[hit * kTokenCols + c]);
            }
        });
}

template <int FMT> struct DownTokenRows : LaneRows<FMT> {
    const LayerArgs &a;
    const Pairs &pairs;
    __device__ __forceinline__ DownTokenRows(const LayerArgs &a, const Pairs &pairs) : a(a), pairs(pairs) {}
    __device__ __forceinline__ void open(int tile, int segment) {
        aim_down<FMT>(*this, a.w2, pairs.expert[segment], tile * 16, a.H);
    }
    __device__ __forceinline__ bool mask(int segment, int column) const { return pairs.slot[segment * kTokenCols + column] >= 0; }
};

template <typename T> constexpr int kHScaled = std::is_same<T, __half>::value ? 2 : 1; // terms of scaled h
template <typename T, int FMT> constexpr int kHTerms = FMT == kWInt4 ? kIntTerms : FMT == kW16 || std::is_same<T, __half>::value ? 2 : 1;

template <typename T, int FMT, int G>
__global__ void __launch_bounds__(32 * kTokenWarps, 1) moe_down_token_kernel(const __grid_constant__ LayerArgs a, int shares) {
    extern __shared__ __align__(16) uint8_t raw[];
    uint8_t *smem = aligned(raw);
    __shared__ Pairs pairs;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, blocks = (a.I + kKB - 1) / kKB;
    // 16-bit weights: the MMA's type is that of h, bf16, whatever x is
    using M = __nv_bfloat16;
    constexpr int kTerms = kHTerms<T, FMT>;
    if (warp == 0) find_pairs(a, pairs);
    __syncthreads();
    few_tokens_walk<M, FMT, G, kTerms, FMT == kW16 && std::is_same<T, __half>::value, true, true>(
        smem, &a.w2.map, a.T, (a.H + 15) / 16, shares, pairs.hits, a.I, DownTokenRows<FMT>(a, pairs),
        [&](uint8_t *x, uint8_t *runs) {
            stage_blocks<M, float, FMT, G, kTerms>(x, runs, pairs.hits * blocks, a.T, [&](int block, int col, int &left) {
                const int hit = block / blocks, kb = block - hit * blocks, slot = pairs.slot[hit * kTokenCols + col];
                left = slot < 0 ? 0 : a.I - kb * kKB; // zeros for a token that does not go there
                return a.h32 + (int64_t) max(slot, 0) * a.I + kb * kKB;
            });
        },
        [&](int tile, auto &&sum) {
            for (int i = lane; i < a.T * 16; i += 32) {
                const int m = i / 16, n = tile * 16 + i % 16;
                if (n < a.H) ((T *) a.out)[(int64_t) m * a.H + n] = from_f32<T>(sum(m, i % 16));
            }
        });
}

// ---- more tokens: gate and up projection -----------------------------------------------------------------------------------------
constexpr int kWarps = 8, kChannels = 8 * kWarps; // of a CTA, eight channels a warp

template <int FMT> struct GateUpRows : LaneRows<FMT> {
    const uint8_t *x0;
    int64_t pitch;
    const int *token; // row of x of a column
    __device__ __forceinline__ const uint8_t *x(int, int col) const { return x0 + token[col] * pitch; }
};

// blockIdx.y counts the experts that are hit.  The CTAs of a cluster share k; the results of column c are share c % shares's to finish.
template <typename T, int FMT, int G, int NT, bool kShared>
__global__ void __launch_bounds__(32 * kWarps, 2) moe_gate_up_kernel(const __grid_constant__ LayerArgs a, int all_shares) {
    const int shares = kShared ? all_shares : 1; // (its own code for one share: 351 instead of 367 us for 48 tokens in 4 bits)
    extern __shared__ __align__(16) uint8_t raw[];
    uint8_t *smem = aligned(raw);
    using W = Walk<FMT, NT, kWarps>;
    constexpr int kPitch = kChannels + 1;
    __shared__ uint64_t bars[W::kBars];
    __shared__ int token[NT * 8];
    float *h_of = reinterpret_cast<float *>(smem + W::kSums); // [column][channel]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dep_wait();
    const int hit = blockIdx.y;
    if (hit >= a.lists.active[0]) return;
    const int64_t e = a.lists.active[1 + hit];
    const int begin = a.lists.first[hit], end = a.lists.first[hit + 1];
    const int share = kShared ? blockIdx.x % shares : 0, r0 = blockIdx.x / shares * kChannels;
    const Share k = kShared ? share_of(a.H, share, shares) : Share{0, (a.H + kKB - 1) / kKB};
    GateUpRows<FMT> src;
    aim_gate_up<FMT>(src, a.w1, e, r0 + warp * 8, a.I);
    src.x0    = kScaledX<FMT> ? a.xs.planes : (const uint8_t *) a.x;
    src.pitch = kScaledX<FMT> ? a.xs.pitch : a.ldx * 2;
    src.token = token;
    for (int s0 = begin; s0 < end; s0 += NT * 8) {
        const int cols = min(NT * 8, end - s0);
        if (threadIdx.x < cols) token[threadIdx.x] = a.lists.token[s0 + threadIdx.x];
        __syncthreads();
        float acc[NT][4] = {};
        if (r0 < a.I) few_rows_walk<T, FMT, G, 128, NT, kWarps, 1, false>(acc, smem, bars, &a.w1.map, a.H, cols, k.begin, k.end, src);
        else grid_dep_open(); // (past the last channel there is only h's padding to write)
        const RowSums<FMT, NT, kWarps> sums(acc, smem);
        if (shares > 1) cluster_sync();
        const int mine = (cols - share + shares - 1) / shares; // columns
        for (int i = threadIdx.x; i < mine * kChannels; i += W::kThreads) {
            const int c = share + i / kChannels * shares, r = i % kChannels, at = r / 8 * 16 + r % 8, slot = s0 + c;
            const float h = r0 + r < a.I ? swiglu_prob(sums.sum(c, at, shares), sums.sum(c, at + 8, shares), a.lists.prob[slot]) : 0.0f;
            if constexpr (kScaledX<FMT>) {
                h_of[i / kChannels * kPitch + r] = h;
            } else if (r0 + r < a.I) {
                const __nv_bfloat16 hi = __float2bfloat16_rn(h);
                a.h_hi[(int64_t) slot * a.I + r0 + r] = hi;
                a.h_lo[(int64_t) slot * a.I + r0 + r] = __float2bfloat16_rn(fabsf(h) < INFINITY ? h - __bfloat162float(hi) : 0.0f);
            }
        }
        if constexpr (kScaledX<FMT>) { // a half-warp scales a token's 64 channels, four a lane
            __syncthreads();
            for (int c2 = warp; 2 * c2 < mine; c2 += kWarps) {
                const int c = min(2 * c2 + (lane >> 4), mine - 1), in = (lane & 15) * 4;
                const int64_t slot = s0 + share + c * shares;
                float v[4], largest = 0.0f, scale, inv;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[j] = h_of[c * kPitch + in + j];
                    if (fabsf(v[j]) < INFINITY) largest = fmaxf(largest, fabsf(v[j]));
                }
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
                block_scale(largest, kTopHalf, scale, inv);
                uint8_t *block = a.hs.planes + slot * a.hs.pitch + (int64_t) (r0 / kKB) * kScaledBlock;
#pragma unroll
                for (int term = 0; term < kHScaled<T>; ++term) put_halves<FMT>(block + term * a.hs.plane, r0 % kKB + in, v, inv, term > 0);
                if ((lane & 15) == 0) reinterpret_cast<float *>(block + 256)[r0 % kKB / 64] = scale;
            }
        }
        if (shares > 1) cluster_sync(); // all of this is read before it is written again, or its CTA leaves
        else if (s0 + NT * 8 < end) __syncthreads();
    }
}

// ---- more tokens: down projection, a row per pair --------------------------------------------------------------------------------
template <int FMT> struct DownRows : LaneRows<FMT> {
    const uint8_t *x0;
    int64_t plane, pitch;
    __device__ __forceinline__ const uint8_t *x(int term, int col) const { return x0 + term * plane + col * pitch; }
};

template <typename T, int FMT> constexpr int kDownTerms = kScaledX<FMT> ? kHScaled<T> : 2;
template <typename T, int FMT, int G, int NT, bool kShared>
__global__ void __launch_bounds__(32 * kWarps, 2) moe_down_kernel(const __grid_constant__ LayerArgs a, int all_shares) {
    const int shares = kShared ? all_shares : 1;
    extern __shared__ __align__(16) uint8_t raw[];
    uint8_t *smem = aligned(raw);
    using W = Walk<FMT, NT, kWarps>;
    __shared__ uint64_t bars[W::kBars];
    const int hit = blockIdx.y; // the lists are from two kernels before
    if (hit >= a.lists.active[0]) {
        grid_dep_wait();
        return;
    }
    const int warp = threadIdx.x >> 5, share = kShared ? blockIdx.x % shares : 0, n0 = blockIdx.x / shares * W::kRows;
    const Share k = kShared ? share_of(a.I, share, shares) : Share{0, (a.I + kKB - 1) / kKB};
    const int begin = a.lists.first[hit], end = a.lists.first[hit + 1];
    DownRows<FMT> src;
    aim_down<FMT>(src, a.w2, a.lists.active[1 + hit], n0 + warp * 16, a.H);
    src.plane = kScaledX<FMT> ? a.hs.plane : (int64_t) ((const uint8_t *) a.h_lo - (const uint8_t *) a.h_hi);
    src.pitch = kScaledX<FMT> ? a.hs.pitch : (int64_t) a.I * 2;
    for (int s0 = begin; s0 < end; s0 += NT * 8) {
        const int cols = min(NT * 8, end - s0);
        src.x0 = (kScaledX<FMT> ? a.hs.planes : (const uint8_t *) a.h_hi) + s0 * src.pitch;
        float acc[NT][4] = {};
        few_rows_walk<__nv_bfloat16, FMT, G, 64, NT, kWarps, kDownTerms<T, FMT>, FMT == kW16 && std::is_same<T, __half>::value>(
            acc, smem, bars, &a.w2.map, a.I, cols, k.begin, k.end, src);
        const RowSums<FMT, NT, kWarps> sums(acc, smem);
        if (shares > 1) cluster_sync();
        for (int i = threadIdx.x + share * W::kThreads; i < cols * W::kRows; i += W::kThreads * shares) {
            const int c = i / W::kRows, n = i % W::kRows;
            if (n0 + n < a.H) a.rows[(int64_t) (s0 + c) * a.H + n0 + n] = sums.sum(c, n, shares);
        }
        if (shares > 1) cluster_sync();
        else if (s0 + NT * 8 < end) __syncthreads();
    }
}

// out[t] = the sum of token t's rows; one thread per eight columns
template <typename T> __global__ void __launch_bounds__(128) moe_merge_kernel(const LayerArgs a) {
    grid_dep_wait();
    grid_dep_open();
    const int n = (blockIdx.x * 128 + threadIdx.x) * 8, token = blockIdx.y;
    if (n >= a.H) return;
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = 0.0f;
    for (int j = 0; j < a.k; ++j) {
        const int slot = a.lists.slot[token * a.k + j];
        if (slot < 0) continue;
        const float4 *r = reinterpret_cast<const float4 *>(a.rows + (int64_t) slot * a.H + n);
        const float4 u = r[0], v = r[1];
        s[0] += u.x; s[1] += u.y; s[2] += u.z; s[3] += u.w;
        s[4] += v.x; s[5] += v.y; s[6] += v.z; s[7] += v.w;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ((T *) a.out)[(int64_t) token * a.H + n + j] = from_f32<T>(s[j]);
}

constexpr int kMostSmem = 227 * 1024 - 4096; // of a CTA, less what is not dynamic

// Whether the two-kernel form has room for x and for h, and the shared memory of its kernels.
template <typename T, int FMT, int G> bool fits_token(const LayerArgs &a, int &up, int &down) {
    if (a.T > kTokenCols || a.T * a.k > kTokenPairs || a.H > 1 << 17 || a.I > 1 << 15) return false;
    up   = token_smem(TokenX<FMT, G>::bytes(FMT == kWInt4 ? kIntTerms : 1, a.T, cdiv(a.H, kKB)), a.T);
    down = token_smem(TokenX<FMT, G>::bytes(kHTerms<T, FMT>, a.T, (int) imin(a.E, a.T * a.k) * cdiv(a.I, kKB)), a.T);
    return up <= kMostSmem && down <= kMostSmem;
}

template <typename T, int FMT, int G> int launch_token(const LayerArgs &a, int up, int down, cudaStream_t st) {
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    const int hits = (int) imin(a.E, a.T * a.k), up_tiles = hits * cdiv(a.I, 8), down_tiles = cdiv(a.H, 16);
    const int up_shares = token_shares(up_tiles, cdiv(a.H, kKB), sms), down_shares = token_shares(down_tiles, hits * cdiv(a.I, kKB), sms);
    const dim3 g1((unsigned) cdiv(up_tiles, kTokenWarps >> up_shares)), g2((unsigned) cdiv(down_tiles, kTokenWarps >> down_shares));
    PTB_CUDA(launch_early(moe_gate_up_token_kernel<T, FMT, G>, g1, 32 * kTokenWarps, up, kMostSmem, st, 1, a, up_shares));
    PTB_LAUNCH_CHECK("moe_gate_up_token_kernel");
    PTB_CUDA(launch_early(moe_down_token_kernel<T, FMT, G>, g2, 32 * kTokenWarps, down, kMostSmem, st, 1, a, down_shares));
    PTB_LAUNCH_CHECK("moe_down_token_kernel");
    return 0;
}

template <typename T, int FMT, int G, int NT> int launch_batch(const LayerArgs &a, cudaStream_t st) {
    using W = Walk<FMT, NT, kWarps>;
    const unsigned hits = (unsigned) imin(a.E, a.T * a.k), splits = kScaledX<FMT> ? (unsigned) cdiv(a.T * cdiv(a.H, kKB), 32) : 0u;
    const int cols = (int) imin(a.T, NT * 8);
    constexpr int kMore = NT * 8 * (kChannels + 1) * 4, kUpMost = W::smem(1, NT * 8, kMore), kDownMost = W::smem(kDownTerms<T, FMT>, NT * 8);
    const int up_smem = W::smem(1, cols, kMore), down_smem = W::smem(kDownTerms<T, FMT>, cols);
    PTB_CUDA(launch_early(moe_list_kernel<T, FMT>, dim3(1 + splits), 1024, 0, 0, st, 1, a.ids, a.probs, a.T, a.k, a.E, a.lists, (const T *) a.x, a.ldx, a.H, a.xs));
    PTB_LAUNCH_CHECK("moe_list_kernel");
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    const unsigned channels = (unsigned) (kScaledX<FMT> ? cdiv(a.I, kKB) * 2 : cdiv(a.I, kChannels)), rows = (unsigned) cdiv(a.H, W::kRows); // CTAs; h's planes are whole blocks
    const unsigned up = (unsigned) shares_for(a.H, (int64_t) channels * hits, 2 * sms), down = (unsigned) shares_for(a.I, (int64_t) rows * hits, 2 * sms);
    PTB_CUDA(launch_early(up > 1 ? moe_gate_up_kernel<T, FMT, G, NT, true> : moe_gate_up_kernel<T, FMT, G, NT, false>, dim3(channels * up, hits), W::kThreads, up_smem, kUpMost, st, up, a, (int) up));
    PTB_LAUNCH_CHECK("moe_gate_up_kernel");
    PTB_CUDA(launch_early(down > 1 ? moe_down_kernel<T, FMT, G, NT, true> : moe_down_kernel<T, FMT, G, NT, false>, dim3(rows * down, hits), W::kThreads, down_smem, kDownMost, st, down, a, (int) down));
    PTB_LAUNCH_CHECK("moe_down_kernel");
    PTB_CUDA(launch_early(moe_merge_kernel<T>, dim3((unsigned) cdiv(a.H, 1024), (unsigned) a.T), 128, 0, 0, st, 1, a));
    PTB_LAUNCH_CHECK("moe_merge_kernel");
    return 0;
}

template <typename T, int FMT, int G> int launch_layer(const LayerArgs &a, cudaStream_t st) {
    int up = 0, down = 0;
    if (fits_token<T, FMT, G>(a, up, down)) return launch_token<T, FMT, G>(a, up, down, st);
    // Columns of a CTA: an expert with more tokens reads its weight again.  With 16 two blocks' code is held in registers, with 32 hardly: so 16 where an
    // expert has ten or fewer on average.  us with 16 and 32: 4-bit, nine on average, 357 and 402; FP8, 1.5, 89 and 95; 16-bit, 16 on average, 150 and 122.
    if (a.T <= 8) return launch_batch<T, FMT, G, 1>(a, st);
    return a.T <= 16 || a.T * a.k <= 10 * a.E ? launch_batch<T, FMT, G, 2>(a, st) : launch_batch<T, FMT, G, 4>(a, st);
}

template <typename T> int launch_format(int format, int group, const LayerArgs &a, cudaStream_t st) {
    switch (format) {
    case PTB_E4M3: return launch_layer<T, kWE4M3, 128>(a, st);
    case PTB_E5M2: return launch_layer<T, kWE5M2, 128>(a, st);
    case PTB_INT4:
        if (group == 32) return launch_layer<T, kWInt4, 32>(a, st);
        if (group == 64) return launch_layer<T, kWInt4, 64>(a, st);
        return launch_layer<T, kWInt4, 128>(a, st);
    default: return launch_layer<T, kW16, 128>(a, st);
    }
}

// The workspace's pieces, one after the other; whichever form runs, there is room for it.
struct Pieces {
    int64_t xs, hs, rows, lists, total;
};
Pieces pieces(int format, int dtype, int64_t T, int64_t k, int64_t H, int64_t I) {
    auto up = [](int64_t n) { return (n + 15) / 16 * 16; };
    const bool scaled = format == PTB_E4M3 || format == PTB_E5M2 || format == PTB_INT4;
    Pieces p{};
    p.hs    = scaled ? up(scaled_bytes(1, T, H)) : 0;
    p.rows  = p.hs + up(imax(scaled ? scaled_bytes(dtype == PTB_F16 ? 2 : 1, T * k, I) : 0, T * k * I * 4));
    p.lists = p.rows + up(T * k * H * 4);
    p.total = p.lists + list_words(T * k) * 4;
    return p;
}

// One weight's description from the arguments of the C call.
int describe(const char *who, const PtbExpertWeight &p, int format, int64_t rows, int64_t K, ExpertWeight &w) {
    PTB_REQUIRE(p.data != nullptr, PTB_ERR_ARG, "moe_few_tokens: %s has no data", who);
    PTB_REQUIRE(aligned16(p.data), PTB_ERR_ALIGN, "moe_few_tokens: %s must be 16-byte aligned", who);
    w = ExpertWeight{};
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

int moe_few_status(int *status, int reset) { return few_status(status, reset); }
} // namespace ptb

using namespace ptb;

extern "C" {
#pragma GCC visibility push(default)

int64_t ptb_moe_few_tokens_workspace(int dtype, int64_t T, int64_t H, int64_t I, int64_t k, int format) {
    if (T < 0 || k < 0 || H < 0 || I < 0 || T > kMaxTokens || T * k > kMaxPairs) return -1;
    return pieces(format, dtype, T, k, H, I).total;
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
    LayerArgs a{};
    if (int rc = describe("the gate and up weight", *gate_up, format, 2 * I, H, a.w1)) return rc;
    if (int rc = describe("the down weight", *down, format, H, I, a.w2)) return rc;
    auto row_bytes = [&](int64_t K) { return format == PTB_INT4 ? cdiv<int64_t>(K, kKB) * kInt4BlockBytes : format == dtype ? 2 * K : K; };
    if (int rc = weight_map(&a.w1.map, gate_up->data, row_bytes(H), I, 2 * E, true)) return rc;
    if (int rc = weight_map(&a.w2.map, down->data, row_bytes(I), H, E, false)) return rc;
    const int64_t pairs = T * k;
    a.x = x; a.ldx = ldx; a.T = (int) T; a.k = (int) k; a.E = (int) E; a.H = (int) H; a.I = (int) I; a.ids = ids; a.probs = probs; a.out = out;
    const Pieces at = pieces(format, dtype, T, k, H, I);
    uint8_t *ws = (uint8_t *) workspace;
    a.xs    = scaled_rows_at(ws + at.xs, T, H);
    a.hs    = scaled_rows_at(ws + at.hs, pairs, I);
    a.h32   = (float *) (ws + at.hs);
    a.h_hi  = (__nv_bfloat16 *) (ws + at.hs);
    a.h_lo  = a.h_hi + pairs * I;
    a.rows  = (float *) (ws + at.rows);
    a.lists = lists_at(ws + at.lists, pairs);
    if (dtype == PTB_BF16) return launch_format<__nv_bfloat16>(format, gate_up->group, a, (cudaStream_t) stream);
    return launch_format<__half>(format, gate_up->group, a, (cudaStream_t) stream);
}

#pragma GCC visibility pop
} // extern "C"
