// The walk over a weight for a token or a few (see ptb_few_rows.cuh for what goes into an MMA).
//
// One CTA of 16 warps an SM.  All of x is scaled into shared memory first, while the first weights are on their way.  A tile is 16 weight
// rows over all of k -- for the down projection of an MoE layer the experts' k one after the other ("segments").  A CTA has one
// tile or up to 16; 16 warps or down to one share a tile's blocks of k, each a run of neighbouring blocks, and add up at the end in a fixed order.
//
// Weights come as boxes of 16 rows and 256 bytes into slots of the warp's own: one thread asks for them, and they do not queue with
// the loads from shared memory (as cp.async they did: an FP8 layer took 88 us, which was 46 of computing plus 42 of copying; row by row as bulk copies
// 82; as boxes 63, where the weights are 54).  Two slots of 4 KB a warp keep 64 to 128 KB an SM on their way, where 23 bytes a clock and a
// latency of some 1000 clocks need about 25.
//
// What bounds it then is instructions: a block of 16 rows (1 KB of 4-bit codes) has 44 clocks of an SM, 176 issue slots.  A scale per group
// and row would be most of them, if the sums of a group had to be scaled before the next group may be added.  With one token
// seven of the MMA's eight columns have nothing to do; so group j of a window of eight goes to column j (zeros go to the others), and
// eight groups are scaled at once, each lane its own.  With two tokens a window is four groups, and so on.
#pragma once

#include "ptb_few_rows.cuh"

namespace ptb {
namespace {

constexpr int kTokenWarps = 16, kTokenCols = 8;
constexpr int kIntTerms = 3; // bytes of x beside 4-bit weights

// x in shared memory: per block kTerms x cols rows (and once more, zeros), then per block and column the scales (and sums).
template <int FMT, int G> struct TokenX {
    static constexpr int kRow = FMT == kWInt4 ? 128 + 16 : FMT == kW16 ? 256 + 64 : 256 + 16; // bytes of a block of a row, shifted from row to row
    static constexpr int kRuns = FMT == kWInt4 ? kKB / G : FMT == kW16 ? 0 : 1;               // float2 each
    __host__ __device__ static constexpr int block_bytes(int terms, int cols) { return terms * cols * kRow; }
    __host__ __device__ static constexpr int run_bytes(int cols) { return cols * kRuns * 8; }
    __host__ __device__ static constexpr int bytes(int terms, int cols, int blocks) { return (blocks + 1) * block_bytes(terms, cols) + blocks * run_bytes(cols); }
};
inline int token_smem(int x_bytes, int cols) { return kTokenWarps * kWeightSlots * kSlotBytes + (x_bytes + 15) / 16 * 16 + kTokenWarps * cols * 17 * 4 + kAlign; }

// Staging: eight lanes share a block of a column, sixteen neighbouring values (two octets) each; a warp has four blocks at a time.  A CTA runs
// this once, on cold instruction caches: few instructions count, and few different ones.
template <typename T> __device__ __forceinline__ void load_sixteen(const T *x, int left, float (&v)[16]) { // left: values to the row's end, a multiple of 8
#pragma unroll
    for (int o = 0; o < 2; ++o) {
        if (o * 8 < left) {
            uint4 u[sizeof(T) / 2];
#pragma unroll
            for (int i = 0; i < (int) sizeof(T) / 2; ++i) u[i] = reinterpret_cast<const uint4 *>(x + o * 8)[i];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[o * 8 + j] = to_f32(reinterpret_cast<const T *>(u)[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[o * 8 + j] = 0.0f;
        }
    }
}

template <typename T, int FMT, int G, int kTerms>
__device__ __forceinline__ void stage_sixteen(uint8_t *x, uint8_t *runs, int block, int cols, int col, const float (&v)[16], bool here) {
    using X = TokenX<FMT, G>;
    const int lane = threadIdx.x & 31, part = lane & 7;
    uint8_t *to = x + block * X::block_bytes(kTerms, cols) + col * X::kRow;
    const int next_term = cols * X::kRow;
    float scale = 1.0f, inv = 1.0f, largest = 0.0f;
    bool fine = true;
    if constexpr (FMT != kW16) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float m = fabsf(v[j]);
            if (m < INFINITY) largest = fmaxf(largest, m);
            else fine = false;
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
        block_scale(largest, FMT == kWInt4 ? kTopInt : kTopHalf, scale, inv);
    }
    if constexpr (FMT == kWInt4) {
        const unsigned bad = __ballot_sync(0xffffffffu, !fine);
        if (bad >> (lane & 24) & 255) scale = NAN; // integers hold no NaN and no infinity: the block's products become NaN
        uint32_t n = 0;
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            uint32_t high[2], mid[2], low[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t i[4];
#pragma unroll
                for (int l = 0; l < 4; ++l) { // rounded to an integer in the low bits of a float's mantissa
                    i[l] = __float_as_uint(v[o * 8 + j * 4 + l] * inv + kFloatBaseValue) - (uint32_t) kFloatBase;
                    n += i[l];
                }
                const uint32_t a = __byte_perm(i[0], i[1], 0x5140), b = __byte_perm(i[2], i[3], 0x5140);
                low[j]  = __byte_perm(a, b, 0x5410);
                mid[j]  = __byte_perm(a, b, 0x7632);
                high[j] = __byte_perm(__byte_perm(i[0], i[1], 0x0062), __byte_perm(i[2], i[3], 0x0062), 0x5410);
            }
            const int at = byte_place(part * 16 + o * 8);
            if (here) {
                *reinterpret_cast<uint2 *>(to + at)                 = make_uint2(high[0], high[1]);
                *reinterpret_cast<uint2 *>(to + next_term + at)     = make_uint2(mid[0], mid[1]);
                *reinterpret_cast<uint2 *>(to + 2 * next_term + at) = make_uint2(low[0], low[1]);
            }
        }
#pragma unroll
        for (int o = 1; o < G / 16; o <<= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
        if (here && part % (G / 16) == 0) reinterpret_cast<float2 *>(runs)[(block * cols + col) * X::kRuns + part / (G / 16)] = make_float2(scale, (float) (int) n);
    } else {
        using H = std::conditional_t<FMT == kW16, T, __half>;
#pragma unroll
        for (int term = 0; term < kTerms; ++term) {
            H h[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float s = v[j] * inv;
                h[j] = term == 0 ? from_f32<H>(s) : from_f32<H>(fabsf(s) < INFINITY ? s - to_f32(from_f32<H>(s)) : 0.0f);
            }
            uint4 u[2];
            memcpy(u, h, 32);
            if (here) {
                reinterpret_cast<uint4 *>(to + term * next_term + part * 32)[0] = u[0];
                reinterpret_cast<uint4 *>(to + term * next_term + part * 32)[1] = u[1];
            }
        }
        if (FMT != kW16 && here && part == 0) reinterpret_cast<float2 *>(runs)[block * cols + col] = make_float2(scale, 0.0f);
    }
}

// n blocks of every column: at(block, column) is where the row's values of that block start and how many are left in the row.
template <typename T, typename V, int FMT, int G, int kTerms, typename At>
__device__ __forceinline__ void stage_blocks(uint8_t *x, uint8_t *runs, int n, int cols, At &&at) {
    const int part = threadIdx.x & 7, first = threadIdx.x >> 3;
#pragma unroll 1
    for (int col = 0; col < cols; ++col)
#pragma unroll 1
        for (int b0 = 0; b0 < n; b0 += 4 * kTokenWarps) {
            const int block = min(b0 + first, n - 1);
            int left        = 0;
            const V *from   = at(block, col, left);
            float v[16];
            load_sixteen(from + part * 16, left - part * 16, v);
            stage_sixteen<T, FMT, G, kTerms>(x, runs, block, cols, col, v, b0 + first < n);
        }
}

// src.open(tile, segment)     from here on row, slab and scale (a LaneRows) are that part's
// src.mask(segment, column)   with kMasked: whether the segment's weight is meant for the column
// stage(x, runs)              stages all of x in shared memory (called by all warps, after grid_dep_wait)
// finish(tile, sum)           called by one warp for each tile; sum(column, row) is there for columns below `cols` and rows below 16
// 1 << log_shares warps a tile; segments * blocks blocks of k a tile; K: length of a weight row (of a segment).
// kEarly: weights may be fetched ahead of grid_dep_wait.
template <typename T, int FMT, int G, int kTerms, bool kSplit, bool kMasked, bool kEarly, typename Src, typename Stage, typename Finish>
__device__ __forceinline__ void few_tokens_walk(uint8_t *smem, const CUtensorMap *map, int cols, int tiles, int log_shares, int segments, int K, const Src &src, Stage &&stage, Finish &&finish) {
    using X = TokenX<FMT, G>;
    using Piece = RowPiece<FMT>;
    constexpr int CB = kChunk<FMT>;
    __shared__ uint64_t full[kTokenWarps * kWeightSlots];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int blocks = (K + kKB - 1) / kKB, total = segments * blocks;
    const int tile = blockIdx.x * (kTokenWarps >> log_shares) + (warp >> log_shares), share = warp & ((1 << log_shares) - 1);
    const uint32_t ring = shared_u32(smem) + warp * (kWeightSlots * kSlotBytes), bars = shared_u32(full) + warp * (kWeightSlots * 8);
    uint8_t *x0 = smem + kTokenWarps * kWeightSlots * kSlotBytes, *runs0 = x0 + (total + 1) * X::block_bytes(kTerms, cols);
    float *part = reinterpret_cast<float *>(x0 + (X::bytes(kTerms, cols, total) + 15) / 16 * 16);
    const int begin = tile < tiles ? share * total >> log_shares : 0, end = tile < tiles ? (share + 1) * total >> log_shares : 0;

    if (lane < kWeightSlots) bar_init(bars + lane * 8, 1);
    bar_init_fence();
    __syncwarp();
    // what is fetched next
    Src ahead = src;
    const int seg0 = segments == 1 ? 0 : begin / blocks, kb0 = begin - seg0 * blocks;
    int left_w = end - begin, seg_w = seg0, kb_w = kb0;
    auto fetch_chunk = [&](int slot) {
        if (left_w <= 0) return;
        const int n = min(min(CB, blocks - kb_w), left_w);
        if (lane == 0) fetch_tile<FMT>(ring + slot * kSlotBytes, map, kb_w, n, ahead.row, ahead.slab, bars + slot * 8);
        left_w -= n;
        kb_w += n;
        if (kb_w == blocks && left_w > 0) {
            kb_w = 0;
            ++seg_w;
            ahead.open(tile, seg_w);
        }
    };
    if constexpr (!kEarly) grid_dep_wait();
    if (left_w > 0) ahead.open(tile, seg_w);
#pragma unroll 1
    for (int i = 0; i < kWeightSlots; ++i) fetch_chunk(i);
    if constexpr (kEarly) grid_dep_wait();
    grid_dep_open();
    for (int i = threadIdx.x * 4; i < X::block_bytes(kTerms, cols); i += 32 * kTokenWarps * 4) *reinterpret_cast<uint32_t *>(x0 + total * X::block_bytes(kTerms, cols) + i) = 0;
    stage(x0, runs0);
    __syncthreads();

    // Columns: token = column % (1 << shift), place in the window = column >> shift.
    const int shift = cols == 1 ? 0 : cols == 2 ? 1 : cols <= 4 ? 2 : 3, window = 8 >> shift, tokens = 1 << shift;
    const int my_token = min(g & (tokens - 1), cols - 1), my_place = g >> shift; // of the column whose x this lane supplies
    constexpr int kLaneX = FMT == kW16 ? 16 : 32;
    const uint32_t x_lane = shared_u32(x0) + my_token * X::kRow + t * kLaneX, zeros = x_lane + total * X::block_bytes(kTerms, cols), term1 = cols * X::kRow;
    int token[2], place[2]; // of the two columns whose sums this lane has
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        token[j] = (2 * t + j) & (tokens - 1);
        place[j] = (2 * t + j) >> shift;
    }
    const uint32_t w_lane = ring + lane_place();
    using Sum = std::conditional_t<FMT == kWInt4, int, float>;
    constexpr int kSums = FMT == kWInt4 ? kIntTerms : 2;
    Sum c[kSums][4]; // 4-bit: products with high, middle and low bytes; otherwise two chains of MMAs, each waiting for its last
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    uint32_t ws[2][2], wz[2][2]; // of the window: scale and zero point [column][row]
    Src here = src;
    int seg = seg0, kb = kb0, filled = 0, first = kb * X::kRuns; // groups in the window; the segment's first group of it
    int left = end - begin, n = 0, i = 0, slot = 0, q0 = 0; // blocks; in the chunk, and done of it; octets done of the block
    // the octets that are worked on before the window is looked at: a block, or less where a window is less
    constexpr int kRun = FMT == kWInt4 ? G / 32 : 4; // octets a group
    const int unit = FMT == kWInt4 ? min(4, window * kRun) : 4;
    uint32_t parity = 0, at = begin * X::block_bytes(kTerms, cols), from = 0;
    bool ok = true, fresh = true;
    if (left > 0) here.open(tile, seg);
#pragma unroll 1
    while (left > 0) {
        if (fresh) { // a new window: its scales are asked for long before they are needed
            fresh = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int i = 0; i < kSums; ++i) c[i][j] = FMT == kWInt4 ? (Sum) kFloatBase : (Sum) 0;
            }
            if constexpr (FMT != kW16) {
                const int groups = FMT == kWInt4 ? here.scale[0].count : blocks;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int w = min(first + place[j], groups - 1);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if constexpr (FMT == kWInt4) {
                            ws[j][h] = here.scale[h].s4[w];
                            wz[j][h] = here.scale[h].z4 != nullptr ? here.scale[h].z4[w] : 8;
                        } else {
                            ws[j][h] = __float_as_uint(here.scale[h].s8[(int64_t) w * here.scale[h].stride]);
                        }
                    }
                }
            }
        }
        if (i == n) { // a new chunk
            n  = min(min(CB, blocks - kb), left);
            i  = 0;
            ok = __all_sync(0xffffffffu, bar_wait(bars + slot * 8, parity));
            if (!ok) break;
            from = w_lane + slot * kSlotBytes;
        }
        const uint32_t x_here = x_lane + at;
        if constexpr (FMT == kWInt4) {
            if (unit == 4) {
                Piece p[2];
                p[0].read(from, i, 0);
                p[1].read(from, i, 8 * 128);
                uint4 u[kIntTerms];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (q % kRun == 0 || q % 2 == 0) {
                        const uint32_t x = (filled + q / kRun == my_place ? x_here : zeros) + q / 2 * 16;
#pragma unroll
                        for (int term = 0; term < kIntTerms; ++term) u[term] = read16(x + term * term1);
                    }
                    uint32_t lo[2], hi[2];
                    p[0].bytes(q, lo[0], hi[0]);
                    p[1].bytes(q, lo[1], hi[1]);
                    mma_8<true>(c[0], lo[0], lo[1], hi[0], hi[1], q % 2 ? u[0].z : u[0].x, q % 2 ? u[0].w : u[0].y);
                    mma_8<false>(c[1], lo[0], lo[1], hi[0], hi[1], q % 2 ? u[1].z : u[1].x, q % 2 ? u[1].w : u[1].y);
                    mma_8<false>(c[kSums - 1], lo[0], lo[1], hi[0], hi[1], q % 2 ? u[2].z : u[2].x, q % 2 ? u[2].w : u[2].y);
                }
            } else { // a window of one or two octets
                const uint32_t w = (from + (i >> 1) * kBoxBytes) ^ (i & 1) * 64;
#pragma unroll 1
                for (int q = q0; q < q0 + unit; ++q) {
                    const uint32_t x = (filled + (q - q0) / kRun == my_place ? x_here : zeros) + q * 8;
                    const uint2 u[kIntTerms] = {read8u(x), read8u(x + term1), read8u(x + 2 * term1)};
                    const uint32_t wa = read4u(w + q * 4), wb = read4u(w + q * 4 + 8 * 128);
                    mma_8<true>(c[0], wa & 0x0f0f0f0fu, wb & 0x0f0f0f0fu, wa >> 4 & 0x0f0f0f0fu, wb >> 4 & 0x0f0f0f0fu, u[0].x, u[0].y);
                    mma_8<false>(c[1], wa & 0x0f0f0f0fu, wb & 0x0f0f0f0fu, wa >> 4 & 0x0f0f0f0fu, wb >> 4 & 0x0f0f0f0fu, u[1].x, u[1].y);
                    mma_8<false>(c[kSums - 1], wa & 0x0f0f0f0fu, wb & 0x0f0f0f0fu, wa >> 4 & 0x0f0f0f0fu, wb >> 4 & 0x0f0f0f0fu, u[2].x, u[2].y);
                }
            }
            filled += unit / kRun;
        } else {
            Piece p[2];
            p[0].read(from, i, 0);
            p[1].read(from, i, 8 * 128);
            const uint32_t x = (FMT == kW16 ? g < cols : filled == my_place) ? x_here : zeros;
            Piece lo[2];
            if constexpr (kSplit) { // fp16 weights become the sum of two bf16, exactly
                const Piece whole[2] = {p[0], p[1]};
                split_half(whole[0], p[0], lo[0]);
                split_half(whole[1], p[1], lo[1]);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t wa[4], wb[4];
                if constexpr (FMT != kW16) {
                    p[0].halves(q, 0, 0, wa);
                    p[1].halves(q, 0, 0, wb);
                }
#pragma unroll
                for (int term = 0; term < kTerms; ++term) {
                    if constexpr (FMT != kW16) {
                        const uint4 u = read16(x + term * term1 + 128 * (q / 2) + 16 * (q % 2));
                        mma_16<__half>(c[q & 1], wa[0], wb[0], wa[1], wb[1], u.x, u.y);
                        mma_16<__half>(c[q & 1], wa[2], wb[2], wa[3], wb[3], u.z, u.w);
                    } else {
                        const uint4 u = read16(x + term * term1 + 64 * q);
                        mma_16<T>(c[q & 1], p[0].v[q].x, p[1].v[q].x, p[0].v[q].y, p[1].v[q].y, u.x, u.y);
                        mma_16<T>(c[q & 1], p[0].v[q].z, p[1].v[q].z, p[0].v[q].w, p[1].v[q].w, u.z, u.w);
                        if (kSplit && term == 0) {
                            mma_16<T>(c[q & 1], lo[0].v[q].x, lo[1].v[q].x, lo[0].v[q].y, lo[1].v[q].y, u.x, u.y);
                            mma_16<T>(c[q & 1], lo[0].v[q].z, lo[1].v[q].z, lo[0].v[q].w, lo[1].v[q].w, u.z, u.w);
                        }
                    }
                }
            }
            ++filled;
        }
        q0 += unit;
        bool segment_ends = false;
        if (q0 == 4) { // the block is done
            q0 = 0;
            at += X::block_bytes(kTerms, cols);
            --left;
            ++kb;
            if (++i == n) { // and the chunk
                __syncwarp();
                fetch_chunk(slot);
                if (++slot == kWeightSlots) {
                    slot = 0;
                    parity ^= 1;
                }
            }
            segment_ends = kb == blocks || left == 0;
        }
        if ((FMT != kW16 && filled >= window) || segment_ends) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                bool there = token[j] < cols;
                if constexpr (kMasked) there = there && src.mask(seg, token[j]);
                if constexpr (FMT == kW16) {
                    if (there && place[j] == 0) // (the other columns hold zeros, or, where a weight is infinite, NaN)
#pragma unroll
                        for (int h = 0; h < 2; ++h) acc[2 * h + j] += c[0][2 * h + j] + c[1][2 * h + j];
                } else if (there && place[j] < filled) {
                    const int group = first + place[j], block = seg * blocks + group / X::kRuns;
                    const float2 xs = reinterpret_cast<const float2 *>(runs0)[(block * cols + token[j]) * X::kRuns + group % X::kRuns];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if constexpr (FMT == kWInt4) {
                            const float high = __int_as_float(c[0][2 * h + j]) - kFloatBaseValue, mid = __int_as_float(c[1][2 * h + j]) - kFloatBaseValue,
                                        low = __int_as_float(c[kSums - 1][2 * h + j]) - kFloatBaseValue;
                            const float bare = __fmaf_rn(high, 65536.0f, __fmaf_rn(mid, 256.0f, low));
                            acc[2 * h + j] += __fmaf_rn(-(float) wz[j][h], xs.y, bare) * (__uint_as_float(ws[j][h] << 16) * xs.x);
                        } else {
                            acc[2 * h + j] += (c[0][2 * h + j] + c[1][2 * h + j]) * (__uint_as_float(ws[j][h]) * xs.x);
                        }
                    }
                }
            }
            first += filled;
            filled = 0;
            fresh  = true;
            if (segment_ends && left > 0) {
                kb    = 0;
                first = 0;
                ++seg;
                here.open(tile, seg);
            }
        }
    }
    if (!ok) { // what is on its way lands before the CTA gives its memory back
        if (lane == 0) atomicExch(&g_few_status, 5);
        for (int i = 0; i < kWeightSlots; ++i) bar_wait(bars + i * 8, i < slot ? parity ^ 1 : parity);
    }
    // columns of one token: their sums meet, then the shares'
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (tokens == 1) acc[2 * h] += acc[2 * h + 1];
#pragma unroll
        for (int o = 1; o <= 2; o <<= 1)
            if (tokens <= 2 * o)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[2 * h + j] += __shfl_xor_sync(0xffffffffu, acc[2 * h + j], o);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (2 * t + j < min(cols, tokens))
#pragma unroll
            for (int h = 0; h < 2; ++h) part[(warp * cols + 2 * t + j) * 17 + lane_row() + 8 * h] = acc[2 * h + j];
    __syncthreads();
    if (share == 0 && tile < tiles)
        finish(tile, [&](int column, int row) {
            float v = 0.0f;
            for (int w = 0; w < 1 << log_shares; ++w) v += part[((warp + w) * cols + column) * 17 + row];
            return v;
        });
}

// Warps a tile (the power of two): few, for long runs, as long as the SMs have their CTA.  A run's set-up and the adding up are worth
// about six blocks.
inline int token_shares(int tiles, int total, int sms) {
    int best = 0;
    int64_t least = INT64_MAX;
    for (int log = 0; 1 << log <= kTokenWarps; ++log) {
        const int64_t waves = cdiv<int64_t>(cdiv(tiles, kTokenWarps >> log), sms), cost = waves * (cdiv(total, 1 << log) + 6);
        if (cost < least) { least = cost; best = log; }
    }
    return best;
}

} // namespace
} // namespace ptb
