// 4-bit weights: quantise, dequantise, and the product of a few rows with one.  The layout is described in ptb_few_rows.cuh.
#include "ptb_few_tokens.cuh"

namespace ptb {
namespace {

// ---- quantise ---------------------------------------------------------------------------------------------------------
// Groups of G = 32, 64 or 128 neighbouring values of a row:
//   symmetric    s = bf16(max |w| / 7),             z = 8
//   zero points  s = bf16(max(w, 0) / 15 - min(w, 0) / 15), z = clamp(rint(-min(w, 0) / s), 0, 15)
//   code = clamp(rint(w / s) + z, 0, 15)
// The scale is rounded before the codes are chosen, so its rounding costs no accuracy beyond a slightly different grid.  A group that
// holds a NaN or an infinity gets the scale NaN, so that it shows; a group of zeros the scale 0.
//
// HBM-bound: 2 bytes in and half a byte out for a value.  A thread takes the four octets of a block that go into one 16-byte piece of the
// layout, four lanes a block: four 16-byte loads at once, one index per 32 values.
struct Blocks { // block -> row, without a division: for n < 2^31, n / d = mulhi(n, mul) >> shift
    uint32_t count, per_row, mul, shift;
};
inline Blocks blocks_of(int64_t rows, int64_t K) {
    Blocks b;
    b.per_row = (uint32_t) cdiv<int64_t>(K, kKB);
    b.count   = (uint32_t) (rows * b.per_row);
    b.shift   = 0;
    while ((1ull << b.shift) < b.per_row) ++b.shift; // 2^shift >= d
    // mul = ceil(2^(31 + shift) / d) < 2^32, its error times n below 2^31 is less than 1 / d of a unit
    b.mul   = (uint32_t) (((1ull << (31 + b.shift)) + b.per_row - 1) / b.per_row);
    return b;
}
__device__ __forceinline__ uint32_t row_of(const Blocks &b, uint32_t n) { return (uint32_t) ((uint64_t) n * b.mul >> (31 + b.shift)); }

// rint(w / s), where the quotient may lie next to a half-integer: the sign of the exact remainder decides
__device__ __forceinline__ float code_steps(float w, float s, float inv) {
    float r       = inv < INFINITY ? w * inv : __fdiv_rn(w, s); // the inverse of a subnormal scale may overflow
    r             = rintf(fminf(fmaxf(r, -16.0f), 16.0f));
    const float d = __fmaf_rn(-r, s, w); // w - r s, rounded once
    const float h = 0.5f * s;
    // |d| == s / 2 is the tie (to even); beyond it the product with the inverse was a rounding off
    if (fabsf(d) > h) r += d > 0.0f ? 1.0f : -1.0f;
    else if (fabsf(d) == h && (((int) r) & 1)) r += d > 0.0f ? 1.0f : -1.0f;
    return r;
}

template <typename T> struct Pair; // two 16-bit values
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct Pair<__half> { using type = __half2; };

template <typename T, int G, bool kZeros>
__global__ void __launch_bounds__(256) int4_quant_kernel(const T *w, const Blocks blocks, int K, uint4 *codes, __nv_bfloat16 *scale, uint8_t *zero) {
    grid_dep_begin();
    const uint32_t n = blockIdx.x * 64 + (threadIdx.x >> 2);
    const bool here  = n < blocks.count;
    const int t      = threadIdx.x & 3;
    const uint32_t row = here ? row_of(blocks, n) : 0;
    const int k0       = here ? (int) (n - row * blocks.per_row) * kKB + 8 * t : K;
    const T *p         = w + (int64_t) row * K + k0;
    constexpr int kGroups = kKB / G, kPer = 4 / kGroups; // groups of the block, octets of the lane a group
    float lo[kGroups], hi[kGroups]; // of min(w, 0) and max(w, 0), or hi of |w|; NaN where there is one
    uint4 u[4][sizeof(T) / 2];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < (int) sizeof(T) / 2; ++i) {
            u[q][i] = make_uint4(0, 0, 0, 0);
            if (k0 + 32 * q < K) u[q][i] = reinterpret_cast<const uint4 *>(p + 32 * q)[i];
        }
#pragma unroll
    for (int f = 0; f < kGroups; ++f) {
        lo[f] = hi[f] = 0.0f;
        if constexpr (sizeof(T) == 2) {
            using P = typename Pair<T>::type;
            P m = __habs2(*reinterpret_cast<const P *>(&u[f * kPer][0])), l = *reinterpret_cast<const P *>(&u[f * kPer][0]);
            if constexpr (kZeros) m = l;
#pragma unroll
            for (int q = f * kPer; q < f * kPer + kPer; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const P v = reinterpret_cast<const P *>(&u[q][0])[j];
                    m         = __hmax2_nan(m, kZeros ? v : __habs2(v));
                    if constexpr (kZeros) l = __hmin2_nan(l, v);
                }
            const float m0 = to_f32(m.x), m1 = to_f32(m.y), l0 = to_f32(l.x), l1 = to_f32(l.y);
            hi[f] = m0 != m0 || m1 != m1 ? NAN : fmaxf(fmaxf(m0, m1), 0.0f);
            if constexpr (kZeros) lo[f] = fminf(fminf(l0, l1), 0.0f);
        } else {
#pragma unroll
            for (int q = f * kPer; q < f * kPer + kPer; ++q)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float v = reinterpret_cast<const float *>(&u[q][0])[j], m = kZeros ? v : fabsf(v);
                    hi[f] = v != v || hi[f] != hi[f] ? NAN : fmaxf(hi[f], m);
                    if constexpr (kZeros) lo[f] = fminf(lo[f], v);
                }
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            const float h = __shfl_xor_sync(0xffffffffu, hi[f], o);
            hi[f]         = h != h || hi[f] != hi[f] ? NAN : fmaxf(hi[f], h);
            if constexpr (kZeros) lo[f] = fminf(lo[f], __shfl_xor_sync(0xffffffffu, lo[f], o));
        }
    }
    // Divisions are dear: lane t divides for group t, all lanes get all groups' results.
    float s[kGroups], inv[kGroups], zf[kGroups];
    {
        const int f   = t % kGroups;
        float h       = hi[0], l = lo[0];
#pragma unroll
        for (int i = 1; i < kGroups; ++i)
            if (f == i) { h = hi[i]; l = lo[i]; }
        const float wide = kZeros ? __fsub_rn(__fdiv_rn(h, 15.0f), __fdiv_rn(l, 15.0f)) : __fdiv_rn(h, 7.0f);
        const bool fine  = h < INFINITY && l > -INFINITY;
        const float sf   = __bfloat162float(__float2bfloat16_rn(fine ? wide : NAN));
        const float iv   = sf > 0.0f ? __fdiv_rn(1.0f, sf) : 0.0f;
        float z          = 8.0f;
        if (kZeros) z = sf > 0.0f ? fminf(fmaxf(rintf(__fdiv_rn(-l, sf)), 0.0f), 15.0f) : 0.0f;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
            const int from = (threadIdx.x & 28) + i;
            s[i]   = __shfl_sync(0xffffffffu, sf, from);
            inv[i] = __shfl_sync(0xffffffffu, iv, from);
            zf[i]  = kZeros ? __shfl_sync(0xffffffffu, z, from) : 8.0f;
        }
    }
    if (!here) return;
    uint32_t word[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int f = q / kPer;
        uint32_t b[8];
        if (sizeof(T) == 2 && inv[f] < INFINITY) {
            // w / s of 16-bit numbers is a half-integer or at least 2^-13 from one, and the product with the inverse is within 2^-19 of it:
            // rounded to a multiple of 2^-16 (next to 192) ties are ties again.  Next to 1.5 * 2^23 it is an integer, in the low bits.
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float r = __fmaf_rn(to_f32(reinterpret_cast<const T *>(&u[q][0])[j]), inv[f], 192.0f) - 192.0f;
                if constexpr (kZeros) r = fminf(fmaxf(r, -zf[f]), 15.0f - zf[f]);
                r += kFloatBaseValue;
                if constexpr (kZeros) r += zf[f];
                b[j] = __float_as_uint(r);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float r = inv[f] > 0.0f ? code_steps(to_f32(reinterpret_cast<const T *>(&u[q][0])[j]), s[f], inv[f]) : 0.0f;
                b[j]          = (uint32_t) (int) fminf(fmaxf(r + zf[f], 0.0f), 15.0f) ^ (kZeros ? 0u : 8u);
            }
        }
        const uint32_t low = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        const uint32_t high = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
        word[q] = (low & 0x0f0f0f0fu) | (high << 4 & 0xf0f0f0f0u);
        if (!kZeros) word[q] ^= 0x88888888u; // -8 .. 7 in four bits, plus 8
        if (!(s[f] > 0.0f)) word[q] = 0x11111111u * (uint32_t) zf[f];
        if (k0 + 32 * q >= K) word[q] = 0;
    }
    codes[(int64_t) n * 4 + t] = make_uint4(word[0], word[1], word[2], word[3]);
    const int groups = (K + G - 1) / G, g = (k0 - 8 * t) / G + t;
    if (t < kGroups && g < groups) {
        float sf = s[0], z = zf[0];
#pragma unroll
        for (int i = 1; i < kGroups; ++i)
            if (t == i) { sf = s[i]; z = zf[i]; }
        scale[(int64_t) row * groups + g] = __float2bfloat16_rn(sf);
        if constexpr (kZeros) zero[(int64_t) row * groups + g] = (uint8_t) z;
    }
}

// ---- dequantise --------------------------------------------------------------------------------------------------------
// The other way, by the same threads.  In bf16 the difference of two codes is exact and its product with the scale is rounded once; in the
// other types the product is 32-bit (and exact) before it is rounded.
template <typename T>
__global__ void __launch_bounds__(256) int4_dequant_kernel(const uint4 *codes, const __nv_bfloat16 *scale, const uint8_t *zero, int log_group, const Blocks blocks, int K, T *out) {
    grid_dep_begin();
    const uint32_t n = blockIdx.x * 64 + (threadIdx.x >> 2);
    if (n >= blocks.count) return;
    const int t        = threadIdx.x & 3;
    const uint32_t row = row_of(blocks, n);
    const int k0       = (int) (n - row * blocks.per_row) * kKB, groups = (K + (1 << log_group) - 1) >> log_group;
    const uint4 c      = codes[(int64_t) n * 4 + t];
    const uint32_t word[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int k = k0 + 32 * q + 8 * t;
        if (k >= K) continue;
        const int64_t at = (int64_t) row * groups + ((k0 + 32 * q) >> log_group);
        const uint32_t z = zero != nullptr ? zero[at] : 8;
        uint4 *to        = reinterpret_cast<uint4 *>(out + (int64_t) row * K + k);
        if (std::is_same<T, __nv_bfloat16>::value && z < 128) { // 128 + zero is a bf16 up to there
            const __nv_bfloat16 s = scale[at];
            const __nv_bfloat162 s2{s, s};
            const uint32_t base = 0x43004300u + z * 0x00010001u; // 128 + zero
            uint32_t p[4]; // codes 0 2, 1 3, 4 6, 5 7
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t v = (word[q] >> ((i & 1) * 8 + (i >> 1) * 4) & 0x000f000fu) | 0x43004300u;
                const __nv_bfloat162 d = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v), *reinterpret_cast<const __nv_bfloat162 *>(&base)), s2);
                p[i] = *reinterpret_cast<const uint32_t *>(&d);
            }
            to[0] = make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[0], p[1], 0x7632), __byte_perm(p[2], p[3], 0x5410), __byte_perm(p[2], p[3], 0x7632));
        } else {
            const float s = __bfloat162float(scale[at]), base = 8388608.0f + (float) z;
            T r[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) r[j] = from_f32<T>((__uint_as_float((word[q] >> int4_shift(j) & 15) | 0x4b000000u) - base) * s);
            uint4 u[sizeof(T) / 2];
            memcpy(u, r, sizeof(r));
#pragma unroll
            for (int i = 0; i < (int) sizeof(T) / 2; ++i) to[i] = u[i];
        }
    }
}

// ---- product of a few rows ----------------------------------------------------------------------------------------------
struct Int4GemmArgs {
    CUtensorMap map; // of the codes
    const void *x;
    int64_t ldx;
    ScaledRows xs;
    int M, N, K;
    const __nv_bfloat16 *scale;
    const uint8_t *zero;
    const void *bias;
    void *out;
};

template <int G> struct Int4Rows : LaneRows<kWInt4> { // the lane's rows of a tile of 16
    __device__ __forceinline__ void aim(const Int4GemmArgs &a, int n0) {
        const int groups = (a.K + G - 1) / G;
        row  = n0;
        slab = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t r = min(n0 + lane_row() + 8 * h, a.N - 1);
            scale[h] = {nullptr, (const uint16_t *) a.scale + r * groups, a.zero ? a.zero + r * groups : nullptr, 0, groups};
        }
    }
};

// Up to eight rows, as far as they fit into shared memory.
template <int G> struct Int4TokenRows : Int4Rows<G> {
    const Int4GemmArgs &a;
    __device__ __forceinline__ Int4TokenRows(const Int4GemmArgs &a) : a(a) {}
    __device__ __forceinline__ void open(int tile, int) { this->aim(a, tile * 16); }
};
template <typename T, int G> __global__ void __launch_bounds__(32 * kTokenWarps, 1) int4_token_kernel(const __grid_constant__ Int4GemmArgs a, int shares) {
    extern __shared__ __align__(16) uint8_t raw[];
    uint8_t *smem = aligned(raw);
    const int lane = threadIdx.x & 31, blocks = (a.K + kKB - 1) / kKB;
    few_tokens_walk<T, kWInt4, G, kIntTerms, false, false, false>(
        smem, &a.map, a.M, (a.N + 15) / 16, shares, 1, a.K, Int4TokenRows<G>(a),
        [&](uint8_t *x, uint8_t *runs) {
            stage_blocks<T, T, kWInt4, G, kIntTerms>(x, runs, blocks, a.M, [&](int block, int col, int &left) {
                left = a.K - block * kKB;
                return (const T *) a.x + col * a.ldx + block * kKB;
            });
        },
        [&](int tile, auto &&sum) {
            for (int i = lane; i < a.M * 16; i += 32) {
                const int m = i / 16, n = tile * 16 + i % 16;
                if (n >= a.N) continue;
                float v = sum(m, i % 16);
                if (a.bias != nullptr) v += to_f32(((const T *) a.bias)[n]);
                ((T *) a.out)[(int64_t) m * a.N + n] = from_f32<T>(v);
            }
        });
}

// More rows: a CTA has WR * 16 weight rows and up to NT * 8 rows of x, at most 32; more rows are shared out among more CTAs, which then read the weight
// again, mostly from L2.  (64 rows a CTA, with 16 warps: 47 instead of 49 us at 8192 x 8192, but 88 instead of 44 at 4096 x 14336 and
// 17 instead of 8 at 1024 x 512, for want of CTAs.)  Up to 16 rows four warps, beyond eight: 9 rows, 5760 x 2880, groups of 128: 11 us with four
// and 12 with eight; 24 rows, 14336 x 4096: 35 and 25.  The CTAs of a cluster share k; each adds up, and writes, its part of the results, in the order of k.
template <int G> struct Int4BatchRows : Int4Rows<G> {
    ScaledRows xs;
    int row0;
    __device__ __forceinline__ const uint8_t *x(int, int col) const { return xs.planes + (row0 + col) * xs.pitch; }
};
template <typename T, int G, int NT, int WR>
__global__ void __launch_bounds__(32 * WR, 16 / WR) int4_gemm_kernel(const __grid_constant__ Int4GemmArgs a, int shares, int per) {
    extern __shared__ __align__(16) uint8_t raw[];
    uint8_t *smem = aligned(raw);
    using W = Walk<kWInt4, NT, WR>;
    __shared__ uint64_t bars[W::kBars];
    const int tile = blockIdx.x / shares, share = blockIdx.x % shares; // (the rank in the cluster)
    const int n0 = tile * W::kRows, m0 = blockIdx.y * per, cols = min(per, a.M - m0);
    const Share k = share_of(a.K, share, shares);
    Int4BatchRows<G> src;
    src.aim(a, n0 + (threadIdx.x >> 5) * 16);
    src.xs   = a.xs;
    src.row0 = m0;
    float acc[NT][4] = {};
    few_rows_walk<T, kWInt4, G, 128, NT, WR, 1, false>(acc, smem, bars, &a.map, a.K, cols, k.begin, k.end, src);
    const RowSums<kWInt4, NT, WR> sums(acc, smem);
    if (shares > 1) cluster_sync();
    for (int i = threadIdx.x + share * W::kThreads; i < cols * W::kRows; i += W::kThreads * shares) {
        const int m = i / W::kRows, n = i % W::kRows;
        if (n0 + n >= a.N) continue;
        float s = sums.sum(m, n, shares);
        if (a.bias != nullptr) s += to_f32(((const T *) a.bias)[n0 + n]);
        ((T *) a.out)[(int64_t) (m0 + m) * a.N + n0 + n] = from_f32<T>(s);
    }
    if (shares > 1) cluster_sync(); // nobody leaves while his sums are read
}

template <typename T, int G, int NT, int WR> int launch_tile(const Int4GemmArgs &a, cudaStream_t st) {
    using W = Walk<kWInt4, NT, WR>;
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    const int per = cdiv(cdiv(a.M, cdiv(a.M, NT * 8)), 8) * 8, sets = cdiv(a.M, per); // rows of x a CTA, eights as even as can be
    const int tiles = cdiv(a.N, W::kRows);
    const int shares = shares_for(a.K, (int64_t) tiles * sets, sms * (16 / WR));
    constexpr int kMost = W::smem(1, NT * 8);
    PTB_CUDA(launch_early(int4_gemm_kernel<T, G, NT, WR>, dim3((unsigned) (tiles * shares), (unsigned) sets), W::kThreads,
                          W::smem(1, (int) imin(a.M, per)), kMost, st, (unsigned) shares, a, shares, per));
    PTB_LAUNCH_CHECK("int4_gemm_kernel");
    return 0;
}

constexpr int kMostSmem = 227 * 1024 - 1024; // of a CTA, less what is not dynamic

template <typename T, int G> int launch_gemm(const Int4GemmArgs &a, cudaStream_t st) {
    const int x_bytes = a.M <= kTokenCols && a.K <= 1 << 20 ? TokenX<kWInt4, G>::bytes(kIntTerms, a.M, cdiv(a.K, kKB)) : kMostSmem;
    if (token_smem(x_bytes, a.M) <= kMostSmem) {
        int sms = 0;
        if (int rc = sm_count(&sms)) return rc;
        const int tiles = cdiv(a.N, 16), shares = token_shares(tiles, cdiv(a.K, kKB), sms);
        PTB_CUDA(launch_early(int4_token_kernel<T, G>, dim3((unsigned) cdiv(tiles, kTokenWarps >> shares)), 32 * kTokenWarps, token_smem(x_bytes, a.M), kMostSmem, st, 1, a, shares));
        PTB_LAUNCH_CHECK("int4_token_kernel");
        return 0;
    }
    const int64_t warps = a.M * cdiv<int64_t>(a.K, kKB);
    PTB_CUDA(launch_early(scale_rows_kernel<T, kWInt4>, dim3((unsigned) cdiv<int64_t>(warps, 4)), 128, 0, 0, st, 1, (const T *) a.x, a.ldx, a.M, a.K, a.xs));
    PTB_LAUNCH_CHECK("scale_rows_kernel");
    if (a.M <= 8) return launch_tile<T, G, 1, 4>(a, st);
    if (a.M <= 16) return launch_tile<T, G, 2, 4>(a, st);
    return launch_tile<T, G, 4, 8>(a, st);
}

bool is_group(int64_t g) { return g == 32 || g == 64 || g == 128; }

#define PTB_SWITCH_INT4_GROUP(g, G, ...)                   \
    switch (g) {                                           \
    case 32: { constexpr int G = 32; __VA_ARGS__; } break; \
    case 64: { constexpr int G = 64; __VA_ARGS__; } break; \
    default: { constexpr int G = 128; __VA_ARGS__; }       \
    }

} // namespace

int int4_status(int *status, int reset) { return few_status(status, reset); }
} // namespace ptb

using namespace ptb;

extern "C" {
#pragma GCC visibility push(default)

int ptb_quant_int4(const void *w, int dtype, int64_t rows, int64_t K, int64_t group, void *codes, void *scale, void *zero, ptb_stream_t stream) {
    PTB_REQUIRE(rows >= 0 && K >= 0, PTB_ERR_ARG, "quant_int4: negative size");
    PTB_REQUIRE(is_hp(dtype), PTB_ERR_ARG, "quant_int4: the weight must be fp32, fp16 or bf16");
    PTB_REQUIRE(is_group(group), PTB_ERR_ARG, "quant_int4: the group size must be 32, 64 or 128");
    PTB_REQUIRE(K % 8 == 0, PTB_ERR_ALIGN, "quant_int4: the row length must be a multiple of 8");
    PTB_REQUIRE(K <= 1 << 24, PTB_ERR_TOO_LARGE, "quant_int4: row too long");
    if (rows == 0 || K == 0) return 0;
    PTB_REQUIRE(w && codes && scale, PTB_ERR_ARG, "quant_int4: null pointer");
    PTB_REQUIRE(aligned16(w) && aligned16(codes), PTB_ERR_ALIGN, "quant_int4: the weight and the codes must be 16-byte aligned");
    PTB_REQUIRE(rows <= 2147483647ll / cdiv<int64_t>(K, kKB), PTB_ERR_TOO_LARGE, "quant_int4: too many values");
    const Blocks blocks = blocks_of(rows, K);
    const dim3 grid((unsigned) cdiv<int64_t>(blocks.count, 64));
    PTB_SWITCH_HP(dtype, T, PTB_SWITCH_INT4_GROUP(group, G, {
        if (zero != nullptr)
            PTB_CUDA(launch_after(int4_quant_kernel<T, G, true>, grid, 256, 0, (cudaStream_t) stream, 1, (const T *) w, blocks, (int) K, (uint4 *) codes,
                                  (__nv_bfloat16 *) scale, (uint8_t *) zero));
        else
            PTB_CUDA(launch_after(int4_quant_kernel<T, G, false>, grid, 256, 0, (cudaStream_t) stream, 1, (const T *) w, blocks, (int) K, (uint4 *) codes,
                                  (__nv_bfloat16 *) scale, (uint8_t *) nullptr));
    }));
    PTB_LAUNCH_CHECK("int4_quant_kernel");
    return 0;
}

int ptb_dequant_int4(const void *codes, const void *scale, const void *zero, int64_t rows, int64_t K, int64_t group, void *out, int out_dtype,
                     ptb_stream_t stream) {
    PTB_REQUIRE(rows >= 0 && K >= 0, PTB_ERR_ARG, "dequant_int4: negative size");
    PTB_REQUIRE(is_hp(out_dtype), PTB_ERR_ARG, "dequant_int4: the output must be fp32, fp16 or bf16");
    PTB_REQUIRE(is_group(group), PTB_ERR_ARG, "dequant_int4: the group size must be 32, 64 or 128");
    PTB_REQUIRE(K % 8 == 0, PTB_ERR_ALIGN, "dequant_int4: the row length must be a multiple of 8");
    PTB_REQUIRE(K <= 1 << 24, PTB_ERR_TOO_LARGE, "dequant_int4: row too long");
    if (rows == 0 || K == 0) return 0;
    PTB_REQUIRE(codes && scale && out, PTB_ERR_ARG, "dequant_int4: null pointer");
    PTB_REQUIRE(aligned16(codes) && aligned16(out), PTB_ERR_ALIGN, "dequant_int4: the codes and the output must be 16-byte aligned");
    PTB_REQUIRE(rows <= 2147483647ll / cdiv<int64_t>(K, kKB), PTB_ERR_TOO_LARGE, "dequant_int4: too many values");
    const Blocks blocks = blocks_of(rows, K);
    const dim3 grid((unsigned) cdiv<int64_t>(blocks.count, 64));
    const int log_group = group == 32 ? 5 : group == 64 ? 6 : 7;
    PTB_SWITCH_HP(out_dtype, T, PTB_CUDA(launch_after(int4_dequant_kernel<T>, grid, 256, 0, (cudaStream_t) stream, 1, (const uint4 *) codes,
                                                       (const __nv_bfloat16 *) scale, (const uint8_t *) zero, log_group, blocks, (int) K, (T *) out)));
    PTB_LAUNCH_CHECK("int4_dequant_kernel");
    return 0;
}

int64_t ptb_gemm_int4_workspace(int dtype, int64_t M, int64_t K, int64_t group) {
    if (M < 0 || K < 1 || (dtype != PTB_BF16 && dtype != PTB_F16) || !is_group(group)) return -1;
    return scaled_bytes(1, M, K);
}

int ptb_gemm_int4(const void *x, int dtype, int64_t ldx, int64_t M, int64_t N, int64_t K, const void *codes, const void *scale, const void *zero,
                  int64_t group, const void *bias, void *workspace, void *out, ptb_stream_t stream) {
    PTB_REQUIRE(M >= 0 && N >= 0 && K >= 1, PTB_ERR_ARG, "gemm_int4: bad shape");
    PTB_REQUIRE(dtype == PTB_BF16 || dtype == PTB_F16, PTB_ERR_ARG, "gemm_int4: x must be bf16 or fp16");
    PTB_REQUIRE(is_group(group), PTB_ERR_ARG, "gemm_int4: the group size must be 32, 64 or 128");
    PTB_REQUIRE(K % 8 == 0 && (M <= 1 || ldx % 8 == 0), PTB_ERR_ALIGN, "gemm_int4: the row length and pitch of x must be multiples of 8");
    PTB_REQUIRE(M <= 1 || ldx >= K, PTB_ERR_ARG, "gemm_int4: rows of x overlap");
    PTB_REQUIRE(K <= 1 << 24 && N <= 1 << 30 && M <= 1 << 20 && M * K <= 1ll << 34, PTB_ERR_TOO_LARGE, "gemm_int4: matrix too large");
    if (M == 0 || N == 0) return 0;
    PTB_REQUIRE(x && codes && scale && workspace && out, PTB_ERR_ARG, "gemm_int4: null pointer");
    PTB_REQUIRE(aligned16(x) && aligned16(codes) && aligned16(workspace), PTB_ERR_ALIGN, "gemm_int4: x, the codes and the workspace must be 16-byte aligned");
    Int4GemmArgs a{{}, x, ldx, scaled_rows_at(workspace, M, K), (int) M, (int) N, (int) K, (const __nv_bfloat16 *) scale, (const uint8_t *) zero, bias, out};
    if (int rc = weight_map(&a.map, codes, cdiv<int64_t>(K, kKB) * kInt4BlockBytes, N, 1, false)) return rc;
    cudaStream_t st = (cudaStream_t) stream;
    PTB_SWITCH_INT4_GROUP(group, G, return dtype == PTB_BF16 ? launch_gemm<__nv_bfloat16, G>(a, st) : launch_gemm<__half, G>(a, st));
    return 0;
}

#pragma GCC visibility pop
} // extern "C"
